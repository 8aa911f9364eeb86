// Low-rank adapters of many requests beside a shared projection:
//   out[b, t, :] = base[b, t, :] + scale_a (hidden[b, t, :] A_a^T) B_a^T,  a = ids[b],
// with A [n, R, D] and B [n, V, R] in bf16, base the shared projection's
// output (the logits) and out = base where ids[b] names no adapter.
//
// On the matrix cores in tiles of 16 rows of one adapter, sums in f32.  The f32
// operands of a product go in as bf16 parts, each the rounded rest of the ones
// before it: three parts are an f32 to 2^-24 of it, two to 2^-16.  f32 hidden
// and u = scale hidden A^T take three; bf16 hidden is one, and its u takes two
// (out rounds to 2^-8).  Parts below 2^-126 are subnormal bf16, which the matrix
// cores keep: nothing is held closer than half the least of them, 2^-134, so f32
// values below 2^-110 lose their last bits.  u's parts stand side by side, as one
// product of two or three times the depth with the same columns of B.
//
// Rows of a tile: of prompts, 16 of one sequence; with up to 16 tokens a
// sequence (generation), gathered from the sequences of one adapter, so that B
// is read once for up to 16 rows.
//
// A workgroup holds its rows' u in LDS and runs over blocks of columns, bound by
// base, out and B: 8 prompts of 512 (D 256, V 32000, R 16, f32) 212 us (4.9 TB/s),
// 3 of 1001 (D 1024, V 50048, R 64, bf16) 184 (3.3 TB/s; at R 16 148, B being read
// again for every 64 rows), 222 at V 50001, whose rows of odd length leave no access
// aligned.  u comes from the workgroup itself (one launch: small calls
// are launches and latency), or, where many workgroups would compute the same
// u, from a launch of its own through the stream's scratch.
#include <type_traits>

#include "bdh_internal.h"

namespace bdh {
namespace {

constexpr int kTile = 16;
constexpr int kGatherTokens = 16;  // up to here tiles gather sequences
constexpr int kWindow = 512;       // sequences of the batch that are gathered together
constexpr int kRowsTokens = 2, kRowsIn = 512;  // up to here, at ranks to 16, adapter_rows_kernel may do without tiles
constexpr int kRowsShare = 8;                  // the sequences it gathers

typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf16x8_u __attribute__((ext_vector_type(8), aligned(2)));

__device__ __forceinline__ int adapter_of(const AdapterArgs& a, int64_t b) {
  const int id = a.ids[b];
  return id >= 0 && id < a.n ? id : -1;
}

// The next bf16 part of an f32 whose rest is x.  first: rounded to a finite value,
// so that nothing finite grows past bf16's largest; an infinity or a NaN is what
// then remains of one, and is the second part.
__device__ __forceinline__ bf16_t next_part(float& x, bool first) {
  if (first) {
    const bf16_t p = (bf16_t)__builtin_amdgcn_fmed3f(x, -0x1.fep127f, 0x1.fep127f);
    x -= (float)p;
    return p;
  }
  const bf16_t p = (bf16_t)x;
  x = fabsf((float)p) < INFINITY ? x - (float)p : 0.0f;
  return p;
}
template <typename T> constexpr int hidden_parts = sizeof(T) == 4 ? 3 : 1;
template <typename T> constexpr int u_parts = sizeof(T) == 4 ? 3 : 2;
// A row of u: its parts of RP, zeros up to a multiple of the product's 32.
template <typename T, int RP> constexpr int u_row = (u_parts<T> * RP + 31) / 32 * 32;

// Eight values of a row of n from index k on (a multiple of 8), zeros past its
// end.  EVEN: n is a multiple of 8 too.
template <bool EVEN>
__device__ __forceinline__ bf16x8 load8_bf16(const bf16_t* row, int64_t k, int64_t n) {
  bf16x8_u v = {};
  if (EVEN ? k < n : k + 8 <= n) {
    v = *(const bf16x8_u*)(row + k);
  } else if (!EVEN) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = k + j < n ? row[k + j] : (bf16_t)0.0f;
  }
  return __builtin_bit_cast(bf16x8, v);
}
template <bool EVEN>
__device__ __forceinline__ void load8_f32(const float* row, int64_t k, int64_t n, float (&x)[8]) {
  if (EVEN ? k < n : k + 8 <= n) {
    const f32x4_u p = *(const f32x4_u*)(row + k), q = *(const f32x4_u*)(row + k + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = p[j];
      x[4 + j] = q[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = !EVEN && k + j < n ? row[k + j] : 0.0f;
  }
}

// The rows of a workgroup: 16 * MT tokens of sequence b, or gathered.
struct Rows {
  int id;         // adapter, -1: none
  int n;          // rows
  int64_t first;  // in [batch, time]; GATHER: unused
};

// The workgroups of a sequence that is the first of its adapter, or the first
// after `share` more of it, gather that one and the next; the others have no
// rows.  list: their rows.  Every wave for itself, without a barrier: all
// write the same list.  Each 512 sequences are gathered by themselves, or every
// workgroup would go through a large batch's ids.
__device__ Rows gather_rows(const AdapterArgs& a, int b, int share, int* list) {
  const int time = (int)a.time, lane = threadIdx.x & 63;
  Rows g{adapter_of(a, b), 0, 0};
  if (g.id < 0 && a.out == a.base) return g;
  int before = 0, n = 0;
  const int window = b / kWindow * kWindow, end = min(window + kWindow, (int)a.batch);
  for (int i0 = window; i0 < end && n < share; i0 += 64) {
    const int i = i0 + lane;
    const bool is = i < end && adapter_of(a, i) == g.id;
    before += __popcll(__ballot(is && i < b));
    const uint64_t from_b = __ballot(is && i >= b);
    if (from_b != 0 && before % share != 0) return g;
    const int at = n + __popcll(from_b & ((1ull << lane) - 1));
    if (is && i >= b && at < share)
      for (int t = 0; t < time; ++t) list[at * time + t] = i * time + t;
    n += __popcll(from_b);
  }
  g.n = (n < share ? n : share) * time;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  return g;
}

// u of 16 * MT rows into LDS, by the four waves of the workgroup.
template <typename T, int RP, int MT>
struct UTile {
  static constexpr int KS = 4 / MT;                 // waves that share a tile's product over D
  static constexpr int ROWS = kTile * MT, DEPTH = u_parts<T> * RP, ROW = u_row<T, RP>;
  static constexpr int PITCH = ROW + 8;             // (bank spread)
  union Memory {
    float part[KS][ROWS][RP];
    bf16_t u[ROWS][PITCH];
  };

  template <bool EVEN, typename RowAt>
  static __device__ __forceinline__ void compute(Memory& mem, const AdapterArgs& a, int id, const RowAt& row_at) {
    constexpr int NT = RP / 16, HP = hidden_parts<T>, UP = u_parts<T>, PER = ROWS * RP / 256;
    const int lane = threadIdx.x & 63, low = lane & 15, high = lane >> 4;
    const int m = wave_id() % MT, ks = wave_id() / MT;
    const T* h = (const T*)a.hidden + row_at(kTile * m + low) * a.in_dim;
    const bf16_t* w = a.a + (int64_t)id * a.rank * a.in_dim;
    floatx4 acc[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j] = zero4();
    // AHEAD steps of 32 at a time: all their loads, then their products.  (One
    // after the other, each step waited for memory: 2.4 us a step.)
    constexpr int AHEAD = NT <= 4 ? 4 : 2;
    for (int d0 = ks * 32; d0 < (int)a.in_dim; d0 += 32 * KS * AHEAD) {
      bf16x8 y[AHEAD][NT], x[AHEAD];
      float f[AHEAD][8];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int d = d0 + 32 * KS * i + 8 * high;
        if constexpr (HP > 1) load8_f32<EVEN>((const float*)h, d, a.in_dim, f[i]);
        else x[i] = load8_bf16<EVEN>((const bf16_t*)h, d, a.in_dim);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const int k = j * 16 + low;
          y[i][j] = load8_bf16<EVEN>(w + (k < a.rank ? k : 0) * a.in_dim, d, a.in_dim);
        }
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        bf16x8 p[HP];
        if constexpr (HP > 1) {
#pragma unroll
          for (int q = 0; q < HP; ++q)
#pragma unroll
            for (int j = 0; j < 8; ++j) p[q][j] = next_part(f[i][j], q == 0);
        } else {
          p[0] = x[i];
        }
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int q = HP - 1; q >= 0; --q) acc[j] = mfma16(p[q], y[i][j], acc[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) mem.part[ks][kTile * m + acc16_row(lane, r)][j * 16 + low] = acc[j][r];
    __syncthreads();
    const float scale = a.scale[id];
    float s[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = threadIdx.x + 256 * i, r = at / RP, k = at % RP;
      s[i] = mem.part[0][r][k];
#pragma unroll
      for (int q = 1; q < KS; ++q) s[i] += mem.part[q][r][k];
      // (Past the rank: zeros, whatever hidden and the rows of A there are.)
      s[i] = k < a.rank ? s[i] * scale : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = threadIdx.x + 256 * i, r = at / RP, k = at % RP;
#pragma unroll
      for (int q = 0; q < UP; ++q) mem.u[r][q * RP + k] = next_part(s[i], q == 0);
      if (ROW > DEPTH) mem.u[r][DEPTH + k] = (bf16_t)0.0f;
    }
    static_assert(ROW == DEPTH || ROW - DEPTH == RP, "one part of zeros");
    __syncthreads();
  }
};

// u of a tile of 16 rows to scratch [batch * time][u_row].
template <typename T, int RP, bool EVEN, bool GATHER>
__global__ __launch_bounds__(256) void adapter_u_kernel(const AdapterArgs a) {
  typedef UTile<T, RP, 1> U;
  __shared__ __attribute__((aligned(16))) typename U::Memory mem;
  __shared__ int list[kTile];
  Rows g;
  if constexpr (GATHER) {
    g = gather_rows(a, (int)blockIdx.y, kTile / (int)a.time, list);
  } else {
    const int64_t t0 = (int64_t)blockIdx.x * kTile;
    g = Rows{adapter_of(a, blockIdx.y), (int)(a.time - t0 < kTile ? a.time - t0 : kTile), blockIdx.y * a.time + t0};
  }
  if (g.id < 0 || g.n == 0) return;
  const auto row_at = [&](int r) -> int64_t {
    r = r < g.n ? r : g.n - 1;
    return GATHER ? (int64_t)list[r] : g.first + r;
  };
  U::template compute<EVEN>(mem, a, g.id, row_at);
  for (int i = threadIdx.x; i < g.n * (U::ROW / 8); i += 256) {
    const int r = i / (U::ROW / 8), k = i % (U::ROW / 8) * 8;
    *(bf16x8*)(a.u + row_at(r) * U::ROW + k) = *(const bf16x8*)&mem.u[r][k];
  }
}

template <typename T> struct Cols;  // a lane's neighbouring columns: 16 bytes at any element's address
template <> struct Cols<float> { typedef f32x4_u type; };
template <> struct Cols<bf16_t> { typedef bf16x8_u type; };
template <typename T> constexpr int kCols = 16 / sizeof(T);
template <typename T> constexpr int kWide = 4 * 16 * kCols<T>;  // columns of a workgroup's four blocks

// 16 * MT rows by every gridDim.x-th run of kWide columns, the waves side by
// side on its blocks of 16 * kCols (of a row 1 KB in one go), so that the
// workgroups that run together cover neighbouring runs.  A wave takes a block's
// rows of B into registers and runs over the row tiles: u from LDS, base one
// tile ahead.  OWN: computes u itself.
template <typename T, int RP, int MT, bool EVEN, bool GATHER, bool OWN>
__global__ __launch_bounds__(256, RP <= 64 ? 2 : 1) void adapter_out_kernel(const AdapterArgs a) {
  typedef UTile<T, RP, MT> U;
  typedef typename Cols<T>::type Vec;
  constexpr int NC = kCols<T>, BLOCK = 16 * NC;
  constexpr int YS = RP >= 32 ? RP / 32 : 1;  // 32-deep slices of B's rows
  __shared__ __attribute__((aligned(16))) typename U::Memory mem;
  __shared__ int list[kTile];
  Rows g;
  if constexpr (GATHER) {
    g = gather_rows(a, (int)blockIdx.z, kTile / (int)a.time, list);
  } else {
    const int64_t t0 = (int64_t)blockIdx.y * U::ROWS;
    g = Rows{adapter_of(a, blockIdx.z), (int)(a.time - t0 < U::ROWS ? a.time - t0 : U::ROWS), blockIdx.z * a.time + t0};
    if (g.id < 0 && a.out == a.base) return;
  }
  if (g.n == 0) return;
  const int id = g.id, last = g.n - 1, tiles = (g.n + kTile - 1) / kTile;
  const auto row_at = [&](int r) -> int64_t {
    r = r < last ? r : last;
    return GATHER ? (int64_t)list[r] : g.first + r;
  };
  const int lane = threadIdx.x & 63, low = lane & 15, high = lane >> 4;
  const int v_end = (int)a.out_dim;
  const bf16_t* w = a.b + (int64_t)(id >= 0 ? id : 0) * a.out_dim * a.rank;
  const auto load_base = [&](auto full, int v, int m, Vec (&x)[4]) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = kTile * m + 4 * high + r;
      if (GATHER && row > last) continue;
      const T* from = (const T*)a.base + row_at(row) * a.out_dim + v;
      if (full) {
        x[r] = *(const Vec*)from;
      } else {
#pragma unroll
        for (int j = 0; j < NC; ++j) x[r][j] = v + j < v_end ? from[j] : (T)0.0f;
      }
    }
  };
  const auto load_b = [&](auto full, int v, bf16x8 (&y)[YS][NC]) {
#pragma unroll
    for (int s = 0; s < YS; ++s) {
      // This lane's eight-deep slice: each of u's parts meets the same columns of B.
      const int kb = (32 * s + 8 * high) % RP;
#pragma unroll
      for (int j = 0; j < NC; ++j)
        y[s][j] = load8_bf16<EVEN>(w + (uint32_t)((full || v + j < v_end ? v + j : v_end - 1) * (int)a.rank), kb,
                                   a.rank);
    }
  };
  const auto product = [&](const bf16x8 (&y)[YS][NC], int m, floatx4 (&acc)[NC]) {
#pragma unroll
    for (int j = 0; j < NC; ++j) acc[j] = zero4();
    if (id < 0) return;
#pragma unroll
    for (int k = U::ROW - 32; k >= 0; k -= 32) {  // the smaller parts first
      const bf16x8 f = *(const bf16x8*)&mem.u[kTile * m + low][k + 8 * high];
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        // (Rank 16: a step holds two parts, the last of three one and zeros,
        // which are not to meet an infinity.)
        const bf16x8 z = {};
        const bool in = k + 32 <= U::DEPTH || k + 8 * high < U::DEPTH;
        acc[j] = mfma16(f, in ? y[k / 32 % YS][j] : z, acc[j]);
      }
    }
  };
  const auto store = [&](auto full, int v, int m, const Vec (&x)[4], const floatx4 (&acc)[NC]) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = kTile * m + 4 * high + r;
      if (row > last) continue;
      T* to = (T*)a.out + row_at(row) * a.out_dim + v;
      Vec o;
#pragma unroll
      for (int j = 0; j < NC; ++j) o[j] = (T)((float)x[r][j] + acc[j][r]);
      if (full) {
        *(Vec*)to = o;
      } else {
#pragma unroll
        for (int j = 0; j < NC; ++j)
          if (v + j < v_end) to[j] = o[j];
      }
    }
  };
  // Column NC * c + j of a block is column c of product tile j, so a lane's
  // results of a row are NC neighbours: 16 bytes.  The first block's B and base
  // are asked for ahead of u, base then comes one tile ahead.
  const int stride = (int)gridDim.x * kWide<T>;
  int v0 = (int)blockIdx.x * kWide<T> + wave_id() * BLOCK;
  Vec x[2][4];
  bf16x8 y[YS][NC];
  if (v0 + BLOCK <= v_end) {
    load_base(std::true_type{}, v0 + NC * low, 0, x[0]);
    if (id >= 0) load_b(std::true_type{}, v0 + NC * low, y);
  }
  if (id >= 0) {
    if constexpr (OWN) {
      U::template compute<EVEN>(mem, a, id, row_at);
    } else {
      for (int i = threadIdx.x; i < tiles * kTile * (U::ROW / 8); i += 256) {
        const int r = i / (U::ROW / 8), k = i % (U::ROW / 8) * 8;
        *(bf16x8*)&mem.u[r][k] = *(const bf16x8*)(a.u + row_at(r) * U::ROW + k);
      }
      __syncthreads();
    }
  }
  for (bool first = true; v0 + BLOCK <= v_end; v0 += stride, first = false) {
    const int v = v0 + NC * low;
    const bool more = v0 + stride + BLOCK <= v_end;
    if (id >= 0 && !first) load_b(std::true_type{}, v, y);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if (m >= tiles) break;
      if (m + 1 < tiles) load_base(std::true_type{}, v, m + 1, x[(m + 1) & 1]);
      else if (more && (m & 1)) load_base(std::true_type{}, v + stride, 0, x[0]);
      floatx4 acc[NC];
      product(y, m, acc);
      store(std::true_type{}, v, m, x[m & 1], acc);
      if (m + 1 == tiles && more && !(m & 1)) load_base(std::true_type{}, v + stride, 0, x[0]);
    }
  }
  if (v0 >= v_end) return;
  // The rows' last columns, fewer than a block.
  const int v = v0 + NC * low;
  if (id >= 0) load_b(std::false_type{}, v, y);
  for (int m = 0; m < tiles; ++m) {
    load_base(std::false_type{}, v, m, x[0]);
    floatx4 acc[NC];
    product(y, m, acc);
    store(std::false_type{}, v, m, x[0], acc);
  }
}

// --- few rows of a small model --------------------------------------------------
// Sum over 16 neighbouring lanes, in the last of them.
template <int CTRL>
__device__ __forceinline__ float add_dpp(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float sum16(float v) {
  return add_dpp<0x118>(add_dpp<0x114>(add_dpp<0x112>(add_dpp<0x111>(v))));
}

// Gathered rows at ranks to 16 without matrix cores, u computed here: a thread
// holds four columns' rows of B and runs over the rows.  Where a tile of the
// product would be mostly empty, what counts is how much a workgroup asks for at
// once: of 64 rows with 32 adapters (D 256, V 32000, R 16) 12.2 us where the
// tiles take 23.7 (at rank 32 and D 512 36 where they take 25).
template <typename T>
__global__ __launch_bounds__(256) void adapter_rows_kernel(const AdapterArgs a) {
  constexpr int RP = 16, VPT = 4;
  __shared__ float u[kRowsShare * kRowsTokens][RP];
  __shared__ int list[kRowsShare * kRowsTokens];
  const Rows g = gather_rows(a, (int)blockIdx.y, kRowsShare, list);
  if (g.n == 0) return;
  const int id = g.id, n = g.n, v_end = (int)a.out_dim;
  // A thread's columns lie 256 apart: a wave's accesses are runs of neighbours.
  const int v = (int)blockIdx.x * (256 * VPT) + threadIdx.x;
  float w[VPT][RP];
  if (id >= 0) {
    // 16 lanes a rank, eight columns of the dot products each; four rows at a time.
    const int lane = threadIdx.x & 15, k = threadIdx.x >> 4;
    const float scale = a.scale[id];
    const bf16_t* wa = a.a + ((int64_t)id * a.rank + (k < a.rank ? k : 0)) * a.in_dim;
    for (int i0 = 0; i0 < n; i0 += 4) {
      float sum[4] = {};
      const T* h[4];
#pragma unroll
      for (int q = 0; q < 4; ++q)
        h[q] = (const T*)a.hidden + (int64_t)__builtin_amdgcn_readfirstlane(list[i0 + q < n ? i0 + q : i0]) * a.in_dim;
#pragma unroll 2
      for (int d = lane * 8; d < (int)a.in_dim; d += 128) {
        const bf16x8 y = load8_bf16<true>(wa, d, a.in_dim);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float x[8];
          if constexpr (sizeof(T) == 4) {
            load8_f32<true>((const float*)h[q], d, a.in_dim, x);
          } else {
            const bf16x8 p = load8_bf16<true>((const bf16_t*)h[q], d, a.in_dim);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = (float)p[j];
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) sum[q] = fmaf(x[j], (float)y[j], sum[q]);
        }
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float s = sum16(sum[q]) * scale;
        // (Past the rank: zeros, whatever hidden and the rows of A there are.)
        if (lane == 15 && i0 + q < n) u[i0 + q][k] = k < a.rank ? s : 0.0f;
      }
    }
    __syncthreads();
    bf16x8 wb[VPT][RP / 8];
    const bf16_t* from = a.b + (int64_t)id * a.out_dim * a.rank;
#pragma unroll
    for (int j = 0; j < VPT; ++j)
#pragma unroll
      for (int k = 0; k < RP; k += 8)
        wb[j][k / 8] = load8_bf16<true>(from + (uint32_t)((v + 256 * j < v_end ? v + 256 * j : v_end - 1) * (int)a.rank),
                                        k, a.rank);
#pragma unroll
    for (int j = 0; j < VPT; ++j)
#pragma unroll
      for (int q = 0; q < RP; ++q) w[j][q] = (float)wb[j][q / 8][q % 8];
  }
  // Four rows' base values at a time, ahead of the stores.
  for (int i0 = 0; i0 < n; i0 += 4) {
    float x[4][VPT];
    int64_t at[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      at[q] = (int64_t)__builtin_amdgcn_readfirstlane(list[i0 + q < n ? i0 + q : i0]) * a.out_dim + v;
#pragma unroll
      for (int j = 0; j < VPT; ++j) x[q][j] = v + 256 * j < v_end ? (float)((const T*)a.base)[at[q] + 256 * j] : 0.0f;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (i0 + q >= n) break;
      if (id >= 0) {
        float sum[VPT] = {};
#pragma unroll
        for (int k = 0; k < RP; ++k) {
          const float uk = u[i0 + q][k];
#pragma unroll
          for (int j = 0; j < VPT; ++j) sum[j] = fmaf(uk, w[j][k], sum[j]);
        }
#pragma unroll
        for (int j = 0; j < VPT; ++j) x[q][j] += sum[j];
      }
#pragma unroll
      for (int j = 0; j < VPT; ++j)
        if (v + 256 * j < v_end) ((T*)a.out)[at[q] + 256 * j] = (T)x[q][j];
    }
  }
}

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

template <typename T, int RP, int MT, bool EVEN, bool GATHER, bool OWN>
void launch_out(const AdapterArgs& a, int64_t runs, hipStream_t st) {
  const dim3 grid((uint32_t)runs, GATHER ? 1u : (uint32_t)cdiv(a.time, kTile * MT), (uint32_t)a.batch);
  hipLaunchKernelGGL((adapter_out_kernel<T, RP, MT, EVEN, GATHER, OWN>), grid, dim3(256), 0, st, a);
}

template <typename T, int RP, bool EVEN>
bdh_status run_typed(AdapterArgs a, hipStream_t st, uint64_t* launches) {
  const bool gather = a.time <= kGatherTokens;
  if constexpr (EVEN && RP == 16) {
    // Without tiles where those would be mostly empty (few rows an adapter of the
    // set) in a call with columns enough.  us in a graph, this / tiles, R 16, by rows,
    // adapters and columns; the ranges are over D of 64 to 512:
    //   f32    64 of 32: V 128000 35-41 / 49-52, 32000 11-16 / 23-24, 4096 9-12 / 8-10
    //          16 of 16: 32000 6.7-8.3 / 11-12;  4 of 4: 128000 6.0-7.7 / 11-12, 32000 5.7-6.8 / 5.6-7.1
    //          64 of 8: 128000 27-32 / 26-29, 32000 12-16 / 15-16, 4096 11-13 / 5.6-8.9
    //          256 of 16: 32000 30-37 / 35-36;  1: 32000 5.1-6.1 / 5.0-5.4
    //   two tokens, D 256: 64 sequences of 32: 128000 47 / 59, 32000 20 / 25;  64 of 8: 32000 24 / 20
    //   bf16, D 256: 64 of 32: 128000 43 / 46, 32000 18.6 / 18.9;  256 of 64: 128000 181 / 138
    // (At D 1024 64 of 32 20 / 25 and 16 of 2 16 / 11; at rank 32 and D 512 36 / 25.)
    const int64_t rows = a.batch * a.time, columns = a.batch * a.out_dim;
    const bool sparse = sizeof(T) == 4
                            ? (rows <= 4 * a.n && columns > (int64_t)1 << 18) ||
                                  (a.time == 1 && rows <= 8 * a.n && columns >= (int64_t)1 << 20)
                            : rows <= 2 * a.n && columns >= (int64_t)1 << 20;
    if (a.time <= kRowsTokens && a.in_dim <= kRowsIn && sparse) {
      hipLaunchKernelGGL((adapter_rows_kernel<T>), dim3((uint32_t)cdiv(a.out_dim, 1024), (uint32_t)a.batch), dim3(256),
                         0, st, a);
      BDH_HIP_TRY(hipGetLastError());
      *launches += 1;
      return BDH_OK;
    }
  }
  // Workgroups along the columns: 2048 in all where there are columns enough
  // (gathered, whose workgroups mostly end at once, 8192).  A run's remainder
  // gets a workgroup of its own only where the chip has room: of 257 columns
  // the last one cost a second pass over hidden (18.5 us, now 14.2, at 16
  // prompts of 1024).
  const auto runs_of = [&](int64_t tiles) {
    const int64_t whole = a.out_dim / kWide<T>, want = cdiv(gather ? 8192 : 2048, tiles);
    const int64_t wide = whole * tiles >= 256 ? whole : cdiv(a.out_dim, kWide<T>);
    return want < wide ? want : wide;
  };
  // Each workgroup that computes u itself spends about D / 128 us on it, of
  // which the chip runs some 512 at a time; a launch of its own costs about 4.
  const int64_t own_tiles = gather ? a.batch : a.batch * cdiv(a.time, 2 * kTile);
  if (EVEN && own_tiles * runs_of(own_tiles) * a.in_dim <= (int64_t)1 << 18) {
    if constexpr (EVEN) {
      if (gather) launch_out<T, RP, 1, true, true, true>(a, runs_of(own_tiles), st);
      else launch_out<T, RP, 2, true, false, true>(a, runs_of(own_tiles), st);
    }
    BDH_HIP_TRY(hipGetLastError());
    *launches += 1;
    return BDH_OK;
  }
  void* u = nullptr;
  const bdh_status s = scratch(st, SLOT_ADAPTER, (size_t)(a.batch * a.time) * u_row<T, RP> * sizeof(bf16_t), &u);
  if (s != BDH_OK) return s;
  a.u = (bf16_t*)u;
  const dim3 u_grid(gather ? 1u : (uint32_t)cdiv(a.time, kTile), (uint32_t)a.batch);
  if (gather) {
    hipLaunchKernelGGL((adapter_u_kernel<T, RP, EVEN, true>), u_grid, dim3(256), 0, st, a);
    launch_out<T, RP, 1, EVEN, true, false>(a, runs_of(a.batch), st);
  } else {
    hipLaunchKernelGGL((adapter_u_kernel<T, RP, EVEN, false>), u_grid, dim3(256), 0, st, a);
    launch_out<T, RP, 4, EVEN, false, false>(a, runs_of(a.batch * cdiv(a.time, 4 * kTile)), st);
  }
  BDH_HIP_TRY(hipGetLastError());
  *launches += 2;
  return BDH_OK;
}

template <typename T, bool EVEN>
bdh_status run_ranked(const AdapterArgs& a, hipStream_t st, uint64_t* launches) {
  if (a.rank <= 16) return run_typed<T, 16, EVEN>(a, st, launches);
  if (a.rank <= 32) return run_typed<T, 32, EVEN>(a, st, launches);
  if (a.rank <= 64) return run_typed<T, 64, EVEN>(a, st, launches);
  return run_typed<T, 128, EVEN>(a, st, launches);
}

}  // namespace

bdh_status apply_adapters(const AdapterArgs& a, hipStream_t st, uint64_t* launches) {
  if (a.rank % 8 == 0 && a.in_dim % 8 == 0)
    return a.bf16 ? run_ranked<bf16_t, true>(a, st, launches) : run_ranked<float, true>(a, st, launches);
  return a.bf16 ? run_ranked<bf16_t, false>(a, st, launches) : run_ranked<float, false>(a, st, launches);
}

}  // namespace bdh
