// Low-rank adapters of many requests beside a shared projection:
//   out[b, t, :] = base[b, t, :] + scale_a (hidden[b, t, :] A_a^T) B_a^T,  a = ids[b],
// with A [n, R, D] and B [n, V, R] in bf16, base the shared projection's
// output (the logits) and out = base where ids[b] names no adapter.
//
// hidden A^T goes to the stream's scratch first (u, R values a row), scaled.
// All sums in f32.  Two forms, by the tokens of a sequence:
//
// Few (generation): a row's products are small and its adapter its own, so
// what counts is that each adapter's B is read once.  u by one workgroup a
// row in f32; then a workgroup takes a block of columns and up to kShare
// sequences of one adapter, holds the block's rows of B in registers and runs
// over the sequences' rows.  Bound by the bytes of B, base and out.
//
// Many (prompts): 16-row tiles of one sequence, so of one adapter, on the
// matrix cores.  Their f32 operands go in as bf16 parts, each the rounded rest
// of the ones before it: three parts are an f32 to 2^-24 of it, two to 2^-16.
// f32 hidden and its u take three; bf16 hidden is one, and its u takes two
// (out rounds to 2^-8).  u's parts stand side by side, as one product of two or
// three times the depth.  Bound by base and out.
#include "bdh_internal.h"

namespace bdh {
namespace {

constexpr int kFewTokens = 16;   // below: the rows' form; from here on: tiles of 16 rows
constexpr int kShare = 8;        // sequences of one adapter that a workgroup serves
constexpr int kMaxRank = 128;

typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x2_u __attribute__((ext_vector_type(2), aligned(4)));
typedef __bf16 bf16x8_u __attribute__((ext_vector_type(8), aligned(2)));
typedef __bf16 bf16x4_u __attribute__((ext_vector_type(4), aligned(2)));
typedef __bf16 bf16x2_u __attribute__((ext_vector_type(2), aligned(2)));

__device__ __forceinline__ int adapter_of(const AdapterArgs& a, int64_t b) {
  const int id = a.ids[b];
  return id >= 0 && id < a.n ? id : -1;
}

// The next bf16 part of an f32 whose rest is x.  (An infinity is one part.)
__device__ __forceinline__ bf16_t next_part(float& x) {
  const bf16_t p = (bf16_t)x;
  x = fabsf((float)p) < INFINITY ? x - (float)p : 0.0f;
  return p;
}
template <typename T> constexpr int hidden_parts = sizeof(T) == 4 ? 3 : 1;
template <typename T> constexpr int u_parts = sizeof(T) == 4 ? 3 : 2;

// Eight values of a row of n from index k on, zeros past its end.
template <typename T>
__device__ __forceinline__ void load8(const T* row, int64_t k, int64_t n, float (&x)[8]);
template <>
__device__ __forceinline__ void load8<float>(const float* row, int64_t k, int64_t n, float (&x)[8]) {
  if (k + 8 <= n) {
    const f32x4_u p = *(const f32x4_u*)(row + k), q = *(const f32x4_u*)(row + k + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = p[j];
      x[4 + j] = q[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = k + j < n ? row[k + j] : 0.0f;
  }
}
__device__ __forceinline__ bf16x8 load8_bf16(const bf16_t* row, int64_t k, int64_t n) {
  bf16x8 v;
  if (k + 8 <= n) {
    const bf16x8_u p = *(const bf16x8_u*)(row + k);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = p[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = k + j < n ? row[k + j] : (bf16_t)0.0f;
  }
  return v;
}
template <>
__device__ __forceinline__ void load8<bf16_t>(const bf16_t* row, int64_t k, int64_t n, float (&x)[8]) {
  const bf16x8 v = load8_bf16(row, k, n);
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = (float)v[j];
}

// --- few tokens ----------------------------------------------------------------
// u[row, k] f32, k < rp (zeros past the rank).  One workgroup a row; a wave
// takes every fourth k, its lanes eight columns of the dot product each.
template <typename T>
__global__ __launch_bounds__(256) void shrink_rows_kernel(const AdapterArgs a) {
  const int64_t row = blockIdx.x;
  const int id = adapter_of(a, row / a.time);
  if (id < 0) return;
  const T* h = (const T*)a.hidden + row * a.in_dim;
  const bf16_t* w = a.a + (int64_t)id * a.rank * a.in_dim;
  const float scale = a.scale[id];
  const int lane = threadIdx.x & 63;
  for (int k = threadIdx.x >> 6; k < a.rp; k += 4) {
    float s = 0.0f;
    if (k < a.rank) {
      for (int64_t d = lane * 8; d < a.in_dim; d += 512) {
        float x[8], y[8];
        load8<T>(h, d, a.in_dim, x);
        load8<bf16_t>(w + k * a.in_dim, d, a.in_dim, y);
#pragma unroll
        for (int j = 0; j < 8; ++j) s = fmaf(x[j], y[j], s);
      }
      s = wave_sum(s) * scale;
    }
    if (lane == 0) a.u[row * a.rp + k] = s;
  }
}

template <typename T, int N> struct Cols;
template <> struct Cols<float, 4> { typedef f32x4_u type; };
template <> struct Cols<float, 2> { typedef f32x2_u type; };
template <> struct Cols<bf16_t, 4> { typedef bf16x4_u type; };
template <> struct Cols<bf16_t, 2> { typedef bf16x2_u type; };
template <typename T> struct Cols<T, 1> { typedef T type __attribute__((ext_vector_type(1))); };

template <typename T, int N>
__device__ __forceinline__ void load_cols(const T* p, int n, float (&x)[N]) {
  if (n == N) {
    const typename Cols<T, N>::type v = *(const typename Cols<T, N>::type*)p;
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = (float)v[j];
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = j < n ? (float)p[j] : 0.0f;
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_cols(T* p, int n, const float (&x)[N]) {
  if (n == N) {
    typename Cols<T, N>::type v;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = (T)x[j];
    *(typename Cols<T, N>::type*)p = v;
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < n) p[j] = (T)x[j];
  }
}

// out of a block of 256 * VPT columns for the sequences of one adapter: the
// workgroups of a sequence that is the first of its adapter, or the first
// after kShare more of it, serve that one and the next kShare - 1; the others
// end at once.
template <typename T, int RP, int VPT>
__global__ __launch_bounds__(256) void expand_rows_kernel(const AdapterArgs a) {
  __shared__ int served[kShare];
  __shared__ int n_before, n_served;
  const int64_t b = blockIdx.y;
  const int id = adapter_of(a, b);
  if (id < 0 && a.out == a.base) return;
  if (threadIdx.x == 0) n_before = n_served = 0;
  __syncthreads();
  int before = 0;
  for (int64_t i = threadIdx.x; i < b; i += 256) before += adapter_of(a, i) == id;
  if (before) atomicAdd(&n_before, before);
  __syncthreads();
  if (n_before % kShare != 0) return;
  // The first kShare sequences of this adapter from b on, in order: one wave.
  if (threadIdx.x < 64) {
    int n = 0;
    for (int64_t i0 = b; i0 < a.batch && n < kShare; i0 += 64) {
      const int64_t i = i0 + threadIdx.x;
      const bool is = i < a.batch && adapter_of(a, i) == id;
      const uint64_t all = __ballot(is);
      const int at = n + __popcll(all & ((1ull << threadIdx.x) - 1));
      if (is && at < kShare) served[at] = (int)i;
      n += __popcll(all);
    }
    if (threadIdx.x == 0) n_served = n < kShare ? n : kShare;
  }
  __syncthreads();
  const int64_t v = ((int64_t)blockIdx.x * 256 + threadIdx.x) * VPT;
  if (v >= a.out_dim) return;
  const int cols = a.out_dim - v < VPT ? (int)(a.out_dim - v) : VPT;
  float w[VPT][RP];
  if (id >= 0) {
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const bf16_t* row = a.b + ((int64_t)id * a.out_dim + v + (j < cols ? j : 0)) * a.rank;
#pragma unroll
      for (int k = 0; k < RP; k += 8) {
        float x[8];
        load8<bf16_t>(row, k, a.rank, x);
#pragma unroll
        for (int q = 0; q < 8; ++q) w[j][k + q] = x[q];
      }
    }
  }
  const int n = n_served * (int)a.time;
  for (int i = 0; i < n; ++i) {
    const int s = i / (int)a.time;
    const int64_t row = (int64_t)__builtin_amdgcn_readfirstlane(served[s]) * a.time + (i - s * (int)a.time);
    const T* from = (const T*)a.base + row * a.out_dim + v;
    float x[VPT];
    load_cols<T, VPT>(from, cols, x);
    if (id >= 0) {
      const float* u = a.u + row * RP;
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < RP; ++k) sum = fmaf(u[k], w[j][k], sum);
        x[j] += sum;
      }
    }
    store_cols<T, VPT>((T*)a.out + row * a.out_dim + v, cols, x);
  }
}

// --- many tokens ---------------------------------------------------------------
// The parts of u, [row][part][rp].  A workgroup takes 16 rows of one sequence,
// its waves every fourth 32-deep step of the product.
template <typename T, int RP>
__global__ __launch_bounds__(256) void shrink_tile_kernel(const AdapterArgs a) {
  constexpr int NT = RP / 16, HP = hidden_parts<T>, UP = u_parts<T>;
  __shared__ float part[4][16][RP];
  const int64_t b = blockIdx.y;
  const int id = adapter_of(a, b);
  if (id < 0) return;
  const int64_t t0 = (int64_t)blockIdx.x * 16;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t t = t0 + (lane & 15) < a.time ? t0 + (lane & 15) : a.time - 1;
  const T* h = (const T*)a.hidden + (b * a.time + t) * a.in_dim;
  const bf16_t* w = a.a + (int64_t)id * a.rank * a.in_dim;
  floatx4 acc[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[j] = zero4();
  for (int64_t d0 = wave * 32; d0 < a.in_dim; d0 += 128) {
    const int64_t d = d0 + 8 * (lane >> 4);
    bf16x8 x[HP];
    if constexpr (HP > 1) {
      float f[8];
      load8<float>((const float*)h, d, a.in_dim, f);
#pragma unroll
      for (int q = 0; q < HP; ++q)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[q][j] = next_part(f[j]);
    } else {
      x[0] = load8_bf16((const bf16_t*)h, d, a.in_dim);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int k = j * 16 + (lane & 15);
      bf16x8 y;
      if (k < a.rank) {
        y = load8_bf16(w + k * a.in_dim, d, a.in_dim);
      } else {
#pragma unroll
        for (int q = 0; q < 8; ++q) y[q] = (bf16_t)0.0f;
      }
#pragma unroll
      for (int q = HP - 1; q >= 0; --q) acc[j] = mfma16(x[q], y, acc[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r) part[wave][acc16_row(lane, r)][j * 16 + acc16_col(lane)] = acc[j][r];
  __syncthreads();
  const float scale = a.scale[id];
  for (int i = threadIdx.x; i < 16 * RP; i += 256) {
    const int r = i / RP, k = i % RP;
    if (t0 + r >= a.time) break;
    // (Past the rank: zeros, whatever hidden holds.)
    float s = k < a.rank ? (part[0][r][k] + part[1][r][k] + part[2][r][k] + part[3][r][k]) * scale : 0.0f;
    bf16_t* u = a.u_parts + (b * a.time + t0 + r) * (UP * RP) + k;
#pragma unroll
    for (int q = 0; q < UP; ++q) u[q * RP] = next_part(s);
  }
}

// A wave's block: 64 rows of one sequence by 16 * NC columns.  Column
// NC * c + j of the block is column c of product tile j, so a lane's results
// of a row are NC neighbours.
template <typename T, int RP, int NC>
__global__ __launch_bounds__(256) void expand_tile_kernel(const AdapterArgs a) {
  constexpr int MT = 4, DEPTH = u_parts<T> * RP;
  const int64_t b = blockIdx.z;
  const int id = adapter_of(a, b);
  if (id < 0 && a.out == a.base) return;
  const int lane = threadIdx.x & 63;
  const int64_t t0 = (int64_t)blockIdx.x * (16 * MT);
  const int64_t v0 = ((int64_t)blockIdx.y * 4 + wave_id()) * (16 * NC);
  if (v0 >= a.out_dim) return;
  floatx4 acc[MT][NC];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int j = 0; j < NC; ++j) acc[m][j] = zero4();
  if (id >= 0) {
    const bf16_t* w = a.b + (int64_t)id * a.out_dim * a.rank;
#pragma unroll
    for (int s = 0; s < DEPTH; s += 32) {
      // Eight-deep slice of this lane: each of u's parts meets the same columns
      // of B.  (A depth of 48 ends half way through the last step: zeros.)
      const int k = s + 8 * (lane >> 4);
      const bool in = DEPTH % 32 == 0 || k < DEPTH;
      bf16x8 y[NC];
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        const int64_t v = v0 + NC * (lane & 15) + j;
        y[j] = load8_bf16(w + (v < a.out_dim ? v : a.out_dim - 1) * a.rank, in ? k % RP : RP, a.rank);
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int64_t t = t0 + 16 * m + (lane & 15);
        bf16x8 x = *(const bf16x8*)(a.u_parts + (b * a.time + (t < a.time ? t : a.time - 1)) * DEPTH + (in ? k : 0));
        if (!in) {
#pragma unroll
          for (int q = 0; q < 8; ++q) x[q] = (bf16_t)0.0f;
        }
#pragma unroll
        for (int j = 0; j < NC; ++j) acc[m][j] = mfma16(x, y[j], acc[m][j]);
      }
    }
  }
  const int64_t v = v0 + NC * (lane & 15);
  if (v >= a.out_dim) return;
  const int cols = a.out_dim - v < NC ? (int)(a.out_dim - v) : NC;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t t = t0 + 16 * m + acc16_row(lane, r);
      if (t >= a.time) continue;
      const int64_t at = (b * a.time + t) * a.out_dim + v;
      float x[NC];
      load_cols<T, NC>((const T*)a.base + at, cols, x);
#pragma unroll
      for (int j = 0; j < NC; ++j) x[j] += acc[m][j][r];
      store_cols<T, NC>((T*)a.out + at, cols, x);
    }
}

int padded_rank(int64_t r) { return r <= 16 ? 16 : r <= 32 ? 32 : r <= 64 ? 64 : 128; }

template <typename T, int RP>
bdh_status run_typed(AdapterArgs a, hipStream_t st, uint64_t* launches) {
  const int64_t rows = a.batch * a.time;
  void* u = nullptr;
  const size_t bytes = (size_t)rows * RP * (a.time < kFewTokens ? sizeof(float) : u_parts<T> * sizeof(bf16_t));
  const bdh_status s = scratch(st, SLOT_ADAPTER, bytes, &u);
  if (s != BDH_OK) return s;
  a.u = (float*)u;
  a.u_parts = (bf16_t*)u;
  a.rp = RP;
  if (a.time < kFewTokens) {
    constexpr int VPT = RP <= 16 ? 4 : RP <= 32 ? 2 : 1;
    hipLaunchKernelGGL((shrink_rows_kernel<T>), dim3((uint32_t)rows), dim3(256), 0, st, a);
    hipLaunchKernelGGL((expand_rows_kernel<T, RP, VPT>),
                       dim3((uint32_t)((a.out_dim + 256 * VPT - 1) / (256 * VPT)), (uint32_t)a.batch), dim3(256), 0,
                       st, a);
  } else {
    constexpr int NC = 4;
    hipLaunchKernelGGL((shrink_tile_kernel<T, RP>), dim3((uint32_t)((a.time + 15) / 16), (uint32_t)a.batch),
                       dim3(256), 0, st, a);
    hipLaunchKernelGGL((expand_tile_kernel<T, RP, NC>),
                       dim3((uint32_t)((a.time + 63) / 64), (uint32_t)((a.out_dim + 64 * NC - 1) / (64 * NC)),
                            (uint32_t)a.batch),
                       dim3(256), 0, st, a);
  }
  BDH_HIP_TRY(hipGetLastError());
  *launches += 2;
  return BDH_OK;
}

template <typename T>
bdh_status run_ranked(const AdapterArgs& a, hipStream_t st, uint64_t* launches) {
  switch (padded_rank(a.rank)) {
    case 16: return run_typed<T, 16>(a, st, launches);
    case 32: return run_typed<T, 32>(a, st, launches);
    case 64: return run_typed<T, 64>(a, st, launches);
    default: return run_typed<T, 128>(a, st, launches);
  }
}

}  // namespace

bdh_status apply_adapters(const AdapterArgs& a, hipStream_t st, uint64_t* launches) {
  return a.bf16 ? run_ranked<bf16_t>(a, st, launches) : run_ranked<float>(a, st, launches);
}

}  // namespace bdh
