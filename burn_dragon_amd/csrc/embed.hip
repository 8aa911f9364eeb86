// Token embedding and its gradient.
//   out[i] = scale E[t_i], or scale LN(E[t_i]) (eps 1e-5, no weights): the model's
//   input norm; zeros where t_i is no row of E.
//   grad[v] = scale sum over i with t_i = v of g_i, in the order of i; with the norm
//   the transposed Jacobian of that sum, since all tokens of an id share one row:
//   J^T s = r (s - mean(s) - x mean(s x)),  x = (E[v] - mean) r,  r = 1 / sqrt(var + eps).
//
// The gradient goes by sorted tokens, without atomics on values, so a call repeats
// bit for bit: the positions are sorted by id (a stable radix sort of up to 9 bits
// a pass: one pass for up to 511 rows of E, two for 2^18 - 1; in one launch up to
// 4096 tokens; up to 64 need no sort), then each wave sums the rows of a run of positions, and
// writes the ids that lie within it.  An id that runs on into the next runs leaves partial sums,
// which a second launch joins in their order.  The rows without a token are cleared
// by the sort's launches beside their own work.
//
// Bound by the bytes (rows in, rows out) where there are many tokens, else by the chain of
// dependent launches: 65536 tokens of 1024 bf16 columns of a table of 32000, 40 us (3.3 TB/s
// of results, 4.0 with the rows); the gradient of 32768 such tokens to 131072 rows, 94 us: two
// sort passes, which clear 268 MB, sums 32 (67 MB read in the order of the ids, the met rows written) and
// join 11; of 16384 tokens to 256 rows of 256 f32 columns, 23 us in four launches.
#include <type_traits>

#include "bdh_internal.h"

namespace bdh {
namespace {

typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf16x4_u __attribute__((ext_vector_type(4), aligned(2)));
typedef __bf16 bf16x8_u __attribute__((ext_vector_type(8), aligned(2)));
template <typename T, int VEC> struct Vec;
template <> struct Vec<float, 4> { typedef f32x4_u type; };
template <> struct Vec<bf16_t, 4> { typedef bf16x4_u type; };
template <> struct Vec<bf16_t, 8> { typedef bf16x8_u type; };

// A row of n columns held by a wave: lane l has columns VEC (l + 64 k) ..+VEC-1, zeros
// past the end.
template <typename T, int VEC, int PER>
struct Row {
  float v[PER][VEC];

  template <typename F>
  __device__ __forceinline__ void each(F&& f) {
#pragma unroll
    for (int k = 0; k < PER; ++k)
#pragma unroll
      for (int j = 0; j < VEC; ++j) f(v[k][j], VEC * 64 * k + j);
  }
  __device__ __forceinline__ void clear() {
    each([](float& x, int) { x = 0.0f; });
  }
  // (The lane is opaque at each row: else the comparisons with the row's end, one a column,
  // are kept for the whole kernel, in more scalar registers than there are.)
  static __device__ __forceinline__ int anew(int lane) {
    asm volatile("" : "+v"(lane));
    return lane;
  }
  template <typename S>  // of T, or partial sums of f32
  __device__ __forceinline__ void load(const S* row, int n, int lane_) {
    const int lane = anew(lane_);
    constexpr int W = sizeof(S) == 4 ? 4 : VEC;
    typedef typename Vec<S, W>::type V;
#pragma unroll
    for (int k = 0; k < PER; ++k)
#pragma unroll
      for (int q = 0; q < VEC; q += W) {
        const int c = VEC * (lane + 64 * k) + q;
        if (c + W <= n) {
          const V x = *(const V*)(row + c);
#pragma unroll
          for (int j = 0; j < W; ++j) v[k][q + j] = (float)x[j];
        } else {
#pragma unroll
          for (int j = 0; j < W; ++j) v[k][q + j] = c + j < n ? (float)row[c + j] : 0.0f;
        }
      }
  }
  template <typename S>
  __device__ __forceinline__ void store(S* row, int n, int lane_) const {
    const int lane = anew(lane_);
    constexpr int W = sizeof(S) == 4 ? 4 : VEC;
    typedef typename Vec<S, W>::type V;
#pragma unroll
    for (int k = 0; k < PER; ++k)
#pragma unroll
      for (int q = 0; q < VEC; q += W) {
        const int c = VEC * (lane + 64 * k) + q;
        if (c + W <= n) {
          V x;
#pragma unroll
          for (int j = 0; j < W; ++j) x[j] = (S)v[k][q + j];
          *(V*)(row + c) = x;
        } else {
#pragma unroll
          for (int j = 0; j < W - 1; ++j)
            if (c + j < n) row[c + j] = (S)v[k][q + j];
        }
      }
  }
  __device__ __forceinline__ float sum() const {
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < PER; ++k)
#pragma unroll
      for (int j = 0; j < VEC; j += 4) s += (v[k][j] + v[k][j + 1]) + (v[k][j + 2] + v[k][j + 3]);
    return wave_sum(s);
  }
  __device__ __forceinline__ float dot(const Row& u) const {
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < PER; ++k)
#pragma unroll
      for (int j = 0; j < VEC; j += 4)
        s += (v[k][j] * u.v[k][j] + v[k][j + 1] * u.v[k][j + 1]) +
             (v[k][j + 2] * u.v[k][j + 2] + v[k][j + 3] * u.v[k][j + 3]);
    return wave_sum(s);
  }
  // Less its mean, zeros past column n; returns 1 / sqrt(var + eps).  The mean is taken
  // twice: the first one's rounding is large beside the values of a row that lies far
  // from zero.
  __device__ __forceinline__ float center(int n, int lane_) {
    const int lane = anew(lane_);
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {
      const float mean = sum() / (float)n;
      each([&](float& x, int c) { x = c + VEC * lane < n ? x - mean : 0.0f; });
    }
    return 1.0f / sqrtf(dot(*this) / (float)n + 1e-5f);
  }
};

// A wave takes EACH neighbouring tokens, their rows asked for together: with one token a
// wave, what counted was the wait for its id, then for its row (65536 tokens, D 1024, bf16:
// 52 us a call, with two 41).
template <typename T, int VEC, int PER, int EACH, bool NORM>
__global__ __launch_bounds__(256) void embed_kernel(const EmbedArgs a) {
  const int64_t i0 = ((int64_t)blockIdx.x * 4 + wave_id()) * EACH;
  if (i0 >= a.n) return;
  const int lane = threadIdx.x & 63, D = (int)a.embd;
  Row<T, VEC, PER> v[EACH];
  bool there[EACH];
  int id[EACH];
#pragma unroll
  for (int q = 0; q < EACH; ++q) id[q] = a.tokens[i0 + q < a.n ? i0 + q : a.n - 1];
#pragma unroll
  for (int q = 0; q < EACH; ++q) {
    there[q] = id[q] >= 0 && id[q] < a.vocab;
    v[q].load((const T*)a.table + (int64_t)(there[q] ? id[q] : 0) * D, D, lane);
  }
#pragma unroll
  for (int q = 0; q < EACH; ++q) {
    if (i0 + q >= a.n) break;
    float f = a.scale;
    if (NORM) f *= v[q].center(D, lane);
    v[q].each([&](float& x, int) { x = there[q] ? x * f : 0.0f; });
    v[q].store((T*)a.out + (i0 + q) * D, D, lane);
  }
}

// --- the order of the positions by id -----------------------------------------------
constexpr int kMostBins = 512;                              // a pass's digits
// A workgroup's positions: 16 waves have ROUNDS times 64 neighbours each.
constexpr int kWaves = 16, kMostRounds = 4;
constexpr int items(int rounds) { return 64 * rounds * kWaves; }
constexpr int kSmall = items(kMostRounds);  // of the sort in one launch

// The key of position i: its id, or vocab (past all ids) where it is none.
__device__ __forceinline__ uint32_t key_of(const SortArgs& s, int64_t i) {
  if (s.keys) return s.keys[i];
  const int id = s.tokens[i];
  return id >= 0 && id < (int)s.vocab ? (uint32_t)id : (uint32_t)s.vocab;
}

// The workgroups past the sort's own clear a share of the table's gradient.
__device__ void clear_share(const SortArgs& s, int block, int blocks) {
  typedef unsigned int u32x4_2 __attribute__((ext_vector_type(4), aligned(2)));
  const int64_t stride = (int64_t)blocks * 16384;
  for (int64_t i = s.clear_from + ((int64_t)block * 1024 + threadIdx.x) * 16; i < s.clear_to; i += stride) {
    if (i + 16 <= s.clear_to) {
      *(u32x4_2*)(s.clear + i) = u32x4_2{0, 0, 0, 0};
    } else {
      for (int64_t j = i; j < s.clear_to; j += 2) *(uint16_t*)(s.clear + j) = 0;
    }
  }
}

// counts[workgroup][digit].
template <int ROUNDS>
__global__ __launch_bounds__(1024) void digit_counts_kernel(const SortArgs s) {
  if ((int)blockIdx.x >= s.blocks) return clear_share(s, (int)blockIdx.x - s.blocks, (int)gridDim.x - s.blocks);
  __shared__ uint32_t bins[kMostBins];
  for (int d = threadIdx.x; d < s.bins; d += 1024) bins[d] = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * items(ROUNDS);
#pragma unroll
  for (int j = 0; j < items(ROUNDS); j += 1024) {
    const int64_t i = i0 + j + threadIdx.x;
    if (i < s.n) atomicAdd(&bins[(key_of(s, i) >> s.shift) & (s.bins - 1)], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < s.bins; d += 1024) s.counts[(int64_t)blockIdx.x * s.bins + d] = bins[d];
}

// The places of a workgroup's positions, stable: wave w has 64 ROUNDS neighbours.
// key(j), 0 <= j < 64 ROUNDS of the lane's wave: -1 where there is none.  first(digit):
// the place of the workgroup's first one.  put(j, key, place).
struct SortMemory {
  uint32_t at[kWaves][kMostBins];  // counts, then next places
  uint32_t total[kMostBins];
  uint32_t sums[8];
};
template <int ROUNDS, typename Key, typename First, typename Put>
__device__ __forceinline__ void sort_step(SortMemory& mem, int shift, int bins, const Key& key, const First& first,
                                          const Put& put) {
  const int lane = threadIdx.x & 63, w = wave_id();
  for (int d = threadIdx.x; d < kWaves * kMostBins; d += 1024) (&mem.at[0][0])[d] = 0;
  __syncthreads();
  int64_t keys[ROUNDS];
  uint32_t rank[ROUNDS];
#pragma unroll
  for (int q = 0; q < ROUNDS; ++q) keys[q] = key(64 * q + lane);
  // Each round's ranks within its digit; the digit's last lane moves the count on.
#pragma unroll
  for (int q = 0; q < ROUNDS; ++q) {
    const int digit = (int)(keys[q] >> shift) & (bins - 1);
    uint64_t same = __ballot(keys[q] >= 0);
    for (int b = 1; b < bins; b <<= 1) {
      const uint64_t set = __ballot((digit & b) != 0);
      same &= (digit & b) ? set : ~set;
    }
    if (keys[q] >= 0) {
      rank[q] = mem.at[w][digit] + __popcll(same & ((1ull << lane) - 1));
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if ((same >> lane) == 1) mem.at[w][digit] = rank[q] + 1;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  __syncthreads();
  // Counts to places: waves in order after the digit's first place.
  first(mem);
  if ((int)threadIdx.x < bins) {
    uint32_t place = mem.total[threadIdx.x];
#pragma unroll
    for (int q = 0; q < kWaves; ++q) {
      const uint32_t c = mem.at[q][threadIdx.x];
      mem.at[q][threadIdx.x] = place;
      place += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < ROUNDS; ++q)
    if (keys[q] >= 0)
      put(64 * q + lane, (uint32_t)keys[q], mem.at[w][(int)(keys[q] >> shift) & (bins - 1)] + rank[q]);
  __syncthreads();
}
// mem.total[d]: the sum over the digits before d, from its own; plus[d] added.  512 threads.
__device__ __forceinline__ void scan_digits(SortMemory& mem, uint32_t own, uint32_t plus, int bins) {
  const int lane = threadIdx.x & 63, w = wave_id();
  uint32_t s = own;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t v = (uint32_t)__shfl_up((int)s, o, 64);
    if (lane >= o) s += v;
  }
  if (lane == 63 && w < 8) mem.sums[w] = s;
  __syncthreads();
  if (w < 8) {
    for (int q = 0; q < w; ++q) s += mem.sums[q];
    if ((int)threadIdx.x < bins) mem.total[threadIdx.x] = s - own + plus;
  }
  __syncthreads();
}

template <int ROUNDS>
__global__ __launch_bounds__(1024) void digit_scatter_kernel(const SortArgs s) {
  if ((int)blockIdx.x >= s.blocks) return clear_share(s, (int)blockIdx.x - s.blocks, (int)gridDim.x - s.blocks);
  __shared__ SortMemory mem;
  __shared__ uint32_t half[2][kMostBins];
  const int mine = (int)blockIdx.x;
  const int64_t i0 = (int64_t)mine * items(ROUNDS) + wave_id() * 64 * ROUNDS;
  // Of a digit: all its positions, and those of earlier workgroups, by two threads.
  uint32_t total = 0, before = 0;
  {
    const int digit = (int)threadIdx.x & (kMostBins - 1);
    if (digit < s.bins) {
#pragma unroll 8
      for (int b = (int)threadIdx.x >> 9; b < s.blocks; b += 2) {
        const uint32_t c = s.counts[(int64_t)b * s.bins + digit];
        total += c;
        before += b < mine ? c : 0;
      }
    }
  }
  uint32_t from[ROUNDS];
#pragma unroll
  for (int q = 0; q < ROUNDS; ++q) {
    const int64_t i = i0 + 64 * q + ((int)threadIdx.x & 63);
    from[q] = s.order && i < s.n ? s.order[i] : (uint32_t)i;
  }
  sort_step<ROUNDS>(
      mem, s.shift, s.bins, [&](int j) { return i0 + j < s.n ? (int64_t)key_of(s, i0 + j) : (int64_t)-1; },
      [&](SortMemory& m) {
        if (threadIdx.x >= kMostBins) {
          half[0][threadIdx.x - kMostBins] = total;
          half[1][threadIdx.x - kMostBins] = before;
        }
        __syncthreads();
        if (threadIdx.x < kMostBins) {
          total += half[0][threadIdx.x];
          before += half[1][threadIdx.x];
        }
        scan_digits(m, threadIdx.x < kMostBins ? total : 0, before, s.bins);
      },
      [&](int j, uint32_t key, uint32_t place) {
        s.keys_out[place] = key;
        s.order_out[place] = from[j >> 6];
      });
}

// All passes of up to 4096 positions.
__global__ __launch_bounds__(1024) void sort_small_kernel(const SortArgs s) {
  if (blockIdx.x >= 1) return clear_share(s, (int)blockIdx.x - 1, (int)gridDim.x - 1);
  __shared__ SortMemory mem;
  __shared__ uint32_t keys[kSmall], order[kSmall];
  const int i0 = wave_id() * 64 * kMostRounds, n = (int)s.n;
  for (int pass = 0; pass < s.passes; ++pass) {
    const bool last = pass + 1 == s.passes;
    uint32_t from[kMostRounds];
#pragma unroll
    for (int q = 0; q < kMostRounds; ++q) {
      const int i = i0 + 64 * q + ((int)threadIdx.x & 63);
      from[q] = pass > 0 && i < n ? order[i] : (uint32_t)i;
    }
    sort_step<kMostRounds>(
        mem, pass * s.shift, s.bins,
        [&](int j) {
          if (i0 + j >= n) return (int64_t)-1;
          return (int64_t)(pass > 0 ? keys[i0 + j] : key_of(s, i0 + j));
        },
        [&](SortMemory& m) {
          uint32_t own = 0;
          if ((int)threadIdx.x < s.bins)
            for (int q = 0; q < kWaves; ++q) own += m.at[q][threadIdx.x];
          scan_digits(m, own, 0, s.bins);
        },
        [&](int j, uint32_t key, uint32_t place) {
          (last ? s.keys_out : keys)[place] = key;
          (last ? s.order_out : order)[place] = from[j >> 6];
        });
  }
}

// --- the sums ---------------------------------------------------------------------------
// The columns of a workgroup: with the norm all of a row, else a slice of it (blockIdx.y),
// so that a wave holds few of each row, and many rows.
struct Columns {
  int row, first, n;
};
__device__ __forceinline__ Columns columns_of(const EmbedArgs& a, int width) {
  const int D = (int)a.embd, first = (int)blockIdx.y * width;
  return Columns{D, first, D - first < width ? D - first : width};
}

// The sum of id's rows, scaled and through the norm, to its row of the gradient.
template <typename T, int VEC, int PER>
__device__ __forceinline__ void write_row(const EmbedArgs& a, const Columns& c, uint32_t id, Row<T, VEC, PER>& s,
                                          int lane) {
  const int D = c.n;
  s.each([&](float& x, int) { x *= a.scale; });
  if (a.norm) {
    Row<T, VEC, PER> x;
    x.load((const T*)a.table + (int64_t)id * c.row, D, lane);
    const float r = x.center(D, lane);
    x.each([&](float& v, int) { v *= r; });
    const float mean = s.sum() / (float)D, along = s.dot(x) / (float)D;
#pragma unroll
    for (int k = 0; k < PER; ++k)
#pragma unroll
      for (int j = 0; j < VEC; ++j) s.v[k][j] = (s.v[k][j] - mean - x.v[k][j] * along) * r;
  }
  T* out = (T*)a.out + (int64_t)id * c.row + c.first;
  if (a.accumulate) {
    Row<T, VEC, PER> old;
    old.load(out, D, lane);
#pragma unroll
    for (int k = 0; k < PER; ++k)
#pragma unroll
      for (int j = 0; j < VEC; ++j) s.v[k][j] += old.v[k][j];
  }
  s.store(out, D, lane);
}

template <typename T, int VEC, int PER>
__device__ __forceinline__ void add(Row<T, VEC, PER>& s, const Row<T, VEC, PER>& g) {
#pragma unroll
  for (int k = 0; k < PER; ++k)
#pragma unroll
    for (int j = 0; j < VEC; ++j) s.v[k][j] += g.v[k][j];
}

// A wave sums the rows of positions [run * a.run, ..), whose ids and places one load each
// takes.  part [runs][2][D]: the sum of the run's first id where that id began before it,
// of its last where it goes on after it; an id that does both is in the first.
template <typename T, int VEC, int PER>
__global__ __launch_bounds__(256) void embed_sums_kernel(const EmbedArgs a) {
  const int run = (int)blockIdx.x * 4 + wave_id(), lane = threadIdx.x & 63;
  const Columns c = columns_of(a, VEC * PER * 64);
  const int64_t p0 = (int64_t)run * a.run;
  if (p0 >= a.n) return;
  const int n = (int)(a.n - p0 < a.run ? a.n - p0 : a.run);
  // Lane l: position p0 + l - 1 (a.run + 2 <= 64 of them).
  const int64_t at = p0 + lane - 1;
  const bool in = at >= 0 && at < a.n && lane <= a.run + 1;
  const uint32_t none = ~0u;
  const uint32_t key = in ? a.keys[at] : none, place = in ? a.order[at] : 0;
  const auto id_at = [&](int p) { return (uint32_t)__builtin_amdgcn_readlane((int)key, p + 1); };
  uint32_t id = id_at(0);
  if (id >= (uint32_t)a.vocab) return;
  bool begun = id_at(-1) == id;  // before this run
  Row<T, VEC, PER> s;
  s.clear();
  const auto to_part = [&](int which) { s.store(a.part + ((int64_t)run * 2 + which) * c.row + c.first, c.n, lane); };
  constexpr int AHEAD = 64 / (VEC * PER);  // rows asked for together
  for (int p = 0; p < n; p += AHEAD) {
    Row<T, VEC, PER> g[AHEAD];
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) {
      const uint32_t i = (uint32_t)__builtin_amdgcn_readlane((int)place, (p + q < n ? p + q : n - 1) + 1);
      g[q].load((const T*)a.grad + (int64_t)i * c.row + c.first, c.n, lane);
    }
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) {
      if (p + q >= n) break;
      if (id_at(p + q) != id) {
        if (begun) to_part(0);
        else write_row(a, c, id, s, lane);
        id = id_at(p + q);
        begun = false;
        if (id >= (uint32_t)a.vocab) return;
        s.clear();
      }
      add(s, g[q]);
    }
  }
  if (begun) to_part(0);
  else if (id_at(n) == id) to_part(1);
  else write_row(a, c, id, s, lane);
}

// A workgroup for each run: joins the id that begins in it and goes on past it.  (An id that most
// tokens have is one workgroup's a slice of columns: 131072 tokens of one id 125 us at 256 f32
// columns with the norm, 236 at 1024 of bf16.)
constexpr int kJoinWaves = 8;
template <typename T, int VEC, int PER>
__global__ __launch_bounds__(64 * kJoinWaves) void embed_join_kernel(const EmbedArgs a) {
  __shared__ float sums[kJoinWaves][VEC * PER * 64];
  const int run = (int)blockIdx.x, lane = threadIdx.x & 63, w = wave_id();
  const Columns c = columns_of(a, VEC * PER * 64);
  const int64_t p0 = (int64_t)run * a.run, end = p0 + a.run;
  if (end >= a.n) return;
  const uint32_t id = a.keys[end], before = a.keys[end - 1], first = a.keys[p0], last = p0 > 0 ? a.keys[p0 - 1] : ~0u;
  if (id >= (uint32_t)a.vocab || before != id) return;
  if (first == id && last == id) return;  // began earlier
  // The runs from the next one on that begin with this id too, 64 at a time.
  const int runs = (int)((a.n + a.run - 1) / a.run);
  int n = 1;
  for (;; n += 64) {
    const int r = run + n + lane;
    const uint64_t is = __ballot(r < runs && a.keys[(int64_t)(r < runs ? r : run) * a.run] == id);
    if (is != ~0ull) {
      n += __builtin_ctzll(~is);
      break;
    }
  }
  // This run's second sum, then the first of each of those, a share a wave.
  const int q0 = (int)((int64_t)n * w / kJoinWaves), q1 = (int)((int64_t)n * (w + 1) / kJoinWaves);
  Row<T, VEC, PER> s;
  s.clear();
  constexpr int AHEAD = 64 / (VEC * PER);
  for (int q = q0; q < q1; q += AHEAD) {
    Row<T, VEC, PER> g[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int r = q + k < q1 ? q + k : q1 - 1;
      g[k].load(a.part + ((int64_t)(run + r) * 2 + (r == 0 ? 1 : 0)) * c.row + c.first, c.n, lane);
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (q + k < q1) add(s, g[k]);
  }
  s.store(sums[w], VEC * PER * 64, lane);
  __syncthreads();
  if (w > 0) return;
  for (int q = 1; q < kJoinWaves; ++q) {
    Row<T, VEC, PER> g;
    g.load(sums[q], VEC * PER * 64, lane);
    add(s, g);
  }
  write_row(a, c, id, s, lane);
}

// Up to 64 tokens in one launch, their ids in the lanes of each wave: wave i < n sums the rows
// of token i's id, if it is the id's first, in order; the waves after them clear the rows
// without a token.
template <typename T, int VEC, int PER>
__global__ __launch_bounds__(256) void embed_few_kernel(const EmbedArgs a) {
  const int lane = threadIdx.x & 63, n = (int)a.n, vocab = (int)a.vocab;
  const int64_t wave = (int64_t)blockIdx.x * 4 + wave_id();
  const Columns c = columns_of(a, VEC * PER * 64);
  const int own = lane < n ? a.tokens[lane] : -1;
  Row<T, VEC, PER> s;
  s.clear();
  if (wave < n) {
    const int id = __builtin_amdgcn_readlane(own, (int)wave);
    uint64_t same = __ballot(own == id);
    if (id < 0 || id >= vocab || __builtin_ctzll(same) != (int)wave) return;
    constexpr int AHEAD = 64 / (VEC * PER);  // rows asked for together
    while (same != 0) {
      Row<T, VEC, PER> g[AHEAD];
      uint64_t rest = same;
#pragma unroll
      for (int q = 0; q < AHEAD; ++q) {
        const int i = __builtin_ctzll(rest);
        if ((rest & (rest - 1)) != 0) rest &= rest - 1;  // (past the last: the last again)
        g[q].load((const T*)a.grad + (int64_t)i * c.row + c.first, c.n, lane);
      }
#pragma unroll
      for (int q = 0; q < AHEAD; ++q) {
        if (same != 0) add(s, g[q]);
        same &= same - 1;
      }
    }
    write_row(a, c, (uint32_t)id, s, lane);
    return;
  }
  if (a.accumulate) return;
  const int64_t waves = (int64_t)gridDim.x * 4 - n;
  for (int64_t v = wave - n; v < vocab; v += waves)
    if (__ballot(own == (int)v) == 0) s.store((T*)a.out + v * c.row + c.first, c.n, lane);
}

unsigned cdiv(int64_t a, int64_t b) { return (unsigned)((a + b - 1) / b); }

// f(VEC, PER) for rows of D columns.
template <typename T, typename F>
void by_columns(int64_t D, F&& f) {
  const auto call = [&](auto vec, auto per) { f(vec, per); };
  typedef std::integral_constant<int, 1> one;
  typedef std::integral_constant<int, 2> two;
  typedef std::integral_constant<int, 4> four;
  typedef std::integral_constant<int, 8> eight;
  if (D <= 256) return call(four{}, one{});
  if constexpr (sizeof(T) == 4) {
    if (D <= 512) return call(four{}, two{});
    if (D <= 1024) return call(four{}, four{});
    return call(four{}, eight{});
  } else {
    if (D <= 512) return call(eight{}, one{});
    if (D <= 1024) return call(eight{}, two{});
    return call(eight{}, four{});
  }
}

template <typename T>
void launch_rows(const EmbedArgs& a, hipStream_t st) {
  by_columns<T>(a.embd, [&](auto vec, auto per) {
    constexpr int VEC = decltype(vec)::value, PER = decltype(per)::value, EACH = VEC * PER >= 16 ? 2 : 4;
    // Several tokens a wave where there are enough for the chip.
    if (a.n >= 16384) {
      const dim3 grid(cdiv(a.n, 4 * EACH));
      if (a.norm) hipLaunchKernelGGL((embed_kernel<T, VEC, PER, EACH, true>), grid, dim3(256), 0, st, a);
      else hipLaunchKernelGGL((embed_kernel<T, VEC, PER, EACH, false>), grid, dim3(256), 0, st, a);
    } else {
      const dim3 grid(cdiv(a.n, 4));
      if (a.norm) hipLaunchKernelGGL((embed_kernel<T, VEC, PER, 1, true>), grid, dim3(256), 0, st, a);
      else hipLaunchKernelGGL((embed_kernel<T, VEC, PER, 1, false>), grid, dim3(256), 0, st, a);
    }
  });
}

// Whether embed_few_kernel takes a call (us, sorted / so: 64 tokens to 256 rows of 1024 f32
// columns 13 / 4, of 256 with the norm 31 / 5, to 250000 rows of 512 bf16 columns 45 / 34; where
// all 64 tokens have one id, 14 / 8, and 24 / 33 at 2048 f32 columns with the norm).
template <typename T>
bool launch_few(const EmbedArgs& a, hipStream_t st) {
  if (a.n > 64) return false;
  const int64_t slice = sizeof(T) == 4 ? 256 : 512;
  by_columns<T>(a.norm || a.embd < slice ? a.embd : slice, [&](auto vec, auto per) {
    constexpr int VEC = decltype(vec)::value, PER = decltype(per)::value;
    const int64_t rows = a.accumulate ? 0 : (a.vocab < 8192 ? a.vocab : 8192);  // waves that clear
    hipLaunchKernelGGL((embed_few_kernel<T, VEC, PER>), dim3(cdiv(a.n + rows, 4), cdiv(a.embd, VEC * PER * 64)),
                       dim3(256), 0, st, a);
  });
  return true;
}

template <typename T>
void launch_sums(const EmbedArgs& a, int64_t runs, hipStream_t st) {
  const int64_t slice = sizeof(T) == 4 ? 256 : 512;
  by_columns<T>(a.norm || a.embd < slice ? a.embd : slice, [&](auto vec, auto per) {
    constexpr int VEC = decltype(vec)::value, PER = decltype(per)::value;
    const unsigned slices = cdiv(a.embd, VEC * PER * 64);
    hipLaunchKernelGGL((embed_sums_kernel<T, VEC, PER>), dim3(cdiv(runs, 4), slices), dim3(256), 0, st, a);
    if (runs > 1)
      hipLaunchKernelGGL((embed_join_kernel<T, VEC, PER>), dim3((unsigned)runs, slices), dim3(64 * kJoinWaves), 0, st,
                         a);
  });
}

}  // namespace

bdh_status embed_tokens(const EmbedArgs& a, hipStream_t st) {
  if (a.bf16) launch_rows<bf16_t>(a, st);
  else launch_rows<float>(a, st);
  BDH_HIP_TRY(hipGetLastError());
  return BDH_OK;
}

bdh_status embed_tokens_vjp(EmbedArgs a, hipStream_t st, uint64_t* launches) {
  if (a.bf16 ? launch_few<bf16_t>(a, st) : launch_few<float>(a, st)) {
    *launches += 1;
    BDH_HIP_TRY(hipGetLastError());
    return BDH_OK;
  }
  int bits = 1;
  while (a.vocab >> bits) ++bits;  // of the keys 0 .. vocab
  const int passes = (bits + 8) / 9, per_pass = (bits + passes - 1) / passes;
  // Short sorts have one round a workgroup, since what counts is a workgroup's chain; many
  // workgroups each read all counts, the square of their number (us a call, one round / four:
  // 16384 tokens of 256 ids 20 / 24, of 131072 44 / 54; 262144 88 / 86 and 148 / 150; 1048576
  // 418 / 346 and 580 / 421).
  const int rounds = a.n <= kSmall || a.n > 131072 ? kMostRounds : 1;
  const int64_t blocks = cdiv(a.n, items(rounds));
  // Short runs where there are few, and where most ids end in one, whose row's norm a wave
  // takes in turn (us, runs of 4 / 8 / 16: 512 tokens to 32000 rows of 256 f32 columns with the
  // norm 27 / 29 / 41, 4096 34 / 40 / 52, 16384 47 / 46 / 56, to 256 rows 25 / 23 / 21; of 1024
  // columns without the norm 4096 tokens 38 / 35 / 35, 16384 85 / 68 / 59).
  a.run = a.n <= 4096 ? 4 : a.n > 32768 ? 32 : a.norm && a.vocab > a.n / 8 ? 8 : 16;
  const int64_t runs = cdiv(a.n, a.run);
  const int64_t words = 4 * a.n + (blocks << per_pass);
  void* buf = nullptr;
  const bdh_status s = scratch(st, SLOT_EMBED, (size_t)(words + 2 * runs * a.embd) * 4, &buf);
  if (s != BDH_OK) return s;
  uint32_t* keys[2] = {(uint32_t*)buf, (uint32_t*)buf + a.n};
  uint32_t* order[2] = {keys[1] + a.n, keys[1] + 2 * a.n};
  a.part = (float*)buf + words;
  SortArgs q{};
  q.tokens = a.tokens;
  q.n = a.n;
  q.vocab = a.vocab;
  q.bins = 1 << per_pass;
  q.passes = passes;
  q.blocks = (int)blocks;
  q.counts = order[1] + a.n;
  q.clear = (char*)a.out;
  // Bytes to clear, an equal share a launch, by up to 1024 workgroups of 1024 threads.
  const int64_t bytes = a.accumulate ? 0 : a.vocab * a.embd * (a.bf16 ? 2 : 4);
  const int sorts = blocks == 1 ? 1 : 2 * passes;
  int launch = 0;
  const auto grid = [&] {
    q.clear_from = bytes * launch / sorts / 16 * 16;
    q.clear_to = launch + 1 == sorts ? bytes : bytes * (launch + 1) / sorts / 16 * 16;
    ++launch;
    const int64_t more = cdiv(q.clear_to - q.clear_from, 16384);
    return dim3((unsigned)(q.blocks + (more < 1024 ? more : 1024)));
  };
  if (blocks == 1) {
    q.shift = per_pass;
    q.keys_out = keys[0];
    q.order_out = order[0];
    hipLaunchKernelGGL(sort_small_kernel, grid(), dim3(1024), 0, st, q);
  } else {
    for (int p = 0; p < passes; ++p) {
      q.shift = p * per_pass;
      q.keys_out = keys[p & 1];
      q.order_out = order[p & 1];
      if (rounds == 1) {
        hipLaunchKernelGGL(digit_counts_kernel<1>, grid(), dim3(1024), 0, st, q);
        hipLaunchKernelGGL(digit_scatter_kernel<1>, grid(), dim3(1024), 0, st, q);
      } else {
        hipLaunchKernelGGL(digit_counts_kernel<kMostRounds>, grid(), dim3(1024), 0, st, q);
        hipLaunchKernelGGL(digit_scatter_kernel<kMostRounds>, grid(), dim3(1024), 0, st, q);
      }
      q.keys = q.keys_out;
      q.order = q.order_out;
    }
  }
  a.keys = q.keys_out;
  a.order = q.order_out;
  if (a.bf16) launch_sums<bf16_t>(a, runs, st);
  else launch_sums<float>(a, runs, st);
  *launches += (uint64_t)sorts + (runs > 1 ? 2 : 1);
  BDH_HIP_TRY(hipGetLastError());
  return BDH_OK;
}

}  // namespace bdh
