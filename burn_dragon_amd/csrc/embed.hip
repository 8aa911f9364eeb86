// Token embedding and its gradient.
//   out[i] = scale E[t_i], or scale LN(E[t_i]) (eps 1e-5, no weights): the model's
//   input norm; zeros where t_i is no row of E.
//   grad[v] = scale sum over i with t_i = v of g_i, in the order of i; with the norm
//   the transposed Jacobian of that sum, since all tokens of an id share one row:
//   J^T s = r (s - mean(s) - x mean(s x)),  x = (E[v] - mean) r,  r = 1 / sqrt(var + eps).
//
// The gradient goes by sorted tokens, without atomics on values, so a call repeats
// bit for bit: the positions are sorted by id (a stable radix sort of up to 9 bits
// a pass: one pass for up to 511 rows of E, two for 2^18 - 1), then each wave sums the rows of a
// run of positions, and writes the ids that lie within it.  An id that runs on into
// the next runs leaves partial sums, which a second launch joins in their order.
#include "bdh_internal.h"

namespace bdh {
namespace {

typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf16x4_u __attribute__((ext_vector_type(4), aligned(2)));

// Four neighbouring values of a row of n from c on, zeros past its end.
__device__ __forceinline__ floatx4 load4(const float* row, int c, int n) {
  if (c + 4 <= n) return *(const f32x4_u*)(row + c);
  floatx4 v = zero4();
#pragma unroll
  for (int j = 0; j < 3; ++j)
    if (c + j < n) v[j] = row[c + j];
  return v;
}
__device__ __forceinline__ floatx4 load4(const bf16_t* row, int c, int n) {
  floatx4 v = zero4();
  if (c + 4 <= n) {
    const bf16x4_u p = *(const bf16x4_u*)(row + c);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = (float)p[j];
  } else {
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (c + j < n) v[j] = (float)row[c + j];
  }
  return v;
}
__device__ __forceinline__ void store4(float* row, int c, int n, const floatx4& v) {
  if (c + 4 <= n) {
    *(f32x4_u*)(row + c) = v;
  } else {
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (c + j < n) row[c + j] = v[j];
  }
}
__device__ __forceinline__ void store4(bf16_t* row, int c, int n, const floatx4& v) {
  if (c + 4 <= n) {
    bf16x4_u p;
#pragma unroll
    for (int j = 0; j < 4; ++j) p[j] = (bf16_t)v[j];
    *(bf16x4_u*)(row + c) = p;
  } else {
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (c + j < n) row[c + j] = (bf16_t)v[j];
  }
}

// A row held by a wave: lane l has columns 4 l + 256 k ..+3.  Sums over the row.
template <int PER>
__device__ __forceinline__ float row_sum(const floatx4 (&v)[PER]) {
  float s = 0.0f;
#pragma unroll
  for (int k = 0; k < PER; ++k) s += (v[k][0] + v[k][1]) + (v[k][2] + v[k][3]);
  return wave_sum(s);
}
template <int PER>
__device__ __forceinline__ float row_dot(const floatx4 (&v)[PER], const floatx4 (&u)[PER]) {
  float s = 0.0f;
#pragma unroll
  for (int k = 0; k < PER; ++k)
    s += (v[k][0] * u[k][0] + v[k][1] * u[k][1]) + (v[k][2] * u[k][2] + v[k][3] * u[k][3]);
  return wave_sum(s);
}
// Less its mean, zeros past column n; returns 1 / sqrt(var + eps).  The mean is taken
// twice: the first one's rounding is large beside the values of a row that lies far
// from zero.
template <int PER>
__device__ __forceinline__ float center(floatx4 (&v)[PER], int n, int lane) {
#pragma unroll
  for (int pass = 0; pass < 2; ++pass) {
    const float mean = row_sum(v) / (float)n;
#pragma unroll
    for (int k = 0; k < PER; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[k][j] = 256 * k + 4 * lane + j < n ? v[k][j] - mean : 0.0f;
  }
  return 1.0f / sqrtf(row_dot(v, v) / (float)n + 1e-5f);
}

// One wave a token.
template <typename T, int PER, bool NORM>
__global__ __launch_bounds__(256) void embed_kernel(const EmbedArgs a) {
  const int64_t i = (int64_t)blockIdx.x * 4 + wave_id();
  if (i >= a.n) return;
  const int lane = threadIdx.x & 63, D = (int)a.embd;
  const int id = a.tokens[i];
  const bool there = id >= 0 && id < a.vocab;
  const T* row = (const T*)a.table + (int64_t)(there ? id : 0) * D;
  T* out = (T*)a.out + i * D;
  floatx4 v[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) v[k] = there ? load4(row, 256 * k + 4 * lane, D) : zero4();
  float f = a.scale;
  if constexpr (NORM) f = there ? f * center(v, D, lane) : 0.0f;
#pragma unroll
  for (int k = 0; k < PER; ++k) store4(out, 256 * k + 4 * lane, D, v[k] * f);
}

// --- the order of the positions by id -----------------------------------------------
constexpr int kMostBins = 512, kItems = 2048;  // a pass's digits; a workgroup's positions

// The key of position i: its id, or vocab (past all ids) where it is none.
__device__ __forceinline__ uint32_t key_of(const SortArgs& s, int64_t i) {
  if (s.keys) return s.keys[i];
  const int id = s.tokens[i];
  return id >= 0 && id < (int)s.vocab ? (uint32_t)id : (uint32_t)s.vocab;
}

// counts[workgroup][digit].
__global__ __launch_bounds__(256) void digit_counts_kernel(const SortArgs s) {
  __shared__ uint32_t bins[kMostBins];
  for (int d = threadIdx.x; d < s.bins; d += 256) bins[d] = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * kItems;
  for (int j = threadIdx.x; j < kItems; j += 256)
    if (i0 + j < s.n) atomicAdd(&bins[(key_of(s, i0 + j) >> s.shift) & (s.bins - 1)], 1u);
  __syncthreads();
  for (int d = threadIdx.x; d < s.bins; d += 256) s.counts[(int64_t)blockIdx.x * s.bins + d] = bins[d];
}

// Stable: within a digit by position.  A wave takes 512 neighbours in rounds of 64.
__global__ __launch_bounds__(256) void digit_scatter_kernel(const SortArgs s) {
  __shared__ uint32_t at[4][kMostBins];  // next place of a wave's digit
  __shared__ uint32_t sums[256];
  const int lane = threadIdx.x & 63, w = wave_id(), blocks = (int)gridDim.x, mine = (int)blockIdx.x;
  // Places before this workgroup's: smaller digits anywhere, this digit in earlier workgroups.
  uint32_t total[2] = {}, before[2] = {};  // of digits 2 t and 2 t + 1
  for (int d = 0; d < 2; ++d) {
    const int digit = 2 * threadIdx.x + d;
    if (digit >= s.bins) break;
    for (int b = 0; b < blocks; ++b) {
      const uint32_t c = s.counts[(int64_t)b * s.bins + digit];
      total[d] += c;
      if (b < mine) before[d] += c;
    }
  }
  sums[threadIdx.x] = total[0] + total[1];
  for (int d = threadIdx.x; d < s.bins; d += 256)
    for (int q = 0; q < 4; ++q) at[q][d] = 0;
  __syncthreads();
  for (int o = 1; o < 256; o <<= 1) {
    const uint32_t v = (int)threadIdx.x >= o ? sums[threadIdx.x - o] : 0;
    __syncthreads();
    sums[threadIdx.x] += v;
    __syncthreads();
  }
  // Each wave's counts, then their places.
  const int64_t i0 = (int64_t)mine * kItems + w * (kItems / 4);
  for (int j = lane; j < kItems / 4; j += 64)
    if (i0 + j < s.n) atomicAdd(&at[w][(key_of(s, i0 + j) >> s.shift) & (s.bins - 1)], 1u);
  __syncthreads();
  for (int d = 0; d < 2; ++d) {
    const int digit = 2 * threadIdx.x + d;
    if (digit >= s.bins) break;
    uint32_t place = (threadIdx.x ? sums[threadIdx.x - 1] : 0) + (d ? total[0] : 0) + before[d];
    for (int q = 0; q < 4; ++q) {
      const uint32_t c = at[q][digit];
      at[q][digit] = place;
      place += c;
    }
  }
  __syncthreads();
  for (int j = lane; j < kItems / 4; j += 64) {
    const int64_t i = i0 + j;
    const bool is = i < s.n;
    const uint32_t key = is ? key_of(s, i) : 0;
    const int digit = (int)(key >> s.shift) & (s.bins - 1);
    uint64_t same = __ballot(is);
    for (int b = 1; b < s.bins; b <<= 1) {
      const uint64_t set = __ballot((digit & b) != 0);
      same &= (digit & b) ? set : ~set;
    }
    if (is) {
      const uint32_t place = at[w][digit] + __popcll(same & ((1ull << lane) - 1));
      // (The last lane of a digit moves its place on, after every lane has read it.)
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if ((same >> lane) == 1) at[w][digit] = place + 1;
      s.keys_out[place] = key;
      s.order_out[place] = s.order ? s.order[i] : (uint32_t)i;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// --- the sums ---------------------------------------------------------------------------
// Rows of absent ids: zeros everywhere, before the sums.
__global__ __launch_bounds__(256) void zero_rows_kernel(uint32_t* out, int64_t words, bool last_half) {
  const int64_t stride = (int64_t)gridDim.x * 1024;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < words; i += stride) {
    if (i + 4 <= words) {
      typedef unsigned int u32x4_w __attribute__((ext_vector_type(4), aligned(4)));
      *(u32x4_w*)(out + i) = u32x4_w{0, 0, 0, 0};
    } else {
      for (int64_t j = i; j < words; ++j) out[j] = 0;
    }
  }
  if (last_half && blockIdx.x == 0 && threadIdx.x == 0) ((uint16_t*)(out + words))[0] = 0;
}

// The sum of id's rows, scaled and through the norm, to its row of the gradient.
template <typename T, int PER>
__device__ __forceinline__ void write_row(const EmbedArgs& a, uint32_t id, floatx4 (&s)[PER], int lane) {
  const int D = (int)a.embd;
#pragma unroll
  for (int k = 0; k < PER; ++k) s[k] *= a.scale;
  if (a.norm) {
    floatx4 x[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) x[k] = load4((const T*)a.table + (int64_t)id * D, 256 * k + 4 * lane, D);
    const float r = center(x, D, lane);
#pragma unroll
    for (int k = 0; k < PER; ++k) x[k] *= r;
    const float mean = row_sum(s) / (float)D, along = row_dot(s, x) / (float)D;
#pragma unroll
    for (int k = 0; k < PER; ++k) s[k] = (s[k] - mean - x[k] * along) * r;
  }
  T* out = (T*)a.out + (int64_t)id * D;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int c = 256 * k + 4 * lane;
    if (a.accumulate) s[k] += load4(out, c, D);
    store4(out, c, D, s[k]);
  }
}

// A wave sums the rows of positions [run * a.run, ..).  part [runs][2][D]: the sum of
// the run's first id where that id began before it, of its last where it goes on
// after it; an id that does both is in the first.
template <typename T, int PER>
__global__ __launch_bounds__(256) void embed_sums_kernel(const EmbedArgs a) {
  const int run = (int)blockIdx.x * 4 + wave_id(), lane = threadIdx.x & 63, D = (int)a.embd;
  const int64_t p0 = (int64_t)run * a.run, p1 = p0 + a.run < a.n ? p0 + a.run : a.n;
  if (p0 >= a.n) return;
  uint32_t id = a.keys[p0];
  if (id >= (uint32_t)a.vocab) return;
  bool begun = p0 > 0 && a.keys[p0 - 1] == id;  // before this run
  floatx4 s[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) s[k] = zero4();
  const auto to_part = [&](int which) {
    float* part = a.part + ((int64_t)run * 2 + which) * D;
#pragma unroll
    for (int k = 0; k < PER; ++k) store4(part, 256 * k + 4 * lane, D, s[k]);
  };
  constexpr int AHEAD = PER <= 2 ? 8 : PER <= 4 ? 4 : 2;  // rows asked for together
  for (int64_t p = p0; p < p1; p += AHEAD) {
    floatx4 g[AHEAD][PER];
    uint32_t ids[AHEAD];
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) {
      const int64_t at = p + q < p1 ? p + q : p1 - 1;
      ids[q] = __builtin_amdgcn_readfirstlane(a.keys[at]);
      const T* row = (const T*)a.grad + (int64_t)__builtin_amdgcn_readfirstlane(a.order[at]) * D;
#pragma unroll
      for (int k = 0; k < PER; ++k) g[q][k] = load4(row, 256 * k + 4 * lane, D);
    }
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) {
      if (p + q >= p1) break;
      if (ids[q] != id) {
        if (begun) to_part(0);
        else write_row<T, PER>(a, id, s, lane);
        id = ids[q];
        begun = false;
        if (id >= (uint32_t)a.vocab) return;
#pragma unroll
        for (int k = 0; k < PER; ++k) s[k] = zero4();
      }
#pragma unroll
      for (int k = 0; k < PER; ++k) s[k] += g[q][k];
    }
  }
  if (begun) to_part(0);
  else if (p1 < a.n && a.keys[p1] == id) to_part(1);
  else write_row<T, PER>(a, id, s, lane);
}

// A workgroup for each run: joins the id that begins in it and goes on past it.
template <typename T, int PER>
__global__ __launch_bounds__(256) void embed_join_kernel(const EmbedArgs a) {
  __shared__ float sums[3][PER * 256];
  const int run = (int)blockIdx.x, lane = threadIdx.x & 63, w = wave_id(), D = (int)a.embd;
  const int64_t end = ((int64_t)run + 1) * a.run;
  if (end >= a.n) return;
  const uint32_t id = a.keys[end];
  if (id >= (uint32_t)a.vocab || a.keys[end - 1] != id) return;
  const int64_t p0 = (int64_t)run * a.run;
  if (a.keys[p0] == id && p0 > 0 && a.keys[p0 - 1] == id) return;  // began earlier
  // The last run that begins with this id.
  const int runs = (int)((a.n + a.run - 1) / a.run);
  int low = run + 1, high = runs - 1;
  while (low < high) {
    const int mid = (low + high + 1) / 2;
    if (a.keys[(int64_t)mid * a.run] == id) low = mid;
    else high = mid - 1;
  }
  // This run's second sum, then the first of each run up to there, a quarter a wave.
  const int n = low - run + 1, q0 = (int)((int64_t)n * w / 4), q1 = (int)((int64_t)n * (w + 1) / 4);
  floatx4 s[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) s[k] = zero4();
#pragma unroll 4
  for (int q = q0; q < q1; ++q) {
    const float* part = a.part + ((int64_t)(run + q) * 2 + (q == 0 ? 1 : 0)) * D;
#pragma unroll
    for (int k = 0; k < PER; ++k) s[k] += load4(part, 256 * k + 4 * lane, D);
  }
  if (w > 0) {
#pragma unroll
    for (int k = 0; k < PER; ++k) *(floatx4*)&sums[w - 1][256 * k + 4 * lane] = s[k];
  }
  __syncthreads();
  if (w > 0) return;
#pragma unroll
  for (int q = 0; q < 3; ++q)
#pragma unroll
    for (int k = 0; k < PER; ++k) s[k] += *(const floatx4*)&sums[q][256 * k + 4 * lane];
  write_row<T, PER>(a, id, s, lane);
}

unsigned cdiv(int64_t a, int64_t b) { return (unsigned)((a + b - 1) / b); }

// f(std::integral_constant PER) for rows of D columns.
template <typename F>
void by_columns(int64_t D, F&& f) {
  if (D <= 256) f(std::integral_constant<int, 1>{});
  else if (D <= 512) f(std::integral_constant<int, 2>{});
  else if (D <= 1024) f(std::integral_constant<int, 4>{});
  else f(std::integral_constant<int, 8>{});
}

}  // namespace

bdh_status embed_tokens(const EmbedArgs& a, hipStream_t st) {
  by_columns(a.embd, [&](auto per) {
    constexpr int PER = decltype(per)::value;
    const dim3 grid(cdiv(a.n, 4)), block(256);
    if (a.bf16 && a.norm) hipLaunchKernelGGL((embed_kernel<bf16_t, PER, true>), grid, block, 0, st, a);
    else if (a.bf16) hipLaunchKernelGGL((embed_kernel<bf16_t, PER, false>), grid, block, 0, st, a);
    else if (a.norm) hipLaunchKernelGGL((embed_kernel<float, PER, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((embed_kernel<float, PER, false>), grid, block, 0, st, a);
  });
  BDH_HIP_TRY(hipGetLastError());
  return BDH_OK;
}

bdh_status embed_tokens_vjp(EmbedArgs a, hipStream_t st, uint64_t* launches) {
  int bits = 1;
  while (a.vocab >> bits) ++bits;  // of the keys 0 .. vocab
  const int passes = (bits + 8) / 9, per_pass = (bits + passes - 1) / passes;
  const int64_t blocks = cdiv(a.n, kItems);
  // Fewer, longer runs of more tokens: their partial sums are joined one after the other.
  a.run = a.n <= 16384 ? 16 : a.n <= 65536 ? 32 : 64;
  const int64_t runs = cdiv(a.n, a.run);
  const int64_t words = 4 * a.n + (blocks << per_pass);
  void* buf = nullptr;
  const bdh_status s = scratch(st, SLOT_EMBED, (size_t)(words + 2 * runs * a.embd) * 4, &buf);
  if (s != BDH_OK) return s;
  uint32_t* keys[2] = {(uint32_t*)buf, (uint32_t*)buf + a.n};
  uint32_t* order[2] = {keys[1] + a.n, keys[1] + 2 * a.n};
  SortArgs q{};
  q.tokens = a.tokens;
  q.n = a.n;
  q.vocab = a.vocab;
  q.bins = 1 << per_pass;
  q.counts = order[1] + a.n;
  a.part = (float*)buf + words;
  if (!a.accumulate) {
    const int64_t halves = a.vocab * a.embd * (a.bf16 ? 1 : 2);
    const int64_t grid = cdiv(halves / 2 + 1, 1024);
    hipLaunchKernelGGL(zero_rows_kernel, dim3((unsigned)(grid < 4096 ? grid : 4096)), dim3(256), 0, st,
                       (uint32_t*)a.out, halves / 2, (halves & 1) != 0);
    *launches += 1;
  }
  for (int p = 0; p < passes; ++p) {
    q.shift = p * per_pass;
    q.keys_out = keys[p & 1];
    q.order_out = order[p & 1];
    hipLaunchKernelGGL(digit_counts_kernel, dim3((unsigned)blocks), dim3(256), 0, st, q);
    hipLaunchKernelGGL(digit_scatter_kernel, dim3((unsigned)blocks), dim3(256), 0, st, q);
    q.keys = q.keys_out;
    q.order = q.order_out;
    *launches += 2;
  }
  a.keys = q.keys;
  a.order = q.order;
  by_columns(a.embd, [&](auto per) {
    constexpr int PER = decltype(per)::value;
    const dim3 grid(cdiv(runs, 4)), join((unsigned)runs), block(256);
    if (a.bf16) {
      hipLaunchKernelGGL((embed_sums_kernel<bf16_t, PER>), grid, block, 0, st, a);
      if (runs > 1) hipLaunchKernelGGL((embed_join_kernel<bf16_t, PER>), join, block, 0, st, a);
    } else {
      hipLaunchKernelGGL((embed_sums_kernel<float, PER>), grid, block, 0, st, a);
      if (runs > 1) hipLaunchKernelGGL((embed_join_kernel<float, PER>), join, block, 0, st, a);
    }
  });
  *launches += runs > 1 ? 2 : 1;
  BDH_HIP_TRY(hipGetLastError());
  return BDH_OK;
}

}  // namespace bdh
