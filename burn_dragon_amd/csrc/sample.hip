// The next token of every row from its logits and a given uniform number:
// temperature, top-k, top-p and min-p.
//
// Of a row: x = logits (NaN as -inf, +inf as the largest finite f32), m the
// largest, t_i = (x_i - m) log2(e) / temperature, w_i = 2^t_i where
// t_i >= -42 and 0 below.  In the order of x descending, ties by index
// ascending: top-k keeps the first k, top-p the ones before which the kept w
// sum to less than top_p of all that top-k kept, min-p those of w >= min_p.
// The token is the first in vocabulary order whose running sum of kept w
// exceeds uniform * (their sum).
//
// No sort.  The weights are integers, w * 2^42 rounded, from a 64-bit 2^t: sums
// of them are exact, so no order of atomics or of partial sums changes a token.
// Up to 2^20 logits, a sum stays below 2^62.
// Long rows sum in chunks, each in units of 2^-42 of its own largest weight, and
// the chunks' sums are scaled to the row's units and rounded (a bin's for the cuts,
// what is kept whole for the draw).  Such a sum is off from the one of the row's
// own integers by up to half a unit a logit, and top-p's total also counts weights
// below 2^-42 of the row's largest that are not below that of their chunk's, up to a
// unit each: a border is right to about V units, 2^-42 V of the largest weight
// (2^-22 at 2^20 logits).  Where a chunk's sum is more than its logits' own, its last kept
// logit has the rest.  Chunks lie by index, so none of it depends on the batch.
//
//   1. A histogram over 512 bins of 1/10 octave of weight below the largest
//      (counts for top-k, weights for top-p) finds the bin in which a cut
//      falls; bins before it are kept whole, bins after it are not.
//   2. The candidates of that bin go to a list.  Up to 64 are compared each with
//      each in a wave, up to 256 by the workgroup; more are narrowed first by
//      histograms of nine bits of (value, index), so equal logits are cut by
//      index.  What a workgroup's list does not hold is read from a longer one in
//      the scratch (long rows), or from the row again.
//   3. The kept weights are summed by wave, and the draw descends into the
//      wave, the stripe, the lane and the element that it falls in.
//
// Rows up to 16384 logits: one workgroup, the row in registers, read once.
// Longer ones in chunks of 8192, four launches (sample_chunk_kernel on).  Where
// top-k keeps few, the first launch already leaves all that can be drawn in
// lists, and the last works on those alone.
//
// Measured (us): 1 row of 256 with top-k and top-p 7, 256 of 8192 14; 64 of 32000
// 23; 256 of 131072 75, with top-p 0.9 alone 111 (134 MB twice: 2.4 TB/s).  Short
// rows are bound by the chain of block-wide steps, long ones by the launches in
// turn up to some 50 rows; past that by the 64-bit 2^t and the histogram's atomics
// of the first launch (2.8 TB/s), and by the second read.
// Flat rows have many candidates in a cut's bin: 256 of 131072 normal logits of
// deviation 0.2 with top-p 0.9 144 (803 where the workgroup went through the row
// for what its list of 4096 could not hold; equal logits, which the scratch's list
// cannot hold either, 971).
#include "bdh_internal.h"

namespace bdh {
namespace {

constexpr int kBins = 512;
constexpr int kBinsPerOctave = 10;  // 420 of the bins: see bin_of
constexpr double kLeastT = -42.0;
constexpr int kSmall = 64;       // candidates that one wave orders
constexpr int kMid = 256;        // that the workgroup compares each with each
constexpr int kListMax = 4096;   // candidates that a workgroup's list holds
constexpr int kFarMax = 32768;   // that a long row's list in the scratch holds
constexpr int kNear = 256;       // logits that a chunk lists for top-k
constexpr int kChunkThreads = 512;
constexpr int kChunkPer = 16;    // logits a thread
constexpr int kChunk = kChunkThreads * kChunkPer;
constexpr int kMaxChunks = (int)(kMaxSampleVocab / kChunk);
constexpr int64_t kGroupBytes = (int64_t)256 << 20;  // of scratch that rows go through at a time
constexpr int kNoLimitIndex = 0x7fffffff;

struct Row {
  double c;      // log2(e) / temperature
  float cb;      // bins per unit of x
  double min_t;  // least t that is kept
  double p;
  int k;
  bool greedy, use_k, use_p;
  float u;
};

__device__ Row row_settings(const SampleArgs& a, int64_t r) {
  const float tau = a.temperature_rows ? a.temperature_rows[r] : a.temperature;
  const float p = a.top_p_rows ? a.top_p_rows[r] : a.top_p;
  const float mp = a.min_p_rows ? a.min_p_rows[r] : a.min_p;
  Row s;
  s.k = a.top_k_rows ? a.top_k_rows[r] : a.top_k;
  s.greedy = !(tau > 0.0f) || s.k == 1;
  s.c = 1.4426950408889634074 / (double)tau;
  // Above 0, so that -inf stays -inf; below the least that a finite temperature
  // gives (4e-38), so that bins are as wide as the weights' at any of them.
  s.cb = (float)fmax(fmin(s.c * kBinsPerOctave, 1e30), 0x1p-126);
  s.use_k = s.k > 0 && s.k < a.vocab;
  s.use_p = p < 1.0f;
  s.p = p > 0.0f ? (double)p : 0.0;
  s.min_t = mp > 0.0f ? fmax(log2((double)fminf(mp, 1.0f)), kLeastT) : kLeastT;
  s.u = a.uniform[r];
  return s;
}

// 2^t * 2^42 as an integer, t in [-42, 0], in 64 bits: 2^f of the fraction by the
// polynomial of degree 9 with the least largest relative error on [-1/2, 1/2]
// (2^-46; its coefficients come out of Remez' exchange).
//
// The loops over a row's logits keep the coefficients in scalar registers, where
// an FMA takes one as its addend; as literals each costs two moves, a third of
// the instructions.
struct Series {
  double c[10];
  __device__ __forceinline__ Series()
      : c{1.0000000000000127,    0.693147180559871,     0.24022650695649653,   0.055504108668685624,
          0.009618129192067193,  0.0013333557617602426, 0.00015403434948103528, 1.5252984839814557e-05,
          1.3259405603573696e-06, 1.0150336495148618e-07} {}
  __device__ __forceinline__ void keep() {
#pragma unroll
    for (int k = 0; k < 10; ++k) asm("" : "+s"(c[k]));
  }
};
__device__ __forceinline__ uint64_t weight42(double t, const Series& series = Series()) {
  const double magic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer
  const double kd = t + magic;
  const int n = __double2loint(kd);
  const double f = t - (kd - magic);
  double e = series.c[9];
#pragma unroll
  for (int k = 8; k >= 0; --k) e = fma(e, f, series.c[k]);
  const double w = __hiloint2double(__double2hiint(e) + (n << 20) + (42 << 20), __double2loint(e));
  const double r = w + 4503599627370496.0;  // 2^52: the integer is in the low bits
  return (uint64_t)(uint32_t)(__double2hiint(r) - 0x43300000) << 32 | (uint32_t)__double2loint(r);
}

// t of a logit.  It is computed again wherever a weight is needed, and all of
// them have to agree to the unit, or a draw falls behind the last weight: its
// product is never fused into what follows it.
__device__ __forceinline__ double t_of(float x, float m, double c) {
#pragma clang fp contract(off)
  return ((double)x - (double)m) * c;
}

// Its weight where t is kept at all.
__device__ __forceinline__ uint64_t weight_from(double t, double least, const Series& series = Series()) {
  return t >= least ? weight42(t, series) : 0;  // (NaN: -inf logits at an infinite temperature)
}

__device__ __forceinline__ float clean(float x) {
  x = x != x ? -INFINITY : x;
  return fminf(x, 3.402823466e38f) + 0.0f;  // -0 as 0: equal logits are equal bits
}

// (value, index) as one number, smaller = earlier in the order.
__device__ __forceinline__ uint64_t order_of(float x, int idx) {
  const uint32_t b = __float_as_uint(x);
  const uint32_t up = b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
  return ((uint64_t)~up << 32) | (uint32_t)idx;
}
__device__ __forceinline__ float value_of(uint64_t o) {
  const uint32_t up = ~(uint32_t)(o >> 32);
  return __uint_as_float((up >> 31) ? up ^ 0x80000000u : ~up);
}

// A grid that all chunks of a row share, of 1/10 octave of weight, and the bin
// of a logit in it, counted down from the bin of the largest; kBins further
// down (weight 0).  Every step is monotone in x, so the bins are ranges of the
// order whatever is rounded.  A weight of 2^-42 lies in bin 420, so f32 leaves
// room to be off by 92 bins together: |x| / temperature up to 2^26; past that
// weights from about 2^-38 down may fall out too.
__device__ __forceinline__ float grid_of(float x, float cb) {
  return __builtin_amdgcn_fmed3f(floorf(x * cb), -3e38f, 3e38f);
}
__device__ __forceinline__ int bin_of(float x, float top, float cb) {
  const float d = top - grid_of(x, cb);
  return d < (float)kBins ? (int)d : kBins;
}
__device__ __forceinline__ bool is_real(float x) { return x > -INFINITY; }

template <typename T>
__device__ __forceinline__ float load1(const T* p) { return clean((float)*p); }

typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf16x4_u __attribute__((ext_vector_type(4), aligned(2)));
template <typename T> struct Vec4;
template <> struct Vec4<float> { typedef f32x4_u type; };
template <> struct Vec4<bf16_t> { typedef bf16x4_u type; };

// A chunk's logits: each wave holds 64 * E consecutive ones in stripes of
// 256, each lane four of a stripe.
template <int E>
__device__ __forceinline__ int index_of(int base, int e) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  return base + wave * (64 * E) + ((e >> 2) * 64 + lane) * 4 + (e & 3);
}
template <typename T, int E>
__device__ __forceinline__ void load_chunk(const T* row, int base, int vocab, float (&x)[E]) {
#pragma unroll
  for (int e = 0; e < E; e += 4) {
    const int i = index_of<E>(base, e);
    if (i + 4 <= vocab) {
      const typename Vec4<T>::type v = *(const typename Vec4<T>::type*)(row + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[e + j] = clean((float)v[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[e + j] = i + j < vocab ? load1(row + i + j) : -INFINITY;
    }
  }
}

// Keeps the compiler from carrying what it has computed of the logits from one
// pass over them to the next (their f64 forms alone would fill the registers).
template <int E>
__device__ __forceinline__ void forget(float (&x)[E]) {
#pragma unroll
  for (int e = 0; e < E; ++e) asm volatile("" : "+v"(x[e]));
}

// What the histogram says about the cuts of a row.
struct Cuts {
  int k_bin;            // holds the k-th in order; kBins: top-k cuts nothing that is drawn
  int p_first, p_last;  // bins that the top-p cut can fall in; kBins: no top-p
  int m_first, m_last;  // (long rows) bins that the least kept t can fall in; kBins: none
  uint64_t k_above;     // logits in bins before k_bin
  uint64_t k_upto;      // and with it
  uint64_t k_mass;      // their weight (all weight: no k_bin)
  uint64_t p_above;     // weight in bins before p_first
};

template <int NT, int LIST>
struct Shared {
  uint64_t mass[kBins];
  uint64_t list[LIST];
  uint64_t small[kSmall], small_w[kMid], kept[kMid];
  uint64_t wave_sum[NT / 64];
  uint64_t lo, hi, sum;  // of a pass over the candidates
  uint32_t cnt[kBins];
  float wave_max[NT / 64];
  int n_list, n_small, arg;
  int bin;
  uint64_t above;
  Cuts cuts;
};

// Neighbours' values by DPP: `none` where there is none.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp32(uint32_t v, uint32_t none) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp64(uint64_t v) {
  return (uint64_t)dpp32<CTRL, ROWS>((uint32_t)(v >> 32), 0) << 32 | dpp32<CTRL, ROWS>((uint32_t)v, 0);
}
__device__ __forceinline__ uint64_t lane_u64(uint64_t v, int lane) {  // lane: uniform
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
__device__ __forceinline__ uint64_t wave_scan_u64(uint64_t v) {  // inclusive
  v += dpp64<0x111, 0xf>(v);  // the lane before, of a row of 16
  v += dpp64<0x112, 0xf>(v);
  v += dpp64<0x114, 0xf>(v);
  v += dpp64<0x118, 0xf>(v);
  v += dpp64<0x142, 0xa>(v);  // row 0's last to row 1, 2's to 3
  v += dpp64<0x143, 0xc>(v);  // row 1's last to rows 2 and 3
  return v;
}
__device__ __forceinline__ uint64_t wave_sum_u64(uint64_t v) { return lane_u64(wave_scan_u64(v), 63); }
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t max_dpp(uint64_t v) {
  const uint64_t w = dpp64<CTRL, ROWS>(v);
  return w > v ? w : v;
}
__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {
  v = max_dpp<0x111, 0xf>(v);
  v = max_dpp<0x112, 0xf>(v);
  v = max_dpp<0x114, 0xf>(v);
  v = max_dpp<0x118, 0xf>(v);
  v = max_dpp<0x142, 0xa>(v);
  v = max_dpp<0x143, 0xc>(v);
  return lane_u64(v, 63);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float max_dpp(float v) {
  return fmaxf(v, __uint_as_float(dpp32<CTRL, ROWS>(__float_as_uint(v), 0xff800000u)));
}
__device__ __forceinline__ float wave_max_f32(float v) {
  v = max_dpp<0x111, 0xf>(v);
  v = max_dpp<0x112, 0xf>(v);
  v = max_dpp<0x114, 0xf>(v);
  v = max_dpp<0x118, 0xf>(v);
  v = max_dpp<0x142, 0xa>(v);
  v = max_dpp<0x143, 0xc>(v);
  return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), 63));
}

template <int NT>
__device__ __forceinline__ float block_max(float v, float* part) {
  v = wave_max_f32(v);
  if (NT == 64) return v;
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = part[0];
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) v = fmaxf(v, part[w]);
  return v;
}

// Appends to a list: one atomic a wave.
__device__ __forceinline__ int append_at(int* n, bool mine) {
  const uint64_t all = __ballot(mine);
  if (all == 0) return -1;
  int first = 0;
  if ((threadIdx.x & 63) == (uint32_t)__builtin_ctzll(all)) first = atomicAdd(n, __popcll(all));
  first = __builtin_amdgcn_readlane(first, __builtin_ctzll(all));
  return mine ? first + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(all >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)all, 0)) : -1;
}

// A histogram in one wave's registers: eight bins a lane, and the sum of what
// lies before them.
struct BinScan {
  uint64_t v[kBins / 64], before, total;

  template <typename H>
  __device__ BinScan(const H* h, int last) {  // bins past `last` count as empty
    const int first = (threadIdx.x & 63) * (kBins / 64);
    uint64_t s = 0;
#pragma unroll
    for (int j = 0; j < kBins / 64; ++j) {
      v[j] = first + j <= last ? h[first + j] : 0;
      s += v[j];
    }
    before = wave_scan_u64(s) - s;
    total = lane_u64(before + s, 63);
  }
  // The first bin at which the running sum reaches `need` (kBins: none), and
  // the sum before it and in it.
  __device__ int cross(uint64_t need, uint64_t* sum_before, uint64_t* in) const {
    uint64_t run = before, b = 0, w = 0;
    int at = -1;
#pragma unroll
    for (int j = 0; j < kBins / 64; ++j) {
      if (at < 0 && run + v[j] >= need) {
        at = j;
        b = run;
        w = v[j];
      }
      run += v[j];
    }
    const uint64_t found = __ballot(at >= 0);
    if (found == 0) {
      *sum_before = total;
      *in = 0;
      return kBins;
    }
    const int lane = __builtin_ctzll(found);
    *sum_before = lane_u64(b, lane);
    *in = lane_u64(w, lane);
    return lane * (kBins / 64) + __builtin_amdgcn_readlane(at, lane);
  }
};

__device__ __forceinline__ uint64_t p_need(const Row& s, uint64_t total) {
  const uint64_t need = (uint64_t)ceil(s.p * (double)total);
  return need > 0 ? need : 1;  // the first in order is always kept
}
__device__ __forceinline__ Cuts no_cuts() {
  Cuts q;
  q.k_bin = q.p_first = q.p_last = q.m_first = q.m_last = kBins;
  q.k_above = q.k_upto = q.k_mass = q.p_above = 0;
  return q;
}
// One wave each.
__device__ __forceinline__ void find_k(const Row& s, const uint32_t* cnt, Cuts& q) {
  uint64_t in;
  q.k_bin = BinScan(cnt, kBins).cross((uint64_t)s.k, &q.k_above, &in);
  q.k_upto = q.k_above + in;
}
// What f does to the cuts, done by one wave for all (sixteen waves that each
// scan the bins for themselves take 4 us of a workgroup's issue).
template <int NT, typename F>
__device__ __forceinline__ void by_one_wave(Cuts& q, Cuts* shared, const F& f) {
  if (NT == 64 || threadIdx.x < 64) f();
  if (NT == 64) return;
  if (threadIdx.x == 0) *shared = q;
  __syncthreads();
  q = *shared;
}
// Counts a chunk's logits by bin into cnt (cleared).
template <int NT, int E>
__device__ __forceinline__ void count_logits(const Row& s, const float (&x)[E], float top, uint32_t* cnt) {
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int b = bin_of(x[e], top, s.cb);
    if (b < kBins) atomicAdd(&cnt[b], 1u);
  }
  __syncthreads();
}
__device__ __forceinline__ void find_p(const Row& s, const uint64_t* mass, Cuts& q) {
  // What top-k keeps weighs between all before k_bin, and that with k_bin.
  const BinScan h(mass, q.k_bin);
  uint64_t in = q.k_bin < kBins ? mass[q.k_bin] : 0;
  q.k_mass = h.total - in;
  q.p_first = min(h.cross(p_need(s, q.k_mass), &q.p_above, &in), q.k_bin);
  uint64_t unused;
  q.p_last = min(h.cross(p_need(s, h.total), &unused, &in), q.k_bin);
}
// (Wider than its one bin by what f32 may be off here and in bin_of.)
__device__ __forceinline__ void find_least(const Row& s, float m, float top, Cuts& q) {
  const float least = (float)((double)m + s.min_t / s.c);
  if (!is_real(least)) return;  // (an infinite temperature)
  const float bin = top - grid_of(least, s.cb);
  const float off = 2.0f + (fabsf(m) + fabsf(least)) * s.cb * 0x1p-22f;
  if (!(bin - off < (float)kBins)) return;
  q.m_first = (int)fmaxf(bin - off, 0.0f);
  q.m_last = (int)fminf(bin + off, (float)(kBins - 1));
}
// The cuts of a list that holds all that can be kept: each may fall anywhere.
__device__ __forceinline__ Cuts cuts_anywhere() {
  Cuts q = no_cuts();
  q.k_bin = q.p_first = -1;
  return q;
}
// Bins before this are kept whole.
__device__ __forceinline__ int sure_bins(const Cuts& q) { return min(min(q.k_bin, q.p_first), q.m_first); }
// Bins that a cut may divide (past k_bin nothing is kept).
__device__ __forceinline__ bool is_candidate(const Cuts& q, int bin) {
  return bin < kBins && bin <= q.k_bin &&
         (bin == q.k_bin || (bin >= q.p_first && bin <= q.p_last) || (bin >= q.m_first && bin <= q.m_last));
}

// The candidates: in the workgroup's list, in the scratch's where they are more,
// or where that overflowed, too, all of the row's logits.
template <typename T, int NT, int LIST>
struct Candidates {
  Shared<NT, LIST>& sh;
  const T* row;
  int vocab;
  float m;
  float top;
  const Row& s;
  int n;  // found; beyond LIST the workgroup's list is not complete, beyond kFarMax the scratch's
  const uint64_t* far;  // the scratch's, or null

  // Calls f(order, bin) for each whose bin lies in [first, last].
  template <typename F>
  __device__ __forceinline__ void each(int first, int last, const F& f) {
    if (n <= LIST) {
      for (int i = threadIdx.x; i < n; i += NT) {
        const uint64_t o = sh.list[i];
        const int b = bin_of(value_of(o), top, s.cb);
        if (b >= first && b <= last) f(o, b);
      }
    } else if (far && n <= kFarMax) {
      for (int i = threadIdx.x; i < n; i += NT) {
        const uint64_t o = far[i];
        const int b = bin_of(value_of(o), top, s.cb);
        if (b >= first && b <= last) f(o, b);
      }
    } else {
      for (int i = threadIdx.x; i < vocab; i += NT) {
        const float x = load1(row + i);
        const int b = bin_of(x, top, s.cb);
        if (b >= first && b <= last) f(order_of(x, i), b);
      }
    }
  }
  __device__ __forceinline__ uint64_t weight(uint64_t o, double least) const {
    return weight_from(t_of(value_of(o), m, s.c), least);
  }

  // The last candidate in order that a cut keeps, among those of bins
  // [first, last]: by count, the one with `need` - 1 logits before it; by
  // weight, the last with less than `need` of weight before it.  `above`:
  // what lies before bin `first`.
  template <bool MASS>
  __device__ uint64_t cut(int first, int last, uint64_t above, uint64_t need) {
    uint64_t lo = 0, hi = ~0ull;
    for (;;) {
      __syncthreads();
      if (threadIdx.x == 0) {
        sh.lo = ~0ull;
        sh.hi = 0;
        sh.n_small = 0;
      }
      __syncthreads();
      uint64_t low = ~0ull, high_o = 0;
      int count = 0;
      each(first, last, [&](uint64_t o, int) {
        if (o < lo || o > hi) return;
        ++count;
        low = o < low ? o : low;
        high_o = o > high_o ? o : high_o;
      });
      low = ~wave_max_u64(~low);
      high_o = wave_max_u64(high_o);
      count = (int)wave_sum_u64((uint64_t)count);
      if ((threadIdx.x & 63) == 0 && count) {
        atomicAdd(&sh.n_small, count);
        atomicMin((unsigned long long*)&sh.lo, (unsigned long long)low);
        atomicMax((unsigned long long*)&sh.hi, (unsigned long long)high_o);
      }
      __syncthreads();
      const int n_in = sh.n_small;
      if (n_in <= kSmall) {
        __syncthreads();
        if (threadIdx.x == 0) sh.n_small = 0;
        __syncthreads();
        each(first, last, [&](uint64_t o, int) {
          const int at = append_at(&sh.n_small, o >= lo && o <= hi);
          if (at >= 0) sh.small[at] = o;
        });
        __syncthreads();
        if (threadIdx.x < 64) {
          const int lane = threadIdx.x;
          const uint64_t mine = lane < n_in ? sh.small[lane] : ~0ull;
          const uint64_t w = lane >= n_in ? 0 : MASS ? weight(mine, kLeastT) : 1;
          uint64_t before = above;
          for (int j = 0; j < n_in; ++j) before += lane_u64(mine, j) < mine ? lane_u64(w, j) : 0;
          const bool kept = lane < n_in && before < need;
          const uint64_t best = wave_max_u64(kept ? mine : 0);
          if (lane == 0) sh.sum = best;
        }
        __syncthreads();
        return sh.sum;
      }
      const uint64_t from = sh.lo, to = sh.hi;
      const int high = 63 - __builtin_clzll(from ^ to);
      const int shift = high > 8 ? high - 8 : 0;
      for (int b = threadIdx.x; b < kBins; b += NT) sh.mass[b] = 0;
      __syncthreads();
      each(first, last, [&](uint64_t o, int) {
        if (o < lo || o > hi) return;
        const uint64_t w = MASS ? weight(o, kLeastT) : 1;
        atomicAdd((unsigned long long*)&sh.mass[(int)((o >> shift) - (from >> shift))], (unsigned long long)w);
      });
      __syncthreads();
      if (threadIdx.x < 64) {
        uint64_t before, in;
        const int bin = BinScan(sh.mass, kBins).cross(need > above ? need - above : 1, &before, &in);
        if (threadIdx.x == 0) {
          // (Weights scaled from chunks may leave the sum short, by up to a unit a
          // logit: the last candidates, of which the end keeps all.)
          sh.bin = bin < kBins ? bin : (int)((to >> shift) - (from >> shift));
          sh.above = bin < kBins ? above + before : above;
        }
      }
      __syncthreads();
      lo = ((from >> shift) + (uint64_t)sh.bin) << shift;
      hi = lo + ((1ull << shift) - 1);
      above = sh.above;
    }
  }

  // The same for up to kSmall candidates, in one wave: a lane compares its own
  // with each other.  (One candidate at least is kept.)
  __device__ uint64_t limit_small(const Cuts& q) {
    const int lane = threadIdx.x & 63;
    const uint64_t mine = lane < n ? sh.list[lane] : ~0ull;
    const int bin = lane < n ? bin_of(value_of(mine), top, s.cb) : kBins;
    const uint64_t w = s.use_p && lane < n ? weight(mine, kLeastT) : 0;
    const bool in_k = lane < n && bin >= q.k_bin, in_p = bin >= q.p_first && bin <= q.p_last;
    const uint64_t wp = in_p ? w : 0;
    uint64_t k_before = q.k_above, p_before = q.p_above;
    for (int j = 0; j < n; ++j) {
      const bool earlier = lane_u64(mine, j) < mine;
      k_before += earlier && __builtin_amdgcn_readlane((int)in_k, j);
      p_before += earlier ? lane_u64(wp, j) : 0;
    }
    bool kept = lane < n && (bin < q.k_bin || k_before < (uint64_t)s.k);
    if (s.use_p) {
      const uint64_t total = q.k_mass + (q.k_bin < kBins ? wave_sum_u64(in_k && kept ? w : 0) : 0);
      kept = kept && (bin < q.p_first || (in_p && p_before < p_need(s, total)));
    }
    return wave_max_u64(kept ? mine : 0);
  }

  // The same for up to kMid, a thread (or at 64 threads four) a candidate.
  __device__ uint64_t limit_mid(const Cuts& q) {
    constexpr int PER = kMid > NT ? kMid / NT : 1;
    constexpr uint64_t in_k_bit = 1ull << 63;  // (weights end below)
    uint64_t mine[PER], w[PER], k_before[PER], p_before[PER];
    int bin[PER];
#pragma unroll
    for (int c = 0; c < PER; ++c) {
      const int i = threadIdx.x + c * NT;
      mine[c] = i < n ? sh.list[i] : ~0ull;
      bin[c] = i < n ? bin_of(value_of(mine[c]), top, s.cb) : kBins;
      w[c] = s.use_p && i < n ? weight(mine[c], kLeastT) : 0;
      k_before[c] = q.k_above;
      p_before[c] = q.p_above;
      if (i < n)
        sh.small_w[i] = (bin[c] >= q.p_first && bin[c] <= q.p_last ? w[c] : 0) | (bin[c] >= q.k_bin ? in_k_bit : 0);
    }
    if (threadIdx.x == 0) sh.sum = sh.hi = 0;
    __syncthreads();
    if (threadIdx.x < n) {
#pragma unroll 4
      for (int j = 0; j < n; ++j) {
        const uint64_t o = sh.list[j], wj = sh.small_w[j];
#pragma unroll
        for (int c = 0; c < PER; ++c) {
          k_before[c] += o < mine[c] ? wj >> 63 : 0;
          p_before[c] += o < mine[c] ? wj & ~in_k_bit : 0;
        }
      }
    }
    uint64_t last = 0;
#pragma unroll
    for (int c = 0; c < PER; ++c) {
      const bool real = threadIdx.x + c * NT < n;
      const bool kept = real && (bin[c] < q.k_bin || k_before[c] < (uint64_t)s.k);
      if (s.use_p && kept && bin[c] >= q.k_bin) atomicAdd((unsigned long long*)&sh.sum, (unsigned long long)w[c]);
      if (!kept) mine[c] = 0;
    }
    __syncthreads();
    const uint64_t need = s.use_p ? p_need(s, q.k_mass + sh.sum) : 0;
#pragma unroll
    for (int c = 0; c < PER; ++c) {
      const bool kept = !s.use_p || bin[c] < q.p_first || (bin[c] <= q.p_last && p_before[c] < need);
      last = kept && mine[c] > last ? mine[c] : last;
    }
    if (last) atomicMax((unsigned long long*)&sh.hi, (unsigned long long)last);
    __syncthreads();
    return sh.hi;
  }

  // The last logit in order that top-k and top-p keep.
  __device__ uint64_t limit(const Cuts& q) {
    if (q.k_bin == kBins && !s.use_p) return ~0ull;  // neither divides anything
    if (n <= kSmall) {
      if (NT == 64) return limit_small(q);
      if (threadIdx.x < 64) {
        const uint64_t last = limit_small(q);
        if (threadIdx.x == 0) sh.sum = last;
      }
      __syncthreads();
      return sh.sum;
    }
    if (n <= kMid) return limit_mid(q);
    uint64_t lim = ~0ull, total = q.k_mass;
    if (q.k_bin < kBins) {
      lim = cut<false>(q.k_bin, q.k_bin, q.k_above, (uint64_t)s.k);
      if (s.use_p) {
        __syncthreads();
        if (threadIdx.x == 0) sh.sum = 0;
        __syncthreads();
        uint64_t w = 0;
        each(q.k_bin, q.k_bin, [&](uint64_t o, int) { w += o <= lim ? weight(o, kLeastT) : 0; });
        if (w) atomicAdd((unsigned long long*)&sh.sum, (unsigned long long)w);
        __syncthreads();
        total += sh.sum;
      }
    }
    if (s.use_p && q.p_first < kBins) {
      const uint64_t lp = cut<true>(q.p_first, q.p_last, q.p_above, p_need(s, total));
      lim = lp < lim ? lp : lim;
    }
    return lim;
  }
};

// The kept weight of a thread's logits: those up to (limit_x, limit_i) in order.
template <int E>
__device__ __forceinline__ uint64_t kept_weight(const Row& s, float x, int i, float m, float limit_x, int limit_i,
                                                const Series& series = Series()) {
  if (!(x > limit_x || (x == limit_x && i <= limit_i))) return 0;
  return weight_from(t_of(x, m, s.c), s.min_t, series);
}

__device__ __forceinline__ uint64_t draw_at(float u, uint64_t total) {
  const uint64_t at = u > 0.0f ? (uint64_t)((double)fminf(u, 0x1.fffffep-1f) * (double)total) : 0;
  return at < total ? at : total - 1;
}

// Finds the logit of the chunk that the draw falls in: the first whose
// running sum of kept weights exceeds `at` (at < their sum).  Returns true in
// the one thread that holds it.
template <int NT, int E, int LIST>
__device__ bool locate(Shared<NT, LIST>& sh, const Row& s, const float (&x)[E], int base, float m, float limit_x,
                       int limit_i, uint64_t at, int* token, double* t) {
  const int wave = threadIdx.x >> 6;
  uint64_t before = 0;
  for (int w = 0; w < NT / 64; ++w) {
    const uint64_t sum = sh.wave_sum[w];
    if (at < before + sum) {
      if (w != wave) return false;
      break;
    }
    before += sum;
  }
  at -= before;
  for (int e = 0; e < E; e += 4) {
    uint64_t w[4], mine = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // (x[e] by a select: the loop is not unrolled, one stripe at a time is few instructions.)
      float v = 0.0f;
#pragma unroll
      for (int q = 0; q < E; q += 4) v = q == e ? x[q + j] : v;
      w[j] = kept_weight<E>(s, v, index_of<E>(base, e) + j, m, limit_x, limit_i);
      mine += w[j];
    }
    const uint64_t incl = wave_scan_u64(mine);
    const uint64_t stripe = lane_u64(incl, 63);
    if (at >= stripe) {
      at -= stripe;
      continue;
    }
    uint64_t run = incl - mine;
    if (at < run || at >= incl) return false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (at < run + w[j]) {
        float v = 0.0f;
#pragma unroll
        for (int q = 0; q < E; q += 4) v = q == e ? x[q + j] : v;
        *token = index_of<E>(base, e) + j;
        *t = t_of(v, m, s.c);
        return true;
      }
      run += w[j];
    }
  }
  return false;
}

template <typename T, int NT, int E>
__global__ __launch_bounds__(NT) void sample_row_kernel(const SampleArgs a) {
  constexpr int LIST = NT * E < kListMax ? NT * E : kListMax;
  __shared__ Shared<NT, LIST> sh;
  const int64_t r = blockIdx.x;
  const T* row = (const T*)a.logits + r * a.row_stride;
  const Row s = row_settings(a, r);
  const int vocab = (int)a.vocab;
  float x[E];
  load_chunk<T, E>(row, 0, vocab, x);
  float best = x[0];
#pragma unroll
  for (int e = 1; e < E; ++e) best = fmaxf(best, x[e]);
  const float m = block_max<NT>(best, sh.wave_max);
  if (!is_real(m)) {
    if (threadIdx.x == 0) {
      a.tokens[r] = -1;
      if (a.logprob) a.logprob[r] = -INFINITY;
    }
    return;
  }
  if (s.greedy) {
    if (threadIdx.x == 0) sh.arg = kNoLimitIndex;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (x[e] == m) atomicMin(&sh.arg, index_of<E>(0, e));
    __syncthreads();
    if (threadIdx.x == 0) {
      a.tokens[r] = sh.arg;
      if (a.logprob) a.logprob[r] = 0.0f;
    }
    return;
  }
  Series series;
  series.keep();
  float limit_x = -INFINITY;
  int limit_i = -1;  // (-inf itself is not kept)
  if (s.use_k || s.use_p) {
    const float top = grid_of(m, s.cb);
    for (int b = threadIdx.x; b < kBins; b += NT) {
      sh.cnt[b] = 0;
      sh.mass[b] = 0;
    }
    if (threadIdx.x == 0) sh.n_list = 0;
    __syncthreads();
    Cuts q = no_cuts();
    if (s.use_k) {
      count_logits<NT, E>(s, x, top, sh.cnt);
      by_one_wave<NT>(q, &sh.cuts, [&] { find_k(s, sh.cnt, q); });
      forget<E>(x);
    }
    if (s.use_p) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int b = bin_of(x[e], top, s.cb);
        if (b < kBins && b <= q.k_bin)  // no weight past the k-th counts
          atomicAdd((unsigned long long*)&sh.mass[b],
                    (unsigned long long)weight_from(t_of(x[e], m, s.c), kLeastT, series));
        if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
      __syncthreads();
      by_one_wave<NT>(q, &sh.cuts, [&] { find_p(s, sh.mass, q); });
      forget<E>(x);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int b = bin_of(x[e], top, s.cb);
      const int at = append_at(&sh.n_list, is_candidate(q, b));
      if (at >= 0 && at < LIST) sh.list[at] = order_of(x[e], index_of<E>(0, e));
    }
    __syncthreads();
    Candidates<T, NT, LIST> cand{sh, row, vocab, m, top, s, sh.n_list, nullptr};
    const uint64_t lim = cand.limit(q);
    if (lim != ~0ull) {
      limit_x = value_of(lim);
      limit_i = (int)(uint32_t)lim;
    }
  }
  forget<E>(x);
  uint64_t mine = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    mine += kept_weight<E>(s, x[e], index_of<E>(0, e), m, limit_x, limit_i, series);
    if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
  }
  mine = wave_sum_u64(mine);
  if ((threadIdx.x & 63) == 0) sh.wave_sum[threadIdx.x >> 6] = mine;
  __syncthreads();
  uint64_t total = 0;
  for (int w = 0; w < NT / 64; ++w) total += sh.wave_sum[w];
  forget<E>(x);
  int token;
  double t;
  if (locate<NT, E, LIST>(sh, s, x, 0, m, limit_x, limit_i, draw_at(s.u, total), &token, &t)) {
    a.tokens[r] = token;
    if (a.logprob) a.logprob[r] = (float)(t * 0.69314718055994530942 - log((double)total * 0x1p-42));
  }
}

// --- long rows ---------------------------------------------------------------
// What a row's launches leave for one another.
struct RowState {
  Cuts cuts;
  float top;
  float m;
  int n_list;
  bool near;  // the chunks' `near` holds all that can be drawn
};
struct SplitArgs {
  SampleArgs a;
  int64_t row0;      // of this group of rows
  int chunks;
  int far;           // what a row's list holds: kFarMax, or its logits where they are fewer
  float* max;        // [rows, chunks]
  int32_t* arg;      // [rows, chunks]: the first index of the chunk's largest
  uint32_t* cnt;     // [rows, chunks, kBins], bins counted from the chunk's own largest
  uint64_t* mass;    // [rows, chunks, kBins], weights relative to it
  int32_t* near_n;   // [rows, chunks]: logits in `near`, -1: they are not all there
  uint64_t* near;    // [rows, chunks, kNear]: the logits up to the bin of the chunk's k-th
  uint64_t* sure;    // [rows, chunks]
  uint64_t* list;    // [rows, far]
  RowState* state;   // [rows]
};

// 1. A chunk's largest logit and its histogram, relative to that.  (48 us for 256
// rows of 131072.)
template <typename T>
__global__ __launch_bounds__(kChunkThreads) void sample_chunk_kernel(const SplitArgs p) {
  constexpr int E = kChunkPer, NT = kChunkThreads;
  __shared__ uint64_t mass[kBins];
  __shared__ uint32_t cnt[kBins];
  __shared__ float part[NT / 64];
  __shared__ int arg, n_near;
  __shared__ Cuts cuts;
  const int64_t lr = blockIdx.y, r = p.row0 + lr;
  const int64_t slot = lr * p.chunks + blockIdx.x;
  const T* row = (const T*)p.a.logits + r * p.a.row_stride;
  const Row s = row_settings(p.a, r);
  const int base = (int)blockIdx.x * kChunk;
  float x[E];
  load_chunk<T, E>(row, base, (int)p.a.vocab, x);
  for (int b = threadIdx.x; b < kBins; b += NT) {
    cnt[b] = 0;
    mass[b] = 0;
  }
  if (threadIdx.x == 0) arg = kNoLimitIndex;
  float best = x[0];
#pragma unroll
  for (int e = 1; e < E; ++e) best = fmaxf(best, x[e]);
  const float m = block_max<NT>(best, part);
  if (threadIdx.x == 0) {
    p.max[slot] = m;
    p.near_n[slot] = s.use_k && s.k <= kNear && !is_real(m) ? 0 : -1;
    n_near = 0;
  }
  if (!is_real(m)) return;
  if (s.greedy) {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (x[e] == m) atomicMin(&arg, index_of<E>(base, e));
    __syncthreads();
    if (threadIdx.x == 0) p.arg[slot] = arg;
    return;
  }
  const float top = grid_of(m, s.cb);
  Cuts q = no_cuts();
  if (s.use_k) {
    // Past the chunk's own k-th no logit is among the row's first k.
    count_logits<NT, E>(s, x, top, cnt);
    by_one_wave<NT>(q, &cuts, [&] { find_k(s, cnt, q); });
    if (q.k_upto <= kNear && s.k <= kNear) {
      if (threadIdx.x == 0) p.near_n[slot] = (int)q.k_upto;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int b = bin_of(x[e], top, s.cb);
        const int at = append_at(&n_near, b < kBins && b <= q.k_bin);
        if (at >= 0) p.near[slot * kNear + at] = order_of(x[e], index_of<E>(base, e));
      }
    }
    for (int b = threadIdx.x; b < kBins; b += NT) p.cnt[slot * kBins + b] = cnt[b];
  }
  // What lies below the least kept t from here lies further below it from the
  // row's largest; only top-p's total counts it.
  const double least = s.use_p ? kLeastT : s.min_t;
  Series series;
  series.keep();
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int b = bin_of(x[e], top, s.cb);
    const double t = t_of(x[e], m, s.c);
    if (b < kBins && b <= q.k_bin && t >= least)
      atomicAdd((unsigned long long*)&mass[b], (unsigned long long)weight42(t, series));
  }
  __syncthreads();
  for (int b = threadIdx.x; b < kBins; b += NT) p.mass[slot * kBins + b] = mass[b];
}

// 2. The row's histogram from its chunks' and the bins that its cuts fall in.  (10
// us there, 3 of few rows.)
__global__ __launch_bounds__(kBins) void sample_merge_kernel(const SplitArgs p) {
  __shared__ uint64_t mass[kBins];
  __shared__ uint32_t cnt[kBins];
  __shared__ double scale[kMaxChunks];  // of a chunk's weights to the row's
  __shared__ int shift[kMaxChunks];     // of its bins; kBins: none of them is drawn
  __shared__ float part[kBins / 64];
  __shared__ int n_near, away;
  const int64_t lr = blockIdx.x, r = p.row0 + lr;
  const Row s = row_settings(p.a, r);
  if (threadIdx.x == 0) n_near = away = 0;
  __syncthreads();
  float mine = -INFINITY;
  for (int g = threadIdx.x; g < p.chunks; g += kBins) {
    mine = fmaxf(mine, p.max[lr * p.chunks + g]);
    const int n = p.near_n[lr * p.chunks + g];
    if (n < 0) away = 1;
    else atomicAdd(&n_near, n);
  }
  const float m = block_max<kBins>(mine, part);  // (waits for all)
  const bool near = !away && n_near <= kListMax;
  const float top = grid_of(m, s.cb);
  Cuts q = no_cuts();
  if (is_real(m) && !s.greedy && !near) {
    for (int g = threadIdx.x; g < p.chunks; g += kBins) {
      const float mg = p.max[lr * p.chunks + g], by = top - grid_of(mg, s.cb);
      shift[g] = is_real(mg) && by < (float)kBins ? (int)by : kBins;
      scale[g] = exp2(t_of(mg, m, s.c));
    }
    __syncthreads();
    if (s.use_k || s.use_p) {
      const int b = threadIdx.x;
      uint32_t n = 0;
      uint64_t w = 0;
#pragma unroll 8
      for (int g = 0; g < p.chunks; ++g) {
        if (b < shift[g]) continue;
        const int64_t at = (lr * p.chunks + g) * kBins + (b - shift[g]);
        if (s.use_k) n += p.cnt[at];
        if (s.use_p) w += (uint64_t)rint((double)p.mass[at] * scale[g]);
      }
      cnt[b] = n;
      mass[b] = w;
      __syncthreads();
      if (threadIdx.x < 64) {
        if (s.use_k) find_k(s, cnt, q);
        if (s.use_p) find_p(s, mass, q);
      }
    }
    find_least(s, m, top, q);
  }
  if (threadIdx.x == 0) p.state[lr] = RowState{q, top, m, 0, near};
}

// 3. From a chunk's histogram the weight that is kept whatever happens in the
// cuts' bins (`sure`), and if it has candidates those to the row's list:
// counted, a place taken for all of them at once, written.  (38 us there with
// top-p, 2 where the chunks' lists hold all that can be drawn.)
template <typename T>
__global__ __launch_bounds__(kChunkThreads) void sample_gather_kernel(const SplitArgs p) {
  constexpr int E = kChunkPer, NT = kChunkThreads;
  static_assert(NT == kBins, "a thread a bin");
  __shared__ uint64_t part[NT / 64];
  __shared__ int n_here, first, some;
  const int64_t lr = blockIdx.y, r = p.row0 + lr;
  const int64_t slot = lr * p.chunks + blockIdx.x;
  const Row s = row_settings(p.a, r);
  RowState* st = p.state + lr;
  const float m = st->m, top = st->top, mg = p.max[slot];
  if (s.greedy || !is_real(m) || st->near) return;
  const Cuts q = st->cuts;
  if (threadIdx.x == 0) n_here = some = 0;
  __syncthreads();
  const float shift = top - grid_of(mg, s.cb);
  uint64_t w = 0;
  if (is_real(mg) && shift < (float)kBins) {  // (a chunk without a logit left no histogram)
    const int64_t at = slot * kBins + threadIdx.x;
    const int b = threadIdx.x + (int)shift;
    w = p.mass[at];
    // (Top-k counts what weighs nothing, too.)
    if (is_candidate(q, b) && (w > 0 || (b == q.k_bin && p.cnt[at] > 0))) some = 1;
    w = b < sure_bins(q) ? w : 0;
  }
  w = wave_sum_u64(w);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = w;
  __syncthreads();
  if (threadIdx.x == 0) {
    uint64_t sum = 0;
    for (int i = 0; i < NT / 64; ++i) sum += part[i];
    p.sure[slot] = sum ? (uint64_t)rint((double)sum * exp2(t_of(mg, m, s.c))) : 0;
  }
  if (!some) return;
  const int base = (int)blockIdx.x * kChunk;
  float x[E];
  load_chunk<T, E>((const T*)p.a.logits + r * p.a.row_stride, base, (int)p.a.vocab, x);
  uint32_t mine = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int b = bin_of(x[e], top, s.cb);
    mine |= (uint32_t)is_candidate(q, b) << e;
  }
  const int n = (int)wave_sum_u64((uint64_t)__popc(mine));
  int at = 0;
  if ((threadIdx.x & 63) == 0 && n) at = atomicAdd(&n_here, n);
  at = __builtin_amdgcn_readfirstlane(at);
  __syncthreads();
  if (threadIdx.x == 0) first = n_here ? atomicAdd(&st->n_list, n_here) : 0;
  __syncthreads();
  at += first + (int)wave_scan_u64((uint64_t)__popc(mine)) - __popc(mine);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if ((mine >> e & 1) && at < kFarMax) p.list[lr * p.far + at] = order_of(x[e], index_of<E>(base, e));
    at += mine >> e & 1;
  }
}

// The draw from a list (sh.list, n of them) of all that can be kept.
template <typename T, int NT, int LIST>
__device__ void draw_from_list(Shared<NT, LIST>& sh, const SampleArgs& a, const Row& s, int64_t r, float m, float top,
                               int n) {
  static_assert(kNear <= kMid && kMid <= NT, "a thread a kept logit");
  constexpr int PER = LIST / NT;
  uint64_t o[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) o[j] = threadIdx.x + j * NT < n ? sh.list[threadIdx.x + j * NT] : ~0ull;
  Cuts q = cuts_anywhere();
  int n_cut = n;
  if (n > kSmall) {
    // As of a row: the bins of the cuts, and their candidates alone to the list.
    for (int b = threadIdx.x; b < kBins; b += NT) {
      sh.cnt[b] = 0;
      sh.mass[b] = 0;
    }
    if (threadIdx.x == 0) sh.n_list = 0;
    __syncthreads();
    q = no_cuts();
    int bin[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      bin[j] = o[j] != ~0ull ? bin_of(value_of(o[j]), top, s.cb) : kBins;
      if (bin[j] < kBins) atomicAdd(&sh.cnt[bin[j]], 1u);
    }
    __syncthreads();
    by_one_wave<NT>(q, &sh.cuts, [&] { find_k(s, sh.cnt, q); });
    if (s.use_p) {
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (bin[j] < kBins && bin[j] <= q.k_bin)
          atomicAdd((unsigned long long*)&sh.mass[bin[j]],
                    (unsigned long long)weight_from(t_of(value_of(o[j]), m, s.c), kLeastT));
      __syncthreads();
      by_one_wave<NT>(q, &sh.cuts, [&] { find_p(s, sh.mass, q); });
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (j * NT >= n) break;
      const int at = append_at(&sh.n_list, is_candidate(q, bin[j]));
      if (at >= 0) sh.list[at] = o[j];
    }
    __syncthreads();
    n_cut = sh.n_list;
  }
  const uint64_t lim = Candidates<T, NT, LIST>{sh, nullptr, 0, m, top, s, n_cut, nullptr}.limit(q);
  __syncthreads();
  if (threadIdx.x == 0) sh.n_small = 0;
  __syncthreads();
  // What is kept: at most k of them, and k is at most kNear.
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    if (j * NT >= n) break;
    const uint64_t w = o[j] != ~0ull && o[j] <= lim
                           ? weight_from(t_of(value_of(o[j]), m, s.c), s.min_t) : 0;
    const int at = append_at(&sh.n_small, w > 0);
    if (at >= 0) {
      sh.small_w[at] = w;
      sh.kept[at] = o[j];
    }
  }
  __syncthreads();
  const int n_kept = sh.n_small;
  if (threadIdx.x >= n_kept) return;
  const uint64_t mine = sh.kept[threadIdx.x];
  uint64_t before = 0, total = 0;
#pragma unroll 4
  for (int j = 0; j < n_kept; ++j) {
    const uint64_t w = sh.small_w[j];
    total += w;
    before += (uint32_t)sh.kept[j] < (uint32_t)mine ? w : 0;
  }
  const uint64_t at = draw_at(s.u, total);
  if (at < before || at >= before + sh.small_w[threadIdx.x]) return;
  a.tokens[r] = (int)(uint32_t)mine;
  if (a.logprob)
    a.logprob[r] = (float)(t_of(value_of(mine), m, s.c) * 0.69314718055994530942 -
                           log((double)total * 0x1p-42));
}

// 4. The cuts among the candidates, the chunk that the draw falls in, its token.
// (22 us there, 10 of few rows: a chain of block-wide steps.)
template <typename T>
__global__ __launch_bounds__(kChunkThreads) void sample_finish_kernel(const SplitArgs p) {
  constexpr int E = kChunkPer, NT = kChunkThreads, LIST = kListMax;
  __shared__ Shared<NT, LIST> sh;
  __shared__ uint64_t chunk_sum[kMaxChunks];
  const int64_t lr = blockIdx.x, r = p.row0 + lr;
  const SampleArgs& a = p.a;
  const T* row = (const T*)a.logits + r * a.row_stride;
  const Row s = row_settings(a, r);
  const RowState st = p.state[lr];
  const float m = st.m;
  if (!is_real(m) || s.greedy) {
    if (threadIdx.x == 0) {
      int token = -1;
      for (int g = p.chunks - 1; g >= 0 && is_real(m); --g)
        if (p.max[lr * p.chunks + g] == m) token = p.arg[lr * p.chunks + g];
      a.tokens[r] = token;
      if (a.logprob) a.logprob[r] = is_real(m) ? 0.0f : -INFINITY;
    }
    return;
  }
  if (st.near) {
    // (chunk_sum holds the lists' lengths here.)
    for (int g = threadIdx.x; g < p.chunks; g += NT) chunk_sum[g] = (uint64_t)p.near_n[lr * p.chunks + g];
    if (threadIdx.x == 0) sh.n_list = 0;
    __syncthreads();
    for (int i0 = 0; i0 < p.chunks * kNear; i0 += NT) {
      const int i = i0 + threadIdx.x, g = i / kNear;
      const bool is = g < p.chunks && i % kNear < (int)chunk_sum[g];
      const uint64_t o = is ? p.near[(lr * p.chunks + g) * kNear + i % kNear] : 0;
      const int at = append_at(&sh.n_list, is);
      if (at >= 0) sh.list[at] = o;
    }
    __syncthreads();
    const int n = sh.n_list;
    __syncthreads();
    draw_from_list<T, NT, LIST>(sh, a, s, r, m, st.top, n);
    return;
  }
  for (int g = threadIdx.x; g < p.chunks; g += NT) chunk_sum[g] = p.sure[lr * p.chunks + g];
  const int n = st.n_list;
  if (n <= LIST)
    for (int i = threadIdx.x; i < n; i += NT) sh.list[i] = p.list[lr * p.far + i];
  __syncthreads();
  Candidates<T, NT, LIST> cand{sh, row, (int)a.vocab, m, st.top, s, n, p.list + lr * p.far};
  const uint64_t lim = cand.limit(st.cuts);
  const float limit_x = lim != ~0ull ? value_of(lim) : -INFINITY;
  const int limit_i = lim != ~0ull ? (int)(uint32_t)lim : -1;  // (-inf itself is not kept)
  cand.each(0, kBins - 1, [&](uint64_t o, int b) {
    if (o > lim || !is_candidate(st.cuts, b)) return;
    const uint64_t w = cand.weight(o, s.min_t);
    if (w) atomicAdd((unsigned long long*)&chunk_sum[(uint32_t)o / kChunk], (unsigned long long)w);
  });
  __syncthreads();
  uint64_t total = 0;
  for (int g = 0; g < p.chunks; ++g) total += chunk_sum[g];
  uint64_t at = draw_at(s.u, total);
  int g = 0;
  for (; g + 1 < p.chunks && at >= chunk_sum[g]; ++g) at -= chunk_sum[g];
  const int base = g * kChunk;
  float x[E];
  load_chunk<T, E>(row, base, (int)a.vocab, x);
  uint64_t mine = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) mine += kept_weight<E>(s, x[e], index_of<E>(base, e), m, limit_x, limit_i);
  mine = wave_sum_u64(mine);
  if ((threadIdx.x & 63) == 0) sh.wave_sum[threadIdx.x >> 6] = mine;
  __syncthreads();
  // (The chunk's sum was scaled as a whole: its logits' own may be less, by half a unit each.)
  uint64_t here = 0;
  for (int w = 0; w < NT / 64; ++w) here += sh.wave_sum[w];
  at = at < here ? at : here - 1;
  int token;
  double t;
  if (locate<NT, E, LIST>(sh, s, x, base, m, limit_x, limit_i, at, &token, &t)) {
    a.tokens[r] = token;
    if (a.logprob) a.logprob[r] = (float)(t * 0.69314718055994530942 - log((double)total * 0x1p-42));
  }
}

template <typename T, int NT, int E>
void launch_row(const SampleArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((sample_row_kernel<T, NT, E>), dim3((uint32_t)a.rows), dim3(NT), 0, st, a);
}

size_t up(size_t bytes) { return (bytes + 255) & ~(size_t)255; }

template <typename T>
bdh_status sample_typed(const SampleArgs& a, hipStream_t st, uint64_t* launches) {
  // Workgroups of up to 1024 threads, 4 to 16 logits a thread.  One for the whole
  // row, against the four launches: 16000 logits with top-k 50 and top-p 0.95,
  // 1 row 14.9 / 18.7 us, 256 rows 18.1 / 24.5, with top-p 0.9 alone 30.4 / 40.8
  // (from some 1000 rows on the launches win, 68.7 / 55.8); rows of 32000, 32 a
  // thread, spill (58, split 23).
  if (a.vocab <= 16384) {
    if (a.vocab <= 256) launch_row<T, 64, 4>(a, st);
    else if (a.vocab <= 1024) launch_row<T, 256, 4>(a, st);
    else if (a.vocab <= 4096) launch_row<T, 1024, 4>(a, st);
    else if (a.vocab <= 8192) launch_row<T, 1024, 8>(a, st);
    else launch_row<T, 1024, 16>(a, st);
    BDH_HIP_TRY(hipGetLastError());
    *launches += 1;
    return BDH_OK;
  }
  SplitArgs p;
  p.a = a;
  p.chunks = (int)((a.vocab + kChunk - 1) / kChunk);
  p.far = a.vocab < kFarMax ? (int)a.vocab : kFarMax;
  // Groups of rows that kGroupBytes of scratch hold (8.2 KB a chunk, up to 256 KB a
  // row; the stream keeps up to a quarter more), as many in each, and smaller ones
  // where there is less to be had.  1024 rows of 20000 in one group 113 us, in two
  // of 512 130; 300 of 2^20 in two groups 1017, in three 1133.
  const int64_t row_bytes = p.chunks * (int64_t)(4 + 4 + kBins * 4 + kBins * 8 + 4 + kNear * 8 + 8) +
                            (int64_t)p.far * 8 + (int64_t)sizeof(RowState);
  const int64_t most = kGroupBytes / row_bytes, groups = (a.rows + most - 1) / most;
  int64_t group = (a.rows + groups - 1) / groups;
  size_t sizes[9];
  void* buf = nullptr;
  for (;; group = (group + 1) / 2) {
    const size_t slots = (size_t)group * (size_t)p.chunks;
    const size_t need[9] = {up(slots * 4), up(slots * 4), up(slots * kBins * 4), up(slots * kBins * 8), up(slots * 4),
                            up(slots * kNear * 8), up(slots * 8), up((size_t)group * (size_t)p.far * 8),
                            up((size_t)group * sizeof(RowState))};
    size_t bytes = 0;
    for (int i = 0; i < 9; ++i) bytes += sizes[i] = need[i];
    const bdh_status s = scratch(st, SLOT_SAMPLE, bytes, &buf);
    if (s == BDH_OK) break;
    if (group == 1 || !scratch_short(s)) return s;
  }
  char* at = (char*)buf;
  p.max = (float*)at; at += sizes[0];
  p.arg = (int32_t*)at; at += sizes[1];
  p.cnt = (uint32_t*)at; at += sizes[2];
  p.mass = (uint64_t*)at; at += sizes[3];
  p.near_n = (int32_t*)at; at += sizes[4];
  p.near = (uint64_t*)at; at += sizes[5];
  p.sure = (uint64_t*)at; at += sizes[6];
  p.list = (uint64_t*)at; at += sizes[7];
  p.state = (RowState*)at;
  for (p.row0 = 0; p.row0 < a.rows; p.row0 += group) {
    const uint32_t n = (uint32_t)(a.rows - p.row0 < group ? a.rows - p.row0 : group);
    const dim3 grid((uint32_t)p.chunks, n);
    hipLaunchKernelGGL((sample_chunk_kernel<T>), grid, dim3(kChunkThreads), 0, st, p);
    hipLaunchKernelGGL(sample_merge_kernel, dim3(n), dim3(kBins), 0, st, p);
    hipLaunchKernelGGL((sample_gather_kernel<T>), grid, dim3(kChunkThreads), 0, st, p);
    hipLaunchKernelGGL((sample_finish_kernel<T>), dim3(n), dim3(kChunkThreads), 0, st, p);
    BDH_HIP_TRY(hipGetLastError());
    *launches += 4;
  }
  return BDH_OK;
}

}  // namespace

bdh_status sample_tokens(const SampleArgs& a, hipStream_t st, uint64_t* launches) {
  return a.bf16 ? sample_typed<bf16_t>(a, st, launches) : sample_typed<float>(a, st, launches);
}

}  // namespace bdh
