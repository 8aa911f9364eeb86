// The gated block of latents and its backward pass, bf16 with f32 sums:
//   p = x U_h - th, q = c_h G_h - th                 per head h, [tokens, N]
//   out = up(p) m * act(q) m                         [tokens, H, N]
// with relu: up = act = ReLU (y of the layer, residual_stream.rs:440-505), m the latent
// mask; silu, gelu: up linear, th 0 and no mask.  c = x where there is no context.
// Backward, with g the gradient of out:
//   dp = g act(q) up'(p) m^2,  dq = g up(p) act'(q) m^2
//   dx = sum_h dp_h U_h^T,  dc_h = dq_h G_h^T,  dU_h = x^T dp_h,  dG_h = c_h^T dq_h.
//
// All products run on v_mfma_f32_32x32x16_bf16 from LDS tiles of 32 k's that direct
// loads fill one or two steps ahead.  A tile holds an operand as it lies in memory:
// rows along k (KC), or rows of k (MC), whose fragments ds_read_b64_tr_b16 transposes
// on the way to the registers; so no operand is ever laid out anew, U and G
// [H, D, N] serve the forward (MC) and dx, dc (KC) alike, dp and dq serve dx (KC) and
// dU (MC).  The first factor of a product is the one whose rows lie along the
// result's rows in memory: a lane's sums are then neighbours there.
#include <algorithm>
#include <type_traits>

#include "bdh_fp8.h"
#include "bdh_internal.h"

namespace bdh {
namespace {

constexpr int BK = 32;
enum { KC, MC };

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4_8 __attribute__((ext_vector_type(4), aligned(8)));
typedef unsigned int u32_1 __attribute__((aligned(1)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}
// 16 bytes from p to LDS at m0 + 16 * lane (M0 needs a wait state before it).
__device__ __forceinline__ void load_lds16(const char* p, uint32_t m0) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "{m0}"(m0) : "memory");
}
// The same from base (of the wave) + at.  (A scalar register that a vector instruction
// wrote needs 5 wait states before the load.)
__device__ __forceinline__ void load_lds16(const char* base, uint32_t at, uint32_t m0) {
  const uint64_t b = (uint64_t)base;
  const uint32_t low = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)b);
  const uint32_t high = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(b >> 32));
  asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(at), "s"(((uint64_t)high << 32) | low), "{m0}"(m0)
               : "memory");
}
// At most n of this wave's loads are in flight and all its LDS accesses are done, in every wave.
template <int N>
__device__ __forceinline__ void wait_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// An operand's tile of 32 k's by W rows (KC) or columns (MC), 64 W bytes of LDS.
//   KC  [W][32]: the 16-byte chunk c of row r lies at c ^ (r >> 1 & 3)
//   MC  [32][W]: the 32-byte piece q of row k lies at q ^ 2 (k & 3)
// which leaves both the fragments' reads without bank conflicts.  A direct load fills
// 1 KB; of the W / 16 that a tile takes each wave issues its share.
template <int MODE, int W, int WAVES = 4>
struct Tile {
  static constexpr int BYTES = 64 * W, LOADS = W / 16 / WAVES;
  static constexpr int PER = 512 / W;  // MC: rows of k in 1 KB
  static constexpr int WAVE_STEP = WAVES;
  // The lane's row (KC) or k (MC) of load j, and its chunk along the row.
  static __device__ __forceinline__ int row(int j, int w, int lane) {
    const int block = w + WAVES * j;
    return MODE == KC ? 16 * block + (lane >> 2) : PER * block + lane / (W / 8);
  }
  static __device__ __forceinline__ int chunk(int w, int lane) {
    if (MODE == KC) return (lane & 3) ^ ((lane >> 3) & 3);
    const int slot = lane % (W / 8), k = row(0, w, lane);
    return slot ^ ((k & 3) << 2);
  }
  // Fragment of 32 rows / columns from at (a multiple of 32), k's 16 kk ..+15.
  static __device__ __forceinline__ bf16x8 frag(const char* tile, int at, int kk, int lane) {
    if constexpr (MODE == KC) {
      const int r = at + (lane & 31), c = 2 * kk + (lane >> 5);
      return *(const bf16x8*)(tile + r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
    } else {
      const int k = 8 * (lane >> 5) + ((lane & 15) >> 2);  // of the lane's first row; the second is 4 on
      const int piece = at / 16 + ((lane >> 4) & 1);
      const char* p = tile + (16 * kk + k) * (2 * W) + ((piece ^ ((k & 3) << 1)) << 5) + ((lane & 3) << 3);
      const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
      const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 8 * W));
      return __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
};

// Load j of a tile from per-lane addresses; lanes that are not in write zeros.
template <class Tl>
__device__ __forceinline__ void fill_one(char* lds, uint32_t tile, int w, int lane, int j, bool in, const char* from) {
  const uint32_t to = tile + (uint32_t)((w + Tl::WAVE_STEP * j) * 1024);
  if (in) load_lds16(from, lds_addr(lds) + to);
  else *(u32x4*)(lds + to + 16 * lane) = u32x4{0, 0, 0, 0};
}
// The same from a base of the wave and the lane's place.
template <class Tl, class Inside>
__device__ __forceinline__ void fill_one(char* lds, uint32_t tile, int w, int lane, int j, Inside, bool in,
                                         const char* base, uint32_t at) {
  const uint32_t to = tile + (uint32_t)((w + Tl::WAVE_STEP * j) * 1024);
  if (Inside::value || in) load_lds16(base, at, lds_addr(lds) + to);
  else *(u32x4*)(lds + to + 16 * lane) = u32x4{0, 0, 0, 0};
}
// All of a tile's.
template <class Tl, class At, class In>
__device__ __forceinline__ void fill(char* lds, uint32_t tile, int w, int lane, bool whole, At&& at, In&& in) {
#pragma unroll
  for (int j = 0; j < Tl::LOADS; ++j) {
    const uint32_t to = tile + (uint32_t)((w + Tl::WAVE_STEP * j) * 1024);
    if (whole || in(j)) load_lds16(at(j), lds_addr(lds) + to);
    else *(u32x4*)(lds + to + 16 * lane) = u32x4{0, 0, 0, 0};
  }
}

// The same from a base and per-lane places, which move with the lanes' own rows alone.
template <class Tl, class In>
__device__ __forceinline__ void fill(char* lds, uint32_t tile, int w, int lane, bool whole, const char* base,
                                     const uint32_t (&at)[Tl::LOADS], In&& in) {
#pragma unroll
  for (int j = 0; j < Tl::LOADS; ++j) {
    const uint32_t to = tile + (uint32_t)((w + Tl::WAVE_STEP * j) * 1024);
    if (whole || in(j)) load_lds16(base, at[j], lds_addr(lds) + to);
    else *(u32x4*)(lds + to + 16 * lane) = u32x4{0, 0, 0, 0};
  }
}

// The products of large calls: four waves, one a SIMD, of 256 f32 sums a lane; of a step of
// 32 k's each takes 2 x 8 fragments and 2 x 16 products.  A ring of five stages of 32 KB;
// at step s the barrier confirms stage s + 1, the loads of step s + 4 go into the stage of
// step s - 1, and fragments are read half a step ahead of their products, a fragment or
// a load after each product: so LDS, loads and the matrix cores
// run side by side in one wave.  Against two workgroups a CU of half the sums, a step moves
// 96 KB in LDS for the same products, not 144, and loads 32 KB, not 48 (4096 tokens of 8192
// latents, D 2048: 279 -> 218-228 us, 1.2-1.26 PFLOP/s).
//   load(inside, s, stage, j) this wave's j-th of LOADS loads of step s; not inside: zeros
//                             past k's end
//   read(set, i, stage, kk)   fragment i of half kk (as many as loads)
//   multiply(set, i)          product i of PRODUCTS
// (12 products, 7 loads and fragments: tiles of three quarters, 28 KB a step.)
constexpr int BIG_STAGE = 32768, BIG_STAGES = 5, BIG_LOADS = 8;
template <int LOADS = BIG_LOADS, int PRODUCTS = 16, class Load, class Read, class Multiply>
__device__ __forceinline__ void big_loop(int s0, int s1, int K, Load&& load, Read&& read, Multiply&& multiply) {
  if (s0 >= s1) return;
  const std::false_type no{};
#pragma unroll
  for (int q = 0; q < 4; ++q)
    if (s0 + q < s1) {
#pragma unroll
      for (int j = 0; j < LOADS; ++j) load(no, s0 + q, q, j);
    }
  wait_barrier<0>();
#pragma unroll
  for (int i = 0; i < LOADS; ++i) read(0, i, 0, 0);
  int stage = 0, s = s0;
  // Fragments after the products 0, 1, 3, 4, 6, 7, 9, 10 (0, 1, 2, 4, 5, 6, 8), so that the
  // last of them has five (three) products' time; loads after the others.
  static_assert((LOADS == 8 && PRODUCTS == 16) || (LOADS == 7 && PRODUCTS == 12), "the places of reads and loads");
  constexpr int GROUP = LOADS == 8 ? 3 : 4, FREE = PRODUCTS - LOADS;
  const auto is_read = [](int i) { return i % GROUP != GROUP - 1 && i < (LOADS == 8 ? 11 : 9); };
  const auto read_of = [](int i) { return i - i / GROUP; };
  const auto other_of = [](int i) {
    int n = 0;
    for (int k = 0; k < i; ++k) n += k % GROUP == GROUP - 1 || k >= (LOADS == 8 ? 11 : 9);
    return n;
  };
  const auto step = [&](auto inside) {
    constexpr bool INSIDE = decltype(inside)::value;
    // In flight: the steps s + 2 and s + 3, where they are whole.
    if (INSIDE || (s + 3 < s1 && (s + 4) * BK <= K)) wait_barrier<2 * LOADS>();
    else wait_barrier<0>();
    const int next = stage == BIG_STAGES - 1 ? 0 : stage + 1, free = stage == 0 ? BIG_STAGES - 1 : stage - 1;
    if (!INSIDE && s + 4 < s1) {
#pragma unroll
      for (int j = 0; j < LOADS; ++j) load(no, s + 4, free, j);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < PRODUCTS; ++i) {
      multiply(0, i);
      if (is_read(i)) read(1, read_of(i), stage, 1);
      else if (INSIDE) load(inside, s + 4, free, other_of(i));
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int i = 0; i < PRODUCTS; ++i) {
      multiply(1, i);
      if (is_read(i)) read(0, read_of(i), next, 0);  // (after the last step: any)
      else if (INSIDE && FREE + other_of(i) < LOADS) load(inside, s + 4, free, FREE + other_of(i));
      __builtin_amdgcn_sched_barrier(0);
    }
    stage = next;
  };
  const int last = min(s1, K / BK) - 1;  // whole step
  for (; s + 4 <= last; ++s) step(std::true_type{});
  for (; s < s1; ++s) step(no);
}

// Sums of the large tiles stay where the matrix cores have them until they are taken: else all
// 256 a lane move to the other registers at once where the loop ends, which pushes what is there
// to memory.  (Memory of its own, which the runtime has to find at a launch, makes a kernel end
// the process where the device has none left.  The products' 440 bytes a lane took 15 us a launch
// besides: the backward of 64 tokens of 8192, D 2048, saved 61 -> 45 us.)
__device__ __forceinline__ void until_here(floatx16& sums) { asm volatile("" : "+a"(sums)); }

// Rows of tokens: token i = (b, t) lies at b * batch + t * step elements.
struct TokenRows {
  int64_t batch, step;
  uint32_t time;
  float inverse;  // 1 / time
  __device__ __forceinline__ int64_t at(uint32_t i) const {
    // (i < 2^24 is exact in f32, so the quotient is off by one at most.)
    int32_t b = (int32_t)((float)i * inverse);
    int32_t t = (int32_t)(i - (uint32_t)b * time);
    if (t < 0) {
      --b;
      t += (int32_t)time;
    } else if (t >= (int32_t)time) {
      ++b;
      t -= (int32_t)time;
    }
    return b * batch + t * step;
  }
};

// Which tile a workgroup has.  Workgroup i runs on XCD i % 8, which has an L2 of its own:
// an XCD takes blocks of up to 8 by 8 tiles (what it runs at a time), along b first, so
// that its a-tiles' operand (8 of the weights' tiles, say) stays in its L2 while the other
// one streams.
struct TileOrder {
  int a_tiles, b_tiles;    // in all
  int a_block, b_block;    // of a block
  int b_blocks, blocks, per_xcd;
  __device__ __forceinline__ bool at(int id, int& a, int& b) const {
    const int k = id >> 3, size = a_block * b_block, local = k / size, r = k - local * size;
    const int block = (id & 7) * per_xcd + local;
    const int ga = block / b_blocks, gb = block - ga * b_blocks;
    a = ga * a_block + r % a_block;
    b = gb * b_block + r / a_block;
    return local < per_xcd && block < blocks && a < a_tiles && b < b_tiles;
  }
};
TileOrder tile_order(int64_t a_tiles, int64_t b_tiles) {
  TileOrder t{};
  t.a_tiles = (int)a_tiles;
  t.b_tiles = (int)b_tiles;
  t.a_block = a_tiles < 8 ? (int)a_tiles : 8;
  t.b_block = b_tiles < 8 ? (int)b_tiles : 8;
  const auto count = [&] {
    t.b_blocks = (t.b_tiles + t.b_block - 1) / t.b_block;
    t.blocks = (t.a_tiles + t.a_block - 1) / t.a_block * t.b_blocks;
    t.per_xcd = (t.blocks + 7) / 8;
    return t.blocks;
  };
  // Smaller blocks where there are too few for the eight XCDs.
  while (count() < 16 && (t.a_block > 1 || t.b_block > 1)) (t.b_block >= t.a_block ? t.b_block : t.a_block) /= 2;
  return t;
}
unsigned grid_of(const TileOrder& t) { return (unsigned)(8 * t.per_xcd * t.a_block * t.b_block); }

// --- activations ---------------------------------------------------------------------
enum { RELU = BDH_RELU, SILU = BDH_SILU, GELU = BDH_GELU };

// (A NaN stays one.)
__device__ __forceinline__ float relu(float x) { return x <= 0.0f ? 0.0f : x; }
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __expf(-x)); }
// The normal distribution at q, Phi(q), and exp(-q^2 / 2).  Of |q| the upper tail is
// exp(-q^2 / 2) f(t), t = 1 / (1 + 0.265 |q|), with f a polynomial of degree 9 without a
// constant, fitted here to the scaled complementary error function (least squares with
// weights moved towards the largest error): with its constants in f32 1e-7 of a tail to
// |q| = 14.5, past which the exponential is 0; in f32 steps within 2.1e-7 of Phi, which is
// 2e-6 of a tail at |q| = 6.  The slope takes the same exponential (the backward's projections
// of 3003 tokens of 4096, D 1024: 94 us with the library's erf, 78-83 so; 8192 tokens of 8192
// saved: 388 -> 366).
struct Normal {
  float cdf, bell;
};
__device__ __forceinline__ Normal normal(float q) {
  const float bell = __expf(-0.5f * q * q), t = __builtin_amdgcn_rcpf(fmaf(0.265f, fabsf(q), 1.0f));
  float f = 0.0306265727f;
  f = fmaf(f, t, -0.143310606f);
  f = fmaf(f, t, 0.215970472f);
  f = fmaf(f, t, -0.114308789f);
  f = fmaf(f, t, 0.136569932f);
  f = fmaf(f, t, 0.0608888119f);
  f = fmaf(f, t, 0.102556631f);
  f = fmaf(f, t, 0.105266571f);
  f = fmaf(f, t, 0.105740413f);
  const float tail = f * t * bell;
  return Normal{q > 0.0f ? 1.0f - tail : tail, bell};
}

// up(p) act(q) with relu's taken already.
template <int ACT>
__device__ __forceinline__ float value_of(float p, float q) {
  if (ACT == RELU) return p * q;
  return p * (q * (ACT == SILU ? sigmoid(q) : normal(q).cdf));
}
// g act(q) up'(p) and g up(p) act'(q), likewise.
template <int ACT>
__device__ __forceinline__ void grads_of(float g, float p, float q, float& dp, float& dq) {
  if (ACT == RELU) {
    dp = p <= 0.0f ? 0.0f : g * q;
    dq = q <= 0.0f ? 0.0f : g * p;
    return;
  }
  float z, slope;
  if (ACT == SILU) {
    z = sigmoid(q);
    slope = z + q * z * (1.0f - z);
  } else {
    const Normal n = normal(q);
    z = n.cdf;
    slope = z + q * n.bell * 0.39894228f;
  }
  dp = g * (q * z);
  dq = g * p * slope;
}

struct GatedArgs {
  const bf16_t *x, *c;      // [M, D]; c (or null) by heads and tokens
  const bf16_t *up, *gate;  // [H, D, N]
  int64_t M, N, D;
  int H;
  int64_t c_head;           // elements from a head of c to the next
  TokenRows c_rows;
  float th;
  const float* mask;        // [N] or null
  bf16_t* out;              // [M, H, N]
  const bf16_t* g;          // [M, H, N]
  uint8_t *up_codes, *up_scales, *gate_codes, *gate_scales;
  // [M, H, N].  Rounded to bf16, as the products' operands have to be: 0.0017 of them in the
  // mean square, as the gradients' own rounding (f32 operands would cost three products for one).
  bf16_t *dp, *dq;
  TileOrder order;          // tiles of latents (of all heads) and of tokens
};

// --- both projections, and what is made of them ------------------------------------------
enum { OUT, SAVE, BACK };

// Two sums that lanes l and l + 32 hold four neighbours each of, to eight neighbours a lane.
__device__ __forceinline__ void join_halves(u32x2 a, u32x2 b, u32x4& v) {
  const auto x = __builtin_amdgcn_permlane32_swap(a.x, b.x, false, false);
  const auto y = __builtin_amdgcn_permlane32_swap(a.y, b.y, false, false);
  v = u32x4{x[0], y[0], x[1], y[1]};
}
__device__ __forceinline__ u32x2 join_halves(uint32_t a, uint32_t b) {
  const auto x = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  return u32x2{x[0], x[1]};
}

// A workgroup: 128 latents (n) of a head by 128 tokens (m), a wave 64 by 64 of both
// products.  NJ 1: by 64 tokens, for calls of few tiles.  NJ 3 and 4 (no context): by 192
// and 256 tokens, a wave 64 by 96 and 128, in big_loop.
template <int ACT, int EPI, bool CTX, int NJ>  // NJ: 32 tokens each of a wave
__global__ __launch_bounds__(256, NJ > 2 ? 1 : 2) void gated_kernel(const GatedArgs a) {
  constexpr bool BIG = NJ > 2;
  static_assert(!(CTX && BIG), "a context's tiles do not fit");
  typedef Tile<MC, 128> W;
  typedef Tile<KC, 64 * NJ> X;
  constexpr int STAGE = 2 * W::BYTES + (CTX ? 2 : 1) * X::BYTES, STAGES = BIG ? BIG_STAGES : CTX ? 2 : 3;
  __shared__ __attribute__((aligned(16))) char lds[STAGES * STAGE];
  const int lane = threadIdx.x & 63, w = wave_id();
  const int D = (int)a.D, N = (int)a.N, M = (int)a.M;
  int an, am;
  if (!a.order.at((int)blockIdx.x, an, am)) return;
  const int n_tiles = (N + 127) / 128;
  // (With the largest tiles all vector registers are taken: the divisions' results, which are
  // the vector unit's, go to scalar ones.)
  const auto scalar = [](int v) { return NJ == 4 ? __builtin_amdgcn_readfirstlane(v) : v; };
  const int n0 = scalar(an % n_tiles) * 128, h = scalar(an / n_tiles), m0 = scalar(am) * 64 * NJ;
  const char* wp[2][2];
  {
    const int c = W::chunk(w, lane) * 8;
    const int col = n0 + c < N ? n0 + c : 0;  // (past the end: any, never stored)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int64_t off = ((int64_t)h * D + W::row(j, w, lane)) * N + col;
      wp[0][j] = (const char*)(a.up + off);
      wp[1][j] = (const char*)(a.gate + off);
    }
  }
  const char* xp[2][X::LOADS];
#pragma unroll
  for (int j = 0; j < X::LOADS; ++j) {
    const int m = m0 + X::row(j, w, lane);
    const uint32_t i = (uint32_t)(m < M ? m : M - 1);
    xp[0][j] = (const char*)(a.x + (int64_t)i * D + X::chunk(w, lane) * 8);
    if (CTX) xp[1][j] = (const char*)(a.c + (int64_t)h * a.c_head + a.c_rows.at(i) + X::chunk(w, lane) * 8);
  }
  const int steps = (D + BK - 1) / BK;
  const auto issue = [&](int s, int stage) {
    const int k0 = s * BK;
    const bool whole = k0 + BK <= D;
    const uint32_t base = (uint32_t)(stage * STAGE);
    const auto w_ok = [&](int j) { return k0 + W::row(j, w, lane) < D; };
    const auto x_ok = [&](int) { return k0 + X::chunk(w, lane) * 8 < D; };
    const int64_t wo = (int64_t)k0 * N * 2;
    fill<W>(lds, base, w, lane, whole, [&](int j) { return wp[0][j] + wo; }, w_ok);
    fill<W>(lds, base + W::BYTES, w, lane, whole, [&](int j) { return wp[1][j] + wo; }, w_ok);
    fill<X>(lds, base + 2 * W::BYTES, w, lane, whole, [&](int j) { return xp[0][j] + 2 * k0; }, x_ok);
    if (CTX)
      fill<X>(lds, base + 2 * W::BYTES + X::BYTES, w, lane, whole, [&](int j) { return xp[1][j] + 2 * k0; }, x_ok);
  };
  floatx16 p[2][NJ], q[2][NJ];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) p[i][j][r] = q[i][j][r] = ACT == RELU ? -a.th : 0.0f;
  const int nw = 64 * (w & 1), mw = 32 * NJ * (w >> 1);
  if constexpr (BIG) {
    struct {
      bf16x8 u[2], g[2], x[NJ];
    } f[2];
    const char* const w_base[2] = {(const char*)(a.up + (int64_t)h * D * N + n0),
                                   (const char*)(a.gate + (int64_t)h * D * N + n0)};
    const char* const x_base = (const char*)(a.x + (int64_t)m0 * D);
    uint32_t w_at[2], x_at[X::LOADS];
    {
      const int c = W::chunk(w, lane) * 8;
#pragma unroll
      for (int j = 0; j < 2; ++j) w_at[j] = 2u * (uint32_t)(W::row(j, w, lane) * N + (n0 + c < N ? c : 0));
#pragma unroll
      for (int j = 0; j < X::LOADS; ++j) {
        const int m = X::row(j, w, lane);
        x_at[j] = 2u * (uint32_t)((m0 + m < M ? m : M - 1 - m0) * D + X::chunk(w, lane) * 8);
      }
    }
    big_loop<2 * W::LOADS + X::LOADS, 4 * NJ>(
        0, steps, D,
        [&](auto inside, int s, int stage, int j) {
          const int k0 = s * BK;
          const uint32_t base = (uint32_t)(stage * STAGE);
          if (j < 4) {
            const int r = j & 1, which = j >> 1;
            fill_one<W>(lds, base + which * W::BYTES, w, lane, r, inside, k0 + W::row(r, w, lane) < D,
                        w_base[which] + 2 * (int64_t)k0 * N, w_at[r]);
          } else {
            fill_one<X>(lds, base + 2 * W::BYTES, w, lane, j - 4, inside, k0 + X::chunk(w, lane) * 8 < D,
                        x_base + 2 * k0, x_at[j - 4]);
          }
        },
        [&](int set, int i, int stage, int kk) {
          const char* t = lds + stage * STAGE;
          if (i < 2) f[set].u[i] = W::frag(t, nw + 32 * i, kk, lane);
          else if (i < 4) f[set].g[i - 2] = W::frag(t + W::BYTES, nw + 32 * (i - 2), kk, lane);
          else f[set].x[i - 4] = X::frag(t + 2 * W::BYTES, mw + 32 * (i - 4), kk, lane);
        },
        [&](int set, int i) {
          const int j = i / 4, e = i & 1;
          if (i & 2) q[e][j] = mfma32(f[set].g[e], f[set].x[j], q[e][j]);
          else p[e][j] = mfma32(f[set].u[e], f[set].x[j], p[e][j]);
        });
  } else {
    issue(0, 0);
    if (STAGES == 3 && steps > 1) issue(1, 1);
    for (int s = 0, stage = 0; s < steps; ++s) {
      if (STAGES == 3 && s + 1 < steps && (s + 2) * BK <= D) wait_barrier<2 * W::LOADS + X::LOADS>();
      else wait_barrier<0>();
      if (s + STAGES - 1 < steps) issue(s + STAGES - 1, stage == 0 ? STAGES - 1 : stage - 1);
      const char* t = lds + stage * STAGE;
      stage = stage == STAGES - 1 ? 0 : stage + 1;
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        bf16x8 u[2], g[2], x[NJ], c[NJ];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          u[i] = W::frag(t, nw + 32 * i, kk, lane);
          if (i < NJ) x[i] = X::frag(t + 2 * W::BYTES, mw + 32 * i, kk, lane);
          g[i] = W::frag(t + W::BYTES, nw + 32 * i, kk, lane);
          if (i < NJ) c[i] = CTX ? X::frag(t + 2 * W::BYTES + X::BYTES, mw + 32 * i, kk, lane) : x[i];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < NJ; ++j) p[i][j] = mfma32(u[i], x[j], p[i][j]);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < NJ; ++j) q[i][j] = mfma32(g[i], c[j], q[i][j]);
      }
    }
  }
  // A lane has token mw + 32 j + (lane & 31) and, of 32 latents, 8 r + 4 (lane >> 5)
  // ..+3 for r of 0..3.  64 of the tile's tokens at a time (j) go through LDS, so that
  // memory sees whole rows of 128 latents, stored past the caches, which they would only
  // empty (16384 tokens, 4 heads of 8192, D 256, saved: 1400 -> 1200 us; with the conversions
  // of bdh_fp8.h 1000-1130: 2.1 GB of results at 2 TB/s beside 0.52 PFLOP/s of products, which
  // eight steps of k a tile, each waited for in full with a context, leave waiting for loads
  // and the ends; without saving 790).
  constexpr int VP = 272, CP = 144;  // row pitches in bytes (bank spread)
  char* const vals = lds;            // [64][VP]: out; the gradient, then dp
  char* const more = lds + 64 * VP;  // [64][VP]: dq; or [2][64][CP] codes, [2][64][4] scales
  char* const bytes = more + 128 * CP;
  static_assert(64 * VP + 128 * CP + 512 <= 2 * STAGE && 128 * VP <= 2 * STAGE, "the stages' memory");
  // (The thread opaque: else places computed from it before the products are kept through them.)
  int tid = (int)threadIdx.x;
  if (NJ == 4) asm volatile("" : "+v"(tid));
  const int high = (NJ == 4 ? tid & 63 : lane) >> 5, nb = (N + kFp8Block - 1) / kFp8Block;
  const int mine = 32 * (w >> 1) + ((NJ == 4 ? tid : lane) & 31);  // the lane's row of the part
  // Row r of part j, and its place in [tokens, H].
  const auto token = [&](int r, int j) { return m0 + 32 * NJ * (r >> 5) + 32 * j + (r & 31); };
  const auto place = [&](int m) { return (int64_t)m * a.H + h; };
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    wait_barrier<0>();
    if (EPI == BACK) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = tid / 16 + 16 * e, c = tid % 16, m = token(r, j);
        u32x4 g = {0, 0, 0, 0};
        if (m < M && n0 + 8 * c < N) g = *(const u32x4*)(a.g + place(m) * N + n0 + 8 * c);
        *(u32x4*)(vals + r * VP + 16 * c) = g;
      }
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int nt = nw + 32 * i;  // in the tile
      if (NJ == 4 && ACT != RELU) {
        until_here(p[i][j]);
        until_here(q[i][j]);
      }
      floatx4 mask[4];
      if (ACT == RELU && a.mask) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int n = n0 + nt + 8 * r + 4 * high;
          mask[r] = *(const floatx4*)(a.mask + (n < N ? n : 0));
          mask[r] *= mask[r];
        }
      }
      if (ACT == RELU) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          p[i][j][r] = relu(p[i][j][r]);
          q[i][j][r] = relu(q[i][j][r]);
        }
      }
      if (EPI == SAVE) {
        // The same 32 latents in 8 bits (those past N do not count).
        const auto keep = [&](const floatx16& v, int which) {
          floatx16 x = v;
          if (n0 + nt + 32 > N) {
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (n0 + nt + 8 * (r >> 2) >= N) x[r] = 0.0f;
          }
          uint32_t top = finite_top<ACT != RELU, 16>(x);
          const auto both = __builtin_amdgcn_permlane32_swap(top, top, false, false);
          top = max((uint32_t)both[0], (uint32_t)both[1]);
          const int scale = fp8_scale(top);
          const float power = fp8_power(scale);
          uint32_t c[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float f[4] = {v[4 * r], v[4 * r + 1], v[4 * r + 2], v[4 * r + 3]};
            fp8_keep_finite(f, scale);
            c[r] = fp8_pack4(f[0], f[1], f[2], f[3], power);
          }
#pragma unroll
          for (int r = 0; r < 2; ++r)
            *(u32x2*)(more + (64 * which + mine) * CP + nt + 16 * r + 8 * high) = join_halves(c[2 * r], c[2 * r + 1]);
          if (high == 0) bytes[(64 * which + mine) * 4 + nt / kFp8Block] = (char)scale;
        };
        keep(p[i][j], 0);
        keep(q[i][j], 1);
      }
#pragma unroll
      for (int r = 0; r < 4; r += 2) {  // two groups of four neighbours, then eight a lane
        char* const at = vals + mine * VP + 2 * (nt + 8 * r + 8 * high);
        u32x2 o[2], oq[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float f[4], fq[4];
          bf16x4 g;
          if (EPI == BACK) g = *(const bf16x4*)(vals + mine * VP + 2 * (nt + 8 * (r + e) + 4 * high));
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int v = 4 * (r + e) + k;
            if (EPI == BACK) {
              float gv = (float)g[k];
              if (ACT == RELU && a.mask) gv *= mask[r + e][k];
              grads_of<ACT>(gv, p[i][j][v], q[i][j][v], f[k], fq[k]);
            } else {
              f[k] = value_of<ACT>(p[i][j][v], q[i][j][v]);
              if (ACT == RELU && a.mask) f[k] *= mask[r + e][k];
            }
          }
          o[e] = u32x2{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3])};
          if (EPI == BACK) oq[e] = u32x2{pack_bf16x2(fq[0], fq[1]), pack_bf16x2(fq[2], fq[3])};
        }
        // (BACK: the two lanes of a row have read its gradients before either writes over them.)
        u32x4 v;
        join_halves(o[0], o[1], v);
        *(u32x4*)at = v;
        if (EPI == BACK) {
          join_halves(oq[0], oq[1], v);
          *(u32x4*)(at + 64 * VP) = v;
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = tid / 16 + 16 * e, c = tid % 16, m = token(r, j);
      if (m >= M || n0 + 8 * c >= N) continue;
      const int64_t to = place(m) * N + n0 + 8 * c;
      const u32x4 v = *(const u32x4*)(vals + r * VP + 16 * c);
      __builtin_nontemporal_store(v, (u32x4*)((EPI == BACK ? a.dp : a.out) + to));
      if (EPI == BACK) *(u32x4*)(a.dq + to) = *(const u32x4*)(more + r * VP + 16 * c);
    }
    if (EPI == SAVE) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int which = e >> 1, r = tid / 8 + 32 * (e & 1), c = tid % 8, m = token(r, j);
        if (m >= M || n0 + 16 * c >= N) continue;
        uint8_t* to = (which ? a.gate_codes : a.up_codes) + place(m) * N + n0 + 16 * c;
        const u32x4 v = *(const u32x4*)(more + (64 * which + r) * CP + 16 * c);
        if (n0 + 16 * c + 16 <= N) __builtin_nontemporal_store(v, (u32x4_8*)to);
        else *(u32x2*)to = u32x2{v[0], v[1]};
      }
      if (tid < 128) {
        const int which = tid >> 6, r = tid & 63, m = token(r, j);
        if (m < M) {
          uint8_t* to = (which ? a.gate_scales : a.up_scales) + place(m) * nb + n0 / kFp8Block;
          const uint32_t v = *(const uint32_t*)(bytes + tid * 4);
          if (n0 + 96 < N) {
            *(u32_1*)to = v;
          } else {
            for (int k = 0; n0 + kFp8Block * k < N; ++k) to[k] = (uint8_t)(v >> (8 * k));
          }
        }
      }
    }
  }
}

// dp and dq from what the forward saved: eight neighbours a thread.
template <int ACT>
__global__ __launch_bounds__(256) void gated_grads_kernel(const GatedArgs a) {
  const int N = (int)a.N, per = N / 8, nb = (N + kFp8Block - 1) / kFp8Block;
  const int64_t total = a.M * a.H * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const uint32_t row = (uint32_t)i / (uint32_t)per;  // (total < 2^32)
    const int n = (int)((uint32_t)i - row * (uint32_t)per) * 8;
    const int64_t at = (int64_t)row * N + n, block = (int64_t)row * nb + n / kFp8Block;
    const bf16x8 g = *(const bf16x8*)(a.g + at);
    const u32x2 cp = *(const u32x2*)(a.up_codes + at), cq = *(const u32x2*)(a.gate_codes + at);
    const float sp = fp8_power(a.up_scales[block]), sq = fp8_power(a.gate_scales[block]);
    bf16x8 dp, dq;
    floatx4 m2[2];
    if (ACT == RELU && a.mask) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        m2[half] = *(const floatx4*)(a.mask + n + 4 * half);
        m2[half] *= m2[half];
      }
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float p[4], q[4];
      fp8_unpack4(cp[half], sp, p);
      fp8_unpack4(cq[half], sq, q);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float gv = (float)g[4 * half + k], fp, fq;
        if (ACT == RELU && a.mask) gv *= m2[half][k];
        grads_of<ACT>(gv, p[k], q[k], fp, fq);
        dp[4 * half + k] = (bf16_t)fp;
        dq[4 * half + k] = (bf16_t)fq;
      }
    }
    *(bf16x8*)(a.dp + at) = dp;
    *(bf16x8*)(a.dq + at) = dq;
  }
}

// --- few tokens -------------------------------------------------------------------------
// Up to 64 tokens are bound by the weights, 4 D bytes a latent, each read once: a workgroup
// has 16 VEC latents of a head and all tokens, its eight waves share the k's, and the
// weights go from memory to registers (one token, 4 heads of 8192 latents, D 256: 8.2 us a call,
// 4.1 TB/s, 5.2 a launch of many in a graph, which find the weights in the caches; 64 tokens of
// 8192, D 2048: 17.4 us, 3.9 TB/s).  A lane reads VEC neighbours of eight rows of k and
// pairs the rows (one v_perm for two values), which leaves it with a fragment for each of
// its latents: 16 lanes hold every VEC-th latent of the tile.
constexpr int kFewTokens = 64, kFewWaves = 8;
template <int VEC> struct Words;
template <> struct Words<2> { typedef uint32_t type; };
template <> struct Words<8> { typedef u32x4 type; };
__device__ __forceinline__ uint32_t word_of(uint32_t v, int) { return v; }
__device__ __forceinline__ uint32_t word_of(const u32x4& v, int i) { return v[i]; }

template <int ACT, bool SAVED, bool CTX, int VEC, int MT>
__global__ __launch_bounds__(64 * kFewWaves) void few_kernel(const GatedArgs a) {
  typedef typename Words<VEC>::type V;
  constexpr int NT = 16 * VEC, PITCH = NT + 1;
  __shared__ float sums[kFewWaves][2][16 * MT * PITCH];
  const int lane = threadIdx.x & 63, w = wave_id(), i = lane & 15, g = lane >> 4;
  const int D = (int)a.D, N = (int)a.N, M = (int)a.M;
  // Neighbouring tiles on one XCD (every eighth workgroup): they share lines.
  const int tiles = (N + NT - 1) / NT, all = tiles * a.H, per_xcd = (all + 7) / 8;
  const int id = ((int)blockIdx.x & 7) * per_xcd + ((int)blockIdx.x >> 3);
  if ((int)blockIdx.x >> 3 >= per_xcd || id >= all) return;
  const int h = id / tiles, n0 = id % tiles * NT;
  const int n = n0 + VEC * i < N ? n0 + VEC * i : N - VEC;
  const bf16_t* const wp[2] = {a.up + (int64_t)h * D * N + n, a.gate + (int64_t)h * D * N + n};
  const bf16_t *xp[MT], *cp[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const uint32_t m = (uint32_t)(16 * t + i < M ? 16 * t + i : M - 1);
    xp[t] = a.x + (int64_t)m * D;
    cp[t] = CTX ? a.c + (int64_t)h * a.c_head + a.c_rows.at(m) : xp[t];
  }
  floatx4 acc[2][MT][VEC];
#pragma unroll
  for (int q = 0; q < 2; ++q)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[q][t][j] = zero4();
  struct Step {
    V rows[2][8];
    bf16x8 x[MT], c[MT];
  };
  const int steps = (D + 31) / 32;
  const auto load = [&](int s, Step& f) {
    // (Past D: any row, and zeros below.)
    const int k = 32 * s + 8 * g < D ? 32 * s + 8 * g : 0;
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int r = 0; r < 8; ++r) f.rows[q][r] = *(const V*)(wp[q] + (int64_t)(k + r) * N);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      f.x[t] = *(const bf16x8*)(xp[t] + k);
      if (CTX) f.c[t] = *(const bf16x8*)(cp[t] + k);
    }
  };
  const auto multiply = [&](int s, const Step& f) {
    const bool in = 32 * s + 8 * g < D;
    const bf16x8 none = {};
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        u32x4 v;
#pragma unroll
        for (int r = 0; r < 4; ++r)
          v[r] = __builtin_amdgcn_perm(word_of(f.rows[q][2 * r + 1], j >> 1), word_of(f.rows[q][2 * r], j >> 1),
                                       j & 1 ? 0x07060302u : 0x05040100u);
        const bf16x8 wf = in ? __builtin_bit_cast(bf16x8, v) : none;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          const bf16x8 xf = CTX && q ? f.c[t] : f.x[t];
          acc[q][t][j] = mfma16(wf, in ? xf : none, acc[q][t][j]);
        }
      }
  };
  // Wave w has every eighth step; the next one is asked for before a step is multiplied.
  Step f[2];
  if (w < steps) load(w, f[0]);
  for (int s = w; s < steps; s += 2 * kFewWaves) {
    if (s + kFewWaves < steps) load(s + kFewWaves, f[1]);
    multiply(s, f[0]);
    if (s + kFewWaves < steps) {
      if (s + 2 * kFewWaves < steps) load(s + 2 * kFewWaves, f[0]);
      multiply(s + kFewWaves, f[1]);
    }
  }
  // A lane has token i of each 16, and of the tile latents VEC (4 g + r) + j.
#pragma unroll
  for (int q = 0; q < 2; ++q)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int j = 0; j < VEC; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) sums[w][q][(16 * t + i) * PITCH + VEC * (4 * g + r) + j] = acc[q][t][j][r];
  __syncthreads();
  // Four (two) neighbours a thread: 32 latents lie in eight (sixteen) lanes.
  constexpr int EACH = VEC == 8 ? 4 : 2;
  for (int at = (int)threadIdx.x * EACH; at < M * NT; at += 64 * kFewWaves * EACH) {
    const int m = at / NT, nt = at % NT, nn = n0 + nt;
    const bool in = nn < N;
    float p[EACH], q[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      p[e] = q[e] = 0.0f;
#pragma unroll
      for (int k = 0; k < kFewWaves; ++k) {
        p[e] += sums[k][0][m * PITCH + nt + e];
        q[e] += sums[k][1][m * PITCH + nt + e];
      }
      if (ACT == RELU) {
        p[e] = relu(p[e] - a.th);
        q[e] = relu(q[e] - a.th);
      }
    }
    const int64_t row = (int64_t)m * a.H + h;
    if (SAVED) {
      const int nb = (N + kFp8Block - 1) / kFp8Block;
      const auto keep = [&](float (&v)[EACH], uint8_t* codes, uint8_t* scales) {
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < EACH; ++e) top = in ? max(top, finite_bits(v[e])) : 0;
#pragma unroll
        for (int o = 1; o < kFp8Block / EACH; o <<= 1)
          top = max(top, (uint32_t)__shfl_xor((int)top, o, kFp8Block / EACH));
        const int scale = fp8_scale(top);
        float f4[4] = {v[0], v[1], EACH == 4 ? v[EACH - 2] : 0.0f, EACH == 4 ? v[EACH - 1] : 0.0f};
        fp8_keep_finite(f4, scale);
        const uint32_t c = fp8_pack4(f4[0], f4[1], f4[2], f4[3], fp8_power(scale));
        if (!in) return;
        if (EACH == 4) *(uint32_t*)(codes + row * N + nn) = c;
        else *(uint16_t*)(codes + row * N + nn) = (uint16_t)c;
        if (nt % kFp8Block == 0) scales[row * nb + nn / kFp8Block] = (uint8_t)scale;
      };
      keep(p, a.up_codes, a.up_scales);
      keep(q, a.gate_codes, a.gate_scales);
    }
    if (!in) continue;
    float o[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      o[e] = value_of<ACT>(p[e], q[e]);
      if (ACT == RELU && a.mask) o[e] *= a.mask[nn + e] * a.mask[nn + e];
    }
#pragma unroll
    for (int e = 0; e < EACH; e += 2) *(uint32_t*)(a.out + row * N + nn + e) = pack_bf16x2(o[e], o[e + 1]);
  }
}

template <int ACT, bool SAVED, bool CTX, int VEC, int MT>
void launch_few_as(const GatedArgs& a, hipStream_t st) {
  const int64_t tiles = (a.N + 16 * VEC - 1) / (16 * VEC) * a.H;
  hipLaunchKernelGGL((few_kernel<ACT, SAVED, CTX, VEC, MT>), dim3((unsigned)((tiles + 7) / 8 * 8)),
                     dim3(64 * kFewWaves), 0, st, a);
}
template <int ACT, bool SAVED, bool CTX>
void launch_few(const GatedArgs& a, hipStream_t st) {
  // Tiles of 128 latents (whole lines a row) where they fill the chip; more tokens leave
  // registers for two latents a lane.
  if (a.M <= 16 && a.H * a.N >= 32768) launch_few_as<ACT, SAVED, CTX, 8, 1>(a, st);
  else if (a.M <= 16) launch_few_as<ACT, SAVED, CTX, 2, 1>(a, st);
  else if (a.M <= 32) launch_few_as<ACT, SAVED, CTX, 2, 2>(a, st);
  else launch_few_as<ACT, SAVED, CTX, 2, 4>(a, st);
}

// --- the four products of the backward pass -----------------------------------------------
// A workgroup: 256 of the result's columns (first factor) by 128 of its rows, a wave
// 128 by 64.  blockIdx.z: job and part of k.
enum { INPUTS, WEIGHTS };
struct ProductArgs {
  const bf16_t *dp, *dq, *x, *c, *up, *gate;  // as GatedArgs
  int64_t M, N, D;
  int H;
  int64_t c_head;
  TokenRows c_rows;
  bool c_apart;             // c's rows of a head do not follow one another
  int in_parts, w_parts;    // of k
  int in_tiles, w_tiles;    // in all, parts counted
  bool weights_first;
  int x_units;              // products (up's or gate's of a head) that a workgroup sums for d_x
  int x_jobs;               // such sums, of a part of k
  int x_parts;              // sums that make up d_x
  bool w_kept, w_more;      // the weights' sums stay in f32 (and go on from those there)
  int64_t x_size, c_size;   // elements of d_x, d_c
  bf16_t *d_x, *d_c, *d_up, *d_gate;
  float *x_sums, *c_sums, *w_sums;
};

// A wave's sums of a product, 32 NA of the result's columns from a0 by 32 NB of its rows
// from b0: to the gradient in bf16, or as one of the parts that join_kernel adds.  job: of
// x_jobs, where they are d_x's.  KEEP: w_kept and w_more count.
template <int WHAT, bool KEEP, int NA, int NB>
__device__ __forceinline__ void store_product(const ProductArgs& a, floatx16 (&acc)[NA][NB], int h, int which,
                                              int part, int job, int a0, int b0, int lane) {
  const int high = lane >> 5;
  const bool ctx = which && a.c;
  const int a_end = (int)(WHAT == INPUTS ? a.D : a.N), b_end = (int)(WHAT == INPUTS ? a.M : a.D);
  bf16_t* out;
  float* sums;
  int64_t out_at = 0;
  bool direct;
  if (WHAT == INPUTS && ctx) {
    out_at = (int64_t)h * a.c_head;
    out = a.d_c;
    sums = a.c_sums + part * a.c_size;
    direct = a.in_parts == 1;
  } else if (WHAT == INPUTS) {
    out = a.d_x;
    sums = a.x_sums + ((int64_t)job * a.in_parts + part) * a.x_size;
    direct = a.x_parts == 1;
  } else {
    out_at = (int64_t)h * a.D * a.N;
    out = which ? a.d_gate : a.d_up;
    sums = a.w_sums + ((int64_t)part * 2 + which) * a.H * a.D * a.N;
    direct = a.w_parts == 1 && !(KEEP && a.w_kept);
  }
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int b = b0 + 32 * j + (lane & 31);
    if (b >= b_end) continue;
    const int64_t row = out_at + (WHAT == WEIGHTS ? b * a.N : ctx ? a.c_rows.at((uint32_t)b) : b * a.D);
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      if (NA * NB == 16) until_here(acc[i][j]);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[i][j][8 * r + e]),
                                                          __float_as_uint(acc[i][j][8 * r + 4 + e]), false, false);
          v[e] = __uint_as_float(x[0]);
          v[4 + e] = __uint_as_float(x[1]);
        }
        const int at = a0 + 32 * i + 16 * r + 8 * high;
        if (at >= a_end) continue;
        if (direct) {
          *(u32x4*)(out + row + at) = u32x4{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                                            pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
        } else {
          if (WHAT == WEIGHTS && KEEP && a.w_more) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += sums[row + at + e];
          }
          *(floatx4*)(sums + row + at) = floatx4{v[0], v[1], v[2], v[3]};
          *(floatx4*)(sums + row + at + 4) = floatx4{v[4], v[5], v[6], v[7]};
        }
      }
    }
  }
}

// Neighbouring ids on one XCD (every eighth workgroup): the id of workgroup b of n, -1: none.
__device__ __forceinline__ int id_of(int b, int n) {
  const int per_xcd = (n + 7) / 8, id = (b & 7) * per_xcd + (b >> 3);
  return b >> 3 < per_xcd && id < n ? id : -1;
}

// BIG: 256 by 256, a wave 128 by 128, in big_loop.  MANY: d_x's sum goes on over x_units
// products, up's of the heads in turn, then gate's (where that reads current too), and the
// weights' sums over several launches.
template <int WHAT, bool BIG, bool MANY>
__device__ __forceinline__ void product_tile(const ProductArgs& a, char* lds, int id) {
  typedef Tile<WHAT == INPUTS ? KC : MC, 256> A;  // U, G rows d / dp, dq columns n
  constexpr int NB = BIG ? 4 : 2;                 // 32 of the result's rows each of a wave
  typedef Tile<WHAT == INPUTS ? KC : MC, 64 * NB> B;  // dp, dq rows m / x, c columns d
  constexpr int STAGE = A::BYTES + B::BYTES, LOADS = A::LOADS + B::LOADS;
  static_assert(!BIG || (STAGE == BIG_STAGE && LOADS == BIG_LOADS), "big_loop's stages");
  const int lane = threadIdx.x & 63, w = wave_id();
  const int D = (int)a.D, N = (int)a.N, M = (int)a.M;
  // The tiles along D, which share the larger operand, are neighbours.
  const int d_tiles = (D + (WHAT == INPUTS ? 256 : 64 * NB) - 1) / (WHAT == INPUTS ? 256 : 64 * NB);
  const int other = WHAT == INPUTS ? (M + 64 * NB - 1) / (64 * NB) : (N + 255) / 256;
  const int parts = WHAT == INPUTS ? a.in_parts : a.w_parts;
  const int di = id % d_tiles, oi = id / d_tiles % other, rest = id / d_tiles / other;
  const int part = rest % parts, job = rest / parts;
  constexpr bool ALONG = WHAT == INPUTS && MANY;
  // The products: d_x's jobs first, then d_c's heads.
  const int first = !ALONG ? job : job < a.x_jobs ? job * a.x_units : a.H + job - a.x_jobs;
  const int end = ALONG && job < a.x_jobs ? min(first + a.x_units, a.c ? a.H : 2 * a.H) : first + 1;
  const int h = first % a.H, which = first / a.H;  // which: 0 up, 1 gate
  const int a0 = (WHAT == INPUTS ? di : oi) * 256, b0 = (WHAT == INPUTS ? oi : di) * 64 * NB;
  const int K = WHAT == INPUTS ? N : M;
  const int64_t d_row = (int64_t)a.H * N;
  const bool ctx = which && a.c;
  // Bases of the workgroup, and the lanes' places (below 2^32 bytes: H N is 2^24 at most, of
  // BIG 2^23).  apart: c's rows go by their tokens; else they follow one another, as x's.
  const bool apart = !BIG && ctx && a.c_apart;
  const char* a_base;
  const char* b_base;
  uint32_t a_at[A::LOADS], b_at[B::LOADS];
  const int ac = A::chunk(w, lane) * 8, bc = B::chunk(w, lane) * 8;
  const auto inputs_of = [&](int h, int which) {
    a_base = (const char*)((which ? a.gate : a.up) + ((int64_t)h * D + a0) * N);
    b_base = (const char*)((which ? a.dq : a.dp) + b0 * d_row + (int64_t)h * N);
  };
  // Goes on to product u, once every wave has read the last stages.  (Opaque: else the
  // parts of its addresses are kept from the start on, in more scalar registers than there are.)
  const auto next_of = [&](int& u) {
    wait_barrier<0>();
    asm volatile("" : "+s"(u));
    inputs_of(u < a.H ? u : u - a.H, u >= a.H);
  };
  if (WHAT == INPUTS) {
    inputs_of(h, which);
  } else {
    a_base = (const char*)((which ? a.dq : a.dp) + (int64_t)h * N + a0);
    b_base = (const char*)(ctx ? a.c + (int64_t)h * a.c_head : a.x);
  }
#pragma unroll
  for (int j = 0; j < A::LOADS; ++j) {
    const int r = A::row(j, w, lane);
    a_at[j] = WHAT == INPUTS ? 2u * (uint32_t)((a0 + r < D ? r : D - 1 - a0) * N + ac)
                             : 2u * ((uint32_t)r * (uint32_t)d_row + (uint32_t)(a0 + ac < N ? ac : 0));
  }
#pragma unroll
  for (int j = 0; j < B::LOADS; ++j) {
    const int r = B::row(j, w, lane), d = b0 + bc < D ? b0 + bc : 0;
    b_at[j] = WHAT == INPUTS ? 2u * ((uint32_t)(b0 + r < M ? r : M - 1 - b0) * (uint32_t)d_row + (uint32_t)bc)
                             : 2u * (uint32_t)((apart ? 0 : r * D) + d);
  }
  const int steps = (K + BK - 1) / BK;
  const int s0 = (int)((int64_t)steps * part / parts), s1 = (int)((int64_t)steps * (part + 1) / parts);
  const auto load = [&](auto inside, int s, int stage, int j) {
    const int k0 = s * BK;
    const uint32_t base = (uint32_t)(stage * STAGE);
    if (j < A::LOADS) {
      fill_one<A>(lds, base, w, lane, j, inside, k0 + (WHAT == INPUTS ? ac : A::row(j, w, lane)) < K,
                  a_base + 2 * (WHAT == INPUTS ? (int64_t)k0 : k0 * d_row), a_at[j]);
    } else {
      const int i = j - A::LOADS;
      const bool in = decltype(inside)::value || k0 + (WHAT == INPUTS ? bc : B::row(i, w, lane)) < K;
      if (WHAT == WEIGHTS && apart)
        fill_one<B>(lds, base + A::BYTES, w, lane, i, in,
                    b_base + 2 * a.c_rows.at((uint32_t)(k0 + B::row(i, w, lane))) + b_at[i]);
      else
        fill_one<B>(lds, base + A::BYTES, w, lane, i, inside, in,
                    b_base + 2 * (WHAT == INPUTS ? (int64_t)k0 : (int64_t)k0 * D), b_at[i]);
    }
  };
  const auto issue = [&](int s, int stage) {
#pragma unroll
    for (int j = 0; j < LOADS; ++j) load(std::false_type{}, s, stage, j);
  };
  floatx16 acc[4][NB];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = zero16();
  const int aw = 128 * (w & 1), bw = 32 * NB * (w >> 1);
  if constexpr (BIG) {
    struct {
      bf16x8 a[4], b[4];
    } f[2];
    for (int u = first;;) {
      big_loop(
          s0, s1, K, load,
          [&](int set, int i, int stage, int kk) {
            const char* t = lds + stage * STAGE;
            if (i < 4) f[set].a[i] = A::frag(t, aw + 32 * i, kk, lane);
            else f[set].b[i - 4] = B::frag(t + A::BYTES, bw + 32 * (i - 4), kk, lane);
          },
          [&](int set, int i) { acc[i / 4][i % 4] = mfma32(f[set].a[i / 4], f[set].b[i % 4], acc[i / 4][i % 4]); });
      if (!ALONG || ++u == end) break;
      next_of(u);
    }
    store_product<WHAT, MANY>(a, acc, h, which, part, ALONG ? job : which * a.H + h, a0 + aw, b0 + bw, lane);
    return;
  }
  // Ring of three stages.  A step's loads may be in flight while the one before it is
  // multiplied, but only whole steps' are counted: a last one leaves out some.
  for (int u = first;;) {
    if (s0 < s1) issue(s0, 0);
    if (s0 + 1 < s1) issue(s0 + 1, 1);
    for (int s = s0, stage = 0; s < s1; ++s) {
      if (s + 1 < s1 && (s + 2) * BK <= K) wait_barrier<LOADS>();
      else wait_barrier<0>();
      if (s + 2 < s1) issue(s + 2, stage == 0 ? 2 : stage - 1);
      const char* t = lds + stage * STAGE;
      stage = stage == 2 ? 0 : stage + 1;
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        bf16x8 fa[4], fb[NB];
#pragma unroll
        for (int j = 0; j < NB; ++j) fb[j] = B::frag(t + A::BYTES, bw + 32 * j, kk, lane);
#pragma unroll
        for (int i = 0; i < 4; ++i) fa[i] = A::frag(t, aw + 32 * i, kk, lane);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < NB; ++j) acc[i][j] = mfma32(fa[i], fb[j], acc[i][j]);
      }
    }
    if (!ALONG || ++u == end) break;
    next_of(u);
  }
  store_product<WHAT, MANY>(a, acc, h, which, part, ALONG ? job : which * a.H + h, a0 + aw, b0 + bw, lane);
}

// Both kinds of products, the one with the longer sums first.
template <bool BIG, bool MANY>
__global__ __launch_bounds__(256, BIG ? 1 : 2) void product_kernel(const ProductArgs a) {
  __shared__ __attribute__((aligned(16))) char lds[BIG ? BIG_STAGES * BIG_STAGE : 3 * 64 * (256 + 128)];
  const int first = ((a.weights_first ? a.w_tiles : a.in_tiles) + 7) / 8 * 8, b = (int)blockIdx.x;
  const bool weights = (b < first) == a.weights_first;
  const int id = id_of(b < first ? b : b - first, weights ? a.w_tiles : a.in_tiles);
  if (id < 0) return;
  if (weights) product_tile<WEIGHTS, BIG, MANY>(a, lds, id);
  else product_tile<INPUTS, BIG, MANY>(a, lds, id);
}

// Both products of a kind straight from what the forward saved, D up to 256: dp and dq are
// made a step or two ahead, between memory and LDS, and never written.  A workgroup has
// eight waves, four for each product: INPUTS  128 tokens of a head by all columns, dx by
// four waves and dc by four; WEIGHTS  128 latents by all columns of dU and of dG.  Beside
// the tiles' direct loads a thread asks for eight neighbours of the gradient and of both
// codes a step, SETS steps ahead: WEIGHTS of 32 tokens by 128 latents; INPUTS of 64 tokens
// by the 64 latents of two steps, so that memory sees 128 (64) bytes of a row.  (The barriers'
// counts leave two steps' of them in flight.)
// 16384 tokens, 4 heads of 8192 latents, D 256: 938 and 730 us (0.59 and 0.75 PFLOP/s), 1.8
// and 1.4 a step.  A step's 146 KB in LDS are 1150 cycles and its products 1024, half a
// microsecond each: the rest is waiting for loads.  One step in four waits for all that are in
// flight (vmcnt 0), since the compiler converts the powers of all four sets of raw values
// there, the last asked for a step ago (not so where LEAN).
template <int WHAT, int ACT, bool MASK>
__global__ __launch_bounds__(512, 1) void fused_kernel(const ProductArgs a, const GatedArgs g) {
  constexpr bool IN = WHAT == INPUTS;
  // An activation's or the mask's own values leave registers for two steps' raw values, not
  // four (SiLU: for four), and none for what can be computed again (4096 tokens as above, us with
  // spilled registers / so: GELU 619 / 545, mask 552 / 535, SiLU 493 / 490, with two sets 524).
  constexpr bool LEAN = IN ? ACT != RELU : ACT == GELU || MASK;
  constexpr int SETS = LEAN && ACT != SILU ? 2 : 4;
  typedef Tile<IN ? KC : MC, 256, 8> F;  // U, G rows d / x, c columns d
  typedef Tile<MC, 128, 8> P;            // WEIGHTS: dp, dq columns n
  constexpr int TILES = 2 * F::BYTES, LOADS = 2 * F::LOADS;
  // dp and dq: INPUTS [128 tokens][64 latents], chunk c of row r at c ^ (r & 7), twice;
  // WEIGHTS a tile of a step, three times.
  constexpr int GRAD = IN ? 128 * 128 : P::BYTES, GRADS = IN ? 2 : 3;
  constexpr int NA = IN ? 4 : 2, NB = 6 - NA;
  __shared__ __attribute__((aligned(16))) char lds[3 * TILES + GRADS * 2 * GRAD];
  char* const grads = lds + 3 * TILES;
  const int lane = threadIdx.x & 63, w = wave_id(), which = w >> 2;
  const int D = (int)a.D, N = (int)a.N, M = (int)a.M;
  const int id = id_of((int)blockIdx.x, IN ? a.in_tiles : a.w_tiles);
  if (id < 0) return;
  const int tiles = ((IN ? M : N) + 127) / 128, parts = IN ? a.in_parts : a.w_parts;
  const int at0 = id % tiles * 128, part = id / tiles % parts, h = id / tiles / parts;
  const int K = IN ? N : M;
  const int nb = (N + kFp8Block - 1) / kFp8Block;
  // The tiles' sources: places in U_h, G_h or x (below 2^32, D being 256 at most); c's
  // rows go by their tokens.
  const int fc = F::chunk(w, lane) * 8, fd = fc < D ? fc : 0;
  uint32_t f_place[F::LOADS];
#pragma unroll
  for (int j = 0; j < F::LOADS; ++j) {
    const int r = F::row(j, w, lane);
    f_place[j] = IN ? 2u * ((uint32_t)(r < D ? r : D - 1) * (uint32_t)N + (uint32_t)fc) : 2u * (uint32_t)(r * D + fd);
  }
  const char* const f_base[2] = {(const char*)(IN ? a.up + (int64_t)h * D * N : a.x),
                                 (const char*)(IN ? a.gate + (int64_t)h * D * N : a.c + (int64_t)h * a.c_head)};
  const bool two = IN || a.c;  // WEIGHTS without a context: x for both
  // Steps of this part: an even number before it.
  const int steps = (K + BK - 1) / BK, pairs = (steps + 1) / 2;
  const int s0 = 2 * (int)((int64_t)pairs * part / parts);
  const int s1 = min(steps, 2 * (int)((int64_t)pairs * (part + 1) / parts));
  const auto issue = [&](auto inside, int s, int stage) {
    const int k0 = s * BK;
    const bool whole = decltype(inside)::value || (s < s1 && k0 + BK <= K);
    const uint32_t base = (uint32_t)(stage * TILES);
    const auto in = [&](int j) { return s < s1 && k0 + (IN ? fc : F::row(j, w, lane)) < K; };
    const int64_t move = 2 * (IN ? (int64_t)k0 : (int64_t)k0 * D);
    fill<F>(lds, base, w, lane, whole, f_base[0] + move, f_place, in);
    if (IN)
      fill<F>(lds, base + F::BYTES, w, lane, whole, f_base[1] + move, f_place, in);
    else if (two)
      fill<F>(lds, base + F::BYTES, w, lane, whole,
              [&](int j) { return f_base[1] + 2 * (a.c_rows.at((uint32_t)(k0 + F::row(j, w, lane))) + fd); }, in);
  };
  // A thread's eight neighbours of step s (their k: where the step's begin, and theirs
  // beyond that).  odd: s & 1.  Where they lie: a base that moves with the step, and the
  // thread's place (rows and latents past the end: the last ones').
  const int row = (int)threadIdx.x / (IN ? 8 : 16), col = 8 * ((int)threadIdx.x % (IN ? 8 : 16));
  const int64_t d_row = (int64_t)a.H * N, b_row = (int64_t)a.H * nb;
  const int64_t d_base = (int64_t)h * N + (IN ? at0 * d_row : 0), b_base = (int64_t)h * nb + (IN ? at0 * b_row : 0);
  const auto k_of = [&](int s) { return IN ? (s >> 1) * 2 * BK + col : s * BK + row; };
  const auto place = [&](int odd, uint32_t& d, uint32_t& b) {
    int r = IN ? row + 64 * odd : row;
    if (LEAN && IN) asm volatile("" : "+v"(r));  // (at each step anew)
    const int m = IN && at0 + r >= M ? M - 1 - at0 : r, n = IN ? col : (at0 + col < N ? at0 + col : N - 8);
    d = (uint32_t)(m * d_row + n);
    b = (uint32_t)(m * b_row + n / kFp8Block);
  };
  uint32_t d_kept[2], b_kept[2];
  place(0, d_kept[0], b_kept[0]);
  place(1, d_kept[1], b_kept[1]);
  struct Raw {
    u32x4 g;
    u32x2 p, q;
    int sp, sq;
  };
  // Always RAW loads, which the waits below count.
  constexpr int RAW = 5;
  const auto load_at = [&](int64_t d, int64_t b, uint32_t d_off, uint32_t b_off, Raw& r) {
    r.g = *(const u32x4*)((const char*)(g.g + d) + 2 * d_off);
    r.p = *(const u32x2*)(g.up_codes + d + d_off);
    r.q = *(const u32x2*)(g.gate_codes + d + d_off);
    r.sp = (g.up_scales + b)[b_off];
    r.sq = (g.gate_scales + b)[b_off];
  };
  // inside: all of a step's k lies within K.
  const auto load = [&](auto inside, int s, int odd, Raw& r) {
    uint32_t d_own = d_kept[odd], b_own = b_kept[odd];
    if (LEAN && IN) place(odd, d_own, b_own);
    const auto d_at = [&](int s) { return d_base + (IN ? (int64_t)(s >> 1) * 2 * BK : s * BK * d_row); };
    const auto b_at = [&](int s) { return b_base + (IN ? (int64_t)(s >> 1) * 2 : s * BK * b_row); };
    if constexpr (decltype(inside)::value) {
      load_at(d_at(s), b_at(s), d_own, b_own, r);
      return;
    }
    // Past the end: INPUTS the last eight latents, WEIGHTS the last token.
    const int k = k_of(s), last = IN ? K - 8 : K - 1;
    if (k <= last) {
      load_at(d_at(s), b_at(s), d_own, b_own, r);
    } else if (IN) {
      load_at(d_base + last - col, b_base + last / kFp8Block - col / kFp8Block, d_own, b_own, r);
    } else {
      load_at(d_base + (last - row) * d_row, b_base + (last - row) * b_row, d_own, b_own, r);
    }
  };
  // MASK: relu's mask, squared, of the thread's latents.
  const auto mask_of = [&](int n, floatx4 (&m2)[2]) {
    const float* at = g.mask + (n < N ? n : N - 8);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      m2[half] = *(const floatx4*)(at + 4 * half);
      m2[half] *= m2[half];
    }
  };
  floatx4 m2[2];
  if (MASK && !IN) mask_of(at0 + col, m2);
  u32x4 dp, dq;
  const auto make = [&](auto inside, int s, const Raw& r) {
    int up = r.sp, gate = r.sq;
    if (LEAN) asm volatile("" : "+v"(up), "+v"(gate));  // (not before)
    const float sp = fp8_power(up), sq = fp8_power(gate);
    const bf16x8 gv = __builtin_bit_cast(bf16x8, r.g);
    if (MASK && IN) mask_of(k_of(s), m2);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float p[4], q[4], fp_[4], fq[4];
      fp8_unpack4(r.p[half], sp, p);
      fp8_unpack4(r.q[half], sq, q);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float v = (float)gv[4 * half + k];
        if (MASK) v *= m2[half][k];
        grads_of<ACT>(v, p[k], q[k], fp_[k], fq[k]);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        dp[2 * half + k] = pack_bf16x2(fp_[2 * k], fp_[2 * k + 1]);
        dq[2 * half + k] = pack_bf16x2(fq[2 * k], fq[2 * k + 1]);
      }
    }
    if constexpr (!decltype(inside)::value)
      if ((IN ? s & ~1 : s) >= s1 || k_of(s) >= K) dp = dq = u32x4{0, 0, 0, 0};
  };
  // In LDS: WEIGHTS as a tile of 32 k's; buffer: of the step or pair.
  const uint32_t to = IN ? (uint32_t)(row * 128 + (((col >> 3) ^ (row & 7)) << 4))
                         : (uint32_t)(row * 256 + (((col >> 3) ^ ((row & 3) << 2)) << 4));
  const auto put = [&](int buffer, int odd) {
    char* t = grads + buffer * 2 * GRAD + to + (IN ? odd * 64 * 128 : 0);
    *(u32x4*)t = dp;
    *(u32x4*)(t + GRAD) = dq;
  };
  floatx16 acc[NA][NB];
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = zero16();
  const int w4 = w & 3;
  const int aw = 32 * NA * (w4 & 1), bw = 32 * NB * (w4 >> 1);
  const uint32_t f_at = which && two ? F::BYTES : 0, p_at = (uint32_t)(which * GRAD);
  const auto grad_frag = [&](const char* t, int at, int odd, int kk) -> bf16x8 {
    if constexpr (!IN) return P::frag(t, at, kk, lane);
    const int r = at + (lane & 31), c = 4 * odd + 2 * kk + (lane >> 5);
    return *(const bf16x8*)(t + r * 128 + ((c ^ (r & 7)) << 4));
  };
  // Fragments of 16 k's, read in the order in which the products take them.
  struct Frags {
    bf16x8 a[NA], b[NB];
  };
  const auto frag_of = [&](Frags& f, int i, const char* t, const char* d, int odd, int kk) {
    if (i < NB) {
      f.b[i] = IN ? grad_frag(d + p_at, bw + 32 * i, odd, kk) : F::frag(t + f_at, bw + 32 * i, kk, lane);
    } else {
      const int j = i - NB;
      f.a[j] = IN ? F::frag(t + f_at, aw + 32 * j, kk, lane) : grad_frag(d + p_at, aw + 32 * j, odd, kk);
    }
  };
  const auto product = [&](const Frags& f, int i) {
    acc[i / NB][i % NB] = mfma32(f.a[i / NB], f.b[i % NB], acc[i / NB][i % NB]);
  };
  // Step s: the tile of step s + 2 is asked for, the gradients of step s + AHEAD are made
  // from what was asked for SETS steps ago, step s is multiplied.  (INPUTS: a pair's
  // gradients are made while the pair before it is multiplied.)  Groups of four steps, in
  // which the raw values keep their registers; inside: all that a group asks for lies
  // within k, and nothing in it branches.  The last groups end with steps of zeros.
  constexpr int AHEAD = IN ? 2 : 1;
  const std::false_type no{};
  Raw raw[SETS];
#pragma unroll
  for (int u = 0; u < SETS; ++u) load(no, s0 + u, u & 1, raw[u]);
  issue(no, s0, 0);
  issue(no, s0 + 1, 1);
#pragma unroll
  for (int u = 0; u < AHEAD; ++u) {
    make(no, s0 + u, raw[u]);
    put(0, u);
    load(no, s0 + SETS + u, u, raw[u]);
  }
  int stage = 0, s = s0;
  const auto group = [&](auto inside) {
    constexpr bool INSIDE = decltype(inside)::value;
#pragma unroll
    for (int u = 0; u < 4; ++u, ++s) {
      // Since this step's tiles were asked for: two steps' raw values, the next step's tiles.
      if (INSIDE || (s > s0 && s + 1 < s1 && (s + 2) * BK <= K)) {
        if (two) wait_barrier<LOADS + 2 * RAW>();
        else wait_barrier<F::LOADS + 2 * RAW>();
      } else {
        wait_barrier<0>();
      }
      const int next = stage == 2 ? 0 : stage + 1, after = next == 2 ? 0 : next + 1;
      const char* t = lds + stage * TILES;
      const char* d = grads + (IN ? u >> 1 : stage) * 2 * GRAD;
      const int to_buffer = IN ? (u >> 1) ^ 1 : next;
      Raw& r = raw[(u + AHEAD) % SETS];
      issue(inside, s + 2, after);
      Frags f;
#pragma unroll
      for (int i = 0; i < NA + NB; ++i) frag_of(f, i, t, d, u & 1, 0);
#pragma unroll
      for (int i = 0; i < 8; ++i) product(f, i);
#pragma unroll
      for (int i = 0; i < NA + NB; ++i) frag_of(f, i, t, d, u & 1, 1);
      make(inside, s + AHEAD, r);
#pragma unroll
      for (int i = 0; i < 8; ++i) product(f, i);
      put(to_buffer, u & 1);
      load(inside, s + AHEAD + SETS, (u + AHEAD) & 1, r);
      stage = next;
    }
  };
  const int last = min(s1, K / BK) - 1;  // whole step
  if (s < s1) group(no);
  while (s + 10 <= last) group(std::true_type{});
  while (s < s1) group(no);
  store_product<WHAT, false>(a, acc, h, which, part, which * a.H + h, (IN ? 0 : at0) + aw, (IN ? at0 : 0) + bw, lane);
}

// out[i] = the sum of n parts, in their order; eight neighbours a thread.  Up to four
// tensors (blockIdx.y).
struct JoinArgs {
  struct {
    const float* sums;
    int n;
    int64_t stride, size;
    bf16_t* out;
  } of[4];
};
__global__ __launch_bounds__(256) void join_kernel(const JoinArgs a) {
  const auto& j = a.of[blockIdx.y];
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8; i < j.size; i += (int64_t)gridDim.x * 2048) {
    floatx4 x = *(const floatx4*)(j.sums + i), y = *(const floatx4*)(j.sums + i + 4);
#pragma unroll 4
    for (int k = 1; k < j.n; ++k) {
      x += *(const floatx4*)(j.sums + k * j.stride + i);
      y += *(const floatx4*)(j.sums + k * j.stride + i + 4);
    }
    *(u32x4*)(j.out + i) =
        u32x4{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
  }
}

unsigned cdiv(int64_t a, int64_t b) { return (unsigned)((a + b - 1) / b); }
int64_t capped(int64_t grid) { return grid < 8192 ? grid : 8192; }

TokenRows token_rows(int64_t time, int64_t batch_stride, int64_t step) {
  return TokenRows{batch_stride, step, (uint32_t)time, 1.0f / (float)time};
}

template <int WHAT>
void launch_fused(const ProductArgs& p, const GatedArgs& a, int act, hipStream_t st) {
  const dim3 grid(cdiv(WHAT == INPUTS ? p.in_tiles : p.w_tiles, 8) * 8);
  if (act == RELU && a.mask) hipLaunchKernelGGL((fused_kernel<WHAT, RELU, true>), grid, dim3(512), 0, st, p, a);
  else if (act == RELU) hipLaunchKernelGGL((fused_kernel<WHAT, RELU, false>), grid, dim3(512), 0, st, p, a);
  else if (act == SILU) hipLaunchKernelGGL((fused_kernel<WHAT, SILU, false>), grid, dim3(512), 0, st, p, a);
  else hipLaunchKernelGGL((fused_kernel<WHAT, GELU, false>), grid, dim3(512), 0, st, p, a);
}

// How long n1 tasks of length l1 and n2 of l2 <= l1 take on `slots`, the longer ones first.
int64_t makespan(int64_t n1, int64_t l1, int64_t n2, int64_t l2, int64_t slots) {
  const int64_t all = n1 / slots * l1, more = n1 % slots;  // every slot; and `more` of them one longer
  int64_t low = all + (more ? l1 : 0), high = low + (n2 + slots - 1) / slots * l2;
  while (low < high) {
    const int64_t t = (low + high) / 2;
    const int64_t room = (t >= all + l1 ? more * ((t - all - l1) / l2) : 0) + (slots - more) * ((t - all) / l2);
    if (room >= n2 && t >= all + (more ? l1 : 0)) high = t;
    else low = t + 1;
  }
  return low;
}

// Tiles and parts of k of the backward's products: what takes the least time by the steps of
// the longest row of tiles on a slot and by the bytes of the partial sums.  Measured: a step of
// 256 by 256 tiles (one a CU) 0.84 us, of 256 by 128 (two a CU) 1.11, a tile's ends about
// six steps; sums 4.5 TB/s and a launch.  (3003 tokens of 4096 latents, D 1024: 160 -> 109-121
// us.  A single workgroup on a CU is priced as one of two: few tiles are not told apart well.)
struct ProductPlan {
  int in_parts, w_parts;
  double us;
};
ProductPlan plan_products(int64_t M, int64_t H, int64_t N, int64_t D, bool ctx, bool big) {
  const int64_t slots = (int64_t)device_cus() * (big ? 1 : 2), b = big ? 256 : 128;
  const int64_t in_tiles = (D + 255) / 256 * ((M + b - 1) / b) * 2 * H;
  const int64_t w_tiles = (N + 255) / 256 * ((D + b - 1) / b) * 2 * H;
  const int64_t in_steps = (N + BK - 1) / BK, w_steps = (M + BK - 1) / BK;
  ProductPlan best{1, 1, 1e30};
  for (const int pi : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
    if (pi > 1 && in_steps / pi < 8) break;
    for (const int pw : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
      if (pw > 1 && w_steps / pw < 8) break;
      const int64_t li = (in_steps + pi - 1) / pi + 6, lw = (w_steps + pw - 1) / pw + 6;
      const int64_t ni = in_tiles * pi, nw = w_tiles * pw;
      const int64_t steps = li >= lw ? makespan(ni, li, nw, lw, slots) : makespan(nw, lw, ni, li, slots);
      const int64_t xp = (ctx ? 1 : 2) * H * pi;
      const double bytes = 8.0 * ((xp > 1 ? (double)xp * M * D : 0.0) + (ctx && pi > 1 ? (double)pi * M * H * D : 0.0) +
                                  (pw > 1 ? 2.0 * pw * H * D * N : 0.0));
      const double us = (double)steps * (big ? 0.84 : 1.11) + bytes / 4.5e6 + (bytes > 0 ? 4.0 : 0.0);
      if (us < best.us) best = ProductPlan{pi, pw, us};
    }
  }
  return best;
}

// The tokens of the projections' tiles: what takes the least time by rounds of workgroups
// (between the whole and the broken number of them) times a step's and the ends' us, as
// measured (M 1024 to 8192, N 4096 and 8192, D 256 to 2048; taken for other sizes too).  The
// ends (activation, 8 bits, memory) run beside another workgroup's products only in the smallest.  Over those 180 cases
// 0.8 % off the fastest in the mean, 18 % at worst (1024 tokens of 8192, D 256: 15 us in 128
// tokens, 18 in 256); without tiles of 192 2.9 % in the mean (the backward's at 3003 tokens of
// 4096, D 1024: 72 us in 192, 79 in 128, 81 in 256).
template <int EPI>
int projection_tokens(const GatedArgs& a, int act) {
  // Up to a tile a CU: half of it (us in 64 / 128 tokens, saved: 385 tokens of 3 x 1000, D 200
  // 10.8 / 15.9, 1024 tokens of 4096, D 1024 33 / 40; 192 tokens of 4 x 8192, two tiles a CU,
  // 20 / 18 at D 200).
  if ((a.N + 127) / 128 * a.H * ((a.M + 127) / 128) <= device_cus()) return 64;
  if (a.c) return 128;
  constexpr double step[3] = {1.07, 0.63, 0.82};
  constexpr double ends[3][3][3] = {{{6.3, 6.5, 10.0}, {11.6, 11.0, 15.5}, {14.5, 14.0, 18.0}},
                                    {{8.0, 7.5, 11.0}, {13.5, 13.5, 18.0}, {15.0, 15.0, 18.8}},
                                    {{9.8, 8.0, 13.5}, {17.8, 19.5, 26.7}, {20.0, 19.5, 25.3}}};
  int best = 128;
  double least = 1e30;
  for (int k = 0; k < 3; ++k) {
    const int64_t slots = (int64_t)device_cus() * (k == 0 ? 2 : 1), m = 128 + 64 * k;
    const int64_t tiles = (a.N + 127) / 128 * a.H * ((a.M + m - 1) / m);
    const double rounds = 0.5 * ((double)((tiles + slots - 1) / slots) + (double)tiles / (double)slots);
    const double us = rounds * ((double)((a.D + BK - 1) / BK) * step[k] + ends[k][EPI][act]);
    if (us < least) {
      least = us;
      best = (int)m;
    }
  }
  return best;
}

template <int ACT, int EPI>
void launch_projections(const GatedArgs& a, hipStream_t st) {
  if constexpr (EPI != BACK) {
    if (a.M <= kFewTokens) {
      if (a.c) launch_few<ACT, EPI == SAVE, true>(a, st);
      else launch_few<ACT, EPI == SAVE, false>(a, st);
      return;
    }
  }
  const int tokens = projection_tokens<EPI>(a, ACT);
  if (tokens != 128) {
    GatedArgs b = a;
    b.order = tile_order((int64_t)cdiv(a.N, 128) * a.H, cdiv(a.M, tokens));
    const dim3 grid(grid_of(b.order));
    if (tokens == 64 && a.c)
      hipLaunchKernelGGL((gated_kernel<ACT, EPI, true, 1>), grid, dim3(256), 0, st, b);
    else if (tokens == 64)
      hipLaunchKernelGGL((gated_kernel<ACT, EPI, false, 1>), grid, dim3(256), 0, st, b);
    else if (tokens == 256)
      hipLaunchKernelGGL((gated_kernel<ACT, EPI, false, 4>), grid, dim3(256), 0, st, b);
    else
      hipLaunchKernelGGL((gated_kernel<ACT, EPI, false, 3>), grid, dim3(256), 0, st, b);
    return;
  }
  const dim3 grid(grid_of(a.order));
  if (a.c) hipLaunchKernelGGL((gated_kernel<ACT, EPI, true, 2>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((gated_kernel<ACT, EPI, false, 2>), grid, dim3(256), 0, st, a);
}
template <int EPI>
void launch_projections(const GatedArgs& a, int act, hipStream_t st) {
  if (act == RELU) launch_projections<RELU, EPI>(a, st);
  else if (act == SILU) launch_projections<SILU, EPI>(a, st);
  else launch_projections<GELU, EPI>(a, st);
}

GatedArgs args_of(const GatedCall& g) {
  GatedArgs a{};
  a.x = g.x;
  a.c = g.c;
  a.up = g.up;
  a.gate = g.gate;
  a.M = g.B * g.T;
  a.H = (int)g.H;
  a.N = g.N;
  a.D = g.D;
  a.c_head = g.T * g.D;
  a.c_rows = token_rows(g.T, g.H * g.T * g.D, g.D);
  a.th = g.th;
  a.mask = g.mask;
  a.out = g.out;
  a.g = g.g;
  a.up_codes = g.up_codes;
  a.up_scales = g.up_scales;
  a.gate_codes = g.gate_codes;
  a.gate_scales = g.gate_scales;
  a.order = tile_order((int64_t)cdiv(g.N, 128) * g.H, cdiv(a.M, 128));
  return a;
}

}  // namespace

bdh_status gated_block(const GatedCall& g, hipStream_t st, uint64_t* launches) {
  const GatedArgs a = args_of(g);
  if (g.up_codes) launch_projections<SAVE>(a, g.act, st);
  else launch_projections<OUT>(a, g.act, st);
  BDH_HIP_TRY(hipGetLastError());
  *launches += 1;
  return BDH_OK;
}

// Partial sums of d_x take no more than this, or the bytes of dp and dq: a sum for each product
// of a head takes D / N of those (2 D / N without a context), past which a workgroup goes on
// over several products (us, a sum for each / so: 8192 tokens, 64 heads of 256, D 4096 without a
// context 13170 / 6220, its sums 17.2 GB / 0.5; 16384 tokens, 64 heads of 64, D 256, saved 1317 /
// 464, with a context 1105 / 793; 8192 tokens, 8 heads of 512, D 2048 1240 / 842; 4096 tokens, 16
// heads of 512, D 1024 704 / 525, with a context, at 2^28 bytes and ungrouped, 650).
constexpr int64_t kMostSums = (int64_t)1 << 28;

namespace {

// How a backward call goes, and the scratch that it takes.
struct VjpPlan {
  bool fused, big;
  int64_t group;   // tokens at a time
  ProductArgs p;   // (the counts of a whole call)
  size_t grads, x_bytes, c_bytes, w_bytes;
};
// The tiles of d_x and d_c of M tokens, parts counted.
int64_t in_tiles_of(const GatedCall& g, const VjpPlan& v, int64_t M) {
  if (v.fused) return cdiv(M, 128) * g.H * v.p.in_parts;
  return (int64_t)cdiv(g.D, 256) * cdiv(M, v.big ? 256 : 128) * (v.p.x_jobs + (g.c ? g.H : 0)) * v.p.in_parts;
}
// less: 0 what is fastest; where there is no memory for that, 1 without parts of k, 2 without
// any partial sums, 3 on with the tokens in 2, 4, .. groups, whose weights' sums add up in f32.
bdh_status plan_vjp(const GatedCall& g, int less, VjpPlan* out) {
  VjpPlan v{};
  ProductArgs& p = v.p;
  const int64_t M = g.B * g.T, H = g.H, N = g.N, D = g.D;
  const int64_t cus = device_cus(), all = (g.c ? 1 : 2) * H;  // products that d_x sums
  const int64_t x_sum = M * D * 4, most_sums = std::max(kMostSums, 4 * M * H * N);
  p.x_units = 1;
  v.group = M;
  // From saved values without dp and dq in memory, where there are latents enough (us, fused /
  // not, 4 heads, D 256: 385 tokens of 1000 latents 64 / 50, of 8192 101 / 116; 4096 of 1000
  // 119 / 136, of 8192 475 / 606; 1 head of 8192: 1024 tokens 94 / 101; D 64: 70 / 70).  (A
  // fused step of 128 tokens' places is held in 32 bits.)
  v.fused = less < 2 && g.up_codes && D <= 256 && M * H * N >= (int64_t)1 << 23 && H * N <= (int64_t)1 << 23;
  if (v.fused) {
    // Parts of k: enough workgroups to fill the chip.
    const auto parts_of = [&](int64_t tiles, int64_t K) {
      if (less) return 1;
      const int64_t want = (cus + tiles - 1) / tiles, most = K / 256 > 1 ? K / 256 : 1;
      const int64_t parts = want < most ? want : most;
      return (int)(parts < 32 ? parts : 32);
    };
    p.in_parts = parts_of(cdiv(M, 128) * H, N);
    p.w_parts = parts_of(cdiv(N, 128) * H, M);
    v.fused = all * p.in_parts == 1 || all * p.in_parts * x_sum <= most_sums;
  }
  if (!v.fused && less) {
    p.in_parts = p.w_parts = 1;
    while (p.x_units < all) p.x_units *= 2;
    for (int n = 2; n < less; ++n) v.group = (v.group + 1) / 2;
    p.w_kept = v.group < M;
  } else if (!v.fused) {
    ProductPlan plan = plan_products(M, H, N, D, g.c != nullptr, false);
    // (What the larger tiles' places in memory are held in takes H N up to 2^23, and rows
    // of c that follow one another.)
    if (H * N <= (int64_t)1 << 23 && (!g.c || g.B == 1 || H == 1)) {
      const ProductPlan other = plan_products(M, H, N, D, g.c != nullptr, true);
      if (other.us < plan.us) {
        plan = other;
        v.big = true;
      }
    }
    p.in_parts = plan.in_parts;
    p.w_parts = plan.w_parts;
    if (all * p.in_parts * x_sum > most_sums && all * p.in_parts > 1) {
      p.in_parts = 1;
      while (p.x_units < all && cdiv(all, p.x_units) * x_sum > most_sums) p.x_units *= 2;
    }
  }
  p.x_jobs = (int)cdiv(all, p.x_units);
  p.x_parts = p.x_jobs * p.in_parts;
  p.weights_first = !v.fused && (M + p.w_parts - 1) / p.w_parts > (N * p.x_units + p.in_parts - 1) / p.in_parts;
  const int64_t w_tiles =
      (v.fused ? cdiv(N, 128) * H : (int64_t)cdiv(N, 256) * cdiv(D, v.big ? 256 : 128) * 2 * H) * p.w_parts;
  // (A launch has fewer than 2^32 threads.)
  if (in_tiles_of(g, v, v.group) > (int64_t)1 << 22 || w_tiles > (int64_t)1 << 22)
    return fail(BDH_UNSUPPORTED, "too large for one launch");
  p.w_tiles = (int)w_tiles;
  v.grads = v.fused ? 0 : (size_t)(2 * v.group * H * N) * sizeof(bf16_t);
  v.x_bytes = p.x_parts > 1 ? (size_t)(p.x_parts * x_sum) : 0;
  v.c_bytes = g.c && p.in_parts > 1 ? (size_t)(p.in_parts * H * x_sum) : 0;
  v.w_bytes = p.w_parts > 1 || p.w_kept ? (size_t)p.w_parts * 2 * H * D * N * 4 : 0;
  *out = v;
  return BDH_OK;
}

// The sequences b .. b + nb - 1 of a call, tokens t .. t + nt - 1 of each (all, where nb > 1).
struct TokenGroup {
  int64_t b, nb, t, nt;
};
GatedArgs args_of(const GatedCall& g, const TokenGroup& k) {
  GatedArgs a = args_of(g);
  const int64_t i = k.b * g.T + k.t;
  if (k.nb == g.B && k.nt == g.T) return a;
  a.M = k.nb * k.nt;
  a.x += i * g.D;
  if (a.c) a.c += k.b * g.H * g.T * g.D + k.t * g.D;
  a.c_rows = token_rows(k.nt, g.H * g.T * g.D, g.D);
  a.g += i * g.H * g.N;
  if (a.up_codes) {
    const int64_t blocks = i * g.H * ((g.N + kFp8Block - 1) / kFp8Block);
    a.up_codes += i * g.H * g.N;
    a.gate_codes += i * g.H * g.N;
    a.up_scales += blocks;
    a.gate_scales += blocks;
  }
  a.order = tile_order((int64_t)cdiv(g.N, 128) * g.H, cdiv(a.M, 128));
  return a;
}

}  // namespace

bdh_status gated_block_vjp(const GatedCall& g, hipStream_t st, uint64_t* launches) {
  const int64_t H = g.H, N = g.N, D = g.D, w_size = H * D * N;
  VjpPlan v;
  void *grads = nullptr, *sums = nullptr;
  bool dropped = false;
  for (int less = 0;;) {
    bdh_status s = plan_vjp(g, less, &v);
    if (s != BDH_OK) return s;
    if (v.grads) s = scratch(st, SLOT_GATED_GRADS, v.grads, &grads);
    const size_t bytes = v.x_bytes + v.c_bytes + v.w_bytes;
    if (s == BDH_OK && bytes) s = scratch(st, SLOT_GATED_SUMS, bytes, &sums);
    if (s == BDH_OK) break;
    if (!scratch_no_memory() || (less > 1 && v.group <= 256)) return s;
    // Once more without what earlier calls have left, then with less.
    const bdh_status d = scratch_drop(st, {SLOT_GATED_GRADS, SLOT_GATED_SUMS});
    if (d != BDH_OK) return d;
    less += dropped;
    dropped = true;
  }
  ProductArgs p = v.p;
  p.up = g.up;
  p.gate = g.gate;
  p.N = N;
  p.D = D;
  p.H = (int)H;
  p.d_up = g.d_up;
  p.d_gate = g.d_gate;
  p.x_sums = (float*)sums;
  p.c_sums = (float*)((char*)sums + v.x_bytes);
  p.w_sums = (float*)((char*)sums + v.x_bytes + v.c_bytes);
  TokenGroup k{0, g.B, 0, g.T};
  if (v.group < g.T) k = TokenGroup{0, 1, 0, v.group};
  else if (v.group < g.B * g.T) k.nb = v.group / g.T;
  while (k.b < g.B) {
    TokenGroup now = k;
    now.nb = std::min(k.nb, g.B - k.b);
    now.nt = std::min(k.nt, g.T - k.t);
    GatedArgs a = args_of(g, now);
    const int64_t M = a.M;
    a.dp = (bf16_t*)grads;
    a.dq = a.dp + M * H * N;
    p.dp = a.dp;
    p.dq = a.dq;
    p.x = a.x;
    p.c = a.c;
    p.M = M;
    p.c_head = a.c_head;
    p.c_rows = a.c_rows;
    p.c_apart = now.nb > 1 && H > 1;
    p.x_size = M * D;
    p.c_size = M * H * D;
    p.d_x = g.d_x + (a.x - g.x);
    p.d_c = g.d_c ? g.d_c + (a.c - g.c) : nullptr;
    p.in_tiles = (int)in_tiles_of(g, v, M);
    if (v.fused) {
      launch_fused<INPUTS>(p, a, g.act, st);
      launch_fused<WEIGHTS>(p, a, g.act, st);
    } else {
      if (g.up_codes) {
        const dim3 grid((unsigned)capped(cdiv(M * H * (N / 8), 256)));
        if (g.act == RELU) hipLaunchKernelGGL((gated_grads_kernel<RELU>), grid, dim3(256), 0, st, a);
        else if (g.act == SILU) hipLaunchKernelGGL((gated_grads_kernel<SILU>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((gated_grads_kernel<GELU>), grid, dim3(256), 0, st, a);
      } else {
        launch_projections<BACK>(a, g.act, st);
      }
      const dim3 grid((cdiv(p.in_tiles, 8) + cdiv(p.w_tiles, 8)) * 8);
      const bool many = p.x_units > 1 || p.w_kept;
      if (v.big && many) hipLaunchKernelGGL((product_kernel<true, true>), grid, dim3(256), 0, st, p);
      else if (v.big) hipLaunchKernelGGL((product_kernel<true, false>), grid, dim3(256), 0, st, p);
      else if (many) hipLaunchKernelGGL((product_kernel<false, true>), grid, dim3(256), 0, st, p);
      else hipLaunchKernelGGL((product_kernel<false, false>), grid, dim3(256), 0, st, p);
    }
    *launches += 2;
    p.w_more = true;
    k.t += now.nt;
    if (k.t == g.T) {
      k.t = 0;
      k.b += now.nb;
    }
  }
  JoinArgs j{};
  int joins = 0;
  int64_t most = 0;
  const auto join = [&](const float* from, int n, int64_t stride, bf16_t* out, int64_t size) {
    j.of[joins++] = {from, n, stride, size, out};
    most = size > most ? size : most;
  };
  // (Partial sums of d_x and d_c are a whole call's.)
  if (v.x_bytes) join(p.x_sums, p.x_parts, p.x_size, g.d_x, p.x_size);
  if (v.c_bytes) join(p.c_sums, p.in_parts, p.c_size, g.d_c, p.c_size);
  if (v.w_bytes) {
    join(p.w_sums, p.w_parts, 2 * w_size, g.d_up, w_size);
    join(p.w_sums + w_size, p.w_parts, 2 * w_size, g.d_gate, w_size);
  }
  if (joins) {
    hipLaunchKernelGGL(join_kernel, dim3((unsigned)capped(cdiv(most, 2048)), (unsigned)joins), dim3(256), 0, st, j);
    *launches += 1;
  }
  BDH_HIP_TRY(hipGetLastError());
  return BDH_OK;
}

}  // namespace bdh
