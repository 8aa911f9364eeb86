// Moves of streams' recurrent states between the slots of a batch: forking a
// prompt's state into samples, closing a batch up after requests ended,
// exchanging and clearing slots.  A slot is one stream's rho of a layer, H*N*D
// contiguous f32 (33.5 MB at H 4 N 8192 D 256).
//
// The call is one parallel assignment slot[dst_i] <- slot[src_i] (all sources
// read before any destination is written; src -1 = zeros), of every layer in
// one launch and without a copy aside: each thread owns the same 16 bytes of
// every slot and runs the same short program on them, so the only order that
// matters is inside a thread.  A step of the program loads up to eight slots
// and then stores each to its destinations.  The host orders them:
//   - every slot is the destination of at most one source, so the assignment
//     forms trees that grow out of a slot or of a cycle of slots;
//   - a tree goes in from the leaves (a slot is overwritten once its own value
//     has gone to its children);
//   - a cycle of up to eight slots is one step; a longer one turns eight at a
//     time, its first slot passing the value on.
//
// Bound by memory: each distinct source read once and each destination
// written once (cycles past eight slots: two more accesses for every seven).
// (Steps of two or four slots measured alike; eight let a cycle of eight turn
// without a second access.)  Of 6 layers of 33.5 MB slots, one to 8 others takes
// 352-385 us (4.7-5.1 TB/s; a large copy here 5.15), closing up 8 of 16 slots
// 575-590 (5.5); of 3 layers of 1 MB slots, 9 exchanged, 9 us; a single small
// state 3 us, its launch.
#include <vector>

#include "bdh_internal.h"

namespace bdh {
namespace {

// Of one launch; they travel as kernel arguments (below 4 KB together).
constexpr int kMaxWords = 840;
constexpr int kMaxLayers = 24;
constexpr int kStep = 8;      // sources a step holds in registers
constexpr int kZeros = -1;    // source: zeros
constexpr int kStays = -2;    // a slot that is no destination

// words: steps, each [K in {1, 2, 4, 8}], K sources [slot | destinations << 16],
// then the sources' destinations in turn; behind the n words of the steps,
// the n_zero slots that are cleared.  (Words of 32 bits: scalar loads.)
struct MoveArgs {
  float* dst[kMaxLayers];
  const float* src[kMaxLayers];
  int64_t slab[kMaxLayers];  // f32 of a slot
  int32_t n, n_zero;
  int32_t words[kMaxWords];
};
static_assert(sizeof(MoveArgs) <= 4000, "kernel arguments");

// 16 bytes at any 4-byte address (slots of odd sizes): a dwordx4 access.
typedef float float4_u __attribute__((ext_vector_type(4), aligned(4)));

// PAST: past the caches.
template <bool PAST, typename V>
__device__ __forceinline__ V load_slot(const float* p) {
  if constexpr (PAST) return __builtin_nontemporal_load((const V*)p);
  else return *(const V*)p;
}

template <bool PAST, typename V>
__device__ __forceinline__ void store_slot(float* p, V v) {
  if constexpr (PAST) __builtin_nontemporal_store(v, (V*)p);
  else *(V*)p = v;
}

template <int K, bool PAST, typename V>
__device__ __forceinline__ int run_step(const int32_t* w, int pc, const float* src, float* dst, int64_t slab) {
  V r[K];
#pragma unroll
  for (int j = 0; j < K; ++j) r[j] = load_slot<PAST, V>(src + (w[pc + j] & 0xffff) * slab);
  // All loads are waited for here, together: a wait inside the loops below
  // would also wait for the stores before it.
#pragma unroll
  for (int j = 0; j < K; ++j) asm volatile("" : "+v"(r[j]));
  int at = pc + K;
#pragma unroll
  for (int j = 0; j < K; ++j)
    for (const int end = at + (w[pc + j] >> 16); at < end; ++at) store_slot<PAST>(dst + w[at] * slab, r[j]);
  return at;
}

template <bool PAST, typename V>
__device__ __forceinline__ void run_program(const MoveArgs& a, const float* src, float* dst, int64_t slab) {
  for (int pc = 0; pc < a.n;) {
    const int k = a.words[pc];
    ++pc;
    if (k == 8) pc = run_step<8, PAST, V>(a.words, pc, src, dst, slab);
    else if (k == 4) pc = run_step<4, PAST, V>(a.words, pc, src, dst, slab);
    else if (k == 2) pc = run_step<2, PAST, V>(a.words, pc, src, dst, slab);
    else pc = run_step<1, PAST, V>(a.words, pc, src, dst, slab);
  }
  for (int i = 0; i < a.n_zero; ++i) store_slot<PAST>(dst + a.words[a.n + i] * slab, V{});
}

template <bool PAST>
__global__ __launch_bounds__(256) void move_streams_kernel(const MoveArgs a) {
  const int64_t slab = a.slab[blockIdx.y];
  const int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (e >= slab) return;
  const float* src = a.src[blockIdx.y] + e;
  float* dst = a.dst[blockIdx.y] + e;
  if (e + 4 <= slab) {
    run_program<PAST, float4_u>(a, src, dst, slab);
  } else {
    for (int64_t k = 0; k < slab - e; ++k) run_program<PAST, float>(a, src + k, dst + k, slab);
  }
}

// The ordered program, cut into launches where one holds too much.
struct Program {
  struct Launch {
    std::vector<int32_t> words;  // of the steps
    std::vector<int32_t> zero;
  };
  struct Move {
    int src;
    std::vector<int> dst;
  };
  std::vector<Launch> launches{1};
  std::vector<Move> open;  // the step being filled
  int64_t reads = 0, writes = 0;  // slots
  bool again = false;             // a slot is read that the call has written

  Launch& room(size_t words) {
    if (launches.back().words.size() + launches.back().zero.size() + words > (size_t)kMaxWords)
      launches.emplace_back();
    return launches.back();
  }
  void flush() {
    if (open.empty()) return;
    // K is filled up with a source that the step loads already and that goes nowhere.
    const size_t n = open.size(), K = n > 4 ? 8 : n > 2 ? 4 : n;
    size_t dsts = 0;
    for (const Move& m : open) dsts += m.dst.size();
    Launch& l = room(1 + K + dsts);
    l.words.push_back((int32_t)K);
    for (size_t j = 0; j < K; ++j)
      l.words.push_back(j < n ? open[j].src | (int32_t)open[j].dst.size() << 16 : open[n - 1].src);
    for (const Move& m : open)
      for (int d : m.dst) l.words.push_back(d);
    open.clear();
  }
  void add(int src, const std::vector<int>& dst) {
    constexpr size_t kMost = 64;  // destinations of one load
    for (size_t at = 0; at < dst.size(); at += kMost) {
      const size_t end = at + kMost < dst.size() ? at + kMost : dst.size();
      ++reads;
      writes += (int64_t)(end - at);
      open.push_back(Move{src, std::vector<int>(dst.begin() + at, dst.begin() + end)});
      if (open.size() == (size_t)kStep) flush();
    }
  }
  // slot[v[i + 1]] <- slot[v[i]] and slot[v[0]] <- slot[v[n - 1]], n <= kStep, in one step.
  void turn(const std::vector<int>& v) {
    if (open.size() + v.size() > (size_t)kStep) flush();
    for (size_t i = 0; i < v.size(); ++i) add(v[i], {v[i + 1 < v.size() ? i + 1 : 0]});
  }
  void clear(const std::vector<int>& slots) {
    flush();
    for (int d : slots) room(1).zero.push_back(d);
  }
};

// from[slot]: the slot whose value it takes, kZeros, or kStays.
void order_moves(const std::vector<int>& from_in, int src_slots, bool in_place, Program* p) {
  std::vector<int> from(from_in);
  const int slots = (int)from.size();
  std::vector<std::vector<int>> to((size_t)(in_place ? slots : src_slots));
  std::vector<int> cleared;
  for (int d = 0; d < slots; ++d) {
    if (in_place && from[d] == d) from[d] = kStays;
    if (from[d] >= 0) to[from[d]].push_back(d);
    if (from[d] == kZeros) cleared.push_back(d);
  }
  if (in_place) {
    // waits[s]: slots that take s's value and whose own value is still wanted.
    std::vector<int> waits(slots, 0), ready;
    std::vector<char> wanted(slots, 0);
    for (int s = 0; s < slots; ++s) wanted[s] = !to[s].empty();
    for (int s = 0; s < slots; ++s) {
      for (int d : to[s]) waits[s] += wanted[d];
      if (wanted[s] && waits[s] == 0) ready.push_back(s);
    }
    for (size_t i = 0; i < ready.size(); ++i) {
      const int s = ready[i], above = from[s];
      p->add(s, to[s]);
      wanted[s] = 0;
      if (above >= 0 && --waits[above] == 0) ready.push_back(above);
    }
    // What is wanted still lies on cycles: each slot's other takers first
    // (their own values have gone), then the cycle.
    for (int s0 = 0; s0 < slots; ++s0) {
      if (!wanted[s0]) continue;
      std::vector<int> cycle;
      for (int s = s0; s >= 0;) {
        cycle.push_back(s);
        std::vector<int> others;
        int next = -1;
        for (int d : to[s]) {
          if (wanted[d]) next = d;
          else others.push_back(d);
        }
        p->add(s, others);
        s = next == s0 ? -1 : next;
      }
      for (int s : cycle) wanted[s] = 0;
      // After its first part has turned, the first slot holds the value that
      // the slot after the part wants.
      for (size_t at = 1; at < cycle.size();) {
        std::vector<int> v{cycle[0]};
        while (v.size() < (size_t)kStep && at < cycle.size()) v.push_back(cycle[at++]);
        p->again |= at < cycle.size();
        p->turn(v);
      }
    }
  } else {
    for (int s = 0; s < src_slots; ++s) p->add(s, to[s]);
  }
  p->clear(cleared);
}

// Whether a call passes the caches by: what it moves is more than the last
// level's 256 MB, so neither finds its slots there nor leaves them for the
// layers.  Of a state of 6 layers (33.5 MB a slot and layer), us through the
// caches / past them, after a call that filled them with other data: 1 slot to
// another 97 / 76, 8 to 8 others 740 / 715, closing up 11 of 16 837 / 768, 4 to 8
// 503 / 426, 1 to 2 126 / 112; but 1 to 8 385 / 434 (2 to 8 422 / 427), and 20 in
// a cycle, which reads a slot again, 1835 / 2007.  Smaller calls whose slots the
// caches hold win by them (2 to 2 others of two layers 39 / 47).
bool past_caches(const Program& p, int64_t slot_bytes) {
  return (p.reads + p.writes) * slot_bytes > (int64_t)256 << 20 && p.writes <= 3 * p.reads && !p.again;
}

}  // namespace

bdh_status copy_streams(const StreamMoves& m, hipStream_t st, uint64_t* launches) {
  std::vector<int> from((size_t)m.dst_batch, kStays);
  for (int i = 0; i < m.n; ++i) from[m.dst[i]] = m.src[i] < 0 ? kZeros : m.src[i];
  Program p;
  order_moves(from, (int)m.src_batch, m.in_place, &p);
  int64_t slot = 0;
  for (int l = 0; l < m.n_layers; ++l) slot += m.slab[l];
  const bool past = past_caches(p, slot * 4);
  for (const Program::Launch& part : p.launches) {
    if (part.words.empty() && part.zero.empty()) continue;
    for (int l0 = 0; l0 < m.n_layers; l0 += kMaxLayers) {
      MoveArgs a;
      int64_t most = 0;
      int n = 0;
      for (int l = l0; l < m.n_layers && n < kMaxLayers; ++l) {
        a.dst[n] = m.dst_rho[l];
        a.src[n] = m.src_rho[l];
        a.slab[n] = m.slab[l];
        most = a.slab[n] > most ? a.slab[n] : most;
        ++n;
      }
      a.n = (int32_t)part.words.size();
      a.n_zero = (int32_t)part.zero.size();
      for (int i = 0; i < a.n; ++i) a.words[i] = part.words[i];
      for (int i = 0; i < a.n_zero; ++i) a.words[a.n + i] = part.zero[i];
      const auto kernel = past ? move_streams_kernel<true> : move_streams_kernel<false>;
      hipLaunchKernelGGL(kernel, dim3((uint32_t)((most + 1023) / 1024), (uint32_t)n), dim3(256), 0, st, a);
      BDH_HIP_TRY(hipGetLastError());
      ++*launches;
    }
  }
  return BDH_OK;
}

}  // namespace bdh
