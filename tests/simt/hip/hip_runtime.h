// Just enough of the HIP runtime to run a kernel's source on the CPU: the threads of a
// workgroup are fibers (x86-64) that run in turn, the lanes of a wave in order.  Operations
// across a wave and barriers switch between them; a wave's live lanes (a workgroup's live
// threads) have to meet in each of them, which holds for kernels that make them in
// uniform flow.  LDS is static memory: workgroups run one after another.
#pragma once

#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <sys/mman.h>

#include <functional>
#include <vector>

#define __global__
#define __device__
#define __host__
#define __shared__ static
#define __forceinline__ inline __attribute__((always_inline))
#define __launch_bounds__(...)
#define __restrict__

typedef int hipError_t;
typedef void* hipStream_t;
enum { hipSuccess = 0 };
inline hipError_t hipGetLastError() { return hipSuccess; }
inline const char* hipGetErrorString(hipError_t) { return ""; }

struct dim3 {
  unsigned x, y, z;
  dim3(unsigned a = 1, unsigned b = 1, unsigned c = 1) : x(a), y(b), z(c) {}
};
extern dim3 threadIdx, blockIdx, blockDim, gridDim;
inline dim3 threadIdx(0, 0, 0), blockIdx(0, 0, 0), blockDim, gridDim;

namespace simt {

// Keeps the caller's stack pointer in *from, and goes on where `to` was kept.
asm(".text\n"
    "simt_switch:\n"
    "pushq %rbp\npushq %rbx\npushq %r12\npushq %r13\npushq %r14\npushq %r15\n"
    "movq %rsp, (%rdi)\nmovq %rsi, %rsp\n"
    "popq %r15\npopq %r14\npopq %r13\npopq %r12\npopq %rbx\npopq %rbp\nretq\n");
extern "C" void simt_switch(void** from, void* to);

struct Fiber {
  void* at;
  char* stack;
  bool live;
  int64_t met;  // wave operations
};
// What the lanes of a wave hand each other, by turns.
struct Wave {
  uint64_t value[2][64];
  bool there[2][64];
  int arrived[2], live;
  int64_t which[2];  // the operation that each turn holds
};
constexpr size_t kStack = 256 << 10;
inline std::vector<Fiber> fibers;
inline std::vector<Wave> waves;
inline int now, at_barrier, alive;
inline unsigned barriers;
inline void* scheduler;
inline std::function<void()> body;

inline void yield() { simt_switch(&fibers[(size_t)now].at, scheduler); }
inline void start() {
  body();
  Fiber& f = fibers[now];
  f.live = false;
  --alive;
  --waves[now / 64].live;
  for (;;) yield();
}

// Hands over a value and waits for the wave's other live lanes; their turn.
inline int exchange(uint64_t v) {
  Fiber& f = fibers[now];
  const int me = now, turn = (int)(++f.met & 1);
  Wave& w = waves[me / 64];
  if (w.which[turn] != f.met) {  // (of two turns ago, which all have left)
    w.which[turn] = f.met;
    w.arrived[turn] = 0;
    memset(w.there[turn], 0, sizeof(w.there[turn]));
  }
  w.value[turn][me & 63] = v;
  w.there[turn][me & 63] = true;
  ++w.arrived[turn];
  do yield();  // (the last one too: they go on in their order)
  while (w.arrived[turn] < w.live);
  return turn;
}
template <typename T>
T from(T v, int lane) {
  static_assert(sizeof(T) <= 8, "");
  uint64_t bits = 0;
  memcpy(&bits, &v, sizeof(T));
  const int me = now, turn = exchange(bits);
  const Wave& w = waves[me / 64];
  if (lane < 0 || lane > 63 || !w.there[turn][lane]) {
    fprintf(stderr, "a value of lane %d, which is not there\n", lane);
    abort();
  }
  T out;
  memcpy(&out, &w.value[turn][lane], sizeof(T));
  return out;
}
inline uint64_t ballot(bool b) {
  const int me = now, turn = exchange(b);
  const Wave& w = waves[me / 64];
  uint64_t bits = 0;
  for (int i = 0; i < 64; ++i) bits |= (uint64_t)(w.there[turn][i] && w.value[turn][i]) << i;
  return bits;
}
inline void barrier() {
  const unsigned mine = barriers;
  ++at_barrier;
  while (barriers == mine) yield();
}

template <typename F>
void launch(dim3 grid, dim3 block, F&& f) {
  const int n = (int)block.x;
  while ((int)fibers.size() < n) {
    fibers.push_back(Fiber{});
    fibers.back().stack = (char*)mmap(nullptr, kStack, PROT_READ | PROT_WRITE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0);
  }
  body = f;
  gridDim = grid;
  blockDim = block;
  for (unsigned y = 0; y < grid.y; ++y)
    for (unsigned x = 0; x < grid.x; ++x) {
      blockIdx = dim3(x, y, 0);
      waves.assign((size_t)(n + 63) / 64, Wave{});
      alive = n;
      at_barrier = 0;
      for (int i = 0; i < n; ++i) {
        Fiber& k = fibers[(size_t)i];
        k.live = true;
        k.met = 0;
        ++waves[(size_t)i / 64].live;
        // (Six registers, the place to go on at, and a word that leaves the stack as after a call.)
        void** top = (void**)(k.stack + kStack) - 8;
        memset(top, 0, 64);
        top[6] = (void*)start;
        k.at = top;
      }
      while (alive > 0) {
        for (now = 0; now < n; ++now) {
          if (!fibers[(size_t)now].live) continue;
          threadIdx = dim3((unsigned)now, 0, 0);
          simt_switch(&scheduler, fibers[(size_t)now].at);
        }
        if (alive > 0 && at_barrier == alive) {
          at_barrier = 0;
          ++barriers;
        }
      }
    }
}

}  // namespace simt

#define hipLaunchKernelGGL(kernel, grid, block, lds, stream, ...) \
  simt::launch(grid, block, [=] { (kernel)(__VA_ARGS__); })

inline void __syncthreads() { simt::barrier(); }
inline uint64_t __ballot(int b) { return simt::ballot(b != 0); }
template <typename T>
T __shfl_xor(T v, int o, int width = 64) {
  return simt::from(v, (int)(threadIdx.x & 63) ^ o);
}
template <typename T>
T __shfl_up(T v, int o, int width = 64) {
  const int lane = (int)(threadIdx.x & 63);
  return simt::from(v, lane >= o ? lane - o : lane);
}
inline int __popcll(uint64_t x) { return __builtin_popcountll(x); }
inline uint32_t atomicAdd(uint32_t* p, uint32_t v) {
  const uint32_t old = *p;
  *p = old + v;
  return old;
}
inline float __uint_as_float(uint32_t x) { return __builtin_bit_cast(float, x); }
inline uint32_t __float_as_uint(float x) { return __builtin_bit_cast(uint32_t, x); }

#define __builtin_amdgcn_readlane(v, lane) simt::from((int)(v), lane)
#define __builtin_amdgcn_readfirstlane(v) (v)
#define __builtin_amdgcn_fence(...) ((void)0)
#define __builtin_amdgcn_fractf(x) ((x) - floorf(x))
#define __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, ...) (c)
#define __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, ...) (c)
