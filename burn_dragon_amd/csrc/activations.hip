// Activations kept between forward and backward in 8 bits (bdh_fp8.h): rows of
// `cols` values (f32 or bf16) to codes [rows, cols] and powers of two [rows,
// ceil(cols / 32)], and back.
//
// Four lanes hold a block, eight neighbours each, so a block's largest magnitude
// takes two exchanges and a wave reads and writes runs of 512 values.  Bound by the
// bytes: 3 (5) of bf16 (f32) a value to save, 3 (5) to restore (16384 rows of 8192 bf16: saved
// in 77-93 us, 4.4-5.3 TB/s, restored in 64-69, 5.9-6.3 TB/s).
#include "bdh_fp8.h"
#include "bdh_internal.h"

namespace bdh {
namespace {

typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf16x8_u __attribute__((ext_vector_type(8), aligned(2)));
typedef unsigned int u32x2_u __attribute__((ext_vector_type(2), aligned(1)));

__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const f32x4_u a = *(const f32x4_u*)p, b = *(const f32x4_u*)(p + 4);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[j] = a[j];
    x[4 + j] = b[j];
  }
}
__device__ __forceinline__ void load8(const bf16_t* p, float (&x)[8]) {
  const bf16x8_u a = *(const bf16x8_u*)p;
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = (float)a[j];
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  *(f32x4_u*)p = f32x4_u{x[0], x[1], x[2], x[3]};
  *(f32x4_u*)(p + 4) = f32x4_u{x[4], x[5], x[6], x[7]};
}
__device__ __forceinline__ void store8(bf16_t* p, const float (&x)[8]) {
  bf16x8_u v;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (bf16_t)x[j];
  *(bf16x8_u*)p = v;
}

// Lane group i of four: block i of the flat [rows, blocks].
struct Where {
  int64_t at;   // of the lane's first value
  int64_t block;
  int n;        // its values: 8, or fewer at a row's end
};
__device__ __forceinline__ Where where(int64_t i, int cols, int blocks) {
  const int sub = (int)(i & 3);
  const int64_t block = i >> 2, row = block / blocks;
  const int c = (int)(block - row * blocks) * kFp8Block + sub * 8;
  return Where{row * cols + c, block, c + 8 <= cols ? 8 : (cols > c ? cols - c : 0)};
}

template <typename T>
__global__ __launch_bounds__(256) void save_kernel(const T* __restrict__ x, uint8_t* __restrict__ codes,
                                                   uint8_t* __restrict__ scales, int64_t total, int cols, int blocks) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const Where w = where(i, cols, blocks);
    float v[8];
    if (w.n == 8) {
      load8(x + w.at, v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = j < w.n ? (float)x[w.at + j] : 0.0f;
    }
    uint32_t top = finite_top<true, 8>(v);
    // (total is a multiple of 4: the lanes of a block are there or not together.)
    top = max(top, (uint32_t)__shfl_xor((int)top, 1, 4));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2, 4));
    const int scale = fp8_scale(top);
    const float power = fp8_power(scale);
    fp8_keep_finite(v, scale);
    const u32x2_u c{fp8_pack4(v[0], v[1], v[2], v[3], power), fp8_pack4(v[4], v[5], v[6], v[7], power)};
    if (w.n == 8) {
      *(u32x2_u*)(codes + w.at) = c;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < w.n) codes[w.at + j] = (uint8_t)(c[j >> 2] >> (8 * (j & 3)));
    }
    if ((i & 3) == 0) scales[w.block] = (uint8_t)scale;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void restore_kernel(const uint8_t* __restrict__ codes,
                                                      const uint8_t* __restrict__ scales, T* __restrict__ out,
                                                      int64_t total, int cols, int blocks) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const Where w = where(i, cols, blocks);
    u32x2_u c{0, 0};
    if (w.n == 8) {
      c = *(const u32x2_u*)(codes + w.at);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < w.n) c[j >> 2] |= (uint32_t)codes[w.at + j] << (8 * (j & 3));
    }
    const float power = fp8_power(scales[w.block]);
    float lo[4], hi[4];
    fp8_unpack4(c.x, power, lo);
    fp8_unpack4(c.y, power, hi);
    const float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    if (w.n == 8) {
      store8(out + w.at, v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < w.n) out[w.at + j] = (T)v[j];
    }
  }
}

// (8192 workgroups are four rounds of the chip's; past that each goes on to further blocks.)
unsigned grid_of(int64_t total) {
  const int64_t g = (total + 255) / 256;
  return (unsigned)(g < 8192 ? g : 8192);
}

}  // namespace

bdh_status save_activations(const void* x, bool bf16, int64_t rows, int64_t cols, uint8_t* codes, uint8_t* scales,
                            hipStream_t st) {
  const int blocks = (int)((cols + kFp8Block - 1) / kFp8Block);
  const int64_t total = rows * blocks * 4;
  if (bf16)
    hipLaunchKernelGGL((save_kernel<bf16_t>), dim3(grid_of(total)), dim3(256), 0, st, (const bf16_t*)x, codes, scales,
                       total, (int)cols, blocks);
  else
    hipLaunchKernelGGL((save_kernel<float>), dim3(grid_of(total)), dim3(256), 0, st, (const float*)x, codes, scales,
                       total, (int)cols, blocks);
  BDH_HIP_TRY(hipGetLastError());
  return BDH_OK;
}

bdh_status restore_activations(const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t cols, bool bf16,
                               void* out, hipStream_t st) {
  const int blocks = (int)((cols + kFp8Block - 1) / kFp8Block);
  const int64_t total = rows * blocks * 4;
  if (bf16)
    hipLaunchKernelGGL((restore_kernel<bf16_t>), dim3(grid_of(total)), dim3(256), 0, st, codes, scales, (bf16_t*)out,
                       total, (int)cols, blocks);
  else
    hipLaunchKernelGGL((restore_kernel<float>), dim3(grid_of(total)), dim3(256), 0, st, codes, scales, (float*)out,
                       total, (int)cols, blocks);
  BDH_HIP_TRY(hipGetLastError());
  return BDH_OK;
}

}  // namespace bdh
