// Row access shared by the scoring, block-joint and 8-bit activation kernels:
// eight values at a time in FP32 from BF16, FP16 or FP32 storage, the packed
// 8-bit row layout, and warp/block sums.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace tn5b {
namespace kernels {

constexpr unsigned kAllLanes = 0xffffffffu;

__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }

// 16 bytes of values as they lie in memory, read once, past L1.
template <typename T>
struct Piece {
  static constexpr int kN = 16 / int(sizeof(T));
  uint4 raw;
  __device__ __forceinline__ void load_once(const T* p) {
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(raw.x), "=r"(raw.y), "=r"(raw.z), "=r"(raw.w)
                 : "l"(reinterpret_cast<const uint4*>(p)));
  }
  __device__ __forceinline__ void get(float* v) const {
    const T* h = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i] = to_float(h[i]);
  }
};

// Packed 8-bit rows: cols E4M3 codes padded with zeros to a multiple of 16
// bytes, then one exponent byte for each group of 128 columns (value =
// code * 2^(byte - 127)), padded with zeros to a multiple of 16.  Every row
// starts on a 16-byte boundary whatever cols is.
constexpr int kPackGroup = 128;
__host__ __device__ __forceinline__ int64_t pack_code_bytes(int64_t cols) { return (cols + 15) / 16 * 16; }
__host__ __device__ __forceinline__ int64_t pack_groups(int64_t cols) { return (cols + kPackGroup - 1) / kPackGroup; }
__host__ __device__ __forceinline__ int64_t pack_row_bytes(int64_t cols) {
  return pack_code_bytes(cols) + (pack_groups(cols) + 15) / 16 * 16;
}

__device__ __forceinline__ float pack_unit(unsigned byte) {  // 2^(byte - 127), byte >= 1
  return __uint_as_float(byte << 23);
}
__device__ __forceinline__ void decode2(unsigned short two, float unit, float* v) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(two), __NV_E4M3);
  const float2 f = __half22float2(__half2(h));
  v[0] = f.x * unit;
  v[1] = f.y * unit;
}
__device__ __forceinline__ void decode8(uint2 codes, float unit, float* v) {
  decode2(codes.x & 0xffffu, unit, v);
  decode2(codes.x >> 16, unit, v + 2);
  decode2(codes.y & 0xffffu, unit, v + 4);
  decode2(codes.y >> 16, unit, v + 6);
}
__device__ __forceinline__ float decode1(unsigned char code, float unit) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw(code, __NV_E4M3);
  return __half2float(__half(h)) * unit;
}

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(kAllLanes, x, d);
  return x;
}

// 2^x with a relative error of a few 2^-23; results below 2^-126 are zero.
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two FP32 values in a register pair, and the instructions that work on both.
using Two = unsigned long long;
__device__ __forceinline__ Two two(float a, float b) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 both(Two v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ Two two_fma(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ Two two_add(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Two two_mul(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// The larger value, NaN where either is NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

}  // namespace kernels
}  // namespace tn5b
