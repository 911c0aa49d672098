// Activations kept in 8 bits between the forward and the backward pass (sm_100a).
//
// A row of values x is kept as E4M3 codes with one power of two for each group
// of 128 columns: 2^e is the smallest power with max|x| <= 448 * 2^e, so the
// scaling is exact and the only rounding is to the nearest code (half a step:
// 2^-4 relative, ties to even).  A power of two loses nothing against a free
// scale, because E4M3 has the same relative steps in every binade.  Non-finite
// values become NaN codes and do not count in the group's maximum.  Magnitudes
// above 240 * 2^120 become that, since the next code up is 2^128.
//
//   pack          x -> packed rows
//   unpack        packed rows -> x
//   unpack_gelu   packed rows -> (x, GeLU(x)) in one pass, the two operands that
//                 the backward pass of an MLP needs from its pre-activation
#include "kernels_api.h"
#include "rowvec.cuh"

namespace tn5b {
namespace kernels {
namespace {

// Exponent byte of a group from its largest finite magnitude: with a = 1.m * 2^k,
// a <= 448 * 2^e = 1.75 * 2^(8 + e) for e = k - 8, or k - 7 where 1.m > 1.75.
__device__ __forceinline__ unsigned unit_byte(float amax) {
  const unsigned bits = __float_as_uint(amax);
  const int k = int(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return unsigned(k < 1 ? 1 : k);
}
__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a <= 3.402823466e38f ? a : 0.f;
}
__device__ __forceinline__ unsigned short encode2(float a, float b, float inverse) {
  // Infinities times the unit's inverse stay infinite; as NaN they keep a code of their own.
  float2 f = make_float2(a * inverse, b * inverse);
  if (!(fabsf(f.x) <= 448.f)) f.x = __int_as_float(0x7fffffff);
  if (!(fabsf(f.y) <= 448.f)) f.y = __int_as_float(0x7fffffff);
  return __nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3);
}

// Half a warp per group, eight columns per lane.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) pack_kernel(const T* x, int64_t ld, unsigned char* data, int rows,
                                                   int cols, unsigned groups, unsigned items) {
  const int lane = threadIdx.x & 15;
  const unsigned item = blockIdx.x * 16u + threadIdx.x / 16u;
  const bool live = item < items;
  const unsigned row = live ? item / groups : 0u, group = live ? item - row * groups : 0u;
  const int col = int(group) * kPackGroup + lane * 8;
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = 0.f;
  const T* src = x + int64_t(row) * ld + col;
  if (VEC) {
    if (live && col < cols) {
      Eight<T> e;
      e.load_once(src);
      e.get(v);
    }
  } else if (live) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < cols) v[i] = to_float(src[i]);
  }
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = fmaxf(amax, finite_abs(v[i]));
#pragma unroll
  for (int d = 8; d; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(kAllLanes, amax, d));
  if (!live) return;
  const unsigned byte = unit_byte(amax);
  const float inverse = __uint_as_float((254u - byte) << 23);
  if (byte >= 247u) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (finite_abs(v[i]) != 0.f) v[i] = copysignf(fminf(fabsf(v[i]), 240.f * 1.329227996e36f), v[i]);
  }
  unsigned char* dst = data + int64_t(row) * pack_row_bytes(cols);
  if (col < pack_code_bytes(cols)) {
    uint2 codes;
    codes.x = encode2(v[0], v[1], inverse) | unsigned(encode2(v[2], v[3], inverse)) << 16;
    codes.y = encode2(v[4], v[5], inverse) | unsigned(encode2(v[6], v[7], inverse)) << 16;
    *reinterpret_cast<uint2*>(dst + col) = codes;
  }
  unsigned char* units = dst + pack_code_bytes(cols);
  if (lane == 0) units[group] = static_cast<unsigned char>(byte);
  if (group == groups - 1) {  // zero padding of the exponent bytes
    const unsigned end = (groups + 15u) / 16u * 16u;
    if (groups + lane < end) units[groups + lane] = 0;
  }
}

// GeLU(v) = v * Phi(v) of a kept value.  Kept values have three mantissa bits,
// so sign, exponent and mantissa (the top twelve bits of the FP32 value) name
// each of them: a table over the magnitudes 2^-24 .. 16 replaces the error
// function, which would cost more than the memory traffic.
constexpr int kTableLow = 127 - 24, kTableHigh = 127 + 4;  // biased exponents [low, high)
constexpr int kTableHalf = (kTableHigh - kTableLow) * 8;
__device__ __forceinline__ void fill_gelu_table(float* table) {
  for (int i = threadIdx.x; i < 2 * kTableHalf; i += blockDim.x) {
    const int k = i % kTableHalf;
    const float v = __uint_as_float((unsigned(kTableLow) << 23) + (unsigned(k) << 20));
    // Phi(-v) = e^(-v^2 / 2) erfcx(v / sqrt 2) / 2 for the negative half: v^2 is exact in
    // FP32 (v has four significant bits), where erfc of a rounded argument would be
    // off by v^2 roundings.
    const float z = 0.70710678118654752440f * v;
    table[i] = i >= kTableHalf ? -0.5f * v * expf(-0.5f * v * v) * erfcxf(z) : 0.5f * v * erfcf(-z);
  }
}
__device__ __forceinline__ float kept_gelu(float v, const float* table) {
  const unsigned bits = __float_as_uint(v);
  const int k = int((bits >> 20) & 0x7ffu) - kTableLow * 8;
  if (k < 0) return 0.5f * v;                                   // Phi(v) = 1/2 within 2^-24
  if (k >= kTableHalf) return v > 0.f ? v : (v == v ? -0.f : v);  // Phi(-16) < 2^-188
  return table[k + int(bits >> 31) * kTableHalf];
}

// Sixteen columns per thread (one 16-byte load of codes).
template <typename T, bool GELU, bool VEC>
__global__ void __launch_bounds__(256) unpack_kernel(const unsigned char* data, T* out, T* act, int rows,
                                                     int cols, unsigned segments, int64_t items) {
  __shared__ float table[GELU ? 2 * kTableHalf : 1];
  if (GELU) {
    fill_gelu_table(table);
    __syncthreads();
  }
  const int64_t row_bytes = pack_row_bytes(cols), code_bytes = pack_code_bytes(cols);
  for (int64_t item = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; item < items;
       item += int64_t(gridDim.x) * blockDim.x) {
    const int64_t row = item / segments;
    const int col = int(item - row * segments) * 16;
    const unsigned char* src = data + row * row_bytes;
    const uint4 codes = *reinterpret_cast<const uint4*>(src + col);
    const float unit = pack_unit(src[code_bytes + col / kPackGroup]);
    float v[16], a[16];
    decode8(make_uint2(codes.x, codes.y), unit, v);
    decode8(make_uint2(codes.z, codes.w), unit, v + 8);
    if (GELU) {
#pragma unroll
      for (int i = 0; i < 16; ++i) a[i] = kept_gelu(v[i], table);
    }
    T* o = out + row * cols + col;
    T* g = act + row * cols + col;
    if (VEC) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (col + h * 8 >= cols) break;
        Eight<T> e;
        e.set(v + h * 8);
        e.store(o + h * 8);
        if (GELU) {
          e.set(a + h * 8);
          e.store(g + h * 8);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (col + i >= cols) break;
        o[i] = from_float<T>(v[i]);
        if (GELU) g[i] = from_float<T>(a[i]);
      }
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T>
int pack_typed(const void* x, int64_t ld, void* data, int64_t rows, int64_t cols, cudaStream_t s) {
  const int64_t groups = pack_groups(cols), items = rows * groups;
  const bool vec = cols % 8 == 0 && ld * int64_t(sizeof(T)) % 16 == 0 && aligned16(x);
  const unsigned grid = unsigned((items + 15) / 16);
  auto launch = [&](auto kernel) {
    kernel<<<grid, 256, 0, s>>>(static_cast<const T*>(x), ld, static_cast<unsigned char*>(data), int(rows),
                                int(cols), unsigned(groups), unsigned(items));
  };
  vec ? launch(pack_kernel<T, true>) : launch(pack_kernel<T, false>);
  return int(cudaGetLastError());
}

template <typename T, bool GELU>
int unpack_typed(const void* data, void* out, void* act, int64_t rows, int64_t cols, cudaStream_t s) {
  const int64_t segments = (cols + 15) / 16, items = rows * segments;
  const bool vec = cols % 8 == 0 && aligned16(out) && (!GELU || aligned16(act));
  int64_t grid = (items + 255) / 256;
  if (GELU && grid > 148 * 8) grid = 148 * 8;  // one table for many rows
  if (grid > 0x7fffffff) grid = 0x7fffffff;
  auto launch = [&](auto kernel) {
    kernel<<<unsigned(grid), 256, 0, s>>>(static_cast<const unsigned char*>(data), static_cast<T*>(out),
                                          static_cast<T*>(act), int(rows), int(cols), unsigned(segments), items);
  };
  vec ? launch(unpack_kernel<T, GELU, true>) : launch(unpack_kernel<T, GELU, false>);
  return int(cudaGetLastError());
}
}  // namespace

int act_pack(const void* x, int type, int64_t ld, void* data, int64_t rows, int64_t cols, cudaStream_t s) {
  if (rows <= 0 || cols <= 0 || cols > 0x7fffff00 || rows > 0x7fffffff ||
      rows * pack_groups(cols) > 0x7fffffff || !aligned16(data))
    return -1;
  if (type == kTypeBF16) return pack_typed<__nv_bfloat16>(x, ld, data, rows, cols, s);
  if (type == kTypeFP32) return pack_typed<float>(x, ld, data, rows, cols, s);
  return -1;
}
int act_unpack(const void* data, void* out, void* act, int type, int64_t rows, int64_t cols, cudaStream_t s) {
  if (rows <= 0 || cols <= 0 || cols > 0x7fffff00 || rows > 0x7fffffff || !aligned16(data)) return -1;
  if (type == kTypeBF16)
    return act ? unpack_typed<__nv_bfloat16, true>(data, out, act, rows, cols, s)
               : unpack_typed<__nv_bfloat16, false>(data, out, act, rows, cols, s);
  if (type == kTypeFP32)
    return act ? unpack_typed<float, true>(data, out, act, rows, cols, s)
               : unpack_typed<float, false>(data, out, act, rows, cols, s);
  return -1;
}
int64_t act_pack_row_bytes(int64_t cols) { return pack_row_bytes(cols); }

}  // namespace kernels
}  // namespace tn5b
