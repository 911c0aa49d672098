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
  return __nv_cvt_float2_to_fp8x2(make_float2(a * inverse, b * inverse), __NV_SATFINITE, __NV_E4M3);
}

// Largest magnitude of eight values, and whether all are finite.
__device__ __forceinline__ float largest(const Eight<__nv_bfloat16>& e) {
  // Magnitudes of BF16 pairs order like unsigned 16-bit numbers.
  const uint4& r = e.raw[0];
  constexpr unsigned kAbs = 0x7fff7fffu;
  const unsigned m = __vmaxu2(__vmaxu2(r.x & kAbs, r.y & kAbs), __vmaxu2(r.z & kAbs, r.w & kAbs));
  return __uint_as_float(max(m & 0xffff0000u, m << 16));
}
__device__ __forceinline__ float largest(const Eight<float>& e) {
  float m = 0.f;
#pragma unroll
  for (int h = 0; h < 2; ++h)
    m = max_nan(max_nan(max_nan(m, fabsf(__uint_as_float(e.raw[h].x))), fabsf(__uint_as_float(e.raw[h].y))),
                max_nan(fabsf(__uint_as_float(e.raw[h].z)), fabsf(__uint_as_float(e.raw[h].w))));
  return m;
}

// Eight lanes per group; a lane has eight columns of each half, so that every
// load and store of a group is one contiguous piece.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) pack_kernel(const T* x, int64_t ld, unsigned char* data, int cols,
                                                   unsigned groups, unsigned items) {
  const int lane = threadIdx.x & 7;
  const unsigned item = blockIdx.x * 32u + threadIdx.x / 8u;
  const bool live = item < items;
  const unsigned row = live ? item / groups : 0u, group = live ? item - row * groups : 0u;
  const int col = int(group) * kPackGroup + lane * 8;
  Eight<T> e[2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < int(sizeof(T) / 2); ++i) e[h].raw[i] = make_uint4(0, 0, 0, 0);
  const T* src = x + int64_t(row) * ld + col;
  if (VEC) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (live && col + h * 64 < cols) e[h].load_once(src + h * 64);
  } else if (live) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      T* v = reinterpret_cast<T*>(e[h].raw);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (col + h * 64 + i < cols) v[i] = src[h * 64 + i];
    }
  }
  float amax = max_nan(largest(e[0]), largest(e[1]));
#pragma unroll
  for (int d = 4; d; d >>= 1) amax = max_nan(amax, __shfl_xor_sync(kAllLanes, amax, d));
  float v[16];
  e[0].get(v);
  e[1].get(v + 8);
  // Ordinary groups end here; the rest (the same for a group's eight lanes) takes the long way.
  const bool odd = !(amax < 240.f * 1.329227996e36f);
  if (__any_sync(kAllLanes, odd)) {
    float finite = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) finite = fmaxf(finite, finite_abs(v[i]));
#pragma unroll
    for (int d = 4; d; d >>= 1) finite = fmaxf(finite, __shfl_xor_sync(kAllLanes, finite, d));
    amax = finite;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      // Infinities as NaN have a code of their own; magnitudes past the last code are that code.
      const float a = fabsf(v[i]);
      v[i] = a <= 3.402823466e38f ? copysignf(fminf(a, 240.f * 1.329227996e36f), v[i]) : __int_as_float(0x7fffffff);
    }
  }
  if (!live) return;
  const unsigned byte = unit_byte(amax);
  const float inverse = __uint_as_float((254u - byte) << 23);
  unsigned char* dst = data + int64_t(row) * pack_row_bytes(cols);
  const int code_bytes = int(pack_code_bytes(cols));
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (col + h * 64 >= code_bytes) break;
    uint2 codes;
    codes.x = encode2(v[h * 8], v[h * 8 + 1], inverse) | unsigned(encode2(v[h * 8 + 2], v[h * 8 + 3], inverse)) << 16;
    codes.y = encode2(v[h * 8 + 4], v[h * 8 + 5], inverse) |
              unsigned(encode2(v[h * 8 + 6], v[h * 8 + 7], inverse)) << 16;
    *reinterpret_cast<uint2*>(dst + col + h * 64) = codes;
  }
  unsigned char* units = dst + code_bytes;
  if (lane == 0) units[group] = static_cast<unsigned char>(byte);
  if (group == groups - 1) {  // zero padding of the exponent bytes
    const unsigned end = (groups + 15u) / 16u * 16u;
    for (unsigned i = groups + lane; i < end; i += 8) units[i] = 0;
  }
}

// GeLU(v) = v * Phi(v) of a kept value.  Kept values have three mantissa bits, so
// binade and mantissa (eight entries a binade) and the sign name each of them: a
// table of Phi over the magnitudes 2^-24 .. 2^8 replaces the error function, which
// would cost more than the memory traffic.  A code as FP16 has its binade and
// mantissa in bits 7 to 14 and the sign above; the group's unit moves the binade,
// that is, the place in the table: entry = bits 7..15 + 8 (e + 9).  Zeros have no
// binade and hit any entry (or the padding below), times zero.
// Table: [pad | positive 256 | negative 256 | end], the end for the NaN codes.
constexpr int kTablePad = 48, kTableHalf = 256, kTableEnd = 64, kTableLow = 127 - 24;
constexpr int kTableSize = kTablePad + 2 * kTableHalf + kTableEnd;
__device__ __forceinline__ void fill_phi_table(float* table) {
  for (int i = threadIdx.x; i < kTableSize; i += blockDim.x) {
    const int k = i - kTablePad;
    const float v = __uint_as_float((unsigned(kTableLow) << 23) + (unsigned(k & 255) << 20));
    // Phi(-v) = e^(-v^2 / 2) erfcx(v / sqrt 2) / 2 for the negative half: v^2 is exact in
    // FP32 (v has four significant bits), where erfc of a rounded argument would be
    // off by v^2 roundings.
    const float z = 0.70710678118654752440f * v;
    table[i] = k < 0 ? 0.5f : k < kTableHalf ? 0.5f * erfcf(-z) : 0.5f * expf(-0.5f * v * v) * erfcxf(z);
  }
}
// Any kept value, from its FP32 bits.
__device__ __forceinline__ float kept_gelu(float v, const float* table) {
  const unsigned bits = __float_as_uint(v);
  const int k = int((bits >> 20) & 0x7ffu) - kTableLow * 8;
  if (k < 0) return 0.5f * v;                                     // Phi(v) = 1/2 within 2^-24
  if (k >= kTableHalf) return v > 0.f ? v : (v == v ? -0.f : v);  // Phi(-256) = 0
  return v * table[kTablePad + k + int(bits >> 31) * kTableHalf];
}

// Sixteen columns per thread (one 16-byte load of codes).
template <typename T, bool GELU, bool VEC>
__global__ void __launch_bounds__(256) unpack_kernel(const unsigned char* data, T* out, T* act, int cols,
                                                     unsigned segments, unsigned items) {
  __shared__ float table[GELU ? kTableSize : 1];
  if (GELU) {
    fill_phi_table(table);
    __syncthreads();
  }
  const int64_t row_bytes = pack_row_bytes(cols);
  const int code_bytes = int(pack_code_bytes(cols));
  for (unsigned item = blockIdx.x * 256u + threadIdx.x; item < items; item += gridDim.x * 256u) {
    const unsigned row = item / segments;
    const int col = int(item - row * segments) * 16;
    const unsigned char* src = data + int64_t(row) * row_bytes;
    const uint4 codes = *reinterpret_cast<const uint4*>(src + col);
    const unsigned byte = src[code_bytes + col / kPackGroup];
    const float unit = pack_unit(byte);
    const unsigned words[4] = {codes.x, codes.y, codes.z, codes.w};
    // e in [-15, -1]: every code's binade lies in the table's window.
    const bool window = byte - 112u <= 14u;
    const float* place = table + kTablePad + 8 * (int(byte) - 127 + 9);
    float v[16], a[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned short code2 = i & 1 ? words[i / 2] >> 16 : words[i / 2] & 0xffffu;
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(code2), __NV_E4M3);
      const float2 f = __half22float2(__half2(h));
      v[2 * i] = f.x * unit;
      v[2 * i + 1] = f.y * unit;
      if (GELU && window) {
        a[2 * i] = v[2 * i] * place[(h.x >> 7) & 0x1ff];
        a[2 * i + 1] = v[2 * i + 1] * place[h.y >> 7];
      }
    }
    if (GELU && !window) {
#pragma unroll
      for (int i = 0; i < 16; ++i) a[i] = kept_gelu(v[i], table);
    }
    T* o = out + int64_t(row) * cols + col;
    T* g = act + int64_t(row) * cols + col;
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
  const unsigned grid = unsigned((items + 31) / 32);
  auto launch = [&](auto kernel) {
    kernel<<<grid, 256, 0, s>>>(static_cast<const T*>(x), ld, static_cast<unsigned char*>(data), int(cols),
                                unsigned(groups), unsigned(items));
  };
  vec ? launch(pack_kernel<T, true>) : launch(pack_kernel<T, false>);
  return int(cudaGetLastError());
}

template <typename T, bool GELU>
int unpack_typed(const void* data, void* out, void* act, int64_t rows, int64_t cols, cudaStream_t s) {
  const int64_t segments = (cols + 15) / 16, items = rows * segments;
  const bool vec = cols % 8 == 0 && aligned16(out) && (!GELU || aligned16(act));
  if (items > 0x7fffffff) return -1;
  int64_t grid = (items + 255) / 256;
  if (GELU && grid > 148 * 8) grid = 148 * 8;  // one table for many rows
  auto launch = [&](auto kernel) {
    kernel<<<unsigned(grid), 256, 0, s>>>(static_cast<const unsigned char*>(data), static_cast<T*>(out),
                                          static_cast<T*>(act), int(cols), unsigned(segments), unsigned(items));
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
