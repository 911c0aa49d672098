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
//
// B200, 8192 x 16384 BF16, inputs in no cache: pack 67 us (6.0 TB/s), unpack 75 us
// (5.4 TB/s), unpack_gelu 124 us (5.4 TB/s); bound by memory, unpack_gelu also by its
// table (shared-memory pipe 71 % busy).  8192 x 4095, value by value: 32, 33 and 63 us
// (2.1, 2.1 and 2.7 TB/s).
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

// A piece of 16 bytes to p.
__device__ __forceinline__ void put(__nv_bfloat16* p, const Two* v) {
  unsigned w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = both(v[i]);
    const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
    w[i] = *reinterpret_cast<const unsigned*>(&h);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void put(float* p, const Two* v) {
  const float2 a = both(v[0]), b = both(v[1]);
  *reinterpret_cast<float4*>(p) = make_float4(a.x, a.y, b.x, b.y);
}

// Largest magnitude of a piece, NaN if it holds one.
__device__ __forceinline__ float largest(const Piece<__nv_bfloat16>& e) {
  // Magnitudes of BF16 pairs order like unsigned 16-bit numbers.
  const uint4& r = e.raw;
  constexpr unsigned kAbs = 0x7fff7fffu;
  const unsigned m = __vmaxu2(__vmaxu2(r.x & kAbs, r.y & kAbs), __vmaxu2(r.z & kAbs, r.w & kAbs));
  return __uint_as_float(max(m & 0xffff0000u, m << 16));
}
__device__ __forceinline__ float largest(const Piece<float>& e) {
  return max_nan(max_nan(fabsf(__uint_as_float(e.raw.x)), fabsf(__uint_as_float(e.raw.y))),
                 max_nan(fabsf(__uint_as_float(e.raw.z)), fabsf(__uint_as_float(e.raw.w))));
}

// The exponent byte of a group from its values' largest magnitude `amax` over the
// lanes that share it (LANES of them, N values each); values that the codes cannot
// hold are replaced on the way.
template <int LANES, int N>
__device__ __forceinline__ unsigned settle(float* v, float amax) {
#pragma unroll
  for (int d = LANES / 2; d; d >>= 1) amax = max_nan(amax, __shfl_xor_sync(kAllLanes, amax, d));
  // Ordinary groups end here; the rest (the same for all lanes of a group) takes the long way.
  const bool odd = !(amax < 240.f * 1.329227996e36f);
  if (__any_sync(kAllLanes, odd)) {
    float finite = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) finite = fmaxf(finite, finite_abs(v[i]));
#pragma unroll
    for (int d = LANES / 2; d; d >>= 1) finite = fmaxf(finite, __shfl_xor_sync(kAllLanes, finite, d));
    amax = finite;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      // Infinities as NaN have a code of their own; magnitudes past the last code are that code.
      const float a = fabsf(v[i]);
      v[i] = a <= 3.402823466e38f ? copysignf(fminf(a, 240.f * 1.329227996e36f), v[i]) : __int_as_float(0x7fffffff);
    }
  }
  return unit_byte(amax);
}
__device__ __forceinline__ float inverse_unit(unsigned byte) { return __uint_as_float((254u - byte) << 23); }

// Eight lanes per group.  A lane has a piece of 16 bytes of every eighth, so that each
// load and store of a group's lanes is one contiguous stretch (pieces of a lane side by
// side would move every sector twice).
template <typename T>
__global__ void __launch_bounds__(256) pack_kernel(const T* x, int64_t ld, unsigned char* data, int cols,
                                                   unsigned groups, unsigned items) {
  using P = Piece<T>;
  constexpr int kPieces = 16 / P::kN;
  const int lane = threadIdx.x & 7;
  const unsigned item = blockIdx.x * 32u + threadIdx.x / 8u;
  const bool live = item < items;
  const unsigned row = live ? item / groups : 0u, group = live ? item - row * groups : 0u;
  const int col = int(group) * kPackGroup + lane * P::kN;
  P e[kPieces];
  float v[16], amax = 0.f;
#pragma unroll
  for (int h = 0; h < kPieces; ++h) {
    e[h].raw = make_uint4(0, 0, 0, 0);
    if (live && col + h * 8 * P::kN < cols) e[h].load_once(x + int64_t(row) * ld + col + h * 8 * P::kN);
  }
#pragma unroll
  for (int h = 0; h < kPieces; ++h) {
    e[h].get(v + h * P::kN);
    amax = max_nan(amax, largest(e[h]));
  }
  const unsigned byte = settle<8, 16>(v, amax);
  if (!live) return;
  const float inverse = inverse_unit(byte);
  unsigned char* dst = data + int64_t(row) * pack_row_bytes(cols);
  const int code_bytes = int(pack_code_bytes(cols));
#pragma unroll
  for (int h = 0; h < kPieces; ++h) {
    if (col + h * 8 * P::kN >= code_bytes) break;
    unsigned codes[P::kN / 4];
#pragma unroll
    for (int i = 0; i < P::kN / 4; ++i) {
      const float* f = v + h * P::kN + i * 4;
      codes[i] = encode2(f[0], f[1], inverse) | unsigned(encode2(f[2], f[3], inverse)) << 16;
    }
    unsigned char* to = dst + col + h * 8 * P::kN;
    if constexpr (P::kN == 8) *reinterpret_cast<uint2*>(to) = make_uint2(codes[0], codes[1]);
    else *reinterpret_cast<unsigned*>(to) = codes[0];
  }
  unsigned char* units = dst + code_bytes;
  if (lane == 0) units[group] = static_cast<unsigned char>(byte);
  if (group == groups - 1) {  // zero padding of the exponent bytes
    const unsigned end = (groups + 15u) / 16u * 16u;
    for (unsigned i = groups + lane; i < end; i += 8) units[i] = 0;
  }
}

// Odd widths and unaligned rows: a warp has four groups, a lane pairs of columns (loaded
// one by one, their codes stored together), all on their way at once.
template <typename T>
__global__ void __launch_bounds__(256) pack_odd_kernel(const T* x, int64_t ld, unsigned char* data, int cols,
                                                       unsigned segments, unsigned items) {
  constexpr int kGroups = 4;
  const int lane = threadIdx.x & 31;
  const unsigned item = blockIdx.x * 8u + threadIdx.x / 32u;
  if (item >= items) return;
  const unsigned row = item / segments, first = (item - row * segments) * kGroups;
  const int col = int(first) * kPackGroup + 2 * lane, groups = int(pack_groups(cols));
  const T* src = x + int64_t(row) * ld;
  float v[kGroups * 4];  // 2 i and 2 i + 1: columns col + 64 i and the next
#pragma unroll
  for (int i = 0; i < kGroups * 4; ++i) {
    const int c = col + i / 2 * 64 + (i & 1);
    v[i] = c < cols ? to_float(src[c]) : 0.f;
  }
  unsigned char* dst = data + int64_t(row) * pack_row_bytes(cols);
  const int code_bytes = int(pack_code_bytes(cols));
  unsigned bytes = 0;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) amax = max_nan(amax, fabsf(v[g * 4 + i]));
    const unsigned byte = settle<32, 4>(v + g * 4, amax);
    const float inverse = inverse_unit(byte);
    bytes |= byte << (8 * g);
#pragma unroll
    for (int i = g * 2; i < g * 2 + 2; ++i)
      if (col + i * 64 < code_bytes)
        *reinterpret_cast<unsigned short*>(dst + col + i * 64) = encode2(v[2 * i], v[2 * i + 1], inverse);
  }
  // Exponent bytes, then zeros up to the padding's end.
  unsigned char* units = dst + code_bytes;
  const int mine = int(first) + lane;
  if (lane < kGroups && mine < groups) units[mine] = static_cast<unsigned char>(bytes >> (8 * lane));
  if (int(first) + kGroups >= groups && groups + lane < (groups + 15) / 16 * 16) units[groups + lane] = 0;
}

// GeLU(v) = v * Phi(v) of a kept value.  Kept values have three mantissa bits, so
// binade and mantissa (eight entries a binade) and the sign name each of them: a
// table of Phi over the magnitudes 2^-24 .. 2^8 replaces the error function, which
// would cost more than the memory traffic.  A code as FP16 has its binade and
// mantissa in bits 7 to 14 and the sign above; the group's unit moves the binade,
// that is, the place in the table: entry = bits 7..15 + 8 (e + 9).  Zeros have no
// binade and hit any entry (or the padding below), times zero.
// Table: [pad | positive 256 | negative 256 | end], the end for the NaN codes.  Eight
// copies, one for every eighth lane, side by side: an entry's copies lie in eight
// banks, so only four lanes can meet in a bank.
constexpr int kTablePad = 48, kTableHalf = 256, kTableEnd = 64, kTableLow = 127 - 24;
constexpr int kTableSize = kTablePad + 2 * kTableHalf + kTableEnd, kCopies = 8;
__device__ __forceinline__ void fill_phi_table(float* table) {
  for (int i = threadIdx.x; i < kTableSize; i += blockDim.x) {
    const int k = i - kTablePad;
    const float v = __uint_as_float((unsigned(kTableLow) << 23) + (unsigned(k & 255) << 20));
    // Phi(-v) = e^(-v^2 / 2) erfcx(v / sqrt 2) / 2 for the negative half: v^2 is exact in
    // FP32 (v has four significant bits), where erfc of a rounded argument would be
    // off by v^2 roundings.
    const float z = 0.70710678118654752440f * v;
    const float phi = k < 0 ? 0.5f : k < kTableHalf ? 0.5f * erfcf(-z) : 0.5f * expf(-0.5f * v * v) * erfcxf(z);
    const float4 four = make_float4(phi, phi, phi, phi);
    reinterpret_cast<float4*>(table)[2 * i] = four;
    reinterpret_cast<float4*>(table)[2 * i + 1] = four;
  }
}
// Any kept value, from its FP32 bits.
__device__ __forceinline__ float kept_gelu(float v, const float* table) {
  const unsigned bits = __float_as_uint(v);
  const int k = int((bits >> 20) & 0x7ffu) - kTableLow * 8;
  if (k < 0) return 0.5f * v;                                     // Phi(v) = 1/2 within 2^-24
  if (k >= kTableHalf) return v > 0.f ? v : (v == v ? -0.f : v);  // Phi(-256) = 0
  return v * table[(kTablePad + k + int(bits >> 31) * kTableHalf) * kCopies];
}

// As many columns per thread and step as fill 16 bytes of an output; the next step's
// codes are loaded ahead.
template <typename T, bool GELU>
__global__ void __launch_bounds__(1024, 2) unpack_kernel(const unsigned char* data, T* out, T* act, int cols,
                                                         unsigned segments, unsigned items) {
  extern __shared__ __align__(16) float table[];
  constexpr int kN = Piece<T>::kN;
  const unsigned row_bytes = unsigned(pack_row_bytes(cols)), code_bytes = unsigned(pack_code_bytes(cols));
  const unsigned stride = gridDim.x * 1024u, row_step = stride / segments, step = stride - row_step * segments;
  unsigned item = blockIdx.x * 1024u + threadIdx.x;
  unsigned row = item / segments, seg = item - row * segments;
  unsigned codes[kN / 4] = {};
  unsigned byte = 1;
  auto load = [&] {
    if (item < items) {
      const unsigned char* src = data + int64_t(row) * row_bytes;
      if constexpr (kN == 8) {
        const uint2 c = *reinterpret_cast<const uint2*>(src + seg * 8);
        codes[0] = c.x;
        codes[1] = c.y;
      } else {
        codes[0] = *reinterpret_cast<const unsigned*>(src + seg * 4);
      }
      byte = src[code_bytes + seg / (kPackGroup / kN)];
    }
  };
  load();
  if (GELU) {  // the table is filled while the first codes are on their way
    fill_phi_table(table);
    __syncthreads();
  }
  while (item < items) {
    unsigned now[kN / 4];
#pragma unroll
    for (int i = 0; i < kN / 4; ++i) now[i] = codes[i];
    const unsigned unit_byte = byte;
    const int64_t at = int64_t(row) * cols + seg * kN;
    item += stride;
    row += row_step;
    seg += step;
    if (seg >= segments) {
      seg -= segments;
      ++row;
    }
    load();
    const float unit = pack_unit(unit_byte);
    // e in [-15, -1]: every code's binade lies in the table's window.
    const bool window = unit_byte - 112u <= 14u;
    const char* place = reinterpret_cast<const char*>(
        table + (kTablePad + 8 * (int(unit_byte) - 127 + 9)) * kCopies + (threadIdx.x & (kCopies - 1)));
    Two v[kN / 2], a[kN / 2];
#pragma unroll
    for (int i = 0; i < kN / 2; ++i) {
      const unsigned word = now[i / 2];
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(i & 1 ? word >> 16 : word & 0xffffu), __NV_E4M3);
      const float2 f = __half22float2(__half2(h));
      v[i] = two_mul(two(f.x, f.y), two(unit, unit));
      if (GELU && window) {
        // Bits 7 .. 15 as an entry of 32 bytes: bits 5 .. 13 of the offset.
        const unsigned w = unsigned(h.y) << 16 | h.x;
        const float lo = *reinterpret_cast<const float*>(place + ((w >> 2) & 0x3fe0u));
        const float hi = *reinterpret_cast<const float*>(place + ((w >> 18) & 0x3fe0u));
        a[i] = two_mul(v[i], two(lo, hi));
      }
    }
    if (GELU && !window) {
#pragma unroll
      for (int i = 0; i < kN / 2; ++i) {
        const float2 f = both(v[i]);
        a[i] = two(kept_gelu(f.x, table), kept_gelu(f.y, table));
      }
    }
    put(out + at, v);
    if (GELU) put(act + at, a);
  }
}

// Odd widths and unaligned outputs: a warp has 512 columns, 32 at a time, so that
// loads and stores of single values are still contiguous over the warp.
template <typename T, bool GELU>
__global__ void __launch_bounds__(256) unpack_odd_kernel(const unsigned char* data, T* out, T* act, int cols,
                                                         unsigned segments, unsigned items) {
  __shared__ __align__(16) float table[GELU ? kTableSize * kCopies : 4];
  if (GELU) {
    fill_phi_table(table);
    __syncthreads();
  }
  const int64_t row_bytes = pack_row_bytes(cols);
  const int code_bytes = int(pack_code_bytes(cols)), lane = threadIdx.x & 31;
  for (unsigned item = blockIdx.x * 8u + threadIdx.x / 32u; item < items; item += gridDim.x * 8u) {
    const unsigned row = item / segments;
    const int col = int(item - row * segments) * 512 + lane;
    const unsigned char* src = data + int64_t(row) * row_bytes;
    unsigned char code[16], byte[4];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if ((i & 3) == 0) byte[i / 4] = col + i * 32 < cols ? src[code_bytes + (col + i * 32) / kPackGroup] : 1;
      code[i] = col + i * 32 < cols ? src[col + i * 32] : 0;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (col + i * 32 >= cols) break;
      const float v = decode1(code[i], pack_unit(byte[i / 4]));
      const int64_t at = int64_t(row) * cols + col + i * 32;
      out[at] = from_float<T>(v);
      if (GELU) act[at] = from_float<T>(kept_gelu(v, table));
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T>
int pack_typed(const void* x, int64_t ld, void* data, int64_t rows, int64_t cols, cudaStream_t s) {
  const bool vec = cols % 8 == 0 && ld * int64_t(sizeof(T)) % 16 == 0 && aligned16(x);
  const int64_t pieces = vec ? pack_groups(cols) : (cols + 511) / 512, items = rows * pieces;
  auto launch = [&](auto kernel, int64_t per_cta) {
    kernel<<<unsigned((items + per_cta - 1) / per_cta), 256, 0, s>>>(
        static_cast<const T*>(x), ld, static_cast<unsigned char*>(data), int(cols), unsigned(pieces), unsigned(items));
  };
  vec ? launch(pack_kernel<T>, 32) : launch(pack_odd_kernel<T>, 8);
  return int(cudaGetLastError());
}

template <typename T, bool GELU>
int unpack_typed(const void* data, void* out, void* act, int64_t rows, int64_t cols, cudaStream_t s) {
  const bool vec = cols % 8 == 0 && aligned16(out) && (!GELU || aligned16(act));
  const int64_t segments = vec ? cols / Piece<T>::kN : (cols + 511) / 512, items = rows * segments;
  if (items > 0x7fffffff) return -1;
  auto launch = [&](auto kernel, int per_cta, int threads, int most, int smem) {
    const int64_t ctas = (items + per_cta - 1) / per_cta;
    kernel<<<unsigned(ctas < most ? ctas : most), threads, smem, s>>>(
        static_cast<const unsigned char*>(data), static_cast<T*>(out), static_cast<T*>(act), int(cols),
        unsigned(segments), unsigned(items));
  };
  // Full SMs, and one table for many rows.
  vec ? launch(unpack_kernel<T, GELU>, 1024, 1024, 148 * 2, GELU ? kTableSize * kCopies * 4 : 0)
      : launch(unpack_odd_kernel<T, GELU>, 8, 256, 148 * 8, 0);
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
