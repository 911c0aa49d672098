// The joint of two blocks (sm_100a): norm after the branch, gate, residual scale
// and the norm before the next branch in one pass, its gradient, and LayerNorm's
// gradient from an input kept in 8 bits.
//
//   u = alpha x + g * (yhat * pw + pb)      yhat = (y - mean_y) rstd_y
//   h = xhat * w + b                        xhat = (u - mean_u) rstd_u
//
// h comes from u in FP32, before u's own rounding to the storage type.
//
//   dt = du + rstd_u (a - <a> - xhat <a xhat>),            a = dh * w
//   dx = alpha dt
//   dy = rstd_y (c - <c> - yhat <c yhat>),                 c = dt * g * pw
//   dw = sum dh xhat, db = sum dh over the rows; with P = sum dt yhat and
//   Q = sum dt: dg = pw P + pb Q, dpw = g P, dpb = g Q (g, pw, pb are constant
//   down a column, so two column sums serve three gradients)
//
// <.> is the mean over the row.  All arithmetic is FP32, two elements an
// instruction (f32x2); column sums add a fixed set of rows per CTA in order and then
// the CTAs in order, without atomics.
//
// Both directions are persistent: a CTA takes the rows row, row + grid, .. and has
// the next one on its way into shared memory (cp.async) while it works on one, so
// loads are in flight all the time and no register holds them.
//   Vector form (width a multiple of 8, rows on 16-byte boundaries): a thread has
// pieces of 16 bytes and copies what it will read itself, so it waits for its own
// copies alone.
//   Otherwise (odd widths, views) the CTA copies the 16-byte pieces that cover the
// row, and threads read single values at the row's offset, columns a CTA's width
// apart: one barrier more a row.
//
// B200, 8192 x 4096 BF16, inputs in no cache: forward 48 us (5.6 TB/s), gradient 70 us
// and 9 us for the column sums (5.1 TB/s), from packed rows with h again 113 and 9 us
// (3.3 TB/s); LayerNorm's gradient from packed rows 50 and 5 us, with its output again
// 64 and 5 us (4.4 TB/s).  What bounds them is the time that a row's reductions and its
// few warps take (issue slots 40-55 %, shared-memory pipe 48-62 % busy); more rows at
// once would need registers (the column sums) or shared memory that an SM has not.
// 4095 columns, one by one: 96 us forward, 124 and 8 us gradient.  Widths between powers
// of two have threads for the next one and check bounds: 8192 x 5120 takes 81 us forward
// (floor 51) and 138 and 8 us gradient (floor 77).
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "kernels_api.h"
#include "rowvec.cuh"

namespace tn5b {
namespace kernels {
namespace {
constexpr int kMaxRing = 200 * 1024;  // of an SM's 227 KB, for all CTAs on it
constexpr int kFwdStages = 2, kBwdStages = 2;
// Threads of all CTAs on an SM, forward: 96 or 80 registers each.  8192 x 4096 BF16: 640
// threads 47 us, 512 with a third row ahead 55, 768 49; two CTAs of 256 against three at
// 4096 x 8192: 60 and 50 us.
__host__ __device__ constexpr int fwd_threads(int nt) { return nt <= 128 ? 640 : 768; }
constexpr int kSmThreads = 512;  // the same for the gradient, at 128 registers each

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// ------------------------------------------------------- sums over the CTA
// The same bits in every thread.  `sh` is read by every thread after a barrier; it
// may be written again after another one.
template <int NT>
__device__ __forceinline__ float cta_sum(float v, float* sh) {
  v = warp_sum(v);
  if constexpr (NT > 32) {
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
      const float2 q = reinterpret_cast<const float2*>(sh)[w];
      v += q.x + q.y;
    }
  }
  return v;
}
// Two sums at once: half the warp finishes each.
template <int NT>
__device__ __forceinline__ float2 cta_sum2(float a, float b, float2* sh) {
  const bool high = threadIdx.x & 16;
  float v = (high ? b : a) + __shfl_xor_sync(kAllLanes, high ? a : b, 16);
#pragma unroll
  for (int d = 8; d; d >>= 1) v += __shfl_xor_sync(kAllLanes, v, d);
  if constexpr (NT == 32) {
    return make_float2(__shfl_sync(kAllLanes, v, 0), __shfl_sync(kAllLanes, v, 16));
  } else {
    if ((threadIdx.x & 15) == 0) reinterpret_cast<float*>(sh)[threadIdx.x >> 4] = v;
    __syncthreads();
    if constexpr (NT <= 128) {
      float2 s = make_float2(0.f, 0.f);
#pragma unroll
      for (int w = 0; w < NT / 64; ++w) {
        const float4 q = reinterpret_cast<const float4*>(sh)[w];
        s.x += q.x + q.z;
        s.y += q.y + q.w;
      }
      return s;
    } else {  // a lane for each warp's pair
      float2 s = sh[threadIdx.x & (NT / 32 - 1)];
#pragma unroll
      for (int d = NT / 64; d; d >>= 1) {
        s.x += __shfl_xor_sync(kAllLanes, s.x, d);
        s.y += __shfl_xor_sync(kAllLanes, s.y, d);
      }
      return s;
    }
  }
}
__device__ __forceinline__ float total(Two v) {
  const float2 f = both(v);
  return f.x + f.y;
}

// -------------------------------------------------- eight values as four pairs
template <typename T> struct Conv;
template <> struct Conv<__nv_bfloat16> {
  static __device__ __forceinline__ void get(const uint4* r, Two* v) {
    const unsigned w[4] = {r->x, r->y, r->z, r->w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = two(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
  static __device__ __forceinline__ void put(const Two* v, uint4* r) {
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = both(v[i]);
      const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
      w[i] = *reinterpret_cast<const unsigned*>(&h);
    }
    *r = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct Conv<float> {
  static __device__ __forceinline__ void get(const uint4* r, Two* v) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      v[2 * i] = two(__uint_as_float(r[i].x), __uint_as_float(r[i].y));
      v[2 * i + 1] = two(__uint_as_float(r[i].z), __uint_as_float(r[i].w));
    }
  }
  static __device__ __forceinline__ void put(const Two* v, uint4* r) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 a = both(v[2 * i]), b = both(v[2 * i + 1]);
      r[i] = make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
    }
  }
};

// ------------------------------------------------------------- asynchronous copies
template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst, const void* src) {
  const unsigned d = unsigned(__cvta_generic_to_shared(dst));
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(d), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

// A load that stays where it is written, before the barrier that follows.
__device__ __forceinline__ uint4 ld_vector(const uint4* p) {
  uint4 r;
  asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}

// A [rows][cols] matrix with a row stride in elements (bytes if packed).
struct Matrix {
  const void* data;
  int64_t ld;
};

// A thread's columns, in groups of eight, and a matrix's row: copied to `region` of
// shared memory, read from there, or written.  Vector form: a group is one or two
// pieces of 16 bytes, and neighbouring threads have neighbouring pieces, so that every
// access of a warp is contiguous; otherwise columns a CTA's width apart.
template <typename T, int NT, int NV, int FORM>
struct Tile {
  static constexpr int kPieces = int(sizeof(T)) / 2, kPer = 8 / kPieces;
  static __host__ __device__ constexpr int bytes(int cols) {
    return FORM ? NT * NV * 8 * int(sizeof(T)) : ((cols * int(sizeof(T)) + 15) / 16 + 1) * 16;
  }
  static __device__ __forceinline__ int column(int g, int i = 0) {
    return FORM ? ((g * kPieces + i / kPer) * NT + int(threadIdx.x)) * kPer + i % kPer : (g * 8 + i) * NT + int(threadIdx.x);
  }
  static __device__ __forceinline__ int piece(int g, int i) { return column(g, i * kPer); }
  static __device__ __forceinline__ bool has(int g, int i, int cols) { return FORM == 2 || piece(g, i) < cols; }
  // Not vectors: the eight columns of group g at p.
  static __device__ __forceinline__ void singles(const T* p, int cols, int g, Two* v) {
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = column(g, i) < cols ? to_float(p[column(g, i)]) : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = two(f[2 * i], f[2 * i + 1]);
  }
  static __device__ __forceinline__ const T* row_of(const Matrix& m, int64_t row) {
    return static_cast<const T*>(m.data) + row * m.ld;
  }
  static __device__ __forceinline__ void fetch(char* region, const Matrix& m, int64_t row, int rows, int cols) {
    const T* r = row_of(m, row);
    if constexpr (FORM) {
#pragma unroll
      for (int g = 0; g < NV; ++g)
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
          if (has(g, i, cols))
            copy_async<16>(region + ((g * kPieces + i) * NT + threadIdx.x) * 16, r + piece(g, i));
    } else {
      // Pieces that reach past the matrix's first or last value are copied value by value.
      const uintptr_t at = reinterpret_cast<uintptr_t>(r) & ~uintptr_t(15);
      const int pieces = int((reinterpret_cast<uintptr_t>(r + cols) - at + 15) / 16);
      const uintptr_t begin = reinterpret_cast<uintptr_t>(m.data),
                      end = begin + ((rows - 1) * m.ld + cols) * int64_t(sizeof(T));
      for (int i = threadIdx.x; i < pieces; i += NT) {
        const uintptr_t src = at + uintptr_t(i) * 16;
        if (src >= begin && src + 16 <= end) {
          copy_async<16>(region + i * 16, reinterpret_cast<const void*>(src));
        } else {
          for (int b = 0; b < 16; b += int(sizeof(T)))
            if (src + b >= begin && src + b < end)
              *reinterpret_cast<T*>(region + i * 16 + b) = *reinterpret_cast<const T*>(src + b);
        }
      }
    }
  }
  // Group g of the row in `region`; zeros past the width (`clear`).
  static __device__ __forceinline__ void get(const char* region, const Matrix& m, int64_t row, int cols, int g, Two* v) {
    if constexpr (FORM) {
      uint4 raw[kPieces];
#pragma unroll
      for (int i = 0; i < kPieces; ++i)
        raw[i] = *reinterpret_cast<const uint4*>(region + ((g * kPieces + i) * NT + threadIdx.x) * 16);
      Conv<T>::get(raw, v);
    } else {
      singles(reinterpret_cast<const T*>(region + (reinterpret_cast<uintptr_t>(row_of(m, row)) & 15)), cols, g, v);
    }
  }
  // A vector over the columns (a norm's weight, ..), from global memory, L1 after the
  // first row.  Vector form: loaded before a reduction and converted after it, so that
  // the loads' latency and the reduction's pass together.  Past the width it holds the
  // first columns' values, or zeros where they are asked for.
  struct Vector {
    uint4 raw[FORM ? NV : 1][kPieces];
    __device__ __forceinline__ void load(const void* base, int cols, bool zeros = false) {
      if constexpr (FORM) {
#pragma unroll
        for (int g = 0; g < NV; ++g)
#pragma unroll
          for (int i = 0; i < kPieces; ++i) {
            const bool in = has(g, i, cols);
            raw[g][i] = ld_vector(reinterpret_cast<const uint4*>(static_cast<const T*>(base) + (in ? piece(g, i) : 0)));
            if (zeros && !in) raw[g][i] = make_uint4(0, 0, 0, 0);
          }
      }
    }
    __device__ __forceinline__ void get(const void* base, int cols, int g, Two* v) const {
      if constexpr (FORM) Conv<T>::get(raw[g], v);
      else singles(static_cast<const T*>(base), cols, g, v);
    }
  };
  // One group of such a vector, where it is needed.
  static __device__ __forceinline__ void group(const void* base, int cols, int g, Two* v) {
    const T* p = static_cast<const T*>(base);
    if constexpr (FORM) {
      uint4 raw[kPieces];
#pragma unroll
      for (int i = 0; i < kPieces; ++i)
        raw[i] = has(g, i, cols) ? *reinterpret_cast<const uint4*>(p + piece(g, i)) : make_uint4(0, 0, 0, 0);
      Conv<T>::get(raw, v);
    } else {
      singles(p, cols, g, v);
    }
  }
  static __device__ __forceinline__ void store(void* base, int64_t ld, int64_t row, int cols, int g, const Two* v) {
    T* p = static_cast<T*>(base) + row * ld;
    if constexpr (FORM) {
      uint4 raw[kPieces];
      Conv<T>::put(v, raw);
#pragma unroll
      for (int i = 0; i < kPieces; ++i)
        if (has(g, i, cols)) *reinterpret_cast<uint4*>(p + piece(g, i)) = raw[i];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = both(v[i]);
        if (column(g, 2 * i) < cols) p[column(g, 2 * i)] = from_float<T>(f.x);
        if (column(g, 2 * i + 1) < cols) p[column(g, 2 * i + 1)] = from_float<T>(f.y);
      }
    }
  }
  // FP32 sums over the rows, at the same columns.
  static __device__ __forceinline__ void store_sums(float* p, int cols, int g, const Two* v) {
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const float2 a = both(v[i]), b = both(v[i + 1]);
      if constexpr (FORM) {
        if (has(g, 2 * i / kPer, cols)) *reinterpret_cast<float4*>(p + column(g, 2 * i)) = make_float4(a.x, a.y, b.x, b.y);
      } else {
        if (column(g, 2 * i) < cols) p[column(g, 2 * i)] = a.x;
        if (column(g, 2 * i + 1) < cols) p[column(g, 2 * i + 1)] = a.y;
        if (column(g, 2 * i + 2) < cols) p[column(g, 2 * i + 2)] = b.x;
        if (column(g, 2 * i + 3) < cols) p[column(g, 2 * i + 3)] = b.y;
      }
    }
  }
};

// The same columns of packed rows.  Vector form: a piece's codes and the four exponent
// bytes with its own among them; otherwise the whole row (it starts on a boundary).
template <typename T, int NT, int NV, int FORM>
struct PackedTile {
  using C = Tile<T, NT, NV, FORM>;
  static constexpr int kPieces = C::kPieces;
  static __host__ __device__ constexpr int bytes(int cols) {
    return FORM ? NT * NV * (8 + 4 * kPieces) : int(pack_row_bytes(cols));
  }
  static __device__ __forceinline__ void fetch(char* region, const Matrix& m, int64_t row, int, int cols) {
    const char* r = static_cast<const char*>(m.data) + row * m.ld;
    if constexpr (FORM) {
#pragma unroll
      for (int k = 0; k < NV * kPieces; ++k) {
        const int col = C::piece(k / kPieces, k % kPieces);
        if (C::has(k / kPieces, k % kPieces, cols)) {
          copy_async<C::kPer>(region + (k * NT + threadIdx.x) * C::kPer, r + col);
          copy_async<4>(region + NT * NV * 8 + (k * NT + threadIdx.x) * 4,
                        r + pack_code_bytes(cols) + (col / kPackGroup & ~3));
        }
      }
    } else {
      for (int i = threadIdx.x; i < int(pack_row_bytes(cols)) / 16; i += NT) copy_async<16>(region + i * 16, r + i * 16);
    }
  }
  static __device__ __forceinline__ void get(const char* region, const Matrix&, int64_t, int cols, int g, Two* v) {
    float f[8];
    if constexpr (FORM) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int k = g * kPieces + i;
        const unsigned four = *reinterpret_cast<const unsigned*>(region + NT * NV * 8 + (k * NT + threadIdx.x) * 4);
        const float unit = pack_unit(four >> (8 * (C::piece(g, i) / kPackGroup & 3)) & 0xffu);
        const unsigned* codes = reinterpret_cast<const unsigned*>(region + (k * NT + threadIdx.x) * C::kPer);
        if constexpr (C::kPer == 8) {
          decode8(*reinterpret_cast<const uint2*>(codes), unit, f);
        } else {
          decode2(*codes & 0xffffu, unit, f + i * 4);
          decode2(*codes >> 16, unit, f + i * 4 + 2);
        }
      }
    } else {
      const unsigned char* r = reinterpret_cast<const unsigned char*>(region);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int col = C::column(g, i);
        f[i] = col < cols ? decode1(r[col], pack_unit(r[pack_code_bytes(cols) + col / kPackGroup])) : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = two(f[2 * i], f[2 * i + 1]);
  }
};

// Vector form: nothing is copied to the places of columns past the width, and what
// is read from there is zero.
template <int NT, int FORM>
__device__ __forceinline__ void clear(char* ring, int bytes) {
  if (FORM == 1) {
    for (int i = threadIdx.x * 16; i < bytes; i += NT * 16) *reinterpret_cast<uint4*>(ring + i) = make_uint4(0, 0, 0, 0);
    __syncthreads();  // other threads' places were cleared here too
  }
}

// Walks over a CTA's rows with the next ones on their way: fetch(row, stage) starts
// the copies of a row, work(row, stage) has them in place.
template <int NT, int FORM, int STAGES, typename Fetch, typename Work>
__device__ __forceinline__ void walk(int rows, Fetch&& fetch, Work&& work) {
  const int64_t step = gridDim.x;
  if constexpr (STAGES == 1) {
    for (int64_t row = blockIdx.x; row < rows; row += step) {
      if constexpr (!FORM) __syncthreads();  // the last row has been read
      fetch(row, 0);
      copies_commit();
      copies_wait<0>();
      if constexpr (!FORM) __syncthreads();
      work(row, 0);
    }
  } else {
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) {
      const int64_t row = blockIdx.x + s * step;
      if (row < rows) fetch(row, s);
      copies_commit();
    }
    int stage = 0;
    for (int64_t row = blockIdx.x; row < rows; row += step) {
      copies_wait<STAGES - 2>();
      // Other threads' copies are in place, and the stage filled next has been read by all.
      if constexpr (!FORM) __syncthreads();
      const int64_t ahead = row + (STAGES - 1) * step;
      if (ahead < rows) fetch(ahead, stage == 0 ? STAGES - 1 : stage - 1);
      copies_commit();
      work(row, stage);
      stage = stage == STAGES - 1 ? 0 : stage + 1;
    }
  }
}

// ------------------------------------------------------------------ forward
struct JoinFwd {
  Matrix x, y;
  const void *pw, *pb, *gate, *w, *b;
  void *u, *h;
  float* stats;  // [4][rows]: mean_y, rstd_y, mean_u, rstd_u
  int64_t ld_h;
  int rows, cols;
  float alpha, eps, inverse;  // inverse: 1 / cols
};

// Mean and reciprocal deviation of a row: two passes over registers.
template <int NT, int NV, int FORM, typename C>
__device__ __forceinline__ float2 row_stats(const Two* v, const JoinFwd& p, float* sh) {
  Two s = 0;
#pragma unroll
  for (int i = 0; i < NV * 4; ++i) s = two_add(s, v[i]);
  const float mean = cta_sum<NT>(total(s), sh) * p.inverse;
  const Two minus = two(-mean, -mean);
  s = 0;
#pragma unroll
  for (int g = 0; g < NV; ++g) {
#pragma unroll
    for (int k = 0; k < C::kPieces; ++k) {
      Two q = 0;
#pragma unroll
      for (int i = k * C::kPer / 2; i < (k + 1) * C::kPer / 2; ++i) {
        Two d = two_add(v[g * 4 + i], minus);
        if (!FORM) {  // single columns may lie past the width
          const float2 f = both(d);
          d = two(C::column(g, 2 * i) < p.cols ? f.x : 0.f, C::column(g, 2 * i + 1) < p.cols ? f.y : 0.f);
        }
        q = two_fma(d, d, q);
      }
      if (!FORM || C::has(g, k, p.cols)) s = two_add(s, q);
    }
  }
  const float var = cta_sum<NT>(total(s), sh + 16) * p.inverse;
  return make_float2(mean, rsqrtf(var + p.eps));
}

template <typename T, int NT, int NV, int FORM, int STAGES>
__global__ void __launch_bounds__(NT, fwd_threads(NT) / NT) join_fwd_kernel(JoinFwd p) {
  extern __shared__ __align__(16) char ring[];
  __shared__ __align__(16) float sh[64];
  using C = Tile<T, NT, NV, FORM>;
  const int bytes = C::bytes(p.cols);
  clear<NT, FORM>(ring, STAGES * 2 * bytes);
  walk<NT, FORM, STAGES>(
      p.rows,
      [&](int64_t row, int stage) {
        C::fetch(ring + (2 * stage) * bytes, p.y, row, p.rows, p.cols);
        C::fetch(ring + (2 * stage + 1) * bytes, p.x, row, p.rows, p.cols);
      },
      [&](int64_t row, int stage) {
        Two y[NV * 4];
#pragma unroll
        for (int g = 0; g < NV; ++g) C::get(ring + (2 * stage) * bytes, p.y, row, p.cols, g, y + g * 4);
        typename C::Vector pw, pb, gate;
        pw.load(p.pw, p.cols);
        pb.load(p.pb, p.cols);
        gate.load(p.gate, p.cols, true);  // columns past the width stay zero in u
        float2 st = row_stats<NT, NV, FORM, C>(y, p, sh);
        if (threadIdx.x == 0) {
          p.stats[row] = st.x;
          p.stats[p.rows + row] = st.y;
        }
        Two scale = two(st.y, st.y), minus = two(-st.x, -st.x);
        const Two alpha = two(p.alpha, p.alpha);
#pragma unroll
        for (int g = 0; g < NV; ++g) {
          Two w[4], b[4], v[4];
          pw.get(p.pw, p.cols, g, w);
          pb.get(p.pb, p.cols, g, b);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            y[g * 4 + i] = two_fma(two_mul(two_add(y[g * 4 + i], minus), scale), w[i], b[i]);
          gate.get(p.gate, p.cols, g, w);
          C::get(ring + (2 * stage + 1) * bytes, p.x, row, p.cols, g, v);
#pragma unroll
          for (int i = 0; i < 4; ++i) y[g * 4 + i] = two_fma(w[i], y[g * 4 + i], two_mul(alpha, v[i]));
          C::store(p.u, p.cols, row, p.cols, g, y + g * 4);
        }
        pw.load(p.w, p.cols);
        pb.load(p.b, p.cols);
        st = row_stats<NT, NV, FORM, C>(y, p, sh + 32);
        if (threadIdx.x == 0) {
          p.stats[2 * int64_t(p.rows) + row] = st.x;
          p.stats[3 * int64_t(p.rows) + row] = st.y;
        }
        scale = two(st.y, st.y), minus = two(-st.x, -st.x);
#pragma unroll
        for (int g = 0; g < NV; ++g) {
          Two w[4], b[4];
          pw.get(p.w, p.cols, g, w);
          pb.get(p.b, p.cols, g, b);
#pragma unroll
          for (int i = 0; i < 4; ++i) b[i] = two_fma(two_mul(two_add(y[g * 4 + i], minus), scale), w[i], b[i]);
          C::store(p.h, p.ld_h, row, p.cols, g, b);
        }
      });
}

// ----------------------------------------------------------------- backward
struct JoinBwd {
  Matrix dh, du, u, y;  // du.data may be null; u and y rows may be packed
  const void *pw, *gate, *w, *b;  // b: only for h
  const float *mean_y, *rstd_y, *mean_u, *rstd_u;
  void *dx, *dy, *h;  // h (optional): the norm's output again
  float* sums;        // [grid][2 or 4][cols]
  int64_t ld_dy, ld_dx;
  int rows, cols;
  float alpha, inverse;
};

template <typename T, int NT, int NV, int FORM, bool BRANCH, bool PACKED>
struct BwdTiles {
  using C = Tile<T, NT, NV, FORM>;
  using K = std::conditional_t<PACKED, PackedTile<T, NT, NV, FORM>, C>;
  static __host__ __device__ constexpr int bytes(int cols) { return 2 * C::bytes(cols) + (BRANCH ? 2 : 1) * K::bytes(cols); }
};

// A row takes two CTA-wide reductions (one without a branch), the second one of
// values that the first decides.  The column sums stay in registers: 64 of them for
// sixteen columns a thread, which is what limits an SM to 512 threads.
template <typename T, int NT, int NV, int FORM, bool BRANCH, bool PACKED, int STAGES>
__global__ void __launch_bounds__(NT, kSmThreads / NT) join_bwd_kernel(JoinBwd p) {
  constexpr int N = NV * 4;
  extern __shared__ __align__(16) char ring[];
  __shared__ __align__(16) float2 sh[2][16];
  using Tiles = BwdTiles<T, NT, NV, FORM, BRANCH, PACKED>;
  using C = typename Tiles::C;
  using K = typename Tiles::K;
  const int whole = C::bytes(p.cols), kept = K::bytes(p.cols), bytes = Tiles::bytes(p.cols);
  clear<NT, FORM>(ring, STAGES * bytes);
  // For this thread's columns, behind the rows: w as stored, and gate * pw in FP32.
  uint4* const weights = reinterpret_cast<uint4*>(ring + STAGES * bytes);
  constexpr int kW = NV * C::kPieces * NT;  // pieces of w
  auto weight = [&](int which, int g, Two* v) {
    if (which == 0) {
      uint4 raw[C::kPieces];
#pragma unroll
      for (int i = 0; i < C::kPieces; ++i) raw[i] = weights[(g * C::kPieces + i) * NT + threadIdx.x];
      Conv<T>::get(raw, v);
    } else {
      uint4 raw[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) raw[i] = weights[kW + (g * 2 + i) * NT + threadIdx.x];
      Conv<float>::get(raw, v);
    }
  };
  {
    typename C::Vector w, pw, gate;
    w.load(p.w, p.cols, true);
    if (BRANCH) {
      pw.load(p.pw, p.cols, true);
      gate.load(p.gate, p.cols, true);
    }
#pragma unroll
    for (int g = 0; g < NV; ++g) {
      Two a[4], b[4];
      uint4 raw[2];
      w.get(p.w, p.cols, g, a);
      Conv<T>::put(a, raw);  // exact: the values came from this type
#pragma unroll
      for (int i = 0; i < C::kPieces; ++i) weights[(g * C::kPieces + i) * NT + threadIdx.x] = raw[i];
      if (BRANCH) {
        pw.get(p.pw, p.cols, g, a);
        gate.get(p.gate, p.cols, g, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = two_mul(a[i], b[i]);
        Conv<float>::put(a, raw);
#pragma unroll
        for (int i = 0; i < 2; ++i) weights[kW + (g * 2 + i) * NT + threadIdx.x] = raw[i];
      }
    }
  }
  Two dw[N], db[N], P[BRANCH ? N : 1], Q[BRANCH ? N : 1];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    dw[i] = db[i] = 0;
    if (BRANCH) P[i] = Q[i] = 0;
  }
  int turn = 0;  // without a branch: the reductions' buffers alternate
  // Lanes 0 to 3 of every warp hold the row's four statistics, loaded a row ahead.
  const int which = threadIdx.x & 3;
  const float* stats = which == 0 ? p.mean_u : which == 1 || !BRANCH ? p.rstd_u : which == 2 ? p.mean_y : p.rstd_y;
  float stat = blockIdx.x < p.rows ? stats[blockIdx.x] : 0.f;
  walk<NT, FORM, STAGES>(
      p.rows,
      [&](int64_t row, int stage) {
        char* r = ring + stage * bytes;
        C::fetch(r, p.dh, row, p.rows, p.cols);
        K::fetch(r + 2 * whole, p.u, row, p.rows, p.cols);
        if (p.du.data) C::fetch(r + whole, p.du, row, p.rows, p.cols);
        if (BRANCH) K::fetch(r + 2 * whole + kept, p.y, row, p.rows, p.cols);
      },
      [&](int64_t row, int stage) {
        const char* r = ring + stage * bytes;
        const float mean_u = __shfl_sync(kAllLanes, stat, 0), rstd_u = __shfl_sync(kAllLanes, stat, 1);
        const float mean_y = __shfl_sync(kAllLanes, stat, 2), rstd_y = __shfl_sync(kAllLanes, stat, 3);
        if (row + gridDim.x < p.rows) stat = stats[row + gridDim.x];
        // hat = (x - mean) rstd, the difference first: a mean far above the spread would
        // otherwise cost hat the digits that they differ by.
        const Two scale_u = two(rstd_u, rstd_u), minus_u = two(-mean_u, -mean_u);
        const Two scale_y = two(rstd_y, rstd_y), minus_y = two(-mean_y, -mean_y);
        Two s0 = 0, s1 = 0;
        // Without a branch there are registers to hold a and hat over the reduction; with
        // one they would spill, and are read and computed again.
        Two held_a[BRANCH ? 1 : N], held_hat[BRANCH ? 1 : N];
#pragma unroll
        for (int g = 0; g < NV; ++g) {
          Two d[4], hat[4], w[4];
          C::get(r, p.dh, row, p.cols, g, d);
          K::get(r + 2 * whole, p.u, row, p.cols, g, hat);
          weight(0, g, w);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            hat[i] = two_mul(two_add(hat[i], minus_u), scale_u);
            dw[g * 4 + i] = two_fma(d[i], hat[i], dw[g * 4 + i]);
            db[g * 4 + i] = two_add(db[g * 4 + i], d[i]);
            d[i] = two_mul(d[i], w[i]);
            s0 = two_add(s0, d[i]);
            s1 = two_fma(d[i], hat[i], s1);
            if constexpr (!BRANCH) {
              held_a[g * 4 + i] = d[i];
              held_hat[g * 4 + i] = hat[i];
            }
          }
          if (p.h) {
            Two b[4];
            C::group(p.b, p.cols, g, b);
#pragma unroll
            for (int i = 0; i < 4; ++i) b[i] = two_fma(hat[i], w[i], b[i]);
            C::store(p.h, p.cols, row, p.cols, g, b);
          }
        }
        float2 m = cta_sum2<NT>(total(s0), total(s1), sh[BRANCH ? 0 : turn]);
        turn ^= 1;
        // dt = du + rstd (a - <a> - hat <a hat>), as du + a rstd + (h q + r) with q and r of
        // the row, where h is hat if it was held, or u - mean (rstd is in q then).
        float q = -m.y * p.inverse * rstd_u, rest = -m.x * p.inverse * rstd_u;
        if constexpr (BRANCH) q *= rstd_u;
        Two q2 = two(q, q), rest2 = two(rest, rest);
        const Two alpha = two(p.alpha, p.alpha);
        Two c[BRANCH ? N : 1];
        s0 = s1 = 0;
#pragma unroll
        for (int g = 0; g < NV; ++g) {
          Two d[4], hat[4], w[4], t[4] = {0, 0, 0, 0};
          if (p.du.data) C::get(r + whole, p.du, row, p.cols, g, t);
          if constexpr (BRANCH) {
            C::get(r, p.dh, row, p.cols, g, d);
            K::get(r + 2 * whole, p.u, row, p.cols, g, hat);
            weight(0, g, w);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              d[i] = two_mul(d[i], w[i]);
              hat[i] = two_add(hat[i], minus_u);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              d[i] = held_a[g * 4 + i];
              hat[i] = held_hat[g * 4 + i];
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            t[i] = two_add(t[i], two_fma(d[i], scale_u, two_fma(hat[i], q2, rest2)));
            d[i] = two_mul(alpha, t[i]);
          }
          C::store(p.dx, p.ld_dx, row, p.cols, g, d);
          if constexpr (BRANCH) {
            K::get(r + 2 * whole + kept, p.y, row, p.cols, g, hat);
            weight(1, g, w);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int k = g * 4 + i;
              hat[i] = two_mul(two_add(hat[i], minus_y), scale_y);
              P[k] = two_fma(t[i], hat[i], P[k]);
              Q[k] = two_add(Q[k], t[i]);
              c[k] = two_mul(t[i], w[i]);
              s0 = two_add(s0, c[k]);
              s1 = two_fma(c[k], hat[i], s1);
            }
          }
        }
        if constexpr (BRANCH) {
          m = cta_sum2<NT>(total(s0), total(s1), sh[1]);
          // dy = rstd (c - <c> - yhat <c yhat>) = c rstd + ((y - mean) q + r)
          q = -m.y * p.inverse * rstd_y * rstd_y;
          rest = -m.x * p.inverse * rstd_y;
          q2 = two(q, q), rest2 = two(rest, rest);
#pragma unroll
          for (int g = 0; g < NV; ++g) {
            Two hat[4];
            K::get(r + 2 * whole + kept, p.y, row, p.cols, g, hat);
#pragma unroll
            for (int i = 0; i < 4; ++i) hat[i] = two_fma(c[g * 4 + i], scale_y, two_fma(two_add(hat[i], minus_y), q2, rest2));
            C::store(p.dy, p.ld_dy, row, p.cols, g, hat);
          }
        }
      });
  cudaTriggerProgrammaticLaunchCompletion();
  float* out = p.sums + int64_t(blockIdx.x) * (BRANCH ? 4 : 2) * p.cols;
#pragma unroll
  for (int g = 0; g < NV; ++g) {
    C::store_sums(out, p.cols, g, dw + g * 4);
    C::store_sums(out + p.cols, p.cols, g, db + g * 4);
    if constexpr (BRANCH) {
      C::store_sums(out + 2 * int64_t(p.cols), p.cols, g, P + g * 4);
      C::store_sums(out + 3 * int64_t(p.cols), p.cols, g, Q + g * 4);
    }
  }
}

struct JoinFinish {
  const float* sums;
  const void *pw, *pb, *gate;
  void *dw, *db, *dpw, *dpb, *dgate;
  int parts, cols;
};

// The CTA's 32 warps add every 32nd partial sum, in order, then one warp adds those.
// WIDE: a lane has all K sums of one column; otherwise one sum, and the CTA 32 / K
// columns (whole sectors of 32 bytes), since narrow widths have few CTAs here and many
// partial sums: 11 us against 14 at 8192 x 256, but 10 against 7 at 8192 x 4096.
template <typename T, bool BRANCH, bool WIDE>
__global__ void __launch_bounds__(1024) join_finish_kernel(JoinFinish p) {
  constexpr int K = BRANCH ? 4 : 2, kCols = WIDE ? 32 : 32 / K, kEach = WIDE ? K : 1;
  __shared__ float sh[kEach][32][33];
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int col = blockIdx.x * kCols + lane % kCols;
  const bool has = col < p.cols;
  float s[kEach] = {};
  cudaGridDependencySynchronize();
  if (has) {
    const float* from = p.sums + int64_t(lane / kCols) * p.cols + col;
#pragma unroll 4
    for (int q = part; q < p.parts; q += 32) {
#pragma unroll
      for (int k = 0; k < kEach; ++k) s[k] += from[(int64_t(q) * K + k) * p.cols];
    }
  }
#pragma unroll
  for (int k = 0; k < kEach; ++k) sh[k][part][lane] = s[k];
  __syncthreads();
  if (part >= kEach) return;
  float v = 0.f;
#pragma unroll
  for (int q = 0; q < 32; ++q) v += sh[part][q][lane];
  // Sum k of the column, from warp k or from this warp's lanes.
  const int k = WIDE ? part : lane / kCols;
  if (!has) return;
  if (k == 0) static_cast<T*>(p.dw)[col] = from_float<T>(v);
  if (k == 1) static_cast<T*>(p.db)[col] = from_float<T>(v);
  if constexpr (BRANCH) {
    if (k < 2) return;
    const float g = to_float(static_cast<const T*>(p.gate)[col]);
    if (k == 3) {
      static_cast<T*>(p.dpb)[col] = from_float<T>(g * v);
      return;
    }
    // k = 2: Q once more, in the same order.
    float Q = 0.f;
#pragma unroll
    for (int q = 0; q < 32; ++q) Q += WIDE ? sh[kEach - 1][q][lane] : sh[0][q][(lane + kCols) & 31];
    const float pw = to_float(static_cast<const T*>(p.pw)[col]), pb = to_float(static_cast<const T*>(p.pb)[col]);
    static_cast<T*>(p.dgate)[col] = from_float<T>(pw * v + pb * Q);
    static_cast<T*>(p.dpw)[col] = from_float<T>(g * v);
  }
}

// -------------------------------------------------------------------- launches
// Shared memory above 48 KB (the kernel's fixed part counts too), once for each kernel and device.
template <auto Kernel>
int opt_in(int smem) {
  if (smem <= 40 * 1024) return 0;
  static std::atomic<uint64_t> opted{0};
  int device = 0;
  cudaGetDevice(&device);
  const uint64_t bit = uint64_t(1) << (device & 63);
  if (opted.load(std::memory_order_relaxed) & bit) return 0;
  const cudaError_t e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxRing);
  if (e == cudaSuccess) opted.fetch_or(bit, std::memory_order_relaxed);
  return int(e);
}
// CTAs that an SM takes by threads or by what their rings leave room for, on every SM.
int most_ctas(int by_threads, int ring) {
  const int fit = kMaxRing / (ring > 0 ? ring : 1);
  return 148 * (fit < by_threads ? (fit < 1 ? 1 : fit) : by_threads);
}

// The form of a call: 0 for odd widths and unaligned rows, 1 for vectors, 2 for vectors
// of a width that fills every thread (no bounds to check).
template <int NT, int NV>
int form_of(bool vec, int cols) {
  return !vec ? 0 : cols == NT * NV * 8 ? 2 : 1;
}

template <typename T, int NT, int NV, int FORM>
int fwd_launch(const JoinFwd& p, cudaStream_t s) {
  const int smem = kFwdStages * 2 * Tile<T, NT, NV, FORM>::bytes(p.cols);
  if (smem > kMaxRing) return -1;
  if (const int r = opt_in<join_fwd_kernel<T, NT, NV, FORM, kFwdStages>>(smem)) return r;
  const int ctas = std::min(p.rows, most_ctas(fwd_threads(NT) / NT, smem));
  join_fwd_kernel<T, NT, NV, FORM, kFwdStages><<<unsigned(ctas), NT, smem, s>>>(p);
  return int(cudaGetLastError());
}
template <typename T, int NT, int NV>
int fwd_form(const JoinFwd& p, bool vec, cudaStream_t s) {
  switch (form_of<NT, NV>(vec, p.cols)) {
    case 2: return fwd_launch<T, NT, NV, 2>(p, s);
    case 1: return fwd_launch<T, NT, NV, 1>(p, s);
    default: return fwd_launch<T, NT, NV, 0>(p, s);
  }
}
template <typename T>
int fwd_pick(const JoinFwd& p, bool vec, cudaStream_t s) {
  // As few threads a row as registers allow: what a row costs beside its columns, the
  // reductions, grows with its warps.
  if (p.cols <= 256) return fwd_form<T, 32, 1>(p, vec, s);
  if (p.cols <= 512) return fwd_form<T, 32, 2>(p, vec, s);
  // FP32 rows leave room for half as many CTAs, so they have twice the threads.
  constexpr int kMore = sizeof(T) == 4 ? 2 : 1;
  if (p.cols <= 1024) return fwd_form<T, 32 * kMore, 4 / kMore>(p, vec, s);
  if (p.cols <= 2048) return fwd_form<T, 64 * kMore, 4 / kMore>(p, vec, s);
  if (p.cols <= 4096) return fwd_form<T, 128 * kMore, 4 / kMore>(p, vec, s);
  return fwd_form<T, 256 * kMore, 4 / kMore>(p, vec, s);
}

// The gradient's CTAs: as many as fit, but some rows each where that leaves every SM one:
// every CTA's column sums are written and read once. 777 x 2048: four rows and two cost the
// same; odd widths, whose rows take longer, 20 us with four and 16 with two at 777 x 2050.
// No other size was compared.
template <typename T, int NT, int NV, int FORM, bool BRANCH, bool PACKED>
int bwd_launch(const JoinBwd& p, JoinFinish f, cudaStream_t s) {
  // Two rows of the widest FP32 tensors are more than an SM holds.
  constexpr int kRows = sizeof(T) == 4 && NT * NV == 1024 ? 1 : kBwdStages;
  const int smem = kRows * BwdTiles<T, NT, NV, FORM, BRANCH, PACKED>::bytes(p.cols) +
                   NT * NV * (8 * int(sizeof(T)) + (BRANCH ? 32 : 0));
  if (smem > kMaxRing) return -1;
  if (const int r = opt_in<join_bwd_kernel<T, NT, NV, FORM, BRANCH, PACKED, kRows>>(smem)) return r;
  f.parts = std::min(std::min(p.rows, most_ctas(kSmThreads / NT, smem)), std::max(p.rows / (FORM ? 4 : 2), 148));
  join_bwd_kernel<T, NT, NV, FORM, BRANCH, PACKED, kRows><<<unsigned(f.parts), NT, smem, s>>>(p);
  if (const int r = int(cudaGetLastError())) return r;
  constexpr bool kWide = NT * NV * 8 > 2048;
  constexpr int kCols = kWide ? 32 : BRANCH ? 8 : 16;
  // Launched while the rows' last CTAs run; it waits for them itself.
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(unsigned((p.cols + kCols - 1) / kCols));
  config.blockDim = dim3(1024);
  config.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attr;
  config.numAttrs = 1;
  return int(cudaLaunchKernelEx(&config, join_finish_kernel<T, BRANCH, kWide>, f));
}
template <typename T, int NT, int NV, bool BRANCH, bool PACKED>
int bwd_form(const JoinBwd& p, const JoinFinish& f, bool vec, cudaStream_t s) {
  switch (form_of<NT, NV>(vec, p.cols)) {
    case 2: return bwd_launch<T, NT, NV, 2, BRANCH, PACKED>(p, f, s);
    case 1: return bwd_launch<T, NT, NV, 1, BRANCH, PACKED>(p, f, s);
    default: return bwd_launch<T, NT, NV, 0, BRANCH, PACKED>(p, f, s);
  }
}
template <typename T, bool BRANCH, bool PACKED>
int bwd_pick(const JoinBwd& p, const JoinFinish& f, bool vec, cudaStream_t s) {
  if (p.cols <= 256) return bwd_form<T, 32, 1, BRANCH, PACKED>(p, f, vec, s);
  // FP32 rows leave room for half as many CTAs, so they have twice the threads.
  constexpr bool kLong = sizeof(T) == 4 && !PACKED;
  if (p.cols <= 512) return bwd_form<T, 32, 2, BRANCH, PACKED>(p, f, vec, s);
  if (p.cols <= 1024) return bwd_form<T, kLong ? 128 : 64, kLong ? 1 : 2, BRANCH, PACKED>(p, f, vec, s);
  if (p.cols <= 2048) return bwd_form<T, kLong ? 256 : 128, kLong ? 1 : 2, BRANCH, PACKED>(p, f, vec, s);
  if (p.cols <= 4096) return bwd_form<T, kLong ? 512 : 256, kLong ? 1 : 2, BRANCH, PACKED>(p, f, vec, s);
  return bwd_form<T, 512, 2, BRANCH, PACKED>(p, f, vec, s);
}
}  // namespace

int64_t join_max_cols() { return kJoinMaxCols; }
int join_bwd_parts(int64_t rows, int64_t cols) {
  // The most that any form launches at this width (threads alone).
  const int nt = cols <= 512 ? 32 : cols <= 1024 ? 64 : cols <= 2048 ? 128 : cols <= 4096 ? 256 : 512;
  return int(std::min<int64_t>(rows, 148 * (kSmThreads / nt)));
}

int join_fwd(const void* x, int64_t ld_x, const void* y, int64_t ld_y, int type, const void* pw, const void* pb,
             const void* gate, const void* w, const void* b, void* u, void* h, int64_t ld_h, float* stats, int64_t rows,
             int64_t cols, float alpha, float eps, cudaStream_t s) {
  if (rows <= 0 || rows > 0x7fffffff || cols <= 0 || cols > kJoinMaxCols) return -1;
  const JoinFwd p{{x, ld_x}, {y, ld_y}, pw, pb, gate, w, b, u, h, stats, ld_h, int(rows), int(cols), alpha, eps,
                  1.f / float(cols)};
  const int64_t size = type == kTypeFP32 ? 4 : 2;
  const bool vec = cols % 8 == 0 && ld_x * size % 16 == 0 && ld_y * size % 16 == 0 && ld_h * size % 16 == 0 &&
                   aligned16(x) && aligned16(y) && aligned16(pw) && aligned16(pb) && aligned16(gate) && aligned16(w) &&
                   aligned16(b) && aligned16(u) && aligned16(h);
  if (type == kTypeBF16) return fwd_pick<__nv_bfloat16>(p, vec, s);
  if (type == kTypeFP32) return fwd_pick<float>(p, vec, s);
  return -1;
}

int join_bwd(const JoinBwdCall& c, cudaStream_t s) {
  if (c.rows <= 0 || c.rows > 0x7fffffff || c.cols <= 0 || c.cols > kJoinMaxCols) return -1;
  const bool branch = c.y != nullptr;
  if (!branch && !c.packed) return -1;
  const JoinBwd p{{c.dh, c.ld_dh}, {c.du, c.ld_du}, {c.u, c.ld_u}, {c.y, c.ld_y}, c.pw, c.gate, c.w, c.b,
                  c.mean_y, c.rstd_y, c.mean_u, c.rstd_u, c.dx, c.dy, c.h, c.workspace, c.ld_dy, c.ld_dx,
                  int(c.rows), int(c.cols), c.alpha, 1.f / float(c.cols)};
  const JoinFinish f{c.workspace, c.pw, c.pb, c.gate, c.dw, c.db, c.dpw, c.dpb, c.dgate, 0, int(c.cols)};
  const int64_t size = c.type == kTypeFP32 ? 4 : 2;
  auto fine = [&](const void* q, int64_t ld) { return !q || (aligned16(q) && ld * size % 16 == 0); };
  const bool vec = c.cols % 8 == 0 && fine(c.dh, c.ld_dh) && fine(c.du, c.ld_du) && fine(c.dx, c.ld_dx) &&
                   fine(c.dy, c.ld_dy) && fine(c.h, c.cols) && fine(c.pw, 0) && fine(c.gate, 0) && fine(c.w, 0) &&
                   fine(c.b, 0) && aligned16(c.workspace) &&
                   (c.packed || (fine(c.u, c.ld_u) && fine(c.y, c.ld_y)));
  auto pick = [&](auto zero) {
    using T = decltype(zero);
    if (!branch) return bwd_pick<T, false, true>(p, f, vec, s);
    return c.packed ? bwd_pick<T, true, true>(p, f, vec, s) : bwd_pick<T, true, false>(p, f, vec, s);
  };
  if (c.type == kTypeBF16) return pick(__nv_bfloat16());
  if (c.type == kTypeFP32) return pick(float());
  return -1;
}

}  // namespace kernels
}  // namespace tn5b
