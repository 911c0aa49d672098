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
// <.> is the mean over the row.  All arithmetic is FP32; column sums add a fixed
// set of rows per CTA in order and then the CTAs in order, without atomics.
#include <atomic>

#include "kernels_api.h"
#include "rowvec.cuh"

namespace tn5b {
namespace kernels {
namespace {
constexpr int kMaxWarps = 16;
constexpr int kMaxRing = 200 * 1024;  // of an SM's 227 KB; two rings of half that share an SM

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Sums of N values over the CTA, the same bits in every thread.
template <int N>
__device__ __forceinline__ void block_sums(float (&v)[N], float (*sh)[kMaxWarps]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
  if (warps == 1) return;
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) sh[i][warp] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float s = 0.f;
    for (int w = 0; w < warps; ++w) s += sh[i][w];
    v[i] = s;
  }
}

// Columns of a thread: NV groups of eight.  Vector form: eight consecutive
// columns; otherwise (odd widths, unaligned rows) columns a CTA's width apart.
template <int NV, bool VEC>
struct Columns {
  int cols;
  __device__ __forceinline__ int at(int i) const {
    return VEC ? ((i / 8) * int(blockDim.x) + int(threadIdx.x)) * 8 + (i & 7)
               : i * int(blockDim.x) + int(threadIdx.x);
  }
  __device__ __forceinline__ bool has(int i) const { return at(VEC ? i & ~7 : i) < cols; }
  template <typename T>
  __device__ __forceinline__ void load8(const T* row, int g, float* v) const {
    if (VEC) {
      Eight<T> e;
      if (has(g * 8)) {
        e.load(row + at(g * 8));
        e.get(v);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.f;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = has(g * 8 + i) ? to_float(row[at(g * 8 + i)]) : 0.f;
    }
  }
  template <typename T>
  __device__ __forceinline__ void store8(T* row, int g, const float* v) const {
    if (VEC) {
      if (!has(g * 8)) return;
      Eight<T> e;
      e.set(v);
      e.store(row + at(g * 8));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (has(g * 8 + i)) row[at(g * 8 + i)] = from_float<T>(v[i]);
    }
  }
};

// A thread's columns of one row as they were loaded (zeros past the width).
template <typename T, int NV, bool VEC>
struct Row {
  Eight<T> e[NV];
  __device__ __forceinline__ void load(const Columns<NV, VEC>& c, const T* row, bool once) {
#pragma unroll
    for (int g = 0; g < NV; ++g) {
#pragma unroll
      for (int i = 0; i < int(sizeof(T) / 2); ++i) e[g].raw[i] = make_uint4(0, 0, 0, 0);
      if (VEC) {
        if (c.has(g * 8)) once ? e[g].load_once(row + c.at(g * 8)) : e[g].load(row + c.at(g * 8));
      } else {
        T* v = reinterpret_cast<T*>(e[g].raw);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c.has(g * 8 + i)) v[i] = row[c.at(g * 8 + i)];
      }
    }
  }
  __device__ __forceinline__ void get(int g, float* v) const { e[g].get(v); }
};
struct JoinFwd {
  const void *x, *y, *pw, *pb, *gate, *w, *b;
  void *u, *h;
  float* stats;  // [4][rows]: mean_y, rstd_y, mean_u, rstd_u
  int64_t ld_x, ld_y, ld_h;
  int rows, cols;
  float alpha, eps;
};

// Mean and reciprocal deviation of the row, from two passes over registers.
template <int NV, bool VEC>
__device__ __forceinline__ void row_stats(const Columns<NV, VEC>& c, const float (&v)[NV * 8], float eps, float& mean,
                                          float& rstd, float (*sh)[kMaxWarps]) {
  float s[1] = {0.f};
#pragma unroll
  for (int i = 0; i < NV * 8; ++i) s[0] += v[i];
  block_sums(s, sh);
  mean = s[0] / c.cols;
  s[0] = 0.f;
#pragma unroll
  for (int i = 0; i < NV * 8; ++i) {
    const float d = v[i] - mean;
    if (c.has(i)) s[0] = fmaf(d, d, s[0]);
  }
  block_sums(s, sh + 1);
  rstd = rsqrtf(s[0] / c.cols + eps);
}

// One CTA a row.  Every thread keeps its columns of y and x as loaded, later of u in
// FP32.  The vectors over the columns (norm weights, biases, gate) come from L1 for
// every row but the CTA's SM's first; the rows themselves bypass it.
template <typename T, int NV, bool VEC>
__global__ void __launch_bounds__(256) join_fwd_kernel(JoinFwd p) {
  __shared__ float sh[4][kMaxWarps];
  const Columns<NV, VEC> c{p.cols};
  const int64_t row = blockIdx.x;
  float y[NV * 8];
  Row<T, NV, VEC> x;
  {
    Row<T, NV, VEC> r;
    r.load(c, static_cast<const T*>(p.y) + row * p.ld_y, true);
    x.load(c, static_cast<const T*>(p.x) + row * p.ld_x, true);
#pragma unroll
    for (int g = 0; g < NV; ++g) r.get(g, y + g * 8);
  }
  float mean, rstd;
  row_stats(c, y, p.eps, mean, rstd, sh);
  if (threadIdx.x == 0) {
    p.stats[row] = mean;
    p.stats[p.rows + row] = rstd;
  }
#pragma unroll
  for (int g = 0; g < NV; ++g) {
    float pw[8], pb[8], gate[8], v[8];
    c.load8(static_cast<const T*>(p.pw), g, pw);
    c.load8(static_cast<const T*>(p.pb), g, pb);
    c.load8(static_cast<const T*>(p.gate), g, gate);
    x.get(g, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float n = fmaf((y[g * 8 + i] - mean) * rstd, pw[i], pb[i]);
      y[g * 8 + i] = fmaf(gate[i], n, p.alpha * v[i]);
    }
    c.store8(static_cast<T*>(p.u) + row * p.cols, g, y + g * 8);
  }
  row_stats(c, y, p.eps, mean, rstd, sh + 2);
  if (threadIdx.x == 0) {
    p.stats[2 * int64_t(p.rows) + row] = mean;
    p.stats[3 * int64_t(p.rows) + row] = rstd;
  }
#pragma unroll
  for (int g = 0; g < NV; ++g) {
    float w[8], b[8];
    c.load8(static_cast<const T*>(p.w), g, w);
    c.load8(static_cast<const T*>(p.b), g, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = fmaf((y[g * 8 + i] - mean) * rstd, w[i], b[i]);
    c.store8(static_cast<T*>(p.h) + row * p.ld_h, g, b);
  }
}

struct JoinBwd {
  const void *dh, *du, *u, *y;  // du may be null; u and y rows are packed in the 8-bit form
  const void *pw, *gate, *w, *b;  // b: only for h
  const float *mean_y, *rstd_y, *mean_u, *rstd_u;
  void *dx, *dy, *h;              // h (optional): the norm's output again
  float* sums;                    // [grid][2 or 4][cols]
  int64_t ld_dh, ld_du, ld_u, ld_y, ld_dy, ld_dx;
  int rows, cols;
  float alpha;
};

__device__ __forceinline__ void copy_async(void* dst, const void* src, int bytes) {
  const unsigned d = unsigned(__cvta_generic_to_shared(dst));
  if (bytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
  else if (bytes == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(d), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(d), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_begin() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

// The rows that a CTA works on next, in shared memory.  A thread copies the columns
// that it will read itself, so waiting for its own copies is all that is needed:
// no barrier, and no register holds a row in flight.
template <typename T, int NV, bool BRANCH, bool PACKED, int STAGES>
struct Ring {
  static constexpr int kWhole = 8 * int(sizeof(T));          // eight values
  static constexpr int kKept = PACKED ? 8 : kWhole;          // eight values of u or y
  static constexpr int kGroup = 2 * kWhole + (BRANCH ? 2 : 1) * (kKept + (PACKED ? 4 : 0));
  static constexpr int bytes(int threads) { return threads * NV * kGroup * STAGES; }
  char* base;
  // Arrays of [NV][threads] pieces of at most 16 bytes, one after another in a stage.
  __device__ __forceinline__ char* piece(int stage, int offset, int g, int size) const {
    return base + (int64_t(stage) * kGroup + offset) * NV * blockDim.x + (g * int(blockDim.x) + int(threadIdx.x)) * size;
  }
  static constexpr int kDh = 0, kDu = kWhole, kU = 2 * kWhole, kY = kU + kKept, kUnitU = kU + (BRANCH ? 2 : 1) * kKept,
                       kUnitY = kUnitU + 4;
  __device__ __forceinline__ void whole(int stage, int offset, int g, const T* src) const {
#pragma unroll
    for (int i = 0; i < kWhole / 16; ++i)
      copy_async(piece(stage, offset + i * 16, g, 16), reinterpret_cast<const char*>(src) + i * 16, 16);
  }
  __device__ __forceinline__ void kept(int stage, int offset, int unit, int g, const void* row, int col, int cols) const {
    if constexpr (PACKED) {
      const unsigned char* r = static_cast<const unsigned char*>(row);
      copy_async(piece(stage, offset, g, 8), r + col, 8);
      copy_async(piece(stage, unit, g, 4), r + pack_code_bytes(cols) + (col / kPackGroup & ~3), 4);
    } else {
      whole(stage, offset, g, static_cast<const T*>(row) + col);
    }
  }
  __device__ __forceinline__ void fetch(const JoinBwd& p, const Columns<NV, true>& c, int64_t row, int stage) const {
    if (row < p.rows) {
#pragma unroll
      for (int g = 0; g < NV; ++g) {
        if (!c.has(g * 8)) continue;
        const int col = c.at(g * 8);
        whole(stage, kDh, g, static_cast<const T*>(p.dh) + row * p.ld_dh + col);
        kept(stage, kU, kUnitU, g, static_cast<const char*>(p.u) + row * p.ld_u * (PACKED ? 1 : sizeof(T)), col, p.cols);
        if (p.du) whole(stage, kDu, g, static_cast<const T*>(p.du) + row * p.ld_du + col);
        if (BRANCH)
          kept(stage, kY, kUnitY, g, static_cast<const char*>(p.y) + row * p.ld_y * (PACKED ? 1 : sizeof(T)), col, p.cols);
      }
    }
    copies_begin();
  }
  __device__ __forceinline__ void get_whole(int stage, int offset, int g, float* v) const {
    Eight<T> e;
#pragma unroll
    for (int i = 0; i < kWhole / 16; ++i) e.raw[i] = *reinterpret_cast<const uint4*>(piece(stage, offset + i * 16, g, 16));
    e.get(v);
  }
  __device__ __forceinline__ void get_kept(int stage, int offset, int unit, int g, int col, float* v) const {
    if constexpr (PACKED) {
      const unsigned four = *reinterpret_cast<const unsigned*>(piece(stage, unit, g, 4));
      const unsigned byte = four >> (8 * (col / kPackGroup & 3)) & 0xffu;
      decode8(*reinterpret_cast<const uint2*>(piece(stage, offset, g, 8)), pack_unit(byte), v);
    } else {
      get_whole(stage, offset, g, v);
    }
  }
};

// One CTA per set of rows (row, row + grid, ..), its column sums in registers.  A row
// takes two CTA-wide reductions, the second one of values that the first decides.
// Vector form: the next STAGES - 1 rows are on their way into shared memory meanwhile.
template <typename T, int NV, bool VEC, bool BRANCH, bool PACKED, int STAGES>
__global__ void __launch_bounds__(NV == 1 ? 128 : 512, NV == 1 ? 4 : 1) join_bwd_kernel(JoinBwd p) {
  constexpr int N = NV * 8;
  extern __shared__ __align__(16) char dynamic[];
  __shared__ float sh[4][kMaxWarps];
  const Columns<NV, VEC> c{p.cols};
  using R = Ring<T, NV, BRANCH, PACKED, STAGES>;
  const R ring{dynamic};
  float dw[N], db[N], P[BRANCH ? N : 1], Q[BRANCH ? N : 1];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    dw[i] = db[i] = 0.f;
    if (BRANCH) P[i] = Q[i] = 0.f;
  }
  const int64_t first = blockIdx.x, step = gridDim.x;
  if constexpr (VEC) {
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) ring.fetch(p, c, first + s * step, s);
  }
  int stage = 0;
  for (int64_t row = first; row < p.rows; row += step) {
    const float mean_u = p.mean_u[row], rstd_u = p.rstd_u[row];
    float mean_y = 0.f, rstd_y = 0.f;
    if (BRANCH) {
      mean_y = p.mean_y[row];
      rstd_y = p.rstd_y[row];
    }
    if constexpr (VEC) {
      ring.fetch(p, c, row + (STAGES - 1) * step, stage == 0 ? STAGES - 1 : stage - 1);
      copies_wait<STAGES - 1>();
    }
    auto get_t = [&](const void* base, int64_t ld, int offset, int g, float* v) {
      if constexpr (VEC) {
        if (c.has(g * 8)) {
          ring.get_whole(stage, offset, g, v);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = 0.f;
        }
      } else {
        c.load8(static_cast<const T*>(base) + row * ld, g, v);
      }
    };
    auto get_kept = [&](const void* base, int64_t ld, int offset, int unit, int g, float* v) {
      if constexpr (VEC) {
        if (c.has(g * 8)) {
          ring.get_kept(stage, offset, unit, g, c.at(g * 8), v);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = 0.f;
        }
      } else if constexpr (PACKED) {
        const unsigned char* r = static_cast<const unsigned char*>(base) + row * ld;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int col = c.at(g * 8 + i);
          v[i] = c.has(g * 8 + i) ? decode1(r[col], pack_unit(r[pack_code_bytes(p.cols) + col / kPackGroup])) : 0.f;
        }
      } else {
        c.load8(static_cast<const T*>(base) + row * ld, g, v);
      }
    };
    float hat[N], a[N];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int g = 0; g < NV; ++g) {
      float d[8], w[8];
      get_t(p.dh, p.ld_dh, R::kDh, g, d);
      get_kept(p.u, p.ld_u, R::kU, R::kUnitU, g, hat + g * 8);
      c.load8(static_cast<const T*>(p.w), g, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int k = g * 8 + i;
        hat[k] = (hat[k] - mean_u) * rstd_u;
        dw[k] = fmaf(d[i], hat[k], dw[k]);
        db[k] += d[i];
        a[k] = d[i] * w[i];
        s[0] += a[k];
        s[1] = fmaf(a[k], hat[k], s[1]);
      }
      if (p.h) {
        c.load8(static_cast<const T*>(p.b), g, d);
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = fmaf(hat[g * 8 + i], w[i], d[i]);
        c.store8(static_cast<T*>(p.h) + row * p.cols, g, d);
      }
    }
    block_sums(s, sh);
    const float s0 = s[0] / p.cols, s1 = s[1] / p.cols;
    s[0] = s[1] = 0.f;
#pragma unroll
    for (int g = 0; g < NV; ++g) {
      float d[8];
      if (p.du) {
        get_t(p.du, p.ld_du, R::kDu, g, d);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int k = g * 8 + i;
        a[k] = fmaf(rstd_u, a[k] - fmaf(hat[k], s1, s0), d[i]);
        d[i] = p.alpha * a[k];
      }
      c.store8(static_cast<T*>(p.dx) + row * p.ld_dx, g, d);
      if constexpr (BRANCH) {
        float w[8];
        get_kept(p.y, p.ld_y, R::kY, R::kUnitY, g, hat + g * 8);
        c.load8(static_cast<const T*>(p.pw), g, w);
        c.load8(static_cast<const T*>(p.gate), g, d);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int k = g * 8 + i;
          hat[k] = (hat[k] - mean_y) * rstd_y;
          P[k] = fmaf(a[k], hat[k], P[k]);
          Q[k] += a[k];
          a[k] *= d[i] * w[i];
          s[0] += a[k];
          s[1] = fmaf(a[k], hat[k], s[1]);
        }
      }
    }
    if constexpr (BRANCH) {
      block_sums(s, sh + 2);
      const float t0 = s[0] / p.cols, t1 = s[1] / p.cols;
#pragma unroll
      for (int g = 0; g < NV; ++g) {
        float d[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = rstd_y * (a[g * 8 + i] - fmaf(hat[g * 8 + i], t1, t0));
        c.store8(static_cast<T*>(p.dy) + row * p.ld_dy, g, d);
      }
    } else if (blockDim.x > 32) {
      __syncthreads();  // sh is written again by the next row
    }
    stage = stage == STAGES - 1 ? 0 : stage + 1;
  }
  float* out = p.sums + int64_t(blockIdx.x) * (BRANCH ? 4 : 2) * p.cols;
#pragma unroll
  for (int g = 0; g < NV; ++g) {
    c.store8(out, g, dw + g * 8);
    c.store8(out + p.cols, g, db + g * 8);
    if constexpr (BRANCH) {
      c.store8(out + 2 * int64_t(p.cols), g, P + g * 8);
      c.store8(out + 3 * int64_t(p.cols), g, Q + g * 8);
    }
  }
}

struct JoinFinish {
  const float* sums;
  const void *pw, *pb, *gate;
  void *dw, *db, *dpw, *dpb, *dgate;
  int parts, cols;
};

// 32 columns a CTA; each of its 8 rows of threads adds every eighth partial sum.
template <typename T, bool BRANCH>
__global__ void __launch_bounds__(256) join_finish_kernel(JoinFinish p) {
  constexpr int K = BRANCH ? 4 : 2;
  __shared__ float sh[K][8][32];
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;
  float s[K] = {};
  if (col < p.cols) {
    for (int q = part; q < p.parts; q += 8) {
#pragma unroll
      for (int k = 0; k < K; ++k) s[k] += p.sums[(int64_t(q) * K + k) * p.cols + col];
    }
  }
#pragma unroll
  for (int k = 0; k < K; ++k) sh[k][part][lane] = s[k];
  __syncthreads();
  if (part || col >= p.cols) return;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    s[k] = 0.f;
#pragma unroll
    for (int q = 0; q < 8; ++q) s[k] += sh[k][q][lane];
  }
  static_cast<T*>(p.dw)[col] = from_float<T>(s[0]);
  static_cast<T*>(p.db)[col] = from_float<T>(s[1]);
  if constexpr (BRANCH) {
    const float pw = to_float(static_cast<const T*>(p.pw)[col]), pb = to_float(static_cast<const T*>(p.pb)[col]);
    const float g = to_float(static_cast<const T*>(p.gate)[col]);
    static_cast<T*>(p.dgate)[col] = from_float<T>(pw * s[2] + pb * s[3]);
    static_cast<T*>(p.dpw)[col] = from_float<T>(g * s[2]);
    static_cast<T*>(p.dpb)[col] = from_float<T>(g * s[3]);
  }
}

// Groups of eight columns a thread has: enough work per thread that the reductions
// over the CTA weigh little, few enough registers that several CTAs share an SM.
int fwd_groups(int64_t cols) { return cols <= 1024 ? 1 : cols <= 2048 ? 2 : 4; }
int bwd_groups(int64_t cols) { return cols <= 1024 ? 1 : 2; }
int threads_for(int64_t cols, int nv) { return int((cols + nv * 8 - 1) / (nv * 8) + 31) / 32 * 32; }

template <typename T>
int fwd_typed(const JoinFwd& p, bool vec, cudaStream_t s) {
  const int nv = fwd_groups(p.cols);
  auto launch = [&](auto kernel) { kernel<<<unsigned(p.rows), threads_for(p.cols, nv), 0, s>>>(p); };
  if (nv == 1) vec ? launch(join_fwd_kernel<T, 1, true>) : launch(join_fwd_kernel<T, 1, false>);
  else if (nv == 2) vec ? launch(join_fwd_kernel<T, 2, true>) : launch(join_fwd_kernel<T, 2, false>);
  else vec ? launch(join_fwd_kernel<T, 4, true>) : launch(join_fwd_kernel<T, 4, false>);
  return int(cudaGetLastError());
}

// Shared memory above 48 KB (the kernel's fixed part counts too), once for each kernel and device.
template <auto Kernel>
int opt_in(int smem) {
  if (smem <= 47 * 1024) return 0;
  static std::atomic<uint64_t> opted{0};
  int device = 0;
  cudaGetDevice(&device);
  const uint64_t bit = uint64_t(1) << (device & 63);
  if (opted.load(std::memory_order_relaxed) & bit) return 0;
  const cudaError_t e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxRing);
  if (e == cudaSuccess) opted.fetch_or(bit, std::memory_order_relaxed);
  return int(e);
}

template <typename T, int NV, bool VEC, bool BRANCH, bool PACKED, int STAGES>
int bwd_launch(const JoinBwd& p, int parts, cudaStream_t s) {
  constexpr auto kernel = join_bwd_kernel<T, NV, VEC, BRANCH, PACKED, STAGES>;
  const int threads = threads_for(p.cols, NV);
  const int smem = VEC ? Ring<T, NV, BRANCH, PACKED, STAGES>::bytes(threads) : 0;
  if (const int r = opt_in<join_bwd_kernel<T, NV, VEC, BRANCH, PACKED, STAGES>>(smem)) return r;
  kernel<<<unsigned(parts), threads, smem, s>>>(p);
  return int(cudaGetLastError());
}

template <typename T, int NV, bool BRANCH, bool PACKED>
int bwd_pick(const JoinBwd& p, int parts, bool vec, cudaStream_t s) {
  if (!vec) return bwd_launch<T, NV, false, BRANCH, PACKED, 1>(p, parts, s);
  if (Ring<T, NV, BRANCH, PACKED, 3>::bytes(threads_for(p.cols, NV)) <= kMaxRing)
    return bwd_launch<T, NV, true, BRANCH, PACKED, 3>(p, parts, s);
  return bwd_launch<T, NV, true, BRANCH, PACKED, 1>(p, parts, s);
}

template <typename T, bool BRANCH, bool PACKED>
int bwd_typed(const JoinBwd& p, const JoinFinish& f, int parts, bool vec, cudaStream_t s) {
  const int r = bwd_groups(p.cols) == 1 ? bwd_pick<T, 1, BRANCH, PACKED>(p, parts, vec, s)
                                        : bwd_pick<T, 2, BRANCH, PACKED>(p, parts, vec, s);
  if (r) return r;
  join_finish_kernel<T, BRANCH><<<unsigned((p.cols + 31) / 32), 256, 0, s>>>(f);
  return int(cudaGetLastError());
}
}  // namespace

int64_t join_max_cols() { return kJoinMaxCols; }
int join_bwd_parts(int64_t rows, int64_t cols) {
  // CTAs that fit the GPU at once by registers (128 a thread) and, at most, four an SM.
  const int threads = threads_for(cols, bwd_groups(cols));
  const int per_sm = threads >= 512 ? 1 : threads >= 256 ? 2 : 4;
  const int64_t most = 148 * per_sm;
  return int(rows < most ? rows : most);
}

int join_fwd(const void* x, int64_t ld_x, const void* y, int64_t ld_y, int type, const void* pw, const void* pb,
             const void* gate, const void* w, const void* b, void* u, void* h, int64_t ld_h, float* stats, int64_t rows,
             int64_t cols, float alpha, float eps, cudaStream_t s) {
  if (rows <= 0 || rows > 0x7fffffff || cols <= 0 || cols > kJoinMaxCols) return -1;
  const JoinFwd p{x, y, pw, pb, gate, w, b, u, h, stats, ld_x, ld_y, ld_h, int(rows), int(cols), alpha, eps};
  const int64_t size = type == kTypeFP32 ? 4 : 2;
  const bool vec = cols % 8 == 0 && ld_x * size % 16 == 0 && ld_y * size % 16 == 0 && ld_h * size % 16 == 0 &&
                   aligned16(x) && aligned16(y) && aligned16(pw) && aligned16(pb) && aligned16(gate) && aligned16(w) &&
                   aligned16(b) && aligned16(u) && aligned16(h);
  if (type == kTypeBF16) return fwd_typed<__nv_bfloat16>(p, vec, s);
  if (type == kTypeFP32) return fwd_typed<float>(p, vec, s);
  return -1;
}

int join_bwd(const JoinBwdCall& c, cudaStream_t s) {
  if (c.rows <= 0 || c.rows > 0x7fffffff || c.cols <= 0 || c.cols > kJoinMaxCols) return -1;
  const bool branch = c.y != nullptr;
  if (!branch && !c.packed) return -1;
  const int parts = join_bwd_parts(c.rows, c.cols);
  const JoinBwd p{c.dh, c.du, c.u, c.y, c.pw, c.gate, c.w, c.b, c.mean_y, c.rstd_y, c.mean_u, c.rstd_u, c.dx, c.dy, c.h, c.workspace,
                  c.ld_dh, c.ld_du, c.ld_u, c.ld_y, c.ld_dy, c.ld_dx, int(c.rows), int(c.cols), c.alpha};
  const JoinFinish f{c.workspace, c.pw, c.pb, c.gate, c.dw, c.db, c.dpw, c.dpb, c.dgate, parts, int(c.cols)};
  const int64_t size = c.type == kTypeFP32 ? 4 : 2;
  auto fine = [&](const void* q, int64_t ld) { return !q || (aligned16(q) && ld * size % 16 == 0); };
  const bool vec = c.cols % 8 == 0 && fine(c.dh, c.ld_dh) && fine(c.du, c.ld_du) && fine(c.dx, c.ld_dx) &&
                   fine(c.dy, c.ld_dy) && fine(c.h, c.cols) && fine(c.pw, 0) && fine(c.gate, 0) && fine(c.w, 0) &&
                   fine(c.b, 0) && aligned16(c.workspace) &&
                   (c.packed || (fine(c.u, c.ld_u) && fine(c.y, c.ld_y)));
  auto pick = [&](auto zero) {
    using T = decltype(zero);
    if (!branch) return bwd_typed<T, false, true>(p, f, parts, vec, s);
    return c.packed ? bwd_typed<T, true, true>(p, f, parts, vec, s) : bwd_typed<T, true, false>(p, f, parts, vec, s);
  };
  if (c.type == kTypeBF16) return pick(__nv_bfloat16());
  if (c.type == kTypeFP32) return pick(float());
  return -1;
}

}  // namespace kernels
}  // namespace tn5b
