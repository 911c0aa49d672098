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
#include "kernels_api.h"
#include "rowvec.cuh"

namespace tn5b {
namespace kernels {
namespace {
constexpr int kMaxWarps = 16;

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
  static constexpr int kN = NV * 8;
  int cols;
  __device__ __forceinline__ int at(int i) const {
    return VEC ? ((i / 8) * int(blockDim.x) + int(threadIdx.x)) * 8 + (i & 7)
               : i * int(blockDim.x) + int(threadIdx.x);
  }
  __device__ __forceinline__ bool has(int i) const { return at(VEC ? i & ~7 : i) < cols; }
  template <typename T>
  __device__ __forceinline__ void load(const T* row, float (&v)[kN], bool once) const {
    if (VEC) {
#pragma unroll
      for (int g = 0; g < NV; ++g) {
        Eight<T> e;
        if (has(g * 8)) {
          once ? e.load_once(row + at(g * 8)) : e.load(row + at(g * 8));
          e.get(v + g * 8);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[g * 8 + i] = 0.f;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < kN; ++i) v[i] = has(i) ? to_float(row[at(i)]) : 0.f;
    }
  }
  template <typename T>
  __device__ __forceinline__ void store(T* row, const float (&v)[kN]) const {
    if (VEC) {
#pragma unroll
      for (int g = 0; g < NV; ++g) {
        if (!has(g * 8)) continue;
        Eight<T> e;
        e.set(v + g * 8);
        e.store(row + at(g * 8));
      }
    } else {
#pragma unroll
      for (int i = 0; i < kN; ++i)
        if (has(i)) row[at(i)] = from_float<T>(v[i]);
    }
  }
  __device__ __forceinline__ void load_packed(const unsigned char* row, float (&v)[kN]) const {
    const unsigned char* units = row + pack_code_bytes(cols);
    if (VEC) {
#pragma unroll
      for (int g = 0; g < NV; ++g) {
        if (has(g * 8)) {
          const int c = at(g * 8);
          decode8(*reinterpret_cast<const uint2*>(row + c), pack_unit(units[c / kPackGroup]), v + g * 8);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[g * 8 + i] = 0.f;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < kN; ++i) v[i] = has(i) ? decode1(row[at(i)], pack_unit(units[at(i) / kPackGroup])) : 0.f;
    }
  }
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

template <typename T, int NV, bool VEC>
__global__ void __launch_bounds__(512) join_fwd_kernel(JoinFwd p) {
  __shared__ float sh[4][kMaxWarps];
  const Columns<NV, VEC> c{p.cols};
  const int64_t row = blockIdx.x;
  float y[NV * 8], u[NV * 8], t[NV * 8];
  c.load(static_cast<const T*>(p.y) + row * p.ld_y, y, true);
  c.load(static_cast<const T*>(p.x) + row * p.ld_x, u, true);
  float mean, rstd;
  row_stats(c, y, p.eps, mean, rstd, sh);
  if (threadIdx.x == 0) {
    p.stats[row] = mean;
    p.stats[p.rows + row] = rstd;
  }
#pragma unroll
  for (int i = 0; i < NV * 8; ++i) y[i] = (y[i] - mean) * rstd;
  c.load(static_cast<const T*>(p.pw), t, false);
#pragma unroll
  for (int i = 0; i < NV * 8; ++i) y[i] *= t[i];
  c.load(static_cast<const T*>(p.pb), t, false);
#pragma unroll
  for (int i = 0; i < NV * 8; ++i) y[i] += t[i];
  c.load(static_cast<const T*>(p.gate), t, false);
#pragma unroll
  for (int i = 0; i < NV * 8; ++i) u[i] = fmaf(t[i], y[i], p.alpha * u[i]);
  c.store(static_cast<T*>(p.u) + row * p.cols, u);
  row_stats(c, u, p.eps, mean, rstd, sh + 2);
  if (threadIdx.x == 0) {
    p.stats[2 * int64_t(p.rows) + row] = mean;
    p.stats[3 * int64_t(p.rows) + row] = rstd;
  }
  c.load(static_cast<const T*>(p.w), t, false);
  c.load(static_cast<const T*>(p.b), y, false);
#pragma unroll
  for (int i = 0; i < NV * 8; ++i) u[i] = fmaf((u[i] - mean) * rstd, t[i], y[i]);
  c.store(static_cast<T*>(p.h) + row * p.ld_h, u);
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

template <typename T, int NV, bool VEC, bool BRANCH, bool PACKED>
__global__ void __launch_bounds__(512) join_bwd_kernel(JoinBwd p) {
  constexpr int N = NV * 8;
  __shared__ float sh[4][kMaxWarps];
  const Columns<NV, VEC> c{p.cols};
  float dw[N], db[N], P[BRANCH ? N : 1], Q[BRANCH ? N : 1];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    dw[i] = db[i] = 0.f;
    if (BRANCH) P[i] = Q[i] = 0.f;
  }
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const float mean_u = p.mean_u[row], rstd_u = p.rstd_u[row];
    float xhat[N], g[N], a[N], t[N];
    if (PACKED) c.load_packed(static_cast<const unsigned char*>(p.u) + row * p.ld_u, xhat);
    else c.load(static_cast<const T*>(p.u) + row * p.ld_u, xhat, true);
    c.load(static_cast<const T*>(p.dh) + row * p.ld_dh, g, true);
    c.load(static_cast<const T*>(p.w), t, false);
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      xhat[i] = (xhat[i] - mean_u) * rstd_u;
      dw[i] = fmaf(g[i], xhat[i], dw[i]);
      db[i] += g[i];
      a[i] = g[i] * t[i];
      s[0] += a[i];
      s[1] = fmaf(a[i], xhat[i], s[1]);
    }
    if (p.h) {
      c.load(static_cast<const T*>(p.b), g, false);
#pragma unroll
      for (int i = 0; i < N; ++i) g[i] = fmaf(xhat[i], t[i], g[i]);
      c.store(static_cast<T*>(p.h) + row * p.cols, g);
    }
    block_sums(s, sh);
    const float s0 = s[0] / p.cols, s1 = s[1] / p.cols;
    if (p.du) c.load(static_cast<const T*>(p.du) + row * p.ld_du, t, true);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      a[i] = rstd_u * (a[i] - s0 - xhat[i] * s1) + (p.du ? t[i] : 0.f);
      g[i] = p.alpha * a[i];
    }
    c.store(static_cast<T*>(p.dx) + row * p.ld_dx, g);
    if constexpr (BRANCH) {
      const float mean_y = p.mean_y[row], rstd_y = p.rstd_y[row];
      float yhat[N];
      if (PACKED) c.load_packed(static_cast<const unsigned char*>(p.y) + row * p.ld_y, yhat);
      else c.load(static_cast<const T*>(p.y) + row * p.ld_y, yhat, true);
      c.load(static_cast<const T*>(p.pw), t, false);
      c.load(static_cast<const T*>(p.gate), g, false);
      s[0] = s[1] = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        yhat[i] = (yhat[i] - mean_y) * rstd_y;
        if (c.has(i)) {
          P[i] = fmaf(a[i], yhat[i], P[i]);
          Q[i] += a[i];
        }
        a[i] *= g[i] * t[i];
        s[0] += a[i];
        s[1] = fmaf(a[i], yhat[i], s[1]);
      }
      block_sums(s, sh + 2);
      const float t0 = s[0] / p.cols, t1 = s[1] / p.cols;
#pragma unroll
      for (int i = 0; i < N; ++i) a[i] = rstd_y * (a[i] - t0 - yhat[i] * t1);
      c.store(static_cast<T*>(p.dy) + row * p.ld_dy, a);
    }
    if (!BRANCH && blockDim.x > 32) __syncthreads();  // sh is written again by the next row
  }
  float* out = p.sums + int64_t(blockIdx.x) * (BRANCH ? 4 : 2) * p.cols;
  c.store(out, dw);
  c.store(out + p.cols, db);
  if constexpr (BRANCH) {
    c.store(out + 2 * int64_t(p.cols), P);
    c.store(out + 3 * int64_t(p.cols), Q);
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

// Threads that cover the columns eight (or sixteen, above 4096 columns) at a time.
int threads_for(int64_t cols, int nv) { return int((cols + nv * 8 - 1) / (nv * 8) + 31) / 32 * 32; }

template <typename T>
int fwd_typed(const JoinFwd& p, bool vec, cudaStream_t s) {
  const int nv = p.cols <= 4096 ? 1 : 2;
  auto launch = [&](auto kernel) { kernel<<<unsigned(p.rows), threads_for(p.cols, nv), 0, s>>>(p); };
  if (nv == 1) vec ? launch(join_fwd_kernel<T, 1, true>) : launch(join_fwd_kernel<T, 1, false>);
  else vec ? launch(join_fwd_kernel<T, 2, true>) : launch(join_fwd_kernel<T, 2, false>);
  return int(cudaGetLastError());
}

template <typename T, bool BRANCH, bool PACKED>
int bwd_typed(const JoinBwd& p, const JoinFinish& f, int parts, bool vec, cudaStream_t s) {
  const int nv = p.cols <= 4096 ? 1 : 2;
  auto launch = [&](auto kernel) { kernel<<<unsigned(parts), threads_for(p.cols, nv), 0, s>>>(p); };
  if (nv == 1)
    vec ? launch(join_bwd_kernel<T, 1, true, BRANCH, PACKED>) : launch(join_bwd_kernel<T, 1, false, BRANCH, PACKED>);
  else
    vec ? launch(join_bwd_kernel<T, 2, true, BRANCH, PACKED>) : launch(join_bwd_kernel<T, 2, false, BRANCH, PACKED>);
  const int r = int(cudaGetLastError());
  if (r) return r;
  join_finish_kernel<T, BRANCH><<<unsigned((p.cols + 31) / 32), 256, 0, s>>>(f);
  return int(cudaGetLastError());
}
}  // namespace

int64_t join_max_cols() { return kJoinMaxCols; }
int join_bwd_parts(int64_t rows, int64_t cols) {
  const int per_sm = cols <= 1024 ? 8 : 2;
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
