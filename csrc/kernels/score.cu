// Scores of given tokens from logits (sm_100a): log probability, entropy and the
// most probable alternatives of every row in one pass, and the gradient of the
// log probability and the entropy.
//
//   m = max z, s = sum e^(z - m), u = sum e^(z - m) (z - m)
//   log p_t = z_t - m - ln s          H = ln s - u / s
//   d z_j = a ([j = t] - p_j) - b p_j (ln p_j + H)      a = d log p_t, b = d H
//
// Forward: a cluster of 1, 2 or 4 CTAs per row, each thread with running (m, s, u)
// in FP32 over 16-byte vectors; a logit of -inf adds nothing.  The alternatives
// need no sort of the row: the k-th largest of the threads' maxima bounds the k-th
// largest logit from below, and only the threads that reach it can hold one, so a
// second look at those threads' vectors collects the few candidates, which one warp
// sorts.  Equal values go to the lowest index.  Where many values are equal, the
// threads' maxima are (value, start of the vector that held it), of which no two are
// the same.
// Ranks of a vocabulary-parallel group exchange one record a row (m, s, u, z_t
// and their own alternatives) and merge them in rank order.
//
// B200, 8192 BF16 rows of 50304 in no cache: 140 us without alternatives (5.9 TB/s; the
// exponentials keep the special-function units 71-76 % busy, which is what bounds it
// next), 160 us with 8 and 192 us with 32 of them (the second look and the sorts,
// between barriers); 11 us less where the call before had the same inputs.  8192 rows of
// 6288: 28, 42 and 73 us, of 1000 with 8 alternatives 26 us: a row's fixed chain of
// steps.  Gradient of 2048 rows of 50304: 70 us (5.9 TB/s).
#include <cooperative_groups.h>

#include <cmath>
#include <type_traits>

#include "kernels_api.h"
#include "rowvec.cuh"

namespace cg = cooperative_groups;

namespace tn5b {
namespace kernels {
namespace {
constexpr int kThreads = 256, kWarps = kThreads / 32;  // of the merge and the gradient
constexpr int kMaxTop = 32;       // alternatives a row: one sorted list per warp
constexpr int kUnroll = 4;
constexpr int kSmThreads = 1536;  // of all CTAs on an SM, at 40 registers each
constexpr float kLog2e = 1.44269504088896340736f;
// e^d with d below this is zero in FP32; it also keeps 0 * (-inf) out of u.
constexpr float kLowest = -200.f;

using Key = unsigned long long;  // order of (value, -index): a larger key comes first

__device__ __forceinline__ unsigned order_of(float v) {
  v += 0.f;  // -0 and 0 are one value
  if (v != v) return 0xffffffffu;
  const unsigned b = __float_as_uint(v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(Key key) {
  const unsigned o = unsigned(key >> 32);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);  // NaN's 0xffffffff gives a NaN
}
__device__ __forceinline__ Key make_key(float v, unsigned index) {
  return Key(order_of(v)) << 32 | Key(~index);
}
__device__ __forceinline__ unsigned index_of(Key key) { return ~unsigned(key); }

__device__ __forceinline__ Key shfl_xor_key(Key k, int d) { return __shfl_xor_sync(kAllLanes, k, d); }
// One compare-exchange across lanes: keeps the larger key where `first`.
__device__ __forceinline__ Key exchange(Key k, int d, bool larger) {
  const Key o = shfl_xor_key(k, d);
  return (o > k) == larger ? o : k;
}
// Descending over the lanes of a warp.
__device__ __forceinline__ Key sort_warp(Key k) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1) {
#pragma unroll
    for (int d = size >> 1; d; d >>= 1) {
      const bool descending = size == 32 || (lane & size) == 0;
      k = exchange(k, d, ((lane & d) == 0) == descending);
    }
  }
  return k;
}
// The 32 largest of two descending lists, descending.
__device__ __forceinline__ Key merge_warp(Key a, Key b) {
  const int lane = threadIdx.x & 31;
  const Key r = __shfl_sync(kAllLanes, b, 31 - lane);
  Key k = a > r ? a : r;
#pragma unroll
  for (int d = 16; d; d >>= 1) k = exchange(k, d, (lane & d) == 0);
  return k;
}

struct Sums {
  float m, s, u;
};
// Joins b's sums to a's; either may be empty (m = -inf, s = u = 0).
__device__ __forceinline__ Sums join(Sums a, Sums b) {
  Sums r;
  r.m = max_nan(a.m, b.m);
  const float base = r.m == -INFINITY ? 0.f : r.m;
  const float da = fmaxf(a.m - base, kLowest), db = fmaxf(b.m - base, kLowest);
  const float fa = fast_exp2(da * kLog2e), fb = fast_exp2(db * kLog2e);
  r.s = a.s * fa + b.s * fb;
  r.u = (a.u + da * a.s) * fa + (b.u + db * b.s) * fb;
  return r;
}

// Where the results of a row go.
struct Out {
  float* logprob;    // [rows]
  float* entropy;    // [rows]
  float* state;      // [3][rows]: m, ln s, H
  float* top_value;  // [rows][k]
  int64_t* top_id;   // [rows][k]
  float* record;     // [rows][4 + 2k]: m, s, u, z_t, values, ids (ranks of a group), or null
  int rows, k;
};

__device__ __forceinline__ void finish_row(const Out& o, int row, Sums a, float picked, int64_t target,
                                           int64_t vocab_total) {
  const float nan = __int_as_float(0x7fffffff);
  float logprob, entropy, m = a.m, ln_s = 0.f;
  if (!(m < INFINITY)) {  // NaN or +inf among the logits
    logprob = entropy = m = nan;
  } else if (m == -INFINITY) {  // nothing left by the mask
    logprob = -INFINITY;
    entropy = 0.f;
  } else {
    ln_s = logf(a.s);
    logprob = (picked - m) - ln_s;
    entropy = ln_s - a.u / a.s;
  }
  if (target < 0) logprob = 0.f;
  if (target >= vocab_total) logprob = nan;
  o.logprob[row] = logprob;
  o.entropy[row] = entropy;
  o.state[row] = m;
  o.state[o.rows + row] = ln_s;
  o.state[2 * int64_t(o.rows) + row] = entropy;
}
__device__ __forceinline__ float top_logprob(float value, Sums a) {
  if (a.m == -INFINITY) return -INFINITY;
  if (!(a.m < INFINITY)) return __int_as_float(0x7fffffff);
  return (value - a.m) - logf(a.s);
}

template <typename T>
struct Vec {  // one 16-byte load
  static constexpr int kN = 16 / int(sizeof(T));
  uint4 raw;
  __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void get(float* v) const {
    const T* h = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i] = to_float(h[i]);
  }
};

// One thread's sums over its part of a row, by the definitions: any values, with
// infinities and NaN.  Rows of ordinary values take `Fast` below.
template <bool TOP>
struct Running {
  Sums a{-INFINITY, 0.f, 0.f};
  unsigned best = 0, best_at = 0xffffffffu;  // order_of the largest value, start of its vector

  // N values that begin at index `at`.
  template <int N>
  __device__ __forceinline__ void add(const float* v, unsigned at) {
    float top = v[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = max_nan(top, v[i]);
    if (TOP) {
      const unsigned o = order_of(top);
      if (o > best) {
        best = o;
        best_at = at;
      }
    }
    const float m = max_nan(a.m, top);
    const float base = m == -INFINITY ? 0.f : m;
    const float d0 = fmaxf(a.m - base, kLowest);
    const float f = fast_exp2(d0 * kLog2e);
    a.u = (a.u + d0 * a.s) * f;
    a.s *= f;
    a.m = m;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float d = fmaxf(v[i] - base, kLowest);
      const float e = fast_exp2(d * kLog2e);
      a.s += e;
      a.u = fmaf(e, d, a.u);
    }
  }
  __device__ __forceinline__ Key key() const { return best ? Key(best) << 32 | Key(~best_at) : 0; }
};

// The same for rows whose largest value lies within +-kPlain, in half the
// instructions: t = z log2 e - R with one fused multiply-add, R = fl(m log2 e) the
// running reference, two elements an instruction (f32x2), the maximum of 16-bit
// types on packed pairs.  R is a function of m, so sums join without further state.
// Its rounding, off = m log2 e - R, stays in every t of a sum and is taken out once per
// row (`natural`).  off is at most half a unit in R's last place: 1/4 for |m| < 2^22,
// 1 for the lowest start (2^24), so t <= off <= 1 and no exponential overflows.  A row
// whose largest value is further out would have an off that ruins its sums (128 at
// 2^31) and takes `Running`.  Values below -kFloor (-inf above all) are lifted to it:
// 2^t is zero there in any row that counts, and t finite.
constexpr float kFloor = 33554432.f, kLow = 16777216.f, kPlain = 4194304.f;  // 2^25, 2^24, 2^22
template <typename T> struct Packed2;
template <> struct Packed2<__nv_bfloat16> {
  static __device__ __forceinline__ unsigned larger(unsigned a, unsigned b) {
    const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const unsigned*>(&r);
  }
  static __device__ __forceinline__ unsigned floor() { return 0xcc00cc00u; }  // -kFloor
  static __device__ __forceinline__ Two floats(unsigned w) {
    return two(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
};
template <> struct Packed2<__half> {
  static __device__ __forceinline__ unsigned larger(unsigned a, unsigned b) {
    const __half2 r = __hmax2_nan(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const unsigned*>(&r);
  }
  static __device__ __forceinline__ unsigned floor() { return 0xfbfffbffu; }  // -65504, the type's lowest
  static __device__ __forceinline__ Two floats(unsigned w) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    return two(f.x, f.y);
  }
};
// Largest value and the values lifted to the floor of one 16-byte vector.
template <typename T>
struct Loaded {
  static constexpr int kPairs = 8 / int(sizeof(T) / 2) / 2;
  static __device__ __forceinline__ void read(const uint4& raw, float& top, Two* z) {
    const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
    using P = Packed2<T>;
    unsigned t = P::larger(P::larger(w[0], w[1]), P::larger(w[2], w[3]));
    t = P::larger(t, t >> 16 | t << 16);
    top = both(P::floats(t)).x;
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = P::floats(P::larger(w[i], P::floor()));
  }
};
template <>
struct Loaded<float> {
  static constexpr int kPairs = 2;
  static __device__ __forceinline__ void read(const uint4& raw, float& top, Two* z) {
    const float v[4] = {__uint_as_float(raw.x), __uint_as_float(raw.y), __uint_as_float(raw.z), __uint_as_float(raw.w)};
    top = max_nan(max_nan(v[0], v[1]), max_nan(v[2], v[3]));
#pragma unroll
    for (int i = 0; i < 2; ++i) z[i] = two(fmaxf(v[2 * i], -kFloor), fmaxf(v[2 * i + 1], -kFloor));
  }
};
// Where the running maximum begins: above every lifted value, and so low that what was
// counted there vanishes in a row whose largest value is above `plain_low` (FP16's floor
// is its lowest number, where lifted values count 1 until then).
template <typename T> __device__ __forceinline__ float start_low() { return -kLow; }
template <> __device__ __forceinline__ float start_low<__half>() { return -65504.f; }
template <typename T> __device__ __forceinline__ float plain_low() { return -kPlain; }
template <> __device__ __forceinline__ float plain_low<__half>() { return -6e4f; }

// R: rounded on its own everywhere (a product contracted into a following
// difference would be another reference).
__device__ __forceinline__ float reference(float m) { return __fmul_rn(m, kLog2e); }

template <typename T>
struct Fast {
  float m = start_low<T>();
  Two s = 0, u = 0;  // of even and odd elements

  __device__ __forceinline__ void raise(float top) {
    const float next = max_nan(m, top);
    const float d = reference(m) - reference(next);
    const float f = fast_exp2(d);
    u = two_mul(two_fma(two(d, d), s, u), two(f, f));
    s = two_mul(s, two(f, f));
    m = next;
  }
  __device__ __forceinline__ void count(Two z, Two scale, Two minus_r) {
    const Two t = two_fma(z, scale, minus_r);
    const float2 f = both(t);
    const Two e = two(fast_exp2(f.x), fast_exp2(f.y));
    s = two_add(s, e);
    u = two_fma(e, t, u);
  }
  template <int COUNT>
  __device__ __forceinline__ void add(const uint4* raw) {
    constexpr int P = Loaded<T>::kPairs;
    Two z[COUNT * P];
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
      float t;
      Loaded<T>::read(raw[i], t, z + i * P);
      top = max_nan(top, t);
    }
    raise(top);
    const float r = -reference(m);
    const Two scale = two(kLog2e, kLog2e), minus_r = two(r, r);
#pragma unroll
    for (int i = 0; i < COUNT * P; ++i) count(z[i], scale, minus_r);
  }
  __device__ __forceinline__ void add_one(float v) {
    raise(v);
    const float t = fmaf(fmaxf(v, -kFloor), kLog2e, -reference(m));
    const float e = fast_exp2(t);
    s = two_add(s, two(e, 0.f));
    u = two_fma(two(e, 0.f), two(t, 0.f), u);
  }
  // The warp's sums relative to its own maximum, in every lane.
  __device__ __forceinline__ Sums warp_total() const {
    float top = m;
#pragma unroll
    for (int d = 16; d; d >>= 1) top = max_nan(top, __shfl_xor_sync(kAllLanes, top, d));
    const float2 ss = both(s), uu = both(u);
    const float d = reference(m) - reference(top), f = fast_exp2(d);
    const float sum = ss.x + ss.y;
    return Sums{top, warp_sum(sum * f), warp_sum((uu.x + uu.y + d * sum) * f)};
  }
};
// From the reference fl(m log2 e) and log2 units to sums of e^(z - m).
__device__ __forceinline__ Sums natural(Sums a) {
  const float off = fmaf(a.m, kLog2e, -reference(a.m));
  const float f = fast_exp2(-off);
  return Sums{a.m, a.s * f, (a.u - off * a.s) * f * 0.69314718055994530942f};
}

// The part of a row that one CTA reads: `head` single values up to a 16-byte
// boundary, `vectors` vectors, `tail` single values.
template <typename T>
struct Part {
  const T* x;
  unsigned lo, head, vectors, tail;
  __device__ __forceinline__ Part(const T* row, unsigned begin, unsigned end) {
    x = row + begin;
    lo = begin;
    const unsigned n = end - begin;
    const unsigned off = unsigned((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    head = off ? min(n, unsigned(Vec<T>::kN) - off) : 0u;
    vectors = (n - head) / Vec<T>::kN;
    tail = n - head - vectors * Vec<T>::kN;
  }
  __device__ __forceinline__ unsigned vector_at(unsigned j) const { return head + j * Vec<T>::kN; }
};

template <int NT>
struct TopShared {
  static constexpr int W = NT / 32;
  Key lists[W][32];
  static constexpr int kCandidates = 4 * NT;  // more than that takes the selection by rounds
  Key candidates[kCandidates];
  Key best[W];
  unsigned active[NT];
  unsigned active_count, count;
};

__device__ __forceinline__ float exchange(float v, int d, bool larger) {
  const float o = __shfl_xor_sync(kAllLanes, v, d);
  return larger ? fmaxf(v, o) : fminf(v, o);
}

// The warp's sorted list of the candidates that were collected.
template <int NT>
__device__ __forceinline__ void sort_candidates(TopShared<NT>& sh, unsigned n) {
  const int lane = threadIdx.x & 31;
  Key list = 0;
  for (unsigned at = 0; at < n; at += 32) {
    const Key next = sort_warp(at + lane < n ? sh.candidates[at + lane] : 0);
    list = at ? merge_warp(list, next) : next;
  }
  sh.lists[0][lane] = list;
}

// The CTA's list for a part of ordinary values: by values alone, the index counts only
// among the candidates.  False (for every thread) where that does not decide: fewer
// than k threads with ordinary values, or more candidates than there is room for
// (many equal values); then `block_top` does.
template <typename T, int NT>
__device__ __forceinline__ bool fast_top(const Part<T>& part, float own, int k, TopShared<NT>& sh) {
  constexpr int W = NT / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  float(*const lists)[32] = reinterpret_cast<float(*)[32]>(sh.lists);
  float v = own;
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1) {
#pragma unroll
    for (int d = size >> 1; d; d >>= 1) v = exchange(v, d, ((lane & d) == 0) == (size == 32 || (lane & size) == 0));
  }
  lists[warp][lane] = v;
  if (tid == 0) sh.active_count = sh.count = 0;
  __syncthreads();
#pragma unroll
  for (int half = W / 2; half; half >>= 1) {
    if (warp < half) {
      v = fmaxf(v, lists[warp + half][31 - lane]);
#pragma unroll
      for (int d = 16; d; d >>= 1) v = exchange(v, d, (lane & d) == 0);
      lists[warp][lane] = v;
    }
    __syncthreads();
  }
  const float bound = lists[0][k - 1];
  if (!(bound > plain_low<T>())) return false;
  if (own >= bound) sh.active[atomicAdd(&sh.active_count, 1u)] = tid;
  __syncthreads();
  auto take = [&](float value, unsigned index) {
    if (value >= bound) {
      const unsigned at = atomicAdd(&sh.count, 1u);
      if (at < TopShared<NT>::kCandidates) sh.candidates[at] = make_key(value, index);
    }
  };
  // A warp for each active thread: its vectors are NT apart.
  for (unsigned a = warp; a < sh.active_count; a += W) {
    for (unsigned j = sh.active[a] + lane * NT; j < part.vectors; j += 32 * NT) {
      const unsigned at = part.vector_at(j);
      const uint4 raw = *reinterpret_cast<const uint4*>(part.x + at);
      Vec<T> vec;
      vec.raw = raw;
      float z[Vec<T>::kN];
      vec.get(z);
      float top = z[0];
#pragma unroll
      for (int e = 1; e < Vec<T>::kN; ++e) top = fmaxf(top, z[e]);
      if (top < bound) continue;  // most vectors hold none
#pragma unroll
      for (int e = 0; e < Vec<T>::kN; ++e) take(z[e], part.lo + at + e);
    }
  }
  for (unsigned c = tid; c < part.head + part.tail; c += NT) {
    const unsigned at = c < part.head ? c : part.vector_at(part.vectors) + (c - part.head);
    take(to_float(part.x[at]), part.lo + at);
  }
  __syncthreads();
  const unsigned n = sh.count;
  if (n > TopShared<NT>::kCandidates) return false;
  if (warp == 0) sort_candidates(sh, n);
  return true;
}

// The same for any values, equal ones and NaN.  Descending list of the CTA's 32 best,
// of which the first k count, in sh.lists[0].
template <typename T, int NT>
__device__ __forceinline__ void block_top(const Part<T>& part, Key own, int k, TopShared<NT>& sh) {
  constexpr int W = NT / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) sh.active_count = sh.count = 0;
  Key list = sort_warp(own);
  sh.lists[warp][lane] = list;
  __syncthreads();
#pragma unroll
  for (int half = W / 2; half; half >>= 1) {
    if (warp < half) {
      list = merge_warp(list, sh.lists[warp + half][lane]);
      sh.lists[warp][lane] = list;
    }
    __syncthreads();
  }
  const Key bound = sh.lists[0][k - 1];
  if (own >= bound) sh.active[atomicAdd(&sh.active_count, 1u)] = tid;
  __syncthreads();

  // Visits every value whose (value, start of vector) reaches the bound; its own
  // key is handed on.  Items: the active threads' vectors, then single values.
  const unsigned per = (part.vectors + NT - 1) / NT;
  const unsigned scalars = part.head + part.tail;
  const unsigned items = sh.active_count * per;
  auto visit = [&](auto&& take) {
    for (unsigned i = tid; i < items + scalars; i += NT) {
      if (i < items) {
        const unsigned a = i / per, j = sh.active[a] + (i - a * per) * NT;
        if (j >= part.vectors) continue;
        const unsigned at = part.vector_at(j);
        Vec<T> vec;
        float v[Vec<T>::kN];
        vec.load(part.x + at);
        vec.get(v);
        float top = v[0];
#pragma unroll
        for (int e = 1; e < Vec<T>::kN; ++e) top = max_nan(top, v[e]);
        if (make_key(top, part.lo + at) < bound) continue;  // most vectors hold none
#pragma unroll
        for (int e = 0; e < Vec<T>::kN; ++e)
          if (make_key(v[e], part.lo + at) >= bound) take(make_key(v[e], part.lo + at + e));
      } else {
        const unsigned c = i - items;
        const unsigned at = c < part.head ? c : part.vector_at(part.vectors) + (c - part.head);
        const Key key = make_key(to_float(part.x[at]), part.lo + at);
        if (key >= bound) take(key);
      }
    }
  };
  visit([&](Key key) {
    const unsigned at = atomicAdd(&sh.count, 1u);
    if (at < TopShared<NT>::kCandidates) sh.candidates[at] = key;
  });
  __syncthreads();
  const unsigned n = sh.count;
  if (n <= TopShared<NT>::kCandidates) {
    if (warp == 0) sort_candidates(sh, n);
  } else {
    // Many candidates in few threads' vectors: the k largest one after another.
    Key below = ~Key(0);
    for (int r = 0; r < k; ++r) {
      Key best = 0;
      visit([&](Key key) {
        if (key < below && key > best) best = key;
      });
#pragma unroll
      for (int d = 16; d; d >>= 1) {
        const Key o = shfl_xor_key(best, d);
        if (o > best) best = o;
      }
      if (lane == 0) sh.best[warp] = best;
      __syncthreads();
      best = sh.best[0];
#pragma unroll
      for (int w = 1; w < W; ++w) best = best > sh.best[w] ? best : sh.best[w];
      below = best;
      if (tid == 0) sh.lists[0][r] = best;
      __syncthreads();
    }
    if (warp == 0 && lane >= k) sh.lists[0][lane] = 0;
  }
  __syncthreads();
}

// grid = rows * C CTAs in clusters of C; the cluster's CTAs take `chunk` columns each.
template <typename T, bool TOP, int NT>
__global__ void __launch_bounds__(NT, kSmThreads / NT) score_kernel(const T* logits, int64_t ld, unsigned vocab,
                                                         const int64_t* targets, int64_t start,
                                                         int64_t vocab_total, unsigned chunk, Out o) {
  constexpr int W = NT / 32;
  __shared__ Sums warp_sums[W];
  __shared__ Sums block_sums;
  __shared__ std::conditional_t<TOP, TopShared<NT>, int> sh;
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned C = cluster.num_blocks(), rank = cluster.block_rank();
  const int row = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* x = logits + int64_t(row) * ld;
  const unsigned begin = min(vocab, rank * chunk), end = min(vocab, begin + chunk);
  const Part<T> part(x, begin, end);
  constexpr int kN = Vec<T>::kN;

  // Sums of the CTA's part: by the fast form, or by the definitions where the
  // largest value says that the fast one does not hold.
  float own;  // the thread's largest value
  {
    Fast<T> run;
    if (unsigned(tid) < part.head) run.add_one(to_float(part.x[tid]));
    const uint4* vectors = reinterpret_cast<const uint4*>(part.x + part.head);
    unsigned j = tid;
    for (; j + (kUnroll - 1) * NT < part.vectors; j += kUnroll * NT) {
      uint4 raw[kUnroll];
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) raw[i] = vectors[j + i * NT];
      run.template add<kUnroll>(raw);
    }
    // What is left, loaded together as well: one after another these would cost a short
    // row most of its time.
    uint4 last[kUnroll - 1];
#pragma unroll
    for (int i = 0; i < kUnroll - 1; ++i)
      if (j + i * NT < part.vectors) last[i] = vectors[j + i * NT];
    float tail = 0.f;
    if (unsigned(tid) < part.tail) tail = to_float(part.x[part.vector_at(part.vectors) + tid]);
#pragma unroll
    for (int i = 0; i < kUnroll - 1; ++i)
      if (j + i * NT < part.vectors) run.template add<1>(last + i);
    if (unsigned(tid) < part.tail) run.add_one(tail);
    const Sums a = run.warp_total();
    own = run.m;
    if (lane == 0) warp_sums[warp] = a;
  }
  __syncthreads();
  float top = warp_sums[0].m;
#pragma unroll
  for (int w = 1; w < W; ++w) top = max_nan(top, warp_sums[w].m);
  bool plain = top > plain_low<T>() && top < kPlain;
  if constexpr (TOP) {
    if (plain) plain = fast_top(part, own, o.k, sh);
  }
  if (plain) {
    if (tid == 0) {
      Sums a{top, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float d = reference(warp_sums[w].m) - reference(top), f = fast_exp2(d);
        a.s += warp_sums[w].s * f;
        a.u += (warp_sums[w].u + d * warp_sums[w].s) * f;
      }
      block_sums = natural(a);
    }
  } else {
    Running<TOP> run;
    if (unsigned(tid) < part.head) {
      const float v = to_float(part.x[tid]);
      run.template add<1>(&v, part.lo + tid);
    }
    for (unsigned j = tid; j < part.vectors; j += NT) {
      Vec<T> vec;
      float v[kN];
      vec.load(part.x + part.vector_at(j));
      vec.get(v);
      run.template add<kN>(v, part.lo + part.vector_at(j));
    }
    if (unsigned(tid) < part.tail) {
      const unsigned i = part.vector_at(part.vectors) + tid;
      const float v = to_float(part.x[i]);
      run.template add<1>(&v, part.lo + i);
    }
    Sums a = run.a;
#pragma unroll
    for (int d = 16; d; d >>= 1) {
      Sums b;
      b.m = __shfl_xor_sync(kAllLanes, a.m, d);
      b.s = __shfl_xor_sync(kAllLanes, a.s, d);
      b.u = __shfl_xor_sync(kAllLanes, a.u, d);
      // The lower lane's sums come first on both sides, so both get the same bits.
      a = lane & d ? join(b, a) : join(a, b);
    }
    __syncthreads();  // every thread has read the fast form's maxima
    if (lane == 0) warp_sums[warp] = a;
    __syncthreads();
    if (tid == 0) {
      a = warp_sums[0];
#pragma unroll
      for (int w = 1; w < W; ++w) a = join(a, warp_sums[w]);
      block_sums = a;
    }
    if constexpr (TOP) block_top(part, run.key(), o.k, sh);  // synchronises
  }
  if (C > 1) cluster.sync();
  else __syncthreads();
  if (rank == 0 && warp == 0) {
    Sums a = block_sums;
    for (unsigned r = 1; r < C; ++r) a = join(a, *cluster.map_shared_rank(&block_sums, r));
    Key list = 0;
    if constexpr (TOP) {
      list = sh.lists[0][lane];
      for (unsigned r = 1; r < C; ++r) list = merge_warp(list, cluster.map_shared_rank(&sh.lists[0][0], r)[lane]);
    }
    const int64_t target = targets[row], local = target - start;
    const float picked = local >= 0 && local < vocab ? to_float(x[local]) : 0.f;
    if (o.record) {
      float* rec = o.record + int64_t(row) * (4 + 2 * o.k);
      if (lane == 0) {
        rec[0] = a.m;
        rec[1] = a.s;
        rec[2] = a.u;
        rec[3] = picked;
      }
      if (TOP && lane < o.k) {
        rec[4 + lane] = value_of(list);
        rec[4 + o.k + lane] = __int_as_float(int(index_of(list) + unsigned(start)));
      }
    } else {
      if (lane == 0) finish_row(o, row, a, picked, target, vocab_total);
      if (TOP && lane < o.k) {
        o.top_value[int64_t(row) * o.k + lane] = top_logprob(value_of(list), a);
        o.top_id[int64_t(row) * o.k + lane] = start + index_of(list);
      }
    }
  }
  if (C > 1) cluster.sync();  // shared memory stays until rank 0 has read it
}

// Records of `parts` ranks, [parts][rows][4 + 2k], one warp a row.
__global__ void __launch_bounds__(kThreads) score_merge_kernel(const float* records, int parts, int64_t vocab,
                                                               const int64_t* targets, Out o) {
  const int row = blockIdx.x * kWarps + threadIdx.x / 32, lane = threadIdx.x & 31;
  if (row >= o.rows) return;
  const int64_t target = targets[row];
  Sums a{-INFINITY, 0.f, 0.f};
  float picked = 0.f;
  Key list = 0;
  for (int p = 0; p < parts; ++p) {
    const float* rec = records + (int64_t(p) * o.rows + row) * (4 + 2 * o.k);
    a = join(a, Sums{rec[0], rec[1], rec[2]});
    if (target >= p * vocab && target < (p + 1) * vocab) picked = rec[3];
    if (o.k) {
      const Key next = lane < o.k ? make_key(rec[4 + lane], unsigned(__float_as_int(rec[4 + o.k + lane]))) : 0;
      list = merge_warp(list, next);
    }
  }
  if (lane == 0) finish_row(o, row, a, picked, target, parts * vocab);
  if (lane < o.k) {
    o.top_value[int64_t(row) * o.k + lane] = top_logprob(value_of(list), a);
    o.top_id[int64_t(row) * o.k + lane] = index_of(list);
  }
}

// One CTA per `kUnroll` vectors of its threads along a row.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) score_bwd_kernel(const T* logits, int64_t ld, unsigned vocab,
                                                             const int64_t* targets, int64_t start,
                                                             int64_t vocab_total, const float* state, int rows,
                                                             const float* dlogprob, const float* dentropy, T* out,
                                                             int64_t ld_out, unsigned blocks) {
  constexpr int kN = Vec<T>::kN;
  // The last rows first: they are what the forward pass, just before this one in most
  // programs, left in L2.
  const unsigned place = blockIdx.x / blocks, block = blockIdx.x - place * blocks;
  const int row = rows - 1 - int(place);
  const float m = state[row], ln_s = state[rows + row], H = state[2 * int64_t(rows) + row];
  const int64_t target = targets[row];
  float a = target >= 0 ? dlogprob[row] : 0.f;
  const float b = dentropy ? dentropy[row] : 0.f;
  if (target >= vocab_total || m != m) a = __int_as_float(0x7fffffff);
  // Without a gradient: a row that the mask emptied, and one that is not scored, whatever
  // its logits hold (`gradient` lifts NaN to kLowest, so that zero factors give zeros).
  const bool empty = m == -INFINITY || (target < 0 && b == 0.f);
  const int64_t local = target - start;
  const unsigned at = local >= 0 && local < vocab ? unsigned(local) : 0xffffffffu;
  // -p (a + b (l + H)) as p (c0 + c1 l), l = ln p.
  const float c1 = empty ? 0.f : -b, c0 = empty ? 0.f : -a - b * H;
  auto gradient = [&](float z, unsigned i) {
    const float l = fmaxf((z - m) - ln_s, kLowest);
    const float g = fast_exp2(l * kLog2e) * fmaf(c1, l, c0);
    return i == at && !empty ? g + a : g;
  };
  const Two minus_m = two(-m, -m), minus_ln_s = two(-ln_s, -ln_s), scale = two(kLog2e, kLog2e);
  const Two c0s = two(c0, c0), c1s = two(c1, c1);
  auto gradients = [&](Two z) {
    const float2 d = both(two_add(two_add(z, minus_m), minus_ln_s));
    const Two l = two(fmaxf(d.x, kLowest), fmaxf(d.y, kLowest));
    const float2 t = both(two_mul(l, scale));
    return two_mul(two(fast_exp2(t.x), fast_exp2(t.y)), two_fma(c1s, l, c0s));
  };
  const T* x = logits + int64_t(row) * ld;
  T* y = out + int64_t(row) * ld_out;
  if (VEC) {  // both rows are off a 16-byte boundary by the same amount
    const Part<T> part(x, 0, vocab);
    Vec<T> vec[kUnroll];
    const unsigned j0 = block * (kUnroll * kThreads) + threadIdx.x;
#pragma unroll
    for (int i = 0; i < kUnroll; ++i)
      if (j0 + i * kThreads < part.vectors) vec[i].load(x + part.vector_at(j0 + i * kThreads));
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const unsigned j = j0 + i * kThreads;
      if (j >= part.vectors) break;
      const unsigned c = part.vector_at(j);
      float v[kN];
      vec[i].get(v);
      T* h = reinterpret_cast<T*>(&vec[i].raw);
#pragma unroll
      for (int e = 0; e < kN; e += 2) {
        const float2 g = both(gradients(two(v[e], v[e + 1])));
        h[e] = from_float<T>(g.x);
        h[e + 1] = from_float<T>(g.y);
      }
      if (at - c < unsigned(kN)) {  // the given token's own vector
#pragma unroll
        for (int e = 0; e < kN; ++e)
          if (c + e == at) h[e] = from_float<T>(gradient(v[e], at));
      }
      *reinterpret_cast<uint4*>(y + c) = vec[i].raw;
    }
    if (block == 0 && threadIdx.x < part.head + part.tail) {
      const unsigned c = threadIdx.x < part.head ? threadIdx.x
                                                 : part.vector_at(part.vectors) + (threadIdx.x - part.head);
      y[c] = from_float<T>(gradient(to_float(x[c]), c));
    }
  } else {
    const unsigned c0 = block * (kUnroll * kThreads * kN) + threadIdx.x;
#pragma unroll 4
    for (int i = 0; i < kUnroll * kN; ++i) {
      const unsigned c = c0 + i * kThreads;
      if (c < vocab) y[c] = from_float<T>(gradient(to_float(x[c]), c));
    }
  }
}

template <typename T, bool TOP, int NT>
int launch_score(const void* logits, int64_t ld, unsigned vocab, const int64_t* targets, int64_t start,
                 int64_t vocab_total, const Out& o, unsigned C, cudaStream_t s) {
  const unsigned step = Vec<T>::kN;  // every part is off a 16-byte boundary by what the row is
  const unsigned chunk = C == 1 ? vocab : ((vocab + C - 1) / C + step - 1) / step * step;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(unsigned(o.rows) * C);
  config.blockDim = dim3(NT);
  config.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  config.attrs = attr;
  config.numAttrs = C > 1 ? 1 : 0;
  return int(cudaLaunchKernelEx(&config, score_kernel<T, TOP, NT>, static_cast<const T*>(logits), ld, vocab, targets,
                                start, vocab_total, chunk, o));
}
template <typename T, int NT>
int score_threads(const void* logits, int64_t ld, unsigned vocab, const int64_t* targets, int64_t start,
                  int64_t vocab_total, const Out& o, unsigned C, cudaStream_t s) {
  return o.k ? launch_score<T, true, NT>(logits, ld, vocab, targets, start, vocab_total, o, C, s)
             : launch_score<T, false, NT>(logits, ld, vocab, targets, start, vocab_total, o, C, s);
}
template <typename T>
int score_typed(const void* logits, int64_t ld, unsigned vocab, const int64_t* targets, int64_t start,
                int64_t vocab_total, const Out& o, cudaStream_t s) {
  // A row is split over a cluster while the rows alone leave SMs idle: 1 row of 50304 takes
  // 9.5 us on four CTAs and 11.6 us on one, 8192 rows 226 us on two each and 150 us on one.
  // In between no split was compared; one CTA each takes 12.1 us for 128 rows and 20.0 us
  // for 592, with 8 alternatives.
  unsigned C = 1;
  while (C < 4 && int64_t(o.rows) * C * 2 <= 148 && vocab / (2 * C) >= 4096) C *= 2;
  // Threads of a row's CTA: what a row costs beside its loads (joining the threads' sums
  // and lists) grows with them, its latency falls.  Many rows take one for every twenty
  // or so vectors, and four for every alternative, so that few candidates pass the bound.
  // 8192 BF16 rows, 8 alternatives: 64 threads 42 us and 256 threads 76 us at 6288 columns,
  // 227 and 161 us at 50304.
  int nt = 256;
  if (o.rows > 148 * 4) {
    const unsigned vectors = vocab / Vec<T>::kN;
    while (nt > 64 && vectors < unsigned(nt) * 20 && nt / 2 >= 4 * o.k) nt /= 2;
  }
  if (nt == 64) return score_threads<T, 64>(logits, ld, vocab, targets, start, vocab_total, o, C, s);
  if (nt == 128) return score_threads<T, 128>(logits, ld, vocab, targets, start, vocab_total, o, C, s);
  return score_threads<T, 256>(logits, ld, vocab, targets, start, vocab_total, o, C, s);
}
template <typename T>
int score_bwd_typed(const void* logits, int64_t ld, int rows, unsigned vocab, const int64_t* targets, int64_t start,
                    int64_t vocab_total, const float* state, const float* dlogprob, const float* dentropy, void* out,
                    int64_t ld_out, cudaStream_t s) {
  constexpr int64_t kE = sizeof(T), kN = Vec<T>::kN;
  const unsigned span = kThreads * kUnroll * unsigned(kN);
  const unsigned blocks = (vocab + span - 1) / span;
  if (int64_t(rows) * blocks > 0x7fffffff) return -1;
  const uintptr_t a = reinterpret_cast<uintptr_t>(logits), b = reinterpret_cast<uintptr_t>(out);
  const bool vec = (a & 15) == (b & 15) && ((ld - ld_out) * kE) % 16 == 0;
  auto launch = [&](auto kernel) {
    kernel<<<unsigned(rows) * blocks, kThreads, 0, s>>>(static_cast<const T*>(logits), ld, vocab, targets, start,
                                                        vocab_total, state, rows, dlogprob, dentropy,
                                                        static_cast<T*>(out), ld_out, blocks);
  };
  vec ? launch(score_bwd_kernel<T, true>) : launch(score_bwd_kernel<T, false>);
  return int(cudaGetLastError());
}
bool sizes_fit(int64_t rows, int64_t vocab, int64_t vocab_total) {
  // Ids travel as 32-bit integers; a launch has a CTA for each row, or 148 in clusters.
  return rows > 0 && vocab > 0 && rows <= 0x7fffffff / 8 && vocab_total <= 0x7fffffff;
}
}  // namespace

int score_fwd(const void* logits, int type, int64_t ld, int64_t rows, int64_t vocab, const int64_t* targets,
              int64_t start, int64_t vocab_total, int k, float* logprob, float* entropy, float* state,
              float* top_value, int64_t* top_id, float* record, cudaStream_t s) {
  if (!sizes_fit(rows, vocab, vocab_total) || k < 0 || k > kMaxTop || k > vocab) return -1;
  const Out o{logprob, entropy, state, top_value, top_id, record, int(rows), k};
  const unsigned v = unsigned(vocab);
  if (type == kTypeBF16) return score_typed<__nv_bfloat16>(logits, ld, v, targets, start, vocab_total, o, s);
  if (type == kTypeFP16) return score_typed<__half>(logits, ld, v, targets, start, vocab_total, o, s);
  if (type == kTypeFP32) return score_typed<float>(logits, ld, v, targets, start, vocab_total, o, s);
  return -1;
}
int score_merge(const float* records, int parts, int64_t rows, int64_t vocab, const int64_t* targets, int k,
                float* logprob, float* entropy, float* state, float* top_value, int64_t* top_id, cudaStream_t s) {
  if (!sizes_fit(rows, vocab, parts * vocab) || parts < 1 || k < 0 || k > kMaxTop) return -1;
  const Out o{logprob, entropy, state, top_value, top_id, nullptr, int(rows), k};
  score_merge_kernel<<<unsigned((rows + kWarps - 1) / kWarps), kThreads, 0, s>>>(records, parts, vocab, targets, o);
  return int(cudaGetLastError());
}
int score_bwd(const void* logits, int type, int64_t ld, int64_t rows, int64_t vocab, const int64_t* targets,
              int64_t start, int64_t vocab_total, const float* state, const float* dlogprob, const float* dentropy,
              void* out, int64_t ld_out, cudaStream_t s) {
  if (!sizes_fit(rows, vocab, vocab_total)) return -1;
  const unsigned v = unsigned(vocab);
  const int r = int(rows);
  if (type == kTypeBF16)
    return score_bwd_typed<__nv_bfloat16>(logits, ld, r, v, targets, start, vocab_total, state, dlogprob, dentropy,
                                          out, ld_out, s);
  if (type == kTypeFP16)
    return score_bwd_typed<__half>(logits, ld, r, v, targets, start, vocab_total, state, dlogprob, dentropy, out,
                                   ld_out, s);
  if (type == kTypeFP32)
    return score_bwd_typed<float>(logits, ld, r, v, targets, start, vocab_total, state, dlogprob, dentropy, out,
                                  ld_out, s);
  return -1;
}

}  // namespace kernels
}  // namespace tn5b
