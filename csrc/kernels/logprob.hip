// Log probabilities of given tokens, entropy and most probable tokens of rows of logits, and the
// gradient of all three.
//
//   lse = log sum_j e^{x_j}      logp = x_t - lse      H = lse - sum_j p_j x_j,  p_j = e^{x_j - lse}
//   dx_j = [j = t] g_logp + sum_i [j = top_i] g_i - p_j (g_logp + sum_i g_i) - g_H p_j (log p_j + H)
//
// Forward: one pass over the row with the running maximum m, S = sum e^{x - m} and
// U = sum e^{x - m} (x - m); two partial results join as
//   S = sum_i S_i e^{m_i - m},   U = sum_i e^{m_i - m} (U_i + (m_i - m) S_i),
// and H = log S - U / S.  Exponentials are taken in base 2; U is kept in base-2 units.
//
// The n largest need no second pass over the row: each thread's largest element is a sample, and
// the n-th largest sample, T, is a lower bound of the n-th largest element.  Only the n threads
// whose sample is at least T can hold an element above it; their elements alone are read again,
// from the cache, and those of at least T (n and a few) are ranked.  Elements compare as one
// 64-bit key of value and index, so equal values go to the lowest index, whatever their number.
//
// A token outside [0, V) or equal to `ignored` leaves its row unread: zeros, and -1 as top ids.
// A row of -inf alone has logp -inf, entropy 0 and no gradient.
#include "common.h"

namespace hetu {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr int kLpThreads = 256;      // a block a row
constexpr int kMaxTop = 64;
constexpr int kCand = 1024;          // candidate keys kept in LDS; more take the slow way

struct Lse { float m, s, u; };       // running maximum, sum, base-2 weighted sum

__device__ __forceinline__ float shift_of(float m) { return m == -INFINITY ? 0.f : m; }

// base-2 exponent's floor in products e * t: e is 0 there, and t may be -inf
constexpr float kFloor2 = -200.f;

__device__ __forceinline__ Lse lse_join(const Lse& a, const Lse& b) {
  Lse r;
  r.m = fmaxf(a.m, b.m);
  const float sh = shift_of(r.m);
  const float da = (a.m - sh) * kLog2e, db = (b.m - sh) * kLog2e;
  const float ea = exp2f(da), eb = exp2f(db);
  r.s = a.s * ea + b.s * eb;
  r.u = ea * (a.u + fmaxf(da, kFloor2) * a.s) + eb * (b.u + fmaxf(db, kFloor2) * b.s);
  return r;
}

// A row of V elements as 16-byte granules from the aligned address at or below its start:
// granule j holds elements j * VE - off + (0 .. VE - 1), of which the first and the last granule
// may lack some.
template <typename T>
struct Row {
  static constexpr int VE = Vec<T>::N;
  const T* x;
  int V, off, ng;
  __device__ __forceinline__ Row(const T* x_, int V_) : x(x_), V(V_) {
    off = (int)(((uintptr_t)x & 15) / sizeof(T));
    ng = (int)(((int64_t)off + V + VE - 1) / VE);
  }
  __device__ __forceinline__ bool full(int j) const {
    const int64_t e0 = (int64_t)j * VE - off;
    return e0 >= 0 && e0 + VE <= V;
  }
  // elements of granule j, -inf where the row has none
  __device__ __forceinline__ void load(int j, float (&v)[VE]) const {
    const int64_t e0 = (int64_t)j * VE - off;
    if (e0 >= 0 && e0 + VE <= V) {
      load_vec<T>(x + e0, v);
    } else {
#pragma unroll
      for (int k = 0; k < VE; ++k) v[k] = (e0 + k >= 0 && e0 + k < V) ? to_f(x[e0 + k]) : -INFINITY;
    }
  }
};

// value (larger first) and index (smaller first) as one number; NaN orders as -inf
__device__ __forceinline__ uint64_t key_of(float v, int e) {
  v = v != v ? -INFINITY : v + 0.f;                      // -0 is 0
  const unsigned b = __float_as_uint(v);
  const unsigned o = b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
  return ((uint64_t)o << 32) | (unsigned)~e;
}
__device__ __forceinline__ float key_value(uint64_t key) {
  const unsigned o = (unsigned)(key >> 32);
  return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ int key_index(uint64_t key) { return (int)~(unsigned)key; }

template <typename T>
__global__ void __launch_bounds__(kLpThreads) token_logprob_k(const T* __restrict__ logits, int64_t stride,
                                                              const int64_t* __restrict__ ids, int V, int n,
                                                              int64_t ignored, float* __restrict__ out,
                                                              float* __restrict__ stats, int64_t* __restrict__ top) {
  constexpr int NT = kLpThreads, VE = Vec<T>::N;
  __shared__ Lse part[NT / 64];
  __shared__ uint64_t keys[NT], cand[kCand], bound;
  __shared__ int flagged[NT], n_flagged, n_cand;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  const int64_t t = ids[row];
  float* o = out + row * (2 + n);
  if (t < 0 || t >= V || t == ignored) {
    for (int i = tid; i < 2 + n; i += NT) o[i] = 0.f;
    for (int i = tid; i < n; i += NT) top[row * n + i] = -1;
    if (tid < 2) stats[row * 2 + tid] = 0.f;
    return;
  }
  const Row<T> r(logits + row * stride, V);
  Lse a = {-INFINITY, 0.f, 0.f};
  int best = tid;
  for (int j = tid; j < r.ng; j += NT) {
    float v[VE];
    r.load(j, v);
    float vm = v[0];
#pragma unroll
    for (int k = 1; k < VE; ++k) vm = fmaxf(vm, v[k]);
    if (vm > a.m) best = j;
    Lse b = {fmaxf(a.m, vm), 0.f, 0.f};
    const float sh = shift_of(b.m);
#pragma unroll
    for (int k = 0; k < VE; ++k) {
      const float d = (v[k] - sh) * kLog2e, e = exp2f(d);
      b.s += e;
      b.u += e * fmaxf(d, kFloor2);
    }
    const float da = (a.m - sh) * kLog2e, ea = exp2f(da);
    a.u = ea * (a.u + fmaxf(da, kFloor2) * a.s) + b.u;
    a.s = a.s * ea + b.s;
    a.m = b.m;
  }
  // this thread's largest element, for the selection below
  uint64_t mine = 0;
  if (n > 0 && tid < r.ng) {
    float v[VE];
    r.load(best, v);
    const int e0 = best * VE - r.off;
#pragma unroll
    for (int k = 0; k < VE; ++k) {
      const uint64_t key = key_of(v[k], e0 + k);
      if (e0 + k >= 0 && e0 + k < V && key > mine) mine = key;
    }
  }
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) {
    const Lse b = {__shfl_xor(a.m, s, 64), __shfl_xor(a.s, s, 64), __shfl_xor(a.u, s, 64)};
    a = lse_join(a, b);
  }
  if ((tid & 63) == 0) part[tid >> 6] = a;
  if (n > 0) keys[tid] = mine;
  if (tid == 0) { bound = 0; n_flagged = 0; n_cand = 0; }
  __syncthreads();
  a = part[0];
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) a = lse_join(a, part[w]);
  const bool empty = a.m == -INFINITY && a.s == 0.f;
  const float log2s = log2f(a.s), logs = log2s * kLn2;
  if (tid == 0) {
    const float xt = to_f(r.x[t]);
    o[0] = empty ? -INFINITY : (xt - a.m) - logs;
    o[1] = empty ? 0.f : (log2s - a.u / a.s) * kLn2;
    stats[row * 2] = a.m;
    stats[row * 2 + 1] = log2s;
  }
  if (n == 0) return;
  int rank = 0;
  for (int i = 0; i < NT; ++i) rank += keys[i] > mine;
  if (mine != 0 && rank == n - 1) bound = mine;
  __syncthreads();
  const uint64_t least = bound;          // 0 where fewer than n threads have an element: all are candidates
  if (mine != 0 && mine >= least) flagged[atomicAdd(&n_flagged, 1)] = tid;
  __syncthreads();
  const int J = (r.ng + NT - 1) / NT, todo = n_flagged * J;
  for (int i = tid; i < todo; i += NT) {
    const int j = (i % J) * NT + flagged[i / J];
    if (j >= r.ng) continue;
    float v[VE];
    r.load(j, v);
    const int e0 = j * VE - r.off;
#pragma unroll
    for (int k = 0; k < VE; ++k) {
      const uint64_t key = key_of(v[k], e0 + k);
      if (e0 + k >= 0 && e0 + k < V && key >= least) {
        const int at = atomicAdd(&n_cand, 1);
        if (at < kCand) cand[at] = key;
      }
    }
  }
  __syncthreads();
  const int C = n_cand;
  if (C <= kCand) {
    for (int c = tid; c < C; c += NT) {
      const uint64_t key = cand[c];
      int at = 0;
      for (int i = 0; i < C; ++i) at += cand[i] > key;
      if (at < n) {
        o[2 + at] = empty ? -INFINITY : (key_value(key) - a.m) - logs;
        top[row * n + at] = key_index(key);
      }
    }
    return;
  }
  // many elements of few threads above the bound: n rounds of the largest below the last one
  uint64_t last = ~0ull;
  for (int i = 0; i < n; ++i) {
    uint64_t most = 0;
    if (mine != 0 && mine >= least) {
      for (int j = tid; j < r.ng; j += NT) {
        float v[VE];
        r.load(j, v);
        const int e0 = j * VE - r.off;
#pragma unroll
        for (int k = 0; k < VE; ++k) {
          const uint64_t key = key_of(v[k], e0 + k);
          if (e0 + k >= 0 && e0 + k < V && key < last && key > most) most = key;
        }
      }
    }
    __syncthreads();
    keys[tid] = most;
    __syncthreads();
    most = 0;
    for (int k = 0; k < NT; ++k) most = keys[k] > most ? keys[k] : most;
    last = most;
    if (tid == 0) {
      o[2 + i] = empty ? -INFINITY : (key_value(most) - a.m) - logs;
      top[row * n + i] = key_index(most);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads) token_logprob_bwd_k(const T* __restrict__ logits, int64_t stride,
                                                                  const int64_t* __restrict__ ids, int V, int n,
                                                                  int64_t ignored, const float* __restrict__ out,
                                                                  const float* __restrict__ stats,
                                                                  const int64_t* __restrict__ top,
                                                                  const float* __restrict__ grad, T* __restrict__ dx) {
  constexpr int NT = kLpThreads, VE = Vec<T>::N;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  const int64_t t = ids[row];
  T* d = dx + row * (int64_t)V;
  const float m = stats[row * 2], log2s = stats[row * 2 + 1];
  const bool dead = t < 0 || t >= V || t == ignored || (m == -INFINITY && log2s == -INFINITY);
  const Row<T> r(logits + row * stride, V), w(d, V);
  const float* g = grad + row * (2 + n);
  float all = 0.f, gh = 0.f, h = 0.f;
  if (!dead) {
    all = g[0];
    for (int i = 0; i < n; ++i) all += g[2 + i];
    gh = g[1] * kLn2;
    h = out[row * (2 + n) + 1];
    all += g[1] * h;
  }
  const float sh = shift_of(m);
  const auto slope = [&](float x) {
    const float l = (x - sh) * kLog2e - log2s;
    return -exp2f(l) * (all + gh * fmaxf(l, kFloor2));
  };
  if (r.off == w.off) {
    for (int j = tid; j < w.ng; j += NT) {
      float v[VE];
      if (!dead) {
        r.load(j, v);
#pragma unroll
        for (int k = 0; k < VE; ++k) v[k] = slope(v[k]);
      } else {
#pragma unroll
        for (int k = 0; k < VE; ++k) v[k] = 0.f;
      }
      const int64_t e0 = (int64_t)j * VE - w.off;
      if (w.full(j)) {
        store_vec<T>(d + e0, v);
      } else {
#pragma unroll
        for (int k = 0; k < VE; ++k)
          if (e0 + k >= 0 && e0 + k < V) d[e0 + k] = from_f<T>(v[k]);
      }
    }
  } else {
    for (int e = tid; e < V; e += NT) d[e] = from_f<T>(dead ? 0.f : slope(to_f(r.x[e])));
  }
  if (dead) return;
  // the given token and the alternatives once more, each with its own terms: rounded once
  __syncthreads();
  for (int i = tid; i <= n; i += NT) {
    const int64_t e = i == 0 ? t : top[row * n + i - 1];
    if (e < 0 || e >= V) continue;
    float s = slope(to_f(r.x[e]));
    if (e == t) s += g[0];
    for (int k = 0; k < n; ++k)
      if (top[row * n + k] == e) s += g[2 + k];
    d[e] = from_f<T>(s);
  }
}

}  // namespace hetu

using namespace hetu;

HETU_API int hetu_token_logprob(const void* logits, int64_t stride, const int64_t* ids, int64_t R, int V, int n,
                                int64_t ignored, float* out, float* stats, int64_t* top, int is_bf16,
                                hipStream_t st) {
  if (R <= 0) return 0;
  if (V < 1 || n < 0 || n > kMaxTop || n > V || R > 0x7fffffff) return (int)hipErrorInvalidValue;
  const dim3 grid((unsigned)R), block(kLpThreads);
  if (is_bf16)
    hipLaunchKernelGGL(token_logprob_k<bf16>, grid, block, 0, st, (const bf16*)logits, stride, ids, V, n, ignored, out, stats, top);
  else
    hipLaunchKernelGGL(token_logprob_k<float>, grid, block, 0, st, (const float*)logits, stride, ids, V, n, ignored, out, stats, top);
  HETU_LAUNCH_CHECK();
  return 0;
}

HETU_API int hetu_token_logprob_bwd(const void* logits, int64_t stride, const int64_t* ids, int64_t R, int V, int n,
                                    int64_t ignored, const float* out, const float* stats, const int64_t* top,
                                    const float* grad, void* dx, int is_bf16, hipStream_t st) {
  if (R <= 0) return 0;
  if (V < 1 || n < 0 || n > kMaxTop || n > V || R > 0x7fffffff) return (int)hipErrorInvalidValue;
  const dim3 grid((unsigned)R), block(kLpThreads);
  if (is_bf16)
    hipLaunchKernelGGL(token_logprob_bwd_k<bf16>, grid, block, 0, st, (const bf16*)logits, stride, ids, V, n, ignored, out, stats, top, grad, (bf16*)dx);
  else
    hipLaunchKernelGGL(token_logprob_bwd_k<float>, grid, block, 0, st, (const float*)logits, stride, ids, V, n, ignored, out, stats, top, grad, (float*)dx);
  HETU_LAUNCH_CHECK();
  return 0;
}
