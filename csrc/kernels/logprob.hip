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
// from the cache, and those of at least T (n and a few, where few values tie) are ranked.  Elements
// compare as one 64-bit key of value and index, so equal values go to the lowest index, whatever
// their number (the samples as a key of value and granule: a bound on elements all the same).  A row
// most of whose values tie, or with fewer tokens above -inf than alternatives, has more at the bound:
// of bf16 rows of 32 KB and more and from 33 alternatives, where four threads share a sample, up to
// 8 (4 (n - 1) + 1), which the list does not hold.  Such a row is read n times (502 x 131072 bf16, 10
// tokens above -inf: top 32 70 us, top 64 1.9 ms, and 43 us without a mask).
//
// A token outside [0, V) or equal to `ignored` leaves its row unread: zeros, and -1 as top ids.
// A row of -inf alone has logp -inf, entropy 0 and no gradient.
#include "wave_ops.h"

namespace hetu {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr int kMaxTop = 64;

// A launch holds fewer than 2^32 threads along x: more blocks than kRowOfBlocks go along y too.
constexpr int64_t kRowOfBlocks = 1 << 20;
constexpr int64_t kMaxBlocks = kRowOfBlocks * 65535;
static dim3 many_blocks(int64_t n) {
  return n <= kRowOfBlocks ? dim3((unsigned)n) : dim3((unsigned)kRowOfBlocks, (unsigned)((n + kRowOfBlocks - 1) / kRowOfBlocks));
}
__device__ __forceinline__ int64_t block_number() { return (int64_t)blockIdx.y * kRowOfBlocks + blockIdx.x; }

struct Lse { float m, s, u; };       // running maximum, sum, base-2 weighted sum

__device__ __forceinline__ float shift_of(float m) { return m == -INFINITY ? 0.f : m; }

// base-2 exponent's floor in products e * t: e is 0 there, and t may be -inf
constexpr float kFloor2 = -200.f;

// v_exp_f32: results below 2^-126 are 0, which sums of at least 1 do not feel
__device__ __forceinline__ float exp2_(float t) { return __builtin_amdgcn_exp2f(t); }

// joins the results of G lanes (aligned, a power of two): the largest first, then two plain sums
__device__ __forceinline__ Lse lse_join(Lse a, int G) {
#pragma clang fp contract(off)   // a product fused into one lane's sum would leave the lanes unequal
  Lse r;
  r.m = group_max(a.m, G);
  const float d = (a.m - shift_of(r.m)) * kLog2e, e = exp2_(d);
  r.s = group_sum(a.s * e, G);
  r.u = group_sum(e * (a.u + fmaxf(d, kFloor2) * a.s), G);
  return r;
}

__device__ __forceinline__ void unpack(const Raw& q, float (&v)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = __uint_as_float(q[k]);
}
__device__ __forceinline__ void unpack(const Raw& q, float (&v)[8]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    v[2 * k] = __uint_as_float(q[k] << 16);
    v[2 * k + 1] = __uint_as_float(q[k] & 0xffff0000u);
  }
}

// A row of V elements as 16-byte granules from the aligned address at or below its start:
// granule j holds elements j * VE - off + (0 .. VE - 1), of which the first and the last granule
// may lack some.
template <typename T>
struct Row {
  static constexpr int VE = Vec<T>::N;
  const T* x;
  int V, off, ng, f0, f1;      // granules 0 .. ng - 1; those of f0 .. f1 - 1 are whole
  __device__ __forceinline__ Row(const T* x_, int V_) : x(x_), V(V_) {
    off = (int)(((uintptr_t)x & 15) / sizeof(T));
    ng = (int)(((int64_t)off + V + VE - 1) / VE);
    f0 = off ? 1 : 0;
    f1 = (int)(((int64_t)off + V) / VE);
  }
  __device__ __forceinline__ bool has_head() const { return f0 > 0; }
  __device__ __forceinline__ bool has_tail() const { return f1 < ng && ng - 1 >= f0; }
  // a whole granule as it is in memory
  __device__ __forceinline__ Raw raw(int j) const {
    return *reinterpret_cast<const Raw*>(x - off + (int64_t)j * VE);
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

// value (larger first) and index (smaller first) as one number, never 0; NaN orders as -inf
__device__ __forceinline__ unsigned order_of(float v) {
  v = v != v ? -INFINITY : v + 0.f;                      // -0 is 0
  const unsigned b = __float_as_uint(v);
  return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ uint64_t key_of(float v, int e) { return ((uint64_t)order_of(v) << 32) | (unsigned)~e; }
__device__ __forceinline__ float key_value(uint64_t key) {
  const unsigned o = (unsigned)(key >> 32);
  return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ int key_index(uint64_t key) { return (int)~(unsigned)key; }

// A bound that n of the wave's keys k reach and, but for fewer keys than n (then 0), no more: found
// two bits at a time from the highest that differs, first by the values (of which LOW bits are the
// same in a sign: bf16), then where they tie by the low words, ~0 .. ~(limit - 1).
template <int Q, int LOW>
__device__ __forceinline__ uint64_t nth_bound(const uint64_t (&k)[Q], int n, unsigned limit) {
  unsigned hi[Q], most = 0, least = ~0u;
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    hi[q] = (unsigned)(k[q] >> 32);
    most = most > hi[q] ? most : hi[q];
    least = least < hi[q] ? least : hi[q];
  }
  most = group_join(most, 64, [](unsigned a, unsigned b) { return a > b ? a : b; });
  least = group_join(least, 64, [](unsigned a, unsigned b) { return a < b ? a : b; });
  most = (unsigned)__builtin_amdgcn_readfirstlane((int)most);       // (uniform: in scalar registers)
  least = (unsigned)__builtin_amdgcn_readfirstlane((int)least);
  const unsigned differ = most ^ least;
  int at = differ ? (31 - __builtin_clz(differ)) & ~1 : -2, reach = -1;
  unsigned b = differ ? (most >> at >> 2) << at << 2 | ((most & least) & (2u << at)) : most;
  for (; at >= LOW && reach != n; at -= 2) {
    const unsigned c1 = b | 1u << at, c2 = b | 2u << at, c3 = b | 3u << at;
    int r1 = 0, r2 = 0, r3 = 0;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      r1 += __popcll(__ballot(hi[q] >= c1));
      r2 += __popcll(__ballot(hi[q] >= c2));
      r3 += __popcll(__ballot(hi[q] >= c3));
    }
    if (r3 >= n) b = c3, reach = r3;
    else if (r2 >= n) b = c2, reach = r2;
    else if (r1 >= n) b = c1, reach = r1;
  }
  if (reach == n) return (uint64_t)b << 32;
  if (LOW && !(b >> 31)) b |= (1u << LOW) - 1;       // below 0 the same bits are ones
  at = (31 - __builtin_clz(limit | 1)) & ~1;
  uint64_t w = (uint64_t)b << 32 | (at >= 30 ? 0u : ~0u << at << 2);
  for (; at >= 0 && reach != n; at -= 2) {
    const uint64_t c1 = w | 1u << at, c2 = w | 2u << at, c3 = w | 3u << at;
    int r1 = 0, r2 = 0, r3 = 0;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      r1 += __popcll(__ballot(k[q] >= c1));
      r2 += __popcll(__ballot(k[q] >= c2));
      r3 += __popcll(__ballot(k[q] >= c3));
    }
    if (r3 >= n) w = c3, reach = r3;
    else if (r2 >= n) w = c2, reach = r2;
    else if (r1 >= n) w = c1, reach = r1;
  }
  return w;
}

// takes U granules v (numbers j, j + step, ..) into the running sums; `best`: the granule with the
// first of the largest values so far
template <int U, int VE, bool TOP>
__device__ __forceinline__ void lse_take(Lse& a, int& best, const float (&v)[U][VE], int j, int step) {
  float m = a.m;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float vm = v[u][0];
#pragma unroll
    for (int k = 1; k < VE; ++k) vm = fmaxf(vm, v[u][k]);
    if (TOP && (vm > m || best < 0)) best = j + u * step;
    m = fmaxf(m, vm);
  }
  const float sh = shift_of(m);
  float s = 0.f, w = 0.f;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int k = 0; k < VE; ++k) {
      const float d = (v[u][k] - sh) * kLog2e, e = exp2_(d);
      s += e;
      w += e * fmaxf(d, kFloor2);
    }
  const float da = (a.m - sh) * kLog2e, ea = exp2_(da);
  a.u = ea * (a.u + fmaxf(da, kFloor2) * a.s) + w;
  a.s = a.s * ea + s;
  a.m = m;
}

// One block of NT threads a row: thread i takes the whole granules f0 + i, f0 + i + NT, .., U of
// them under way at once; thread 0 the head and the last thread the tail that are not whole.
// (More than 80 scalar registers leave a SIMD 7 waves, and a CU one block of 1024 threads instead of
// two: 1000 x 131072 top 20 took 80 us instead of 62.)
template <typename T, int NT, bool TOP>
__attribute__((amdgpu_num_sgpr(80))) __global__ void __launch_bounds__(NT) token_logprob_k(const T* __restrict__ logits, int64_t stride,
                                                      const int64_t* __restrict__ ids, int64_t R, int V, int n,
                                                      int64_t ignored, float* __restrict__ out,
                                                      int64_t* __restrict__ top) {
  constexpr int VE = Vec<T>::N, U = 4, NW = NT / 64;
  constexpr int NG = TOP ? 256 : 1, PER = TOP ? NT / NG : 1;   // groups of threads that give a sample
  constexpr int CAND = 1024;                        // candidates kept in LDS; more take the slow way
  __shared__ Lse part[NW];
  __shared__ __align__(16) uint64_t cand[TOP ? CAND + 1 : 1];
  __shared__ uint64_t keys[NG], bound;
  __shared__ int flagged[NG], n_flagged, n_cand;
  const int tid = threadIdx.x;
  const int64_t row = block_number();
  if (row >= R) return;
  float* o = out + row * (4 + n);
  const Row<T> r(logits + row * stride, V);
  int j = r.f0 + tid;
  // with few rows the first loads do not wait for the token: one latency less
  const bool ahead = NT > 256 && j + (U - 1) * NT < r.f1;
  Raw q[U];
  if (ahead) {
#pragma unroll
    for (int u = 0; u < U; ++u) q[u] = r.raw(j + u * NT);
  }
  const int64_t t = ids[row];
  if (t < 0 || t >= V || t == ignored) {
    for (int i = tid; i < 4 + n; i += NT) o[i] = 0.f;
    for (int i = tid; i < n; i += NT) top[row * n + i] = -1;
    return;
  }
  const float xt = to_f(r.x[t]);
  Lse a = {-INFINITY, 0.f, 0.f};
  int best = -1;
  if (ahead) {
    float v[U][VE];
#pragma unroll
    for (int u = 0; u < U; ++u) unpack(q[u], v[u]);
    lse_take<U, VE, TOP>(a, best, v, j, NT);
    j += U * NT;
  }
  for (; j + (U - 1) * NT < r.f1; j += U * NT) {
    float v[U][VE];
#pragma unroll
    for (int u = 0; u < U; ++u) q[u] = r.raw(j + u * NT);
#pragma unroll
    for (int u = 0; u < U; ++u) unpack(q[u], v[u]);
    lse_take<U, VE, TOP>(a, best, v, j, NT);
  }
  if (j < r.f1) {                     // fewer than U are left: the others' places hold -inf
    float v[U - 1][VE];
#pragma unroll
    for (int u = 0; u < U - 1; ++u) q[u] = r.raw(j + u * NT < r.f1 ? j + u * NT : j);
#pragma unroll
    for (int u = 0; u < U - 1; ++u) {
      unpack(q[u], v[u]);
#pragma unroll
      for (int k = 0; k < VE; ++k) v[u][k] = j + u * NT < r.f1 ? v[u][k] : -INFINITY;
    }
    lse_take<U - 1, VE, TOP>(a, best, v, j, NT);
  }
  if (tid == 0 && r.has_head()) {
    float v[1][VE];
    r.load(0, v[0]);
    if (TOP) {                        // the row's first elements, taken last: where they tie, they are the sample
      float vm = -INFINITY;
#pragma unroll
      for (int k = 0; k < VE; ++k) vm = fmaxf(vm, v[0][k]);
      if (vm >= a.m) best = 0;
    }
    lse_take<1, VE, TOP>(a, best, v, 0, NT);
  }
  if (tid == NT - 1 && r.has_tail()) {
    float v[1][VE];
    r.load(r.ng - 1, v[0]);
    lse_take<1, VE, TOP>(a, best, v, r.ng - 1, NT);
  }
  uint64_t mine = 0;                  // this thread's sample; 0: it has no element
  if (TOP && best >= 0) mine = key_of(a.m, best);
  a = lse_join(a, 64);
  if ((tid & 63) == 0) part[tid >> 6] = a;
  if (TOP) {
#pragma unroll
    for (int s = 1; s < PER; s <<= 1) {
      const uint64_t other = __shfl_xor((unsigned long long)mine, s, 64);
      if (other > mine) mine = other;
    }
    if (tid % PER == 0) keys[tid / PER] = mine;
    if (tid == 0) { n_flagged = 0; n_cand = 0; }
  }
  __syncthreads();
  a = lse_join(part[tid & (NW - 1)], NW);
  const bool empty = a.m == -INFINITY && a.s == 0.f;
  const float log2s = log2f(a.s), logs = log2s * kLn2;
  if (tid == NT - 1) {
    o[0] = empty ? -INFINITY : (xt - a.m) - logs;
    o[1] = empty ? 0.f : (log2s - a.u / a.s) * kLn2;
    o[2 + n] = a.m;
    o[3 + n] = log2s;
  }
  if constexpr (TOP) {
    // the n-th largest sample (0 where fewer than n threads have an element: all are candidates)
    if (tid < 64) {
      uint64_t k[NG / 64];
#pragma unroll
      for (int q = 0; q < NG / 64; ++q) k[q] = keys[tid + q * 64];
      const uint64_t b = nth_bound<NG / 64, sizeof(T) == 2 ? 16 : 0>(k, n, r.ng);
      if (tid == 0) bound = b;
    }
    __syncthreads();
    const uint64_t least = bound;
    if (tid < NG && keys[tid] != 0 && keys[tid] >= least) flagged[atomicAdd(&n_flagged, 1)] = tid;
    __syncthreads();
    // granules of a flagged group: its threads' whole ones, then the head or tail that is theirs
    const int J = r.f1 > r.f0 ? (r.f1 - r.f0 + NT - 1) / NT * PER : 0;
    const int bits = 32 - __clz(J), todo = n_flagged << bits;      // J + 1 <= 1 << bits
    for (int i = tid; i < todo; i += NT) {
      const int f = flagged[i >> bits], jj = i & ((1 << bits) - 1);
      int j = r.f0 + (jj / PER) * NT + f * PER + jj % PER;
      if (jj == J) {
        if (f == 0 && r.has_head()) j = 0;
        else if (f == NG - 1 && r.has_tail()) j = r.ng - 1;
        else continue;
      } else if (jj > J || j >= r.f1) {
        continue;
      }
      float v[VE];
      r.load(j, v);
      const int e0 = j * VE - r.off;
#pragma unroll
      for (int k = 0; k < VE; ++k) {
        if (e0 + k >= 0 && e0 + k < V && key_of(v[k], j) >= least) {
          const int at = atomicAdd(&n_cand, 1);
          if (at < CAND) cand[at] = key_of(v[k], e0 + k);
        }
      }
    }
    __syncthreads();
    const int C = n_cand;
    if (C <= CAND) {
      if (C & 1) {                 // read in pairs
        if (tid == 0) cand[C] = 0;
        __syncthreads();
      }
      for (int c = tid; c < C; c += NT) {
        const uint64_t key = cand[c];
        int at = 0;
#pragma unroll 4
        for (int i = 0; i < C; i += 2) {
          const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(&cand[i]);
          at += (two.x > key) + (two.y > key);
        }
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
#pragma unroll
      for (int s = 32; s > 0; s >>= 1) {
        const uint64_t other = __shfl_xor((unsigned long long)most, s, 64);
        if (other > most) most = other;
      }
      __syncthreads();
      if ((tid & 63) == 0) keys[tid >> 6] = most;
      __syncthreads();
      for (int w = 0; w < NT / 64; ++w) most = keys[w] > most ? keys[w] : most;
      last = most;
      if (tid == 0) {
        o[2 + i] = empty ? -INFINITY : (key_value(most) - a.m) - logs;
        top[row * n + i] = key_index(most);
      }
    }
  }
}

// ---- rows of at most kShortBytes: a wave a row, held in registers ----------------------------
constexpr int kShortBytes = 4080, kShortGranules = 4;      // at most 256 granules with the head's: 4 a lane
constexpr int kShortWaves = 4;

// sorts one key a lane, the largest first
__device__ __forceinline__ uint64_t wave_sort(uint64_t key, int lane) {
#pragma unroll
  for (int size = 2; size <= 64; size <<= 1)
#pragma unroll
    for (int d = size >> 1; d > 0; d >>= 1) {
      const uint64_t other = __shfl_xor((unsigned long long)key, d, 64);
      const bool larger = ((lane & d) == 0) == ((lane & size) == 0);      // this lane keeps the larger one
      key = (key > other) == larger ? key : other;
    }
  return key;
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(kShortWaves * 64) token_logprob_short_k(const T* __restrict__ logits, int64_t stride,
                                                                          const int64_t* __restrict__ ids, int64_t R,
                                                                          int V, int n, int64_t ignored,
                                                                          float* __restrict__ out,
                                                                          int64_t* __restrict__ top) {
  constexpr int VE = Vec<T>::N, Q = kShortGranules, CAND = kMaxTop * VE, K = CAND / 64;
  __shared__ uint64_t found[kShortWaves][TOP ? CAND : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = block_number() * kShortWaves + wave;
  if (row >= R) return;
  float* o = out + row * (4 + n);
  const int64_t t = ids[row];
  if (t < 0 || t >= V || t == ignored) {
    for (int i = lane; i < 4 + n; i += 64) o[i] = 0.f;
    for (int i = lane; i < n; i += 64) top[row * n + i] = -1;
    return;
  }
  const Row<T> r(logits + row * stride, V);
  const float xt = to_f(r.x[t]);
  float v[Q][VE];
#pragma unroll
  for (int q = 0; q < Q; ++q) r.load(lane + 64 * q, v[q]);        // -inf beyond the row
  uint64_t k[Q];
  float m = -INFINITY;
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    float vm = v[q][0];
#pragma unroll
    for (int e = 1; e < VE; ++e) vm = fmaxf(vm, v[q][e]);
    if (TOP) k[q] = lane + 64 * q < r.ng ? key_of(vm, lane + 64 * q) : 0;
    m = fmaxf(m, vm);
  }
  Lse a = {group_max(m, 64), 0.f, 0.f};
  const float sh = shift_of(a.m);
#pragma unroll
  for (int q = 0; q < Q; ++q)
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const float d = (v[q][e] - sh) * kLog2e, x = exp2_(d);
      a.s += x;
      a.u += x * fmaxf(d, kFloor2);
    }
  a.s = group_sum(a.s, 64);
  a.u = group_sum(a.u, 64);
  const bool empty = a.m == -INFINITY && a.s == 0.f;
  const float log2s = log2f(a.s), logs = log2s * kLn2;
  if (lane == 0) {
    o[0] = empty ? -INFINITY : (xt - a.m) - logs;
    o[1] = empty ? 0.f : (log2s - a.u / a.s) * kLn2;
    o[2 + n] = a.m;
    o[3 + n] = log2s;
  }
  if constexpr (TOP) {
    // the granules of the n largest samples, or all where they are fewer: at most 64 VE elements
    const uint64_t least = nth_bound<Q, sizeof(T) == 2 ? 16 : 0>(k, n, r.ng), below = (1ull << lane) - 1;
    uint64_t* cand = found[wave];
    int C = 0;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int j = lane + 64 * q, e0 = j * VE - r.off;
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const bool in = k[q] != 0 && k[q] >= least && e0 + e >= 0 && e0 + e < V && key_of(v[q][e], j) >= least;
        const uint64_t mask = __ballot(in);
        if (in) cand[C + __popcll(mask & below)] = key_of(v[q][e], e0 + e);
        C += __popcll(mask);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    uint64_t key = 0;
    if (C <= 64) {
      if (lane < C) key = cand[lane];
    } else {                       // more than a wave sorts: the n largest of them
      uint64_t c[K];
#pragma unroll
      for (int i = 0; i < K; ++i) c[i] = lane + 64 * i < C ? cand[lane + 64 * i] : 0;
      const uint64_t bound = nth_bound<K, sizeof(T) == 2 ? 16 : 0>(c, n, V);
      __builtin_amdgcn_wave_barrier();
      int at = 0;
#pragma unroll
      for (int i = 0; i < K; ++i) {
        const bool in = c[i] != 0 && c[i] >= bound;
        const uint64_t mask = __ballot(in);
        if (in) cand[at + __popcll(mask & below)] = c[i];
        at += __popcll(mask);
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      if (lane < n) key = cand[lane];
    }
    key = wave_sort(key, lane);
    if (lane < n) {
      o[2 + lane] = empty ? -INFINITY : (key_value(key) - a.m) - logs;
      top[row * n + lane] = key_index(key);
    }
  }
}

// A block takes kBwdGranules granules of a row, the last row first: the logits that the forward
// pass read last are still in the last-level cache.  Bound by memory: 164 us at 8192 x 30522 bf16, 6.1 TB/s.
//   ST_PAST: the gradient goes past that cache (both passes 282 -> 242 us at 8192 x 30522 bf16, for
//            the next forward pass reads at 5.6 instead of 4 TB/s; 777 x 50021 fp32 89 -> 65 us).
//   LD_PAST: the logits too, where most of them cannot be there (this pass 354 -> 322 us at 4096 x
//            131072 bf16, 1 GB; at 8192 x 30522, half of that, 166 -> 176).
constexpr int kBwdThreads = 256, kBwdU = 4, kBwdGranules = kBwdThreads * kBwdU;

template <typename T, bool LD_PAST, bool ST_PAST>
__global__ void __launch_bounds__(kBwdThreads) token_logprob_bwd_k(const T* __restrict__ logits, int64_t stride,
                                                                   const int64_t* __restrict__ ids, int64_t R, int V,
                                                                   int n, int64_t ignored, int chunks,
                                                                   const float* __restrict__ out,
                                                                   const int64_t* __restrict__ top,
                                                                   const float* __restrict__ grad, T* __restrict__ dx) {
  constexpr int NT = kBwdThreads, VE = Vec<T>::N, U = kBwdU;
  const int tid = threadIdx.x;
  const int64_t at = R * chunks - 1 - block_number();
  if (at < 0) return;
  const int64_t row = at / chunks;
  const int chunk = (int)(at - row * chunks);
  const int64_t t = ids[row];
  T* d = dx + row * (int64_t)V;
  const float* o = out + row * (4 + n);
  const float m = o[2 + n], log2s = o[3 + n];
  const bool dead = t < 0 || t >= V || t == ignored || (m == -INFINITY && log2s == -INFINITY);
  const Row<T> r(logits + row * stride, V), w(d, V);
  const float* g = grad + row * (2 + n);
  float all = 0.f, gh = 0.f;
  if (!dead) {
    all = g[0];
    for (int i = 0; i < n; ++i) all += g[2 + i];
    gh = g[1] * kLn2;
    all += g[1] * o[1];
  }
  const float sh = shift_of(m);
  const auto slope = [&](float x) {
    const float l = (x - sh) * kLog2e - log2s;
    return -exp2_(l) * (all + gh * fmaxf(l, kFloor2));
  };
  const int j0 = chunk * kBwdGranules, j1 = j0 + kBwdGranules < w.ng ? j0 + kBwdGranules : w.ng;
  const auto take = [&](int j) {       // one granule, whole or not
    float v[VE];
    const int64_t e0 = (int64_t)j * VE - w.off;
    if (dead) {
#pragma unroll
      for (int k = 0; k < VE; ++k) v[k] = 0.f;
    } else {
      r.load(j, v);
#pragma unroll
      for (int k = 0; k < VE; ++k) v[k] = slope(v[k]);
    }
    if (j >= w.f0 && j < w.f1) {
      store_raw<ST_PAST>(d + e0, pack_raw(v));
    } else {
#pragma unroll
      for (int k = 0; k < VE; ++k)
        if (e0 + k >= 0 && e0 + k < V) d[e0 + k] = from_f<T>(v[k]);
    }
  };
  if (dead) {
    for (int j = j0 + tid; j < j1; j += NT) take(j);
  } else if (r.off == w.off) {
    const int a0 = j0 < w.f0 ? w.f0 : j0, a1 = j1 < w.f1 ? j1 : w.f1;
    int j = a0 + tid;
    for (; j + (U - 1) * NT < a1; j += U * NT) {
      Raw q[U];
#pragma unroll
      for (int u = 0; u < U; ++u) q[u] = load_raw<LD_PAST>(r.x - r.off + (int64_t)(j + u * NT) * VE);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float v[VE];
        unpack(q[u], v);
#pragma unroll
        for (int k = 0; k < VE; ++k) v[k] = slope(v[k]);
        store_raw<ST_PAST>(d + (int64_t)(j + u * NT) * VE - w.off, pack_raw(v));
      }
    }
    for (; j < a1; j += NT) take(j);
    // (the tail to the chunk that holds it, whose block writes the tokens below too: the last chunk may
    // be empty)
    if (tid == 0 && j0 == 0 && w.has_head()) take(0);
    if (tid == NT - 1 && w.ng - 1 >= j0 && w.ng - 1 < j1 && w.has_tail()) take(w.ng - 1);
  } else {         // rows of another alignment than the gradient's
    const int a0 = j0 * VE - w.off, b0 = a0 < 0 ? 0 : a0;                       // (b0 + NT may pass 32 bits, the count not)
    const int64_t a1 = (int64_t)j1 * VE - w.off;
    const int count = (int)(a1 < V ? a1 : V) - b0;
    const T* xs = r.x + b0;
    T* ds = d + b0;
    for (int e = tid; e < count; e += NT) ds[e] = from_f<T>(slope(to_f(xs[e])));
  }
  if (dead) return;
  // this chunk's part of the given token and the alternatives once more, each with its own terms:
  // rounded once
  __syncthreads();
  for (int i = tid; i <= n; i += NT) {
    const int64_t e = i == 0 ? t : top[row * n + i - 1];
    if (e < 0 || e >= V) continue;
    const int j = (int)((e + w.off) / VE);
    if (j < j0 || j >= j1) continue;
    float s = slope(to_f(r.x[e]));
    if (e == t) s += g[0];
    for (int k = 0; k < n; ++k)
      if (top[row * n + k] == e) s += g[2 + k];
    d[e] = from_f<T>(s);
  }
}

}  // namespace hetu

using namespace hetu;

template <typename T>
static void launch_fwd(const void* logits, int64_t stride, const int64_t* ids, int64_t R, int V, int n, int64_t ignored,
                       float* out, int64_t* top, hipStream_t st) {
#define GO(NT, TOP) hipLaunchKernelGGL((token_logprob_k<T, NT, TOP>), many_blocks(R), dim3(NT), 0, st, \
                                       (const T*)logits, stride, ids, R, V, n, ignored, out, top)
  const int64_t bytes = (int64_t)V * sizeof(T);
  // 1024 threads for long rows that are few, or that have alternatives to find (a thread's elements are
  // read again: 1000 x 131072 top 20 57 us, with 256 threads 71 against 63 then); 256 threads else (8192
  // x 30522: 117 us, with 128 130, with 512 124, all before the gradient went past the cache, 74 to 81
  // since); a wave for rows that it holds in registers (16384 x 2000 bf16: 16 us, with 5 alternatives 39,
  // with 20 44, with 64 64, of which the row's 64-key sort and bit searches are all but the 16)
  if (bytes <= kShortBytes) {
    const dim3 grid = many_blocks((R + kShortWaves - 1) / kShortWaves), block(64 * kShortWaves);
    if (n) hipLaunchKernelGGL((token_logprob_short_k<T, true>), grid, block, 0, st, (const T*)logits, stride, ids, R, V, n, ignored, out, top);
    else hipLaunchKernelGGL((token_logprob_short_k<T, false>), grid, block, 0, st, (const T*)logits, stride, ids, R, V, n, ignored, out, top);
  } else if (bytes >= 32768 && (R <= 512 || n)) {
    if (n) GO(1024, true); else GO(1024, false);
  } else {
    if (n) GO(256, true); else GO(256, false);
  }
#undef GO
}

// out: a row of 4 + n: logp, entropy, the n largest log probabilities, then the row's maximum and
// the base-2 log of its sum for the backward pass
HETU_API int hetu_token_logprob(const void* logits, int64_t stride, const int64_t* ids, int64_t R, int V, int n,
                                int64_t ignored, float* out, int64_t* top, int is_bf16,
                                hipStream_t st) {
  if (R <= 0) return 0;
  if (V < 1 || n < 0 || n > kMaxTop || n > V || R > kMaxBlocks) return (int)hipErrorInvalidValue;
  if (is_bf16) launch_fwd<bf16>(logits, stride, ids, R, V, n, ignored, out, top, st);
  else launch_fwd<float>(logits, stride, ids, R, V, n, ignored, out, top, st);
  HETU_LAUNCH_CHECK();
  return 0;
}

HETU_API int hetu_token_logprob_bwd(const void* logits, int64_t stride, const int64_t* ids, int64_t R, int V, int n,
                                    int64_t ignored, const float* out, const int64_t* top,
                                    const float* grad, void* dx, int is_bf16, hipStream_t st) {
  if (R <= 0) return 0;
  const int VE = is_bf16 ? 8 : 4;
  const int64_t chunks = ((int64_t)V + 2 * VE - 2 + (int64_t)VE * kBwdGranules - 1) / ((int64_t)VE * kBwdGranules);
  if (V < 1 || n < 0 || n > kMaxTop || n > V || R > kMaxBlocks / chunks) return (int)hipErrorInvalidValue;
  const dim3 grid = many_blocks(R * chunks), block(kBwdThreads);
  const int64_t bytes = R * V * (is_bf16 ? 2 : 4);
#define GO(T, LD, ST) hipLaunchKernelGGL((token_logprob_bwd_k<T, LD, ST>), grid, block, 0, st, (const T*)logits, stride, ids, \
                                         R, V, n, ignored, (int)chunks, out, top, grad, (T*)dx)
  if (bytes > 3 * kLastCacheBytes) { if (is_bf16) GO(bf16, true, true); else GO(float, true, true); }
  else if (2 * bytes > kLastCacheBytes) { if (is_bf16) GO(bf16, false, true); else GO(float, false, true); }
  else { if (is_bf16) GO(bf16, false, false); else GO(float, false, false); }
#undef GO
  HETU_LAUNCH_CHECK();
  return 0;
}
