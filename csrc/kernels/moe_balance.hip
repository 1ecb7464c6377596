// Mixture-of-experts balance loss from the router's logits, per-expert counts, and its gradient.
//
// Over the N valid tokens t, with p_t = softmax(x_t), P_e = sum_t p_{t,e} and c_e the number of
// choices that fall on expert e:
//   loss = E / N^2 sum_e c_e P_e,     w_e = E c_e / N^2
//   dx_{t,e} = g p_{t,e} (w_e - sum_f p_{t,f} w_f)       (the counts carry no gradient)
//
// A row of E logits is held by a group of G lanes (a power of two, at most a wave) in registers:
// lane l of a group holds elements (j G + l) V + k for j < NJ, k < V, V elements a load.  Column
// sums stay in the lanes' registers over all rows of a block, join by shuffles and LDS, and go to
// a row of partial sums a block; one block adds those up in a fixed order.  No atomics on floats:
// the same inputs give the same bits.
#include "wave_ops.h"

namespace hetu {

constexpr int kBlThreads = 256;
constexpr int kMaxExperts = 1024;

// validity of token t from a mask of 1-byte (0), fp32 (1), bf16 (2), int64 (3) or int32 (4) values
__device__ __forceinline__ bool token_on(const void* valid, int kind, int64_t t) {
  if (!valid) return true;
  switch (kind) {
    case 0: return ((const unsigned char*)valid)[t] != 0;
    case 1: return ((const float*)valid)[t] != 0.f;
    case 2: return (((const unsigned short*)valid)[t] & 0x7FFFu) != 0;
    case 3: return ((const int64_t*)valid)[t] != 0;
    default: return ((const int*)valid)[t] != 0;
  }
}

template <typename T, int V>
__device__ __forceinline__ void load_n(const T* p, float (&v)[V]) {
  if constexpr (V == 1) v[0] = to_f(p[0]);
  else load_vec<T>(p, v);
}
template <typename T, int V>
__device__ __forceinline__ void store_n(T* p, const float (&v)[V]) {
  if constexpr (V == 1) p[0] = from_f<T>(v[0]);
  else store_vec<T>(p, v);
}

// the lane's elements of row x, -inf beyond E
template <typename T, int V, int NJ>
__device__ __forceinline__ void row_load(const T* x, int E, int G, int lane, float (&p)[NJ * V]) {
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int e = (j * G + lane) * V;
    float v[V];
    if (e < E) {
      load_n<T, V>(x + e, v);
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = -INFINITY;
    }
#pragma unroll
    for (int k = 0; k < V; ++k) p[j * V + k] = v[k];
  }
}

// exponentials in place, 0 beyond E, and the reciprocal of their sum over the row
template <int N>
__device__ __forceinline__ float row_exp(int G, float (&p)[N]) {
  float m = p[0];
#pragma unroll
  for (int i = 1; i < N; ++i) m = fmaxf(m, p[i]);
  m = group_max(m, G);
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    p[i] = __expf(p[i] - m);
    s += p[i];
  }
  return 1.f / group_sum(s, G);
}

// Partial sums of block b: psum [b][E], counts [b][E + 1] (the last: valid tokens).  U rows a
// group are under way at once: their loads and the exchanges of their two reductions overlap.
template <typename T, int V, int NJ>
__global__ void __launch_bounds__(kBlThreads) balance_part_k(const T* __restrict__ x, int64_t stride, int64_t T_, int E,
                                                             int G, const int64_t* __restrict__ idx, int k,
                                                             const void* valid, int kind, int64_t rows,
                                                             float* __restrict__ psum, int* __restrict__ pcnt,
                                                             unsigned* __restrict__ ticket) {
  constexpr int N = NJ * V, U = N <= 8 ? 4 : (N <= 16 ? 2 : 1);
  __shared__ float cols[4][kMaxExperts];
  __shared__ int hist[kMaxExperts + 1];
  const int tid = threadIdx.x, lane = tid & (G - 1), group = tid / G, groups = kBlThreads / G;
  const int64_t t0 = (int64_t)blockIdx.x * rows, t1 = t0 + rows < T_ ? t0 + rows : T_;
  if (blockIdx.x == 0 && tid == 0) *ticket = 0;       // for the joining launch
  for (int e = tid; e <= E; e += kBlThreads) hist[e] = 0;
  __syncthreads();
  float acc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
  // the choices, one a thread: (token, choice) advances by 256 choices without a division
  {
    const int dt = kBlThreads / k, dc = kBlThreads - dt * k;
    int64_t t = t0 + tid / k;
    int c = tid % k;
    while (t < t1) {
      if (token_on(valid, kind, t)) {
        const int64_t e = idx[t * k + c];
        if (e >= 0 && e < E) atomicAdd(&hist[e], 1);
      }
      t += dt;
      c += dc;
      if (c >= k) { c -= k; ++t; }
    }
  }
  int count = 0;
  for (int64_t t = t0 + group; t < t1; t += (int64_t)groups * U) {
    float p[U][N];
    bool on[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {      // a token that is not valid: the row of t0 in its place, unused
      const int64_t tu = t + (int64_t)u * groups;
      on[u] = tu < t1 && token_on(valid, kind, tu);
      row_load<T, V, NJ>(x + (on[u] ? tu : t0) * stride, E, G, lane, p[u]);
      count += on[u];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float inv = row_exp<N>(G, p[u]);
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] += on[u] ? p[u][i] * inv : 0.f;
    }
  }
  if (lane == 0 && count) atomicAdd(&hist[E], count);
  // groups of a wave, then waves
#pragma unroll
  for (int i = 0; i < N; ++i)
    for (int o = G; o < 64; o <<= 1) acc[i] += __shfl_xor(acc[i], o, 64);
  if ((tid & 63) < G) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int e = (j * G + lane) * V;
      if (e < E) {
#pragma unroll
        for (int q = 0; q < V; ++q) cols[tid >> 6][e + q] = acc[j * V + q];
      }
    }
  }
  __syncthreads();
  for (int e = tid; e < E; e += kBlThreads)
    psum[(int64_t)blockIdx.x * E + e] = (cols[0][e] + cols[1][e]) + (cols[2][e] + cols[3][e]);
  for (int e = tid; e <= E; e += kBlThreads) pcnt[(int64_t)blockIdx.x * (E + 1) + e] = hist[e];
}

// Counts, the weights of the backward pass and the loss from the blocks' sums: EB experts a
// block, the partial sums of one expert over 1024 / EB threads, all in a fixed order.  The block
// that comes last adds up the blocks' parts of the loss, in order too.
constexpr int kJoinThreads = 1024, kJoinExperts = 16;

__global__ void __launch_bounds__(kJoinThreads) balance_join_k(const float* __restrict__ psum,
                                                               const int* __restrict__ pcnt, int blocks, int E, int EB,
                                                               int64_t* __restrict__ counts, float* __restrict__ weight,
                                                               float* __restrict__ loss, double* part, unsigned* ticket) {
  __shared__ double sums[kJoinThreads];
  __shared__ int64_t cnts[kJoinThreads];
  __shared__ int64_t wave_n[kJoinThreads / 64];
  __shared__ bool last;
  const int tid = threadIdx.x, e = blockIdx.x * EB + (tid & (EB - 1)), seg = tid / EB, segs = kJoinThreads / EB;
  int64_t n = 0;
  for (int b = tid; b < blocks; b += kJoinThreads) n += pcnt[(int64_t)b * (E + 1) + E];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
  if ((tid & 63) == 0) wave_n[tid >> 6] = n;
  double s = 0.0;
  int64_t c = 0;
  if (e < E) {
#pragma unroll 8
    for (int b = seg; b < blocks; b += segs) {
      s += psum[(int64_t)b * E + e];
      c += pcnt[(int64_t)b * (E + 1) + e];
    }
  }
  sums[tid] = s;
  cnts[tid] = c;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int i = 0; i < kJoinThreads / 64; ++i) total += wave_n[i];
  for (int h = segs >> 1; h > 0; h >>= 1) {
    if (seg < h) {
      sums[tid] += sums[tid + h * EB];
      cnts[tid] += cnts[tid + h * EB];
    }
    __syncthreads();
  }
  if (tid < EB) {
    double l = 0.0;
    if (e < E) {
      const double d = (double)total, w = total > 0 ? (double)E * (double)cnts[tid] / (d * d) : 0.0;
      counts[e] = cnts[tid];
      weight[e] = (float)w;
      l = total > 0 ? w * sums[tid] : 0.0;
    }
    sums[tid] = l;
  }
  __syncthreads();
  if (tid < 64) {
    double l = tid < EB ? sums[tid] : 0.0;
#pragma unroll
    for (int o = kJoinExperts / 2; o > 0; o >>= 1) l += __shfl_xor(l, o, 64);
    sums[tid] = l;
  }
  if (tid == 0) {
    double l = sums[0];
    __hip_atomic_store(part + blockIdx.x, l, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
    if (last) {
      l = 0.0;
      for (unsigned i = 0; i < gridDim.x; ++i) l += __hip_atomic_load(part + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      loss[0] = (float)l;
    }
  }
}

template <typename T, int V, int NJ>
__global__ void __launch_bounds__(kBlThreads) balance_bwd_k(const T* __restrict__ x, int64_t stride, int64_t T_, int E,
                                                            int G, const float* __restrict__ weight,
                                                            const float* __restrict__ g, const void* valid, int kind,
                                                            T* __restrict__ dx) {
  const int tid = threadIdx.x, lane = tid & (G - 1), group = tid / G, groups = kBlThreads / G;
  float w[NJ * V];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int e = (j * G + lane) * V;
#pragma unroll
    for (int q = 0; q < V; ++q) w[j * V + q] = e < E ? weight[e + q] : 0.f;
  }
  const float gr = g[0];
  for (int64_t t = (int64_t)blockIdx.x * groups + group; t < T_; t += (int64_t)gridDim.x * groups) {
    float p[NJ * V];
    if (token_on(valid, kind, t)) {
      row_load<T, V, NJ>(x + t * stride, E, G, lane, p);
      const float inv = row_exp<NJ * V>(G, p);
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < NJ * V; ++i) dot += p[i] * w[i];
      dot = group_sum(dot, G) * inv;
      const float c = gr * inv;
#pragma unroll
      for (int i = 0; i < NJ * V; ++i) p[i] = c * p[i] * (w[i] - dot);
    } else {
#pragma unroll
      for (int i = 0; i < NJ * V; ++i) p[i] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int e = (j * G + lane) * V;
      if (e < E) {
        float v[V];
#pragma unroll
        for (int q = 0; q < V; ++q) v[q] = p[j * V + q];
        store_n<T, V>(dx + t * (int64_t)E + e, v);
      }
    }
  }
}

struct RowPlan { int V, G, NJ; };

// V elements a load where rows and buffers allow 16-byte accesses, G lanes a row, NJ loads a lane
static RowPlan plan_rows(int E, int64_t stride, const void* x, const void* y, int vec) {
  RowPlan r;
  r.V = (E % vec == 0 && stride % vec == 0 && (((uintptr_t)x | (uintptr_t)y) & 15) == 0) ? vec : 1;
  const int units = (E + r.V - 1) / r.V;
  r.G = 1;
  while (r.G < units && r.G < 64) r.G <<= 1;
  const int nj = (units + r.G - 1) / r.G;
  r.NJ = 1;
  while (r.NJ < nj) r.NJ <<= 1;
  return r;
}

}  // namespace hetu

using namespace hetu;

// Rows a block of the partial sums takes: as many blocks as keep the chip's waves busy (4 blocks a
// CU), but at least 8 rows a group of lanes, for each block costs E partial sums.
constexpr int kMaxParts = 1024;
static int64_t balance_rows(int64_t T, int G) {
  const int64_t groups = kBlThreads / G;
  int64_t blocks = (T + groups * 8 - 1) / (groups * 8);
  blocks = blocks < 1 ? 1 : (blocks > kMaxParts ? kMaxParts : blocks);
  return (T + blocks - 1) / blocks;
}

#define BALANCE_CASES(GO)                                                            \
  if (is_bf16) {                                                                     \
    if (r.V == 8) { if (r.NJ == 1) GO(bf16, 8, 1); else GO(bf16, 8, 2); }            \
    else if (r.NJ == 1) GO(bf16, 1, 1); else if (r.NJ == 2) GO(bf16, 1, 2);          \
    else if (r.NJ == 4) GO(bf16, 1, 4); else if (r.NJ == 8) GO(bf16, 1, 8);          \
    else GO(bf16, 1, 16);                                                            \
  } else {                                                                           \
    if (r.V == 4) { if (r.NJ == 1) GO(float, 4, 1); else if (r.NJ == 2) GO(float, 4, 2); else GO(float, 4, 4); } \
    else if (r.NJ == 1) GO(float, 1, 1); else if (r.NJ == 2) GO(float, 1, 2);        \
    else if (r.NJ == 4) GO(float, 1, 4); else if (r.NJ == 8) GO(float, 1, 8);        \
    else GO(float, 1, 16);                                                           \
  }

// number of 4-byte words of workspace (8-byte aligned) that hetu_moe_balance_fwd needs: each
// block's sums and counts, the joining blocks' parts of the loss, their ticket
HETU_API int64_t hetu_moe_balance_ws(int64_t T, int E) {
  if (T < 0 || E < 1 || E > kMaxExperts) return 0;
  const int64_t groups_least = kBlThreads / 64;
  int64_t parts = (T + groups_least * 8 - 1) / (groups_least * 8);
  parts = parts < 1 ? 1 : (parts > kMaxParts ? kMaxParts : parts);
  return 2 * (kMaxExperts / kJoinExperts) + 2 + parts * (2 * E + 1);
}

HETU_API int hetu_moe_balance_fwd(const void* x, int64_t stride, int64_t T, int E, const int64_t* idx, int k,
                                  const void* valid, int kind, int64_t* counts, float* weight, float* loss, void* ws,
                                  int is_bf16, hipStream_t st) {
  if (T < 0 || E < 1 || E > kMaxExperts || k < 1) return (int)hipErrorInvalidValue;
  const RowPlan r = plan_rows(E, stride, x, nullptr, is_bf16 ? 8 : 4);
  const int64_t rows = T > 0 ? balance_rows(T, r.G) : 1;
  const int blocks = T > 0 ? (int)((T + rows - 1) / rows) : 1;
  double* part = (double*)ws;
  unsigned* ticket = (unsigned*)(part + kMaxExperts / kJoinExperts);
  float* psum = (float*)(ticket + 2);
  int* pcnt = (int*)(psum + (int64_t)blocks * E);
#define GO(TT, VV, JJ) hipLaunchKernelGGL((balance_part_k<TT, VV, JJ>), dim3(blocks), dim3(kBlThreads), 0, st, \
                                          (const TT*)x, stride, T, E, r.G, idx, k, valid, kind, rows, psum, pcnt, ticket)
  BALANCE_CASES(GO)
#undef GO
  HETU_LAUNCH_CHECK();
  int EB = 1;
  while (EB < E && EB < kJoinExperts) EB <<= 1;
  hipLaunchKernelGGL(balance_join_k, dim3((E + EB - 1) / EB), dim3(kJoinThreads), 0, st, psum, pcnt, blocks, E, EB,
                     counts, weight, loss, part, ticket);
  HETU_LAUNCH_CHECK();
  return 0;
}

HETU_API int hetu_moe_balance_bwd(const void* x, int64_t stride, int64_t T, int E, const float* weight, const float* g,
                                  const void* valid, int kind, void* dx, int is_bf16, hipStream_t st) {
  if (T <= 0) return 0;
  if (E < 1 || E > kMaxExperts) return (int)hipErrorInvalidValue;
  const RowPlan r = plan_rows(E, stride, x, dx, is_bf16 ? 8 : 4);
  const int64_t groups = kBlThreads / r.G;
  const int64_t want = (T + groups - 1) / groups;
  const dim3 grid((unsigned)(want < 2048 ? want : 2048));
#define GO(TT, VV, JJ) hipLaunchKernelGGL((balance_bwd_k<TT, VV, JJ>), grid, dim3(kBlThreads), 0, st, (const TT*)x, \
                                          stride, T, E, r.G, weight, g, valid, kind, (TT*)dx)
  BALANCE_CASES(GO)
#undef GO
  HETU_LAUNCH_CHECK();
  return 0;
}
