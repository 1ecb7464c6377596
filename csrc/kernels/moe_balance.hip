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
#include "common.h"

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

// this lane's part of softmax(row), 0 beyond E
template <typename T, int V, int NJ>
__device__ __forceinline__ void row_softmax(const T* x, int E, int G, int lane, float (&p)[NJ * V]) {
  float m = -INFINITY;
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
    for (int k = 0; k < V; ++k) {
      p[j * V + k] = v[k];
      m = fmaxf(m, v[k]);
    }
  }
  for (int o = G >> 1; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NJ * V; ++i) {
    p[i] = __expf(p[i] - m);
    s += p[i];
  }
#pragma unroll
  for (int j = 0; j < NJ; ++j)
    if ((j * G + lane) * V >= E) {
#pragma unroll
      for (int k = 0; k < V; ++k) p[j * V + k] = 0.f;
    }
  for (int o = G >> 1; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  const float inv = 1.f / s;
#pragma unroll
  for (int i = 0; i < NJ * V; ++i) p[i] *= inv;
}

// partial sums of block b: psum [b][E], counts [b][E + 1] (the last: valid tokens)
template <typename T, int V, int NJ>
__global__ void __launch_bounds__(kBlThreads) balance_part_k(const T* __restrict__ x, int64_t stride, int64_t T_, int E,
                                                             int G, const int64_t* __restrict__ idx, int k,
                                                             const void* valid, int kind, int64_t rows,
                                                             float* __restrict__ psum, int* __restrict__ pcnt) {
  __shared__ float cols[4][kMaxExperts];
  __shared__ int hist[kMaxExperts + 1];
  const int tid = threadIdx.x, lane = tid & (G - 1), group = tid / G, groups = kBlThreads / G;
  const int64_t t0 = (int64_t)blockIdx.x * rows, t1 = t0 + rows < T_ ? t0 + rows : T_;
  for (int e = tid; e <= E; e += kBlThreads) hist[e] = 0;
  __syncthreads();
  float acc[NJ * V];
#pragma unroll
  for (int i = 0; i < NJ * V; ++i) acc[i] = 0.f;
  int on = 0;
  for (int64_t t = t0 + group; t < t1; t += groups) {
    if (!token_on(valid, kind, t)) continue;      // the whole group: its lanes share t
    ++on;
    float p[NJ * V];
    row_softmax<T, V, NJ>(x + t * stride, E, G, lane, p);
#pragma unroll
    for (int i = 0; i < NJ * V; ++i) acc[i] += p[i];
  }
  if (lane == 0 && on) atomicAdd(&hist[E], on);
  for (int64_t i = t0 * k + tid; i < t1 * k; i += kBlThreads) {
    if (!token_on(valid, kind, i / k)) continue;
    const int64_t e = idx[i];
    if (e >= 0 && e < E) atomicAdd(&hist[e], 1);
  }
  // groups of a wave, then waves
#pragma unroll
  for (int i = 0; i < NJ * V; ++i)
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

// counts, the weights of the backward pass and the loss, from the blocks' sums in order
__global__ void __launch_bounds__(1024) balance_join_k(const float* __restrict__ psum, const int* __restrict__ pcnt,
                                                       int blocks, int E, int64_t* __restrict__ counts,
                                                       float* __restrict__ weight, float* __restrict__ loss) {
  __shared__ int64_t total;
  __shared__ double part[16];
  const int tid = threadIdx.x;
  int64_t c = 0;
  double s = 0.0;
  if (tid < E) {
    for (int b = 0; b < blocks; ++b) {
      c += pcnt[(int64_t)b * (E + 1) + tid];
      s += psum[(int64_t)b * E + tid];
    }
    counts[tid] = c;
  }
  if (tid == 0) {
    int64_t n = 0;
    for (int b = 0; b < blocks; ++b) n += pcnt[(int64_t)b * (E + 1) + E];
    total = n;
  }
  __syncthreads();
  const double n = (double)total;
  const double w = total > 0 ? (double)E * (double)c / (n * n) : 0.0;
  if (tid < E) weight[tid] = (float)w;
  double l = total > 0 ? w * s : 0.0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o, 64);
  if ((tid & 63) == 0) part[tid >> 6] = l;
  __syncthreads();
  if (tid == 0) {
    double r = 0.0;
    for (int i = 0; i < 16; ++i) r += part[i];
    loss[0] = (float)r;
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
      row_softmax<T, V, NJ>(x + t * stride, E, G, lane, p);
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < NJ * V; ++i) dot += p[i] * w[i];
      for (int o = G >> 1; o > 0; o >>= 1) dot += __shfl_xor(dot, o, 64);
#pragma unroll
      for (int i = 0; i < NJ * V; ++i) p[i] = gr * p[i] * (w[i] - dot);
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
static RowPlan plan_rows(int E, int64_t stride, const void* x, const void* y, int vec, int size) {
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

// blocks of the partial sums: at least 16 rows a group of lanes, at most 512 blocks
static int64_t balance_rows(int64_t T, int G) {
  const int64_t groups = kBlThreads / G;
  int64_t blocks = (T + groups * 16 - 1) / (groups * 16);
  blocks = blocks < 1 ? 1 : (blocks > 512 ? 512 : blocks);
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

// number of 4-byte words of workspace that hetu_moe_balance_fwd needs
HETU_API int64_t hetu_moe_balance_ws(int64_t T, int E) {
  if (T <= 0 || E < 1 || E > kMaxExperts) return 0;
  return (int64_t)512 * (2 * E + 1);
}

HETU_API int hetu_moe_balance_fwd(const void* x, int64_t stride, int64_t T, int E, const int64_t* idx, int k,
                                  const void* valid, int kind, int64_t* counts, float* weight, float* loss, void* ws,
                                  int is_bf16, hipStream_t st) {
  if (T < 0 || E < 1 || E > kMaxExperts || k < 1) return (int)hipErrorInvalidValue;
  const RowPlan r = plan_rows(E, stride, x, nullptr, is_bf16 ? 8 : 4, is_bf16 ? 2 : 4);
  const int64_t rows = T > 0 ? balance_rows(T, r.G) : 1;
  const int blocks = T > 0 ? (int)((T + rows - 1) / rows) : 0;
  float* psum = (float*)ws;
  int* pcnt = (int*)ws + (int64_t)512 * E;
  if (blocks > 0) {
#define GO(TT, VV, JJ) hipLaunchKernelGGL((balance_part_k<TT, VV, JJ>), dim3(blocks), dim3(kBlThreads), 0, st, \
                                          (const TT*)x, stride, T, E, r.G, idx, k, valid, kind, rows, psum, pcnt)
    BALANCE_CASES(GO)
#undef GO
    HETU_LAUNCH_CHECK();
  }
  hipLaunchKernelGGL(balance_join_k, dim3(1), dim3(1024), 0, st, psum, pcnt, blocks, E, counts, weight, loss);
  HETU_LAUNCH_CHECK();
  return 0;
}

HETU_API int hetu_moe_balance_bwd(const void* x, int64_t stride, int64_t T, int E, const float* weight, const float* g,
                                  const void* valid, int kind, void* dx, int is_bf16, hipStream_t st) {
  if (T <= 0) return 0;
  if (E < 1 || E > kMaxExperts) return (int)hipErrorInvalidValue;
  const RowPlan r = plan_rows(E, stride, x, dx, is_bf16 ? 8 : 4, is_bf16 ? 2 : 4);
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
