// Mixture-of-experts balance loss from the router's logits, per-expert counts, and its gradient.
//
// Over the N valid tokens t, with p_t = softmax(x_t), P_e = sum_t p_{t,e} and c_e the number of
// choices that fall on expert e:
//   loss = E / N^2 sum_e c_e P_e,     w_e = E c_e / N^2
//   dx_{t,e} = g p_{t,e} (w_e - sum_f p_{t,f} w_f)       (the counts carry no gradient)
//
// A row of E logits is held by a group of G lanes (a power of two, at most a wave) in registers:
// lane l of a group holds elements (j G + l) V + k for j < NJ, k < V, V elements a load.  G, V and
// NJ are known at compile time, so that the exchanges of several rows' reductions interleave.  Column
// sums stay in the lanes' registers over all rows of a block, join by shuffles and LDS, and go to
// a row of partial sums a block; one block adds those up in a fixed order.  No atomics on floats:
// the same inputs give the same bits.
#include "wave_ops.h"

namespace hetu {

constexpr int kBlThreads = 256;
constexpr int kMaxExperts = 1024;

// validity of tokens t, t + step, .. (U of them, those below t1) from a mask of 1-byte (0), fp32
// (1), bf16 (2), int64 (3) or int32 (4) values
template <int U, typename M>
__device__ __forceinline__ void mask_on(const M* mask, M bits, int64_t t, int64_t step, int64_t t1, bool (&on)[U]) {
  M v[U];
#pragma unroll
  for (int u = 0; u < U; ++u) v[u] = mask[t + u * step < t1 ? t + u * step : t1 - 1];
#pragma unroll
  for (int u = 0; u < U; ++u) on[u] = t + u * step < t1 && (v[u] & bits) != 0;
}
template <int U>
__device__ __forceinline__ void tokens_on(const void* valid, int kind, int64_t t, int64_t step, int64_t t1, bool (&on)[U]) {
  if (!valid) {
#pragma unroll
    for (int u = 0; u < U; ++u) on[u] = t + u * step < t1;
  } else if (kind == 0) {
    mask_on<U, unsigned char>((const unsigned char*)valid, 0xFF, t, step, t1, on);
  } else if (kind == 2) {
    mask_on<U, unsigned short>((const unsigned short*)valid, 0x7FFF, t, step, t1, on);     // -0 is 0
  } else if (kind == 3) {
    mask_on<U, uint64_t>((const uint64_t*)valid, ~0ull, t, step, t1, on);
  } else {
    mask_on<U, unsigned>((const unsigned*)valid, kind == 1 ? 0x7FFFFFFFu : ~0u, t, step, t1, on);
  }
}

template <typename T, int V, bool PAST>
__device__ __forceinline__ void store_n(T* p, const float (&v)[V]) {
  if constexpr (V == 1) p[0] = from_f<T>(v[0]);
  else store_raw<PAST>(p, pack_raw(v));
}

// A lane's elements of a row as they are in memory: converted when they are used, so that loads
// can be under way across other work.  V = 1, or the 4 fp32 or 8 bf16 of 16 bytes.  Lanes beyond E
// hold the row's first elements again: they leave the maximum as it is, and are left out of sums.
template <typename T, int V, int NJ, int G>
struct RowRaw {
  Raw q[V == 1 ? 1 : NJ];
  T s[V == 1 ? NJ : 1];
  __device__ __forceinline__ void load(const T* x, int E, int lane) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      int e = (j * G + lane) * V;
      e = e < E ? e : 0;
      if constexpr (V == 1) s[j] = x[e];
      else q[j] = *reinterpret_cast<const Raw*>(x + e);
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      if constexpr (V == 1) s[j] = from_f<T>(0.f);
      else q[j] = Raw{0, 0, 0, 0};
    }
  }
  __device__ __forceinline__ void unpack(float (&p)[NJ * V]) const {
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        if constexpr (V == 1) p[j] = to_f(s[j]);
        else if constexpr (V == 4) p[j * V + k] = __uint_as_float(q[j][k]);
        else p[j * V + k] = __uint_as_float(k & 1 ? q[j][k >> 1] & 0xffff0000u : q[j][k >> 1] << 16);
      }
  }
};

// exponentials of U rows in place and the reciprocals of their sums (v_rcp_f32, off by a unit)
template <int U, int V, int NJ, int G>
__device__ __forceinline__ void rows_exp(int E, int lane, float (&p)[U][NJ * V], float (&inv)[U]) {
  float m[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    m[u] = p[u][0];
#pragma unroll
    for (int i = 1; i < NJ * V; ++i) m[u] = fmaxf(m[u], p[u][i]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) m[u] = group_max(m[u], G);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      float part = 0.f;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        p[u][j * V + k] = __expf(p[u][j * V + k] - m[u]);
        part += p[u][j * V + k];
      }
      s += (j * G + lane) * V < E ? part : 0.f;
    }
    inv[u] = s;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) inv[u] = __builtin_amdgcn_rcpf(group_sum(inv[u], G));
}

// Partial sums of block b, a row of 2 pitch + 4 words: E sums, E counts, the valid tokens, each part
// starting 16-byte aligned; of a single block the results (counts: hetu_moe_balance_fwd).  A group takes
// U rows at a time: the next U rows' loads and the validity of those after them are under way
// while these are summed.
__host__ __device__ inline int part_pitch(int E) { return (E + 3) & ~3; }
constexpr int kPartThreads = 512, kPartWaves = kPartThreads / 64;

template <typename T, int V, int NJ, int G>
__global__ void __launch_bounds__(kPartThreads) balance_part_k(const T* __restrict__ x, int64_t stride, int64_t T_,
                                                               int E, const int64_t* __restrict__ idx, int k,
                                                               const void* valid, int kind, int64_t rows,
                                                               float* __restrict__ parts, unsigned* __restrict__ ticket,
                                                               int64_t* __restrict__ counts) {
  constexpr int N = NJ * V, U = N <= 8 ? 4 : 1, CU = 4, groups = kPartThreads / G;
  constexpr int64_t step = groups * U;
  extern __shared__ __align__(16) int lds[];
  int* hist = lds;                                       // [E + 1]
  float* cols = reinterpret_cast<float*>(lds + E + 1);   // [kPartWaves][E]
  const int tid = threadIdx.x, lane = tid & (G - 1), group = tid / G;
  const int64_t t0 = (int64_t)blockIdx.x * rows, t1 = t0 + rows < T_ ? t0 + rows : T_;
  if (blockIdx.x == 0 && tid == 0) *ticket = 0;       // for the joining launch
  for (int e = tid; e <= E; e += kPartThreads) hist[e] = 0;
  __syncthreads();
  RowRaw<T, V, NJ, G> raw[U];
  const T *base = x + t0 * stride, *at = x + (t0 + group) * stride;
  const int64_t between = groups * stride;
  const auto load = [&](const bool (&on)[U]) {          // not valid: the row of t0 in its place, unused
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u].load(on[u] ? at + u * between : base, E, lane);
  };
  float acc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
  int count = 0;
  bool on[U], next[U];
  int64_t t = t0 + group;
  if (t < t1) {
    tokens_on<U>(valid, kind, t, groups, t1, on);
    load(on);
    tokens_on<U>(valid, kind, t + step, groups, t1, next);
  }
  // the choices, one a thread, CU of them under way: (token, choice) advances by the block's
  // threads without a division
  {
    const int dt = kPartThreads / k, dc = kPartThreads - dt * k;
    int64_t tc = t0 + tid / k;
    int c = tid % k;
    while (tc < t1) {
      int64_t e[CU];
      bool in[CU][1];
#pragma unroll
      for (int u = 0; u < CU; ++u) {
        e[u] = tc < t1 ? idx[tc * k + c] : -1;
        tokens_on<1>(valid, kind, tc, 0, t1, in[u]);
        tc += dt;
        c += dc;
        if (c >= k) { c -= k; ++tc; }
      }
#pragma unroll
      for (int u = 0; u < CU; ++u)
        if (in[u][0] && e[u] >= 0 && e[u] < E) atomicAdd(&hist[e[u]], 1);
    }
  }
  for (; t < t1; t += step) {
    float p[U][N], inv[U];
    bool now[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!on[u]) raw[u].clear();
      raw[u].unpack(p[u]);
      now[u] = on[u];
      on[u] = next[u];
    }
    if (t + step < t1) {
      at += step * stride;
      load(on);
      tokens_on<U>(valid, kind, t + 2 * step, groups, t1, next);
    }
    rows_exp<U, V, NJ, G>(E, lane, p, inv);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float c = now[u] ? inv[u] : 0.f;          // (a row in another's place is finite: zeroed)
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] += p[u][i] * c;
      count += now[u];
    }
  }
  if (lane == 0 && count) atomicAdd(&hist[E], count);
  // groups of a wave, then waves
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = place_sum<G>(acc[i]);
  if ((tid & 63) < G) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int e = (j * G + lane) * V;
      if (e < E) {
#pragma unroll
        for (int q = 0; q < V; ++q) cols[(tid >> 6) * E + e + q] = acc[j * V + q];
      }
    }
  }
  __syncthreads();
  if (gridDim.x == 1) {                // nothing to join: the results themselves
    const double n = (double)hist[E];
    double l = 0.0;
    for (int e = tid; e < E; e += kPartThreads) {
      double s = 0.0;
#pragma unroll
      for (int w = 0; w < kPartWaves; ++w) s += cols[w * E + e];
      const double c = n > 0.0 ? (double)E * hist[e] / (n * n) : 0.0;
      counts[e] = hist[e];
      reinterpret_cast<float*>(counts + E)[e] = (float)c;
      l += c * s;
    }
    l = quad_place_sum(l);
    __syncthreads();                   // (cols are read: their place holds the waves' parts now)
    double* part = reinterpret_cast<double*>(lds);
    if ((tid & 63) < 4) part[(tid >> 6) * 4 + (tid & 3)] = l;
    __syncthreads();
    if (tid == 0) {
      l = 0.0;
      for (int i = 0; i < kPartWaves * 4; ++i) l += part[i];
      reinterpret_cast<float*>(counts + E)[E] = (float)l;
    }
    return;
  }
  const int pitch = part_pitch(E);
  float* sums = parts + (int64_t)blockIdx.x * (2 * pitch + 4);
  int* cnts = reinterpret_cast<int*>(sums) + pitch;
  for (int e = tid; e < pitch; e += kPartThreads) {
    float s = 0.f;
    if (e < E) {
#pragma unroll
      for (int w = 0; w < kPartWaves; ++w) s += cols[w * E + e];
    }
    sums[e] = s;
    cnts[e] = e < E ? hist[e] : 0;
  }
  if (tid == 0) cnts[pitch] = hist[E];
}

// Counts, the weights of the backward pass and the loss from the blocks' sums: 16 experts a block,
// 4 a thread and the blocks' rows over 256 threads, joined in a fixed order.  The block that
// comes last adds up the blocks' parts of the loss, in order too.
constexpr int kJoinThreads = 1024, kJoinExperts = 16, kJoinWaves = kJoinThreads / 64;

__global__ void __launch_bounds__(kJoinThreads) balance_join_k(const float* __restrict__ parts, int blocks, int E,
                                                               int64_t* __restrict__ counts, float* __restrict__ weight,
                                                               float* __restrict__ loss, double* loss_part,
                                                               unsigned* ticket) {
  __shared__ double sums[kJoinWaves][kJoinExperts];
  __shared__ int64_t cnts[kJoinWaves][kJoinExperts], valid[kJoinWaves][4];
  const int tid = threadIdx.x, pitch = part_pitch(E), words = 2 * pitch + 4;
  const int e0 = blockIdx.x * kJoinExperts + (tid & 3) * 4, seg = tid >> 2;
  int64_t n = 0;
  for (int b = tid; b < blocks; b += kJoinThreads)
    n += reinterpret_cast<const int*>(parts)[(int64_t)b * words + 2 * pitch];
  double s[4] = {0.0, 0.0, 0.0, 0.0};
  int64_t c[4] = {0, 0, 0, 0};
  if (e0 < E) {
#pragma unroll 4
    for (int b = seg; b < blocks; b += kJoinThreads / 4) {
      const float* p = parts + (int64_t)b * words + e0;
      const float4 v = *reinterpret_cast<const float4*>(p);
      const int4 w = *reinterpret_cast<const int4*>(p + pitch);
      s[0] += v.x; s[1] += v.y; s[2] += v.z; s[3] += v.w;
      c[0] += w.x; c[1] += w.y; c[2] += w.z; c[3] += w.w;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s[i] = quad_place_sum(s[i]);
    c[i] = quad_place_sum(c[i]);
  }
  n = quad_place_sum(n);
  if ((tid & 63) < 4) {
    valid[tid >> 6][tid & 3] = n;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sums[tid >> 6][(tid & 3) * 4 + i] = s[i];
      cnts[tid >> 6][(tid & 3) * 4 + i] = c[i];
    }
  }
  __syncthreads();
  if (tid >= kJoinExperts) return;
  double l = 0.0;
  int64_t total = 0, count = 0;
#pragma unroll
  for (int w = 0; w < kJoinWaves; ++w) {
    l += sums[w][tid];
    count += cnts[w][tid];
    total += (valid[w][0] + valid[w][1]) + (valid[w][2] + valid[w][3]);
  }
  const int e = blockIdx.x * kJoinExperts + tid;
  const double d = (double)total, w = total > 0 ? (double)E * (double)count / (d * d) : 0.0;
  l = total > 0 && e < E ? w * l : 0.0;
  if (e < E) {
    counts[e] = count;
    weight[e] = (float)w;
  }
#pragma unroll
  for (int o = 1; o < kJoinExperts; o <<= 1) l += __shfl_xor(l, o, 64);
  if (tid == 0) {
    if (gridDim.x == 1) {
      loss[0] = (float)l;
      return;
    }
    __hip_atomic_store(loss_part + blockIdx.x, l, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (__hip_atomic_fetch_add(ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1) {
      l = 0.0;
      for (unsigned i = 0; i < gridDim.x; ++i)
        l += __hip_atomic_load(loss_part + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      loss[0] = (float)l;
    }
  }
}

// U rows a group at a time; PAST: the gradient goes past the last-level cache, in whole 16 bytes
// (262144 x 256 bf16: the next call's partial sums 45 -> 37 us; single elements would take twice as long)
template <typename T, int V, int NJ, int G, bool PAST>
__global__ void __launch_bounds__(kBlThreads) balance_bwd_k(const T* __restrict__ x, int64_t stride, int64_t T_, int E,
                                                            const float* __restrict__ weight,
                                                            const float* __restrict__ g, const void* valid, int kind,
                                                            T* __restrict__ dx) {
  constexpr int N = NJ * V, U = N <= 8 ? 2 : 1, groups = kBlThreads / G;
  const int tid = threadIdx.x, lane = tid & (G - 1), group = tid / G;
  float w[N];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int e = (j * G + lane) * V;
#pragma unroll
    for (int q = 0; q < V; ++q) w[j * V + q] = e < E ? weight[e + q] : 0.f;
  }
  const float gr = g[0];
  for (int64_t t = (int64_t)blockIdx.x * groups * U + group; t < T_; t += (int64_t)gridDim.x * groups * U) {
    RowRaw<T, V, NJ, G> raw[U];
    float p[U][N], inv[U], dot[U];
    bool on[U];
    tokens_on<U>(valid, kind, t, groups, T_, on);
    bool any = false;
#pragma unroll
    for (int u = 0; u < U; ++u) any |= on[u];
    if (any) {
#pragma unroll
      for (int u = 0; u < U; ++u) {       // one that is not valid: its fellow's row in its place, unused
        const int64_t tu = on[u] ? t + u * groups : (on[0] ? t : t + (U - 1) * groups);
        raw[u].load(x + tu * stride, E, lane);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u].unpack(p[u]);
      rows_exp<U, V, NJ, G>(E, lane, p, inv);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        dot[u] = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) dot[u] += p[u][i] * w[i];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) dot[u] = group_sum(dot[u], G) * inv[u];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t tu = t + u * groups;
      const float c = on[u] ? gr * inv[u] : 0.f;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int e = (j * G + lane) * V;
        if (tu < T_ && e < E) {
          float v[V];
#pragma unroll
          for (int q = 0; q < V; ++q) v[q] = on[u] ? c * p[u][j * V + q] * (w[j * V + q] - dot[u]) : 0.f;
          store_n<T, V, PAST>(dx + tu * (int64_t)E + e, v);
        }
      }
    }
  }
}

struct RowPlan { int V, G, NJ; };

// V elements a load where rows and buffers allow 16-byte accesses, G lanes a row, NJ loads a lane.
// The vector unit bounds these kernels (about 9 issue slots an element, 5 more for each exchange of
// a reduction and 15 for a row, in every lane), so a lane takes up to 16 elements and G is what they
// leave (262144 x 256 bf16: partial sums 46 us with 16 lanes a row, 52 with 32; 100003 x 161 fp32: 18
// us with 16 lanes, 30 with 64).
static RowPlan plan_rows(int E, int64_t stride, const void* x, const void* y, int vec) {
  RowPlan r;
  r.V = (E % vec == 0 && stride % vec == 0 && (((uintptr_t)x | (uintptr_t)y) & 15) == 0) ? vec : 1;
  r.G = 1;
  while (16 * r.G < E) r.G <<= 1;
  r.NJ = (E + r.V * r.G - 1) / (r.V * r.G);
  if (r.V == 1) r.NJ = r.NJ <= 2 ? 2 : r.NJ <= 4 ? 4 : r.NJ <= 8 ? 8 : r.NJ <= 12 ? 12 : 16;
  return r;
}

}  // namespace hetu

using namespace hetu;

// Rows a block of the partial sums takes: as many blocks as keep the chip's waves busy (2 blocks of 8
// waves a CU; 1024 blocks gain the partial sums nothing and cost the join 2 us), but at least 2 rows a
// group of lanes, for each block costs E partial sums.
constexpr int kMaxParts = 512;
static int64_t balance_rows(int64_t T, int G) {
  const int64_t groups = kPartThreads / G;
  int64_t blocks = (T + groups * 2 - 1) / (groups * 2);
  // one block has no join: that is worth up to 4 rows a group (96 x 8: 4.5 us for both launches' 8)
  if (T <= groups * 4) blocks = 1;
  blocks = blocks < 1 ? 1 : (blocks > kMaxParts ? kMaxParts : blocks);
  return (T + blocks - 1) / blocks;
}

// calls f(V, NJ, G) as compile-time numbers for the plan: more than one lane a row have 9 to 16
// elements each
template <int N> struct Const { static constexpr int value = N; };
template <int V, int NJ, typename F>
static void with_group(int G, F f) {
  if (G == 1) f(Const<V>(), Const<NJ>(), Const<1>());
  if constexpr (V * NJ > 8) {
    if (G == 2) f(Const<V>(), Const<NJ>(), Const<2>());
    if (G == 4) f(Const<V>(), Const<NJ>(), Const<4>());
    if (G == 8) f(Const<V>(), Const<NJ>(), Const<8>());
    if (G == 16) f(Const<V>(), Const<NJ>(), Const<16>());
    if (G == 32) f(Const<V>(), Const<NJ>(), Const<32>());
    if (G == 64) f(Const<V>(), Const<NJ>(), Const<64>());
  }
}
template <int VEC, typename F>      // VEC: elements of 16 bytes
static void with_plan(const RowPlan& r, F f) {
  if (r.V == VEC) {
    if (r.NJ == 1) with_group<VEC, 1>(r.G, f);
    if (r.NJ == 2) with_group<VEC, 2>(r.G, f);
    if constexpr (VEC == 4) {
      if (r.NJ == 3) with_group<VEC, 3>(r.G, f);
      if (r.NJ == 4) with_group<VEC, 4>(r.G, f);
    }
  } else {
    if (r.NJ == 2) with_group<1, 2>(r.G, f);
    if (r.NJ == 4) with_group<1, 4>(r.G, f);
    if (r.NJ == 8) with_group<1, 8>(r.G, f);
    if (r.NJ == 12) with_group<1, 12>(r.G, f);
    if (r.NJ == 16) with_group<1, 16>(r.G, f);
  }
}

// number of 4-byte words of workspace (16-byte aligned) that hetu_moe_balance_fwd needs: the
// joining blocks' parts of the loss, their ticket, each block's sums and counts
HETU_API int64_t hetu_moe_balance_ws(int64_t T, int E) {
  if (T < 0 || E < 1 || E > kMaxExperts) return 0;
  const int64_t groups_least = kPartThreads / 64;
  int64_t parts = (T + groups_least * 2 - 1) / (groups_least * 2);
  parts = parts < 1 ? 1 : (parts > kMaxParts ? kMaxParts : parts);
  return 2 * (kMaxExperts / kJoinExperts) + 4 + parts * (2 * part_pitch(E) + 4);
}

// counts: a buffer of E int64, then (as fp32) E weights and the loss
HETU_API int hetu_moe_balance_fwd(const void* x, int64_t stride, int64_t T, int E, const int64_t* idx, int k,
                                  const void* valid, int kind, int64_t* counts, void* ws, int is_bf16,
                                  hipStream_t st) {
  if (T < 0 || E < 1 || E > kMaxExperts || k < 1) return (int)hipErrorInvalidValue;
  const RowPlan r = plan_rows(E, stride, x, nullptr, is_bf16 ? 8 : 4);
  const int64_t rows = T > 0 ? balance_rows(T, r.G) : 1;
  const int blocks = T > 0 ? (int)((T + rows - 1) / rows) : 1;
  float *weight = (float*)(counts + E), *loss = weight + E;
  double* part = (double*)ws;
  unsigned* ticket = (unsigned*)(part + kMaxExperts / kJoinExperts);
  float* sums = (float*)(ticket + 4);
  size_t lds = sizeof(int) * (size_t)(E + 1 + kPartWaves * E);
  if (lds < sizeof(double) * kPartWaves * 4) lds = sizeof(double) * kPartWaves * 4;
  const auto go = [&](auto zero, auto v, auto nj, auto g) {
    typedef decltype(zero) TT;
    hipLaunchKernelGGL((balance_part_k<TT, decltype(v)::value, decltype(nj)::value, decltype(g)::value>), dim3(blocks),
                       dim3(kPartThreads), lds, st, (const TT*)x, stride, T, E, idx, k, valid, kind, rows, sums, ticket, counts);
  };
  if (is_bf16) with_plan<8>(r, [&](auto v, auto nj, auto g) { go(bf16(), v, nj, g); });
  else with_plan<4>(r, [&](auto v, auto nj, auto g) { go(0.f, v, nj, g); });
  HETU_LAUNCH_CHECK();
  if (blocks > 1)
    hipLaunchKernelGGL(balance_join_k, dim3((E + kJoinExperts - 1) / kJoinExperts), dim3(kJoinThreads), 0, st, sums,
                     blocks, E, counts, weight, loss, part, ticket);
  HETU_LAUNCH_CHECK();
  return 0;
}

HETU_API int hetu_moe_balance_bwd(const void* x, int64_t stride, int64_t T, int E, const float* weight, const float* grad,
                                  const void* valid, int kind, void* dx, int is_bf16, hipStream_t st) {
  if (T <= 0) return 0;
  if (E < 1 || E > kMaxExperts) return (int)hipErrorInvalidValue;
  const RowPlan r = plan_rows(E, stride, x, dx, is_bf16 ? 8 : 4);
  const int64_t groups = kBlThreads / r.G * (r.NJ * r.V <= 8 ? 2 : 1);
  const int64_t want = (T + groups - 1) / groups;
  // 8 blocks a CU loop over the rows, for each block reads the weights: 262144 x 256 bf16 57 us, with
  // 8192 blocks 75, with one for each of its rows 122
  const dim3 grid((unsigned)(want < 2048 ? want : 2048));
  const bool past = 2 * T * E * (is_bf16 ? 2 : 4) >= kLastCacheBytes;
  const auto go = [&](auto zero, auto v, auto nj, auto g) {
    typedef decltype(zero) TT;
    constexpr int V = decltype(v)::value, NJ = decltype(nj)::value, G = decltype(g)::value;
    if (V > 1 && past)
      hipLaunchKernelGGL((balance_bwd_k<TT, V, NJ, G, (V > 1)>), grid, dim3(kBlThreads), 0, st, (const TT*)x, stride, T,
                         E, weight, grad, valid, kind, (TT*)dx);
    else
      hipLaunchKernelGGL((balance_bwd_k<TT, V, NJ, G, false>), grid, dim3(kBlThreads), 0, st, (const TT*)x, stride, T, E,
                         weight, grad, valid, kind, (TT*)dx);
  };
  if (is_bf16) with_plan<8>(r, [&](auto v, auto nj, auto g) { go(bf16(), v, nj, g); });
  else with_plan<4>(r, [&](auto v, auto nj, auto g) { go(0.f, v, nj, g); });
  HETU_LAUNCH_CHECK();
  return 0;
}
