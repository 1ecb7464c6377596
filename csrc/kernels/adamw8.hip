// AdamW over a flat fp32 buffer with both moments held in 8 bits.
//
//   m' = beta1 m + (1 - beta1) g        v' = beta2 v + (1 - beta2) g^2
//   p -= lr ((m' / (1 - beta1^t)) / (sqrt(v' / (1 - beta2^t)) + eps) + wd p)
//
// The update uses m' and v' in 32 bits; what is kept of them for the next step is one byte each
// and one fp32 scale for each 256 elements: the first moment as e4m3 (4 exponent, 3 mantissa
// bits), the second as e5m2.  Why these choices:
//   * The second moment moves by (1 - beta2) of itself a step, 0.1 %, far below half a step of
//     any 8-bit grid: rounded to the nearest it would never move again.  Both are rounded up or
//     down at random, with the probability of the part cut off, so that the mean is exact.
//   * The scale is a power of two, so that a block's grid stays where it is from step to step and
//     a stored value lies on it exactly: a small change d then costs a variance of d * (step of
//     the grid), not of a step squared.  It also makes decoding exact in 32 bits.
//   * Squares need the range: e5m2 spans 2^30 below a block's largest v, 2^15 in sqrt(v).  A v'
//     above 0 is never stored as 0, for m / (sqrt(0) + eps) would be a step without measure.
//   * The largest of a block is scaled into [128, 256) of e4m3's 448 and [2^14, 2^15) of e5m2's
//     57344: rounding up cannot overflow.
// NaN and Inf in a gradient stay with their elements (the e4m3 NaN, the e5m2 Inf or NaN), as with
// 32-bit moments: the scale is taken over the finite elements of the block.
#include "wave_ops.h"

namespace hetu {

struct Adam8Args {
  // omb..: one less beta, one less its power, as the caller's 64 bits give them (1 - 0.999 in
  // 32 bits is off by 1e-5 of itself)
  float lr, beta1, beta2, omb1, omb2, omb1t, omb2t, eps, wd, gscale;
  // {lr, -, -, gscale, step, omb1t, omb2t} on the device, or null: a captured step's own.  The
  // step number, modulo the 2^24 that fp32 holds, moves the seed, as the caller moves it without dyn.
  const float* dyn;
  uint64_t seed;
};

constexpr int kBlock8 = 256;   // elements that share a scale: 8 a lane, half a wave
constexpr int kLane8 = 8;

// a 32-bit mix (multiply, xor-shift; the multipliers and shifts of C. Wellons, "Prospecting for Hash
// Functions", 2018) of a number made from the element's index and the step's seed: the low half
// rounds m, the high half v
__device__ __forceinline__ unsigned round_bits(unsigned h) {
  h = (h ^ (h >> 16)) * 0x7FEB352Du;
  h = (h ^ (h >> 15)) * 0x846CA68Bu;
  return h ^ (h >> 16);
}

// Codes in the top byte of a word (a sign bit of 0).  The value is scaled so that the format's
// smallest normal number becomes fp32's: its bits then are the code's, the subnormals' too, with
// the rest of the mantissa below.  To these the 16 random bits are added, aligned with the highest
// bit cut off, and half a unit of them, so that 16 bits round without bias.
//   e4m3 (bias 7): x 2^(7 - se), the code from bit 20 up;  e5m2 (bias 15): x 2^(15 - se), bit 21
// where 2^(se - 127) is the block's scale.
__device__ __forceinline__ unsigned encode_m(float m, int se, unsigned h) {
  const unsigned bits = __float_as_uint(__builtin_amdgcn_ldexpf(fabsf(m), 7 - se));
  const unsigned t = (bits + (((h << 4) & 0xFFFF0u) | 8u)) << 4;
  return t | (__float_as_uint(m) & 0x80000000u);
}
__device__ __forceinline__ unsigned encode_v(float v, int se, unsigned h) {
  const unsigned bits = __float_as_uint(__builtin_amdgcn_ldexpf(v, 15 - se));
  const unsigned t = (bits + (((h >> 11) & 0x1FFFE0u) | 16u)) << 3;
  const unsigned least = v > 0.f ? 1u << 24 : 0u;
  return t > least ? t : least;
}

// the top bytes of four words as one
__device__ __forceinline__ unsigned top_bytes(unsigned a, unsigned b, unsigned c, unsigned d) {
  const unsigned lo = __builtin_amdgcn_perm(b, a, 0x0C0C0703u), hi = __builtin_amdgcn_perm(d, c, 0x07030C0Cu);
  return lo | hi;
}

// Half a wave a block of 256 elements, 8 a lane: the block's largest exponents are five lane
// exchanges.  VEC: every buffer lets a lane move its elements in 16 and 8 bytes at once.
//
// What bounds it: 16 bytes an element to move (18 with the copy), and about 60 issue slots of the
// vector unit, where 128 would take as long as the memory.  So no division and no exact root in
// the update, where a unit of fp32 does not matter (v_rcp_f32, v_sqrt_f32: 1 unit each; the root
// of a v below 2^-126 is 0, which an eps of 1e-12 or more does not feel).
template <bool SHADOW, bool VEC>
__global__ void __launch_bounds__(256) adamw8_k(float* __restrict__ p, const float* __restrict__ g,
                                                 unsigned char* __restrict__ mc, unsigned char* __restrict__ vc,
                                                 float* __restrict__ ms, float* __restrict__ vs,
                                                 unsigned short* __restrict__ shadow, int64_t n, int64_t nb,
                                                 Adam8Args a) {
#pragma clang fp contract(off)   // the moments are rounded operation by operation, as documented
  constexpr int N = kLane8;
  const int lane = threadIdx.x & 31;
  const int64_t half = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), halves = (int64_t)gridDim.x * 8;
  float lr = a.lr, c1 = a.omb1t, c2 = a.omb2t, gsc = a.gscale;
  uint64_t key = a.seed;
  if (a.dyn) {
    lr = a.dyn[0]; gsc = a.dyn[3]; c1 = a.dyn[5]; c2 = a.dyn[6];
    key += ((uint64_t)a.dyn[4] & 0xFFFFFFu) * kRngMix;
  }
  const float r1 = 1.f / c1, r2 = 1.f / c2;
  const unsigned seed = (unsigned)key ^ (unsigned)(key >> 32);
  for (int64_t b = half; b < nb; b += halves) {
    const int64_t i0 = b * kBlock8 + lane * N;
    const int cnt = n - i0 >= N ? N : (n > i0 ? (int)(n - i0) : 0);
    float pv[N], gv[N], m[N], v[N];
    unsigned mq[2] = {0, 0}, vq[2] = {0, 0};
    if (VEC && cnt == N) {
      load_vec<float>(p + i0, reinterpret_cast<float(&)[4]>(pv[0]));
      load_vec<float>(p + i0 + 4, reinterpret_cast<float(&)[4]>(pv[4]));
      load_vec<float>(g + i0, reinterpret_cast<float(&)[4]>(gv[0]));
      load_vec<float>(g + i0 + 4, reinterpret_cast<float(&)[4]>(gv[4]));
      const uint2 x = *reinterpret_cast<const uint2*>(mc + i0), y = *reinterpret_cast<const uint2*>(vc + i0);
      mq[0] = x.x; mq[1] = x.y;
      vq[0] = y.x; vq[1] = y.y;
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        pv[k] = k < cnt ? p[i0 + k] : 0.f;
        gv[k] = k < cnt ? g[i0 + k] : 0.f;
        mq[k >> 2] |= (unsigned)(k < cnt ? mc[i0 + k] : 0) << (8 * (k & 3));
        vq[k >> 2] |= (unsigned)(k < cnt ? vc[i0 + k] : 0) << (8 * (k & 3));
      }
    }
    // beta times the scale, a power of two: exact
    const float bm = a.beta1 * ms[b], bv = a.beta2 * vs[b];
    unsigned mtop = 0, vtop = 0;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int w = k >> 2;
      const float gr = gv[k] * gsc;
      const auto dm = (k & 2) ? __builtin_amdgcn_cvt_pk_f32_fp8((int)mq[w], true) : __builtin_amdgcn_cvt_pk_f32_fp8((int)mq[w], false);
      const auto dv = (k & 2) ? __builtin_amdgcn_cvt_pk_f32_bf8((int)vq[w], true) : __builtin_amdgcn_cvt_pk_f32_bf8((int)vq[w], false);
      m[k] = dm[k & 1] * bm + a.omb1 * gr;
      v[k] = dv[k & 1] * bv + a.omb2 * gr * gr;
      const float root = __builtin_amdgcn_sqrtf(v[k] * r2) + a.eps;
      const float u = m[k] * r1 * __builtin_amdgcn_rcpf(root);
      pv[k] = __builtin_fmaf(-lr, __builtin_fmaf(a.wd, pv[k], u), pv[k]);
      const unsigned am = __float_as_uint(m[k]) & 0x7FFFFFFFu, av = __float_as_uint(v[k]);
      mtop = mtop > am ? mtop : am;
      vtop = vtop > av ? vtop : av;
    }
    const auto larger = [](unsigned x, unsigned y) { return x > y ? x : y; };
    mtop = group_join(mtop, 32, larger);
    vtop = group_join(vtop, 32, larger);
    const bool odd = mtop >= 0x7F800000u || vtop >= 0x7F800000u;
    if (odd) {                     // an Inf or NaN in the block: the largest of the others
      mtop = vtop = 0;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const unsigned am = __float_as_uint(m[k]) & 0x7FFFFFFFu, av = __float_as_uint(v[k]) & 0x7FFFFFFFu;
        if (am < 0x7F800000u) mtop = larger(mtop, am);
        if (av < 0x7F800000u) vtop = larger(vtop, av);
      }
      mtop = group_join(mtop, 32, larger);
      vtop = group_join(vtop, 32, larger);
    }
    // the scales 2^(floor(log2(largest)) - 7), - 14, not below the smallest normal number
    int me = (int)(mtop >> 23) - 7, ve = (int)(vtop >> 23) - 14;
    me = me < 1 ? 1 : me;
    ve = ve < 1 ? 1 : ve;
    unsigned em[N], ev[N];
    const unsigned h0 = (unsigned)i0 * 0x9E3779B1u + seed;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const unsigned h = round_bits(h0 + (unsigned)k * 0x9E3779B1u);
      em[k] = encode_m(m[k], me, h);
      ev[k] = encode_v(v[k], ve, h);
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      mq[w] = top_bytes(em[4 * w], em[4 * w + 1], em[4 * w + 2], em[4 * w + 3]);
      vq[w] = top_bytes(ev[4 * w], ev[4 * w + 1], ev[4 * w + 2], ev[4 * w + 3]);
    }
    if (VEC && cnt == N) {
      store_vec<float>(p + i0, reinterpret_cast<const float(&)[4]>(pv[0]));
      store_vec<float>(p + i0 + 4, reinterpret_cast<const float(&)[4]>(pv[4]));
      *reinterpret_cast<uint2*>(mc + i0) = make_uint2(mq[0], mq[1]);
      *reinterpret_cast<uint2*>(vc + i0) = make_uint2(vq[0], vq[1]);
      if (SHADOW) store_vec<bf16>(reinterpret_cast<bf16*>(shadow) + i0, pv);
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        if (k < cnt) {
          p[i0 + k] = pv[k];
          mc[i0 + k] = (unsigned char)(em[k] >> 24);
          vc[i0 + k] = (unsigned char)(ev[k] >> 24);
          if (SHADOW) shadow[i0 + k] = f_to_bf16_bits(pv[k]);
        }
      }
    }
    if (odd) {                     // their codes, over what the arithmetic above made of them
#pragma unroll
      for (int k = 0; k < N; ++k) {
        if (k < cnt && !(fabsf(m[k]) < INFINITY)) mc[i0 + k] = 0x7F;
        if (k < cnt && !(v[k] < INFINITY)) vc[i0 + k] = v[k] != v[k] ? 0x7F : 0x7C;
      }
    }
    if (lane == 0) {
      ms[b] = __uint_as_float((unsigned)me << 23);
      vs[b] = __uint_as_float((unsigned)ve << 23);
    }
  }
}

}  // namespace hetu

using namespace hetu;

HETU_API int hetu_adamw8(float* p, const float* g, void* m, void* v, float* ms, float* vs, void* shadow, int64_t n,
                         float lr, float beta1, float beta2, float omb1, float omb2, float omb1t, float omb2t,
                         float eps, float wd, float gscale, const float* dyn, int64_t seed, hipStream_t st) {
  if (n <= 0) return 0;
  const int64_t nb = (n + kBlock8 - 1) / kBlock8;
  const Adam8Args a = {lr, beta1, beta2, omb1, omb2, omb1t, omb2t, eps, wd, gscale, dyn, (uint64_t)seed};
  // a block of 8 half waves for each 8 blocks of elements: 109 M weights take 345 us, with 2048 that
  // loop over them 389 (they load and store in step), with non-temporal accesses 395 to 405
  const int64_t want = (nb + 7) / 8;
  const dim3 grid((unsigned)(want < 1 << 22 ? want : 1 << 22));     // 8.6e9 elements; more: a loop
  const bool vec = (((uintptr_t)p | (uintptr_t)g) & 15) == 0 && (((uintptr_t)m | (uintptr_t)v) & 7) == 0 &&
                   ((uintptr_t)shadow & 15) == 0;
#define GO(S, V) hipLaunchKernelGGL((adamw8_k<S, V>), grid, dim3(256), 0, st, p, g, (unsigned char*)m, (unsigned char*)v, \
                                    ms, vs, (unsigned short*)shadow, n, nb, a)
  if (shadow) { if (vec) GO(true, true); else GO(true, false); }
  else { if (vec) GO(false, true); else GO(false, false); }
#undef GO
  HETU_LAUNCH_CHECK();
  return 0;
}
