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
#include "common.h"

namespace hetu {

struct Adam8Args {
  // omb..: one less beta, one less its power, as the caller's 64 bits give them (1 - 0.999 in
  // 32 bits is off by 1e-5 of itself)
  float lr, beta1, beta2, omb1, omb2, omb1t, omb2t, eps, wd, gscale;
  // {lr, -, -, gscale, step, omb1t, omb2t} on the device, or null: a captured step's own.  The
  // step number moves the seed, as the caller moves it without dyn.
  const float* dyn;
  uint64_t seed;
};

constexpr int kBlock8 = 256;   // elements that share a scale: 4 a lane, one wave

// a 32-bit mix (multiply, xor-shift) of the element's index and the step's seed: the low half
// rounds m, the high half v
__device__ __forceinline__ unsigned round_bits(unsigned idx, unsigned seed) {
  unsigned h = idx * 0x9E3779B1u + seed;
  h = (h ^ (h >> 16)) * 0x7FEB352Du;
  h = (h ^ (h >> 15)) * 0x846CA68Bu;
  return h ^ (h >> 16);
}

// |y| (finite, below the format's largest power of two) as a code of MANT mantissa bits, exponent
// bias BIAS: r16 is added below the last bit kept (half a unit of r16 on top, so that 16 bits
// round without bias), in the mantissa of a normal, in fixed point where the code is a subnormal
template <int MANT, int BIAS>
__device__ __forceinline__ unsigned encode8(float y, unsigned r16) {
  constexpr int CUT = 23 - MANT;
  const unsigned r = (r16 << (CUT - 16)) | (1u << (CUT - 17));
  const unsigned normal = ((__float_as_uint(y) + r) >> CUT) - ((127u - BIAS) << MANT);
  const float least = __uint_as_float((unsigned)(128 - BIAS) << 23);            // 2^(1 - BIAS)
  const float units = __uint_as_float((unsigned)(127 + BIAS + 22) << 23);       // 2^(BIAS + 22)
  const unsigned small = ((unsigned)(int)(y * units) + r) >> CUT;
  return y < least ? small : normal;
}

__device__ __forceinline__ float decode_m(unsigned c) {
  return __builtin_amdgcn_cvt_f32_fp8((int)c, 0);
}
__device__ __forceinline__ float decode_v(unsigned c) {
  return __builtin_amdgcn_cvt_f32_bf8((int)c, 0);
}

// One wave a block of 256 elements, 4 a lane: the block's largest exponents are one reduction
// over the wave.  VEC: every buffer lets a lane move its 4 elements at once.
template <bool SHADOW, bool VEC>
__global__ void __launch_bounds__(256) adamw8_k(float* __restrict__ p, const float* __restrict__ g,
                                                 unsigned char* __restrict__ mc, unsigned char* __restrict__ vc,
                                                 float* __restrict__ ms, float* __restrict__ vs,
                                                 unsigned short* __restrict__ shadow, int64_t n, int64_t nb,
                                                 Adam8Args a) {
#pragma clang fp contract(off)   // the moments are rounded operation by operation, as documented
  const int lane = threadIdx.x & 63;
  const int64_t wave = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), waves = (int64_t)gridDim.x * 4;
  float lr = a.lr, c1 = a.omb1t, c2 = a.omb2t, gsc = a.gscale;
  uint64_t key = a.seed;
  if (a.dyn) {
    lr = a.dyn[0]; gsc = a.dyn[3]; c1 = a.dyn[5]; c2 = a.dyn[6];
    key += (uint64_t)a.dyn[4] * kRngMix;
  }
  const unsigned seed = (unsigned)key ^ (unsigned)(key >> 32);
  for (int64_t b = wave; b < nb; b += waves) {
    const int64_t i0 = b * kBlock8 + lane * 4;
    const int cnt = n - i0 >= 4 ? 4 : (n > i0 ? (int)(n - i0) : 0);
    float pv[4] = {0, 0, 0, 0}, gv[4] = {0, 0, 0, 0}, m[4], v[4];
    unsigned mq = 0, vq = 0;
    if (VEC && cnt == 4) {
      const float4 x = *reinterpret_cast<const float4*>(p + i0), y = *reinterpret_cast<const float4*>(g + i0);
      pv[0] = x.x; pv[1] = x.y; pv[2] = x.z; pv[3] = x.w;
      gv[0] = y.x; gv[1] = y.y; gv[2] = y.z; gv[3] = y.w;
      mq = *reinterpret_cast<const unsigned*>(mc + i0);
      vq = *reinterpret_cast<const unsigned*>(vc + i0);
    } else {
      for (int k = 0; k < cnt; ++k) {
        pv[k] = p[i0 + k];
        gv[k] = g[i0 + k];
        mq |= (unsigned)mc[i0 + k] << (8 * k);
        vq |= (unsigned)vc[i0 + k] << (8 * k);
      }
    }
    const float msc = ms[b], vsc = vs[b];
    float mtop = 0.f, vtop = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float gr = gv[k] * gsc;
      m[k] = a.beta1 * (decode_m((mq >> (8 * k)) & 255u) * msc) + a.omb1 * gr;
      v[k] = a.beta2 * (decode_v((vq >> (8 * k)) & 255u) * vsc) + a.omb2 * gr * gr;
      const float u = (m[k] / c1) / (sqrtf(v[k] / c2) + a.eps);
      pv[k] -= lr * (u + a.wd * pv[k]);
      if (k >= cnt) m[k] = v[k] = 0.f;
      const float am = fabsf(m[k]);
      if (am < INFINITY) mtop = fmaxf(mtop, am);
      if (v[k] < INFINITY) vtop = fmaxf(vtop, v[k]);
    }
    mtop = wave_max(mtop);
    vtop = wave_max(vtop);
    // 2^(floor(log2(largest)) - 7), - 14, not below the smallest normal
    int me = (int)(__float_as_uint(mtop) >> 23) - 7, ve = (int)(__float_as_uint(vtop) >> 23) - 14;
    me = me < 1 ? 1 : me;
    ve = ve < 1 ? 1 : ve;
    const float minv = __uint_as_float((unsigned)(254 - me) << 23), vinv = __uint_as_float((unsigned)(254 - ve) << 23);
    mq = vq = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const unsigned r = round_bits((unsigned)(i0 + k), seed);
      const float am = fabsf(m[k]);
      unsigned cm = am < INFINITY ? encode8<3, 7>(am * minv, r & 0xFFFFu) : 0x7Fu;
      unsigned cv = v[k] < INFINITY ? encode8<2, 15>(v[k] * vinv, r >> 16) : (v[k] != v[k] ? 0x7Fu : 0x7Cu);
      if (m[k] < 0.f) cm |= 0x80u;
      if (v[k] > 0.f && cv == 0u) cv = 1u;
      mq |= cm << (8 * k);
      vq |= cv << (8 * k);
    }
    if (VEC && cnt == 4) {
      *reinterpret_cast<float4*>(p + i0) = make_float4(pv[0], pv[1], pv[2], pv[3]);
      *reinterpret_cast<unsigned*>(mc + i0) = mq;
      *reinterpret_cast<unsigned*>(vc + i0) = vq;
      if (SHADOW)
        *reinterpret_cast<uint2*>(shadow + i0) =
            make_uint2((unsigned)f_to_bf16_bits(pv[0]) | ((unsigned)f_to_bf16_bits(pv[1]) << 16),
                       (unsigned)f_to_bf16_bits(pv[2]) | ((unsigned)f_to_bf16_bits(pv[3]) << 16));
    } else {
      for (int k = 0; k < cnt; ++k) {
        p[i0 + k] = pv[k];
        mc[i0 + k] = (unsigned char)(mq >> (8 * k));
        vc[i0 + k] = (unsigned char)(vq >> (8 * k));
        if (SHADOW) shadow[i0 + k] = f_to_bf16_bits(pv[k]);
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
  const int64_t want = (nb + 3) / 4;
  const dim3 grid((unsigned)(want < 2048 ? want : 2048));
  const bool vec = (((uintptr_t)p | (uintptr_t)g) & 15) == 0 && (((uintptr_t)m | (uintptr_t)v) & 3) == 0 &&
                   ((uintptr_t)shadow & 7) == 0;
#define GO(S, V) hipLaunchKernelGGL((adamw8_k<S, V>), grid, dim3(256), 0, st, p, g, (unsigned char*)m, (unsigned char*)v, \
                                    ms, vs, (unsigned short*)shadow, n, nb, a)
  if (shadow) { if (vec) GO(true, true); else GO(true, false); }
  else { if (vec) GO(false, true); else GO(false, false); }
#undef GO
  HETU_LAUNCH_CHECK();
  return 0;
}
