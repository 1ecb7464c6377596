// Reductions over aligned groups of lanes of a wave (2, 4, .. 64 lanes; every lane gets the
// result), by lane exchanges of the vector unit instead of LDS permutes: lanes 1 and 2 apart within
// a quad, then quads and halves of a row of 16 mirrored, then rows and halves of the wave swapped
// (v_permlane16_swap, v_permlane32_swap).
#pragma once
#include "common.h"

namespace hetu {

// ---- 16-byte accesses that leave the last-level cache alone -------------------------------------
// What a kernel writes stays in that cache (256 MB) as dirty lines, which the next kernel's reads
// have to push out.  Where a result cannot be found there anyway, for it and its input are larger than
// the cache, it goes past it.  (Known at compile time: a branch between the two kinds is merged into
// one plain access.)
constexpr int64_t kLastCacheBytes = 256ll << 20;
typedef unsigned Raw __attribute__((ext_vector_type(4)));

template <bool PAST>
__device__ __forceinline__ Raw load_raw(const void* p) {
  const Raw* q = reinterpret_cast<const Raw*>(p);
  if constexpr (PAST) return __builtin_nontemporal_load(q);
  else return *q;
}
template <bool PAST>
__device__ __forceinline__ void store_raw(void* p, const Raw& v) {
  Raw* q = reinterpret_cast<Raw*>(p);
  if constexpr (PAST) __builtin_nontemporal_store(v, q);
  else *q = v;
}
__device__ __forceinline__ Raw pack_raw(const float (&v)[4]) {
  return Raw{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
}
__device__ __forceinline__ Raw pack_raw(const float (&v)[8]) {
  Raw r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = (unsigned)f_to_bf16_bits(v[2 * i]) | ((unsigned)f_to_bf16_bits(v[2 * i + 1]) << 16);
  return r;
}

// ---- reductions -------------------------------------------------------------------------------

template <int CTRL>
__device__ __forceinline__ unsigned dpp(unsigned v) {
  return (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xF, 0xF, false);
}

// joins v with the value of the lane (or of an equal group of lanes) that step O pairs it with:
// after steps 1, 2, .. G / 2 all lanes of a group of G hold the same
template <int O, typename F>
__device__ __forceinline__ unsigned lane_join(unsigned v, F f) {
  if constexpr (O == 1) return f(v, dpp<0xB1>(v));         // quad_perm 1 0 3 2
  else if constexpr (O == 2) return f(v, dpp<0x4E>(v));    // quad_perm 2 3 0 1
  else if constexpr (O == 4) return f(v, dpp<0x141>(v));   // row_half_mirror: the other quad
  else if constexpr (O == 8) return f(v, dpp<0x140>(v));   // row_mirror: the other half row
  else if constexpr (O == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return f(r[0], r[1]);
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return f(r[0], r[1]);
  }
}

template <typename F>
__device__ __forceinline__ unsigned group_join(unsigned v, int G, F f) {
  if (G > 1) v = lane_join<1>(v, f);
  if (G > 2) v = lane_join<2>(v, f);
  if (G > 4) v = lane_join<4>(v, f);
  if (G > 8) v = lane_join<8>(v, f);
  if (G > 16) v = lane_join<16>(v, f);
  if (G > 32) v = lane_join<32>(v, f);
  return v;
}

__device__ __forceinline__ float group_max(float v, int G) {
  return __uint_as_float(group_join(__float_as_uint(v), G, [](unsigned a, unsigned b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
}
// (v as it is: where the compiler may fuse v's last product into the first sum, lanes differ by a rounding)
__device__ __forceinline__ float group_sum(float v, int G) {
#pragma clang fp contract(off)
  return __uint_as_float(group_join(__float_as_uint(v), G, [](unsigned a, unsigned b) {
#pragma clang fp contract(off)
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}

// sum over the lanes of a wave with the same place in their group of G
template <int G>
__device__ __forceinline__ float place_sum(float v) {
#pragma clang fp contract(off)
  const auto add = [](unsigned a, unsigned b) {
#pragma clang fp contract(off)
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  };
  unsigned b = __float_as_uint(v);
  if constexpr (G < 2) b = lane_join<1>(b, add);
  if constexpr (G < 4) b = lane_join<2>(b, add);
  if constexpr (G < 16) b = add(b, dpp<0x128>(b));       // row_ror:8
  if constexpr (G < 8) b = add(b, dpp<0x124>(b));        // row_ror:4
  if constexpr (G < 32) b = lane_join<16>(b, add);
  if constexpr (G < 64) b = lane_join<32>(b, add);
  return __uint_as_float(b);
}

// sum over the lanes with the same place in their quad (16 of a wave), of a 64-bit number or double
template <typename T>
__device__ __forceinline__ T quad_place_sum(T v) {
  static_assert(sizeof(T) == 8, "two words");
  const auto pair = [](unsigned lo, unsigned hi) {
    const uint64_t b = ((uint64_t)hi << 32) | lo;
    T r;
    __builtin_memcpy(&r, &b, 8);
    return r;
  };
  const auto words = [](T x) {
    uint64_t b;
    __builtin_memcpy(&b, &x, 8);
    return b;
  };
  uint64_t b = words(v);
  v += pair(dpp<0x128>((unsigned)b), dpp<0x128>((unsigned)(b >> 32)));      // row_ror:8
  b = words(v);
  v += pair(dpp<0x124>((unsigned)b), dpp<0x124>((unsigned)(b >> 32)));      // row_ror:4
  b = words(v);
  const auto l = __builtin_amdgcn_permlane16_swap((unsigned)b, (unsigned)b, false, false);
  const auto h = __builtin_amdgcn_permlane16_swap((unsigned)(b >> 32), (unsigned)(b >> 32), false, false);
  v = pair(l[0], h[0]) + pair(l[1], h[1]);
  b = words(v);
  const auto l2 = __builtin_amdgcn_permlane32_swap((unsigned)b, (unsigned)b, false, false);
  const auto h2 = __builtin_amdgcn_permlane32_swap((unsigned)(b >> 32), (unsigned)(b >> 32), false, false);
  return pair(l2[0], h2[0]) + pair(l2[1], h2[1]);
}

}  // namespace hetu
