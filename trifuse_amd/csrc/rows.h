// Rows of storage elements in a team of lanes' registers: loads and stores of
// eight elements, sums and maxima over the team, and 8-bit codes (residual.hip
// has their definition).
#pragma once

#include "tfm_device.h"

namespace tfm {

// Eight storage elements, as loaded.
struct Vec8 {
  uint32_t w[4];
};

// Elements [0, n) of a vector of eight (n >= 8: all). UNALIGNED: rows start
// at any element and the last vector may be partial.
template <bool UNALIGNED>
__device__ __forceinline__ Vec8 load8(const uint16_t* p, int n) {
  Vec8 v{{0, 0, 0, 0}};
  if constexpr (!UNALIGNED) {
    if (n > 0) {
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      v = Vec8{{u.x, u.y, u.z, u.w}};
    }
  } else if (n >= 8) {
    __builtin_memcpy(v.w, p, 16);
  } else {
#pragma unroll
    for (int j = 0; j < 7; ++j)
      if (j < n) v.w[j / 2] |= (uint32_t)p[j] << (16 * (j & 1));
  }
  return v;
}

template <bool UNALIGNED>
__device__ __forceinline__ void store8(uint16_t* p, const Vec8& v, int n) {
  if constexpr (!UNALIGNED) {
    if (n > 0) *reinterpret_cast<uint4*>(p) = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
  } else if (n >= 8) {
    __builtin_memcpy(p, v.w, 16);
  } else {
#pragma unroll
    for (int j = 0; j < 7; ++j)
      if (j < n) p[j] = (uint16_t)(v.w[j / 2] >> (16 * (j & 1)));
  }
}

template <bool UNALIGNED>
__device__ __forceinline__ void store_codes8(int8_t* p, uint2 v, int n) {
  if constexpr (!UNALIGNED) {
    if (n > 0) *reinterpret_cast<uint2*>(p) = v;
  } else if (n >= 8) {
    __builtin_memcpy(p, &v, 8);
  } else {
#pragma unroll
    for (int j = 0; j < 7; ++j)
      if (j < n) p[j] = (int8_t)((j < 4 ? v.x : v.y) >> (8 * (j & 3)));
  }
}

template <bool F16>
__device__ __forceinline__ float elem(const Vec8& v, int j) {
  return j & 1 ? hi_st<F16>(v.w[j / 2]) : lo_st<F16>(v.w[j / 2]);
}

// Sum of one value per lane over a team of TEAM lanes; every lane gets it.
// `part` (TEAM / 64 floats of LDS, one array per call site) joins the waves.
template <int TEAM>
__device__ __forceinline__ float team_sum(float v, float* part) {
  v = wave_tree_sum64(v);
  const float s = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
  if constexpr (TEAM == 64) return s;
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  float total = part[0];
#pragma unroll
  for (int w = 1; w < TEAM / 64; ++w) total += part[w];
  return total;
}

template <int CTRL, int ROW_MASK>
__device__ __forceinline__ uint32_t dpp_umax(uint32_t v) {
  const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROW_MASK, 0xf, false);
  return v > o ? v : o;
}

template <int TEAM>
__device__ __forceinline__ uint32_t team_umax(uint32_t v, uint32_t* part) {
  v = dpp_umax<0xb1, 0xf>(v);
  v = dpp_umax<0x4e, 0xf>(v);
  v = dpp_umax<0x141, 0xf>(v);
  v = dpp_umax<0x140, 0xf>(v);
  v = dpp_umax<0x142, 0xa>(v);
  v = dpp_umax<0x143, 0xc>(v);
  const uint32_t m = (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
  if constexpr (TEAM == 64) return m;
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
  __syncthreads();
  uint32_t best = part[0];
#pragma unroll
  for (int w = 1; w < TEAM / 64; ++w) best = best > part[w] ? best : part[w];
  return best;
}

// A row's scale and the factor its values take before rounding, from the
// bits of max|x| (as integers they order like the magnitudes, NaN on top).
struct RowScale {
  float scale, factor;
  bool finite;
};
__device__ __forceinline__ RowScale row_scale(uint32_t amax_bits) {
  RowScale r;
  r.finite = amax_bits < 0x7f800000u;
  const float a = fmaxf(__uint_as_float(amax_bits), 0x1p-100f);
  r.scale = r.finite ? a / 127.0f : __uint_as_float(0x7fc00000u);
  r.factor = 127.0f / a;
  return r;
}

// Eight codes. v * factor + 1.5 * 2^23 rounds half to even at its last bit and the
// sum's low byte is the code; the product is rounded first, as the codes are
// defined, so the two are not contracted into one operation.
__device__ __forceinline__ uint2 codes8(const float* v, const RowScale& r) {
#pragma clang fp contract(off)
  uint32_t b[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) b[j] = __float_as_uint(v[j] * r.factor + 12582912.0f);
  uint2 c;
  c.x = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400u), __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), 0x05040100u);
  c.y = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[7], b[6], 0x0c0c0400u), __builtin_amdgcn_perm(b[5], b[4], 0x0c0c0400u), 0x05040100u);
  return r.finite ? c : make_uint2(0, 0);
}

// Bits of the largest magnitude of a vector's elements, two at a time: as
// integers the magnitudes of either storage type order like themselves, NaN on top.
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u16x2_t abs_max(u16x2_t big, const Vec8& v) {
#pragma unroll
  for (int k = 0; k < 4; ++k)
    big = __builtin_elementwise_max(big, __builtin_bit_cast(u16x2_t, v.w[k] & 0x7fff7fffu));
  return big;
}
// The same as the bits of a float.
template <bool F16>
__device__ __forceinline__ uint32_t abs_bits(u16x2_t big) {
  const uint16_t m = big.x > big.y ? big.x : big.y;
  return __float_as_uint(st2f<F16>(m));
}

// One wave's codes of a row of any width that is a multiple of 8, its start
// 2-byte aligned: the row is read twice (the second time from the cache), written
// to `codes` (8-byte aligned).
template <bool F16>
__device__ __forceinline__ RowScale quantize_row_wave(const uint16_t* x, int width, int8_t* codes, int lane) {
  u16x2_t big = {0, 0};
#pragma unroll 4
  for (int c = 8 * lane; c < width; c += 512) big = abs_max(big, load8<true>(x + c, 8));
  const RowScale rs = row_scale(team_umax<64>(abs_bits<F16>(big), nullptr));
#pragma unroll 4
  for (int c = 8 * lane; c < width; c += 512) {
    const Vec8 v = load8<true>(x + c, 8);
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = elem<F16>(v, j);
    *reinterpret_cast<uint2*>(codes + c) = codes8(f, rs);
  }
  return rs;
}

}  // namespace tfm
