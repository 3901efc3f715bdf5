// mx_device.hpp -- blocks of 32 entries that share a power of two (OCP Microscaling
// Formats v1.0): elements e4m3 or e2m1, the scale a byte s, 2^(s - 127), 255 NaN.
#pragma once
#include "npu_device.hpp"

namespace npu {

enum { kToBf16 = 0, kToE4m3 = 1, kToE2m1 = 2 };

// The larger of |m| over the four lanes of a quad, as bits: NaN above Inf above all else.
__device__ __forceinline__ uint32_t quad_max(uint32_t m) {
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xb1, 0xf, 0xf, false));
  return max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4e, 0xf, 0xf, false));
}
template <int N>
__device__ __forceinline__ uint32_t magnitude(const float (&y)[N]) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < N; ++e) m = max(m, __float_as_uint(y[e]) & 0x7fffffffu);
  return m;
}

// The scale takes a whole step where the largest magnitude passes a power of two.  Whether it does,
// f32's roundings (together below 2^-20) decide next to one: there the entries count as they are
// in 64 bits, by the upper halves of those (cut off, not rounded).
__device__ __forceinline__ bool next_to_power(uint32_t mag) {
  return ((mag + 8) & 0x7fffffu) < 16 && mag >= 0x00800000u && mag < 0x7f7ffff0u;
}
__device__ __forceinline__ uint32_t upper_magnitude(double y) { return (uint32_t)__double2hiint(y) & 0x7fffffffu; }
// A magnitude of that exponent.
__device__ __forceinline__ uint32_t from_upper(uint32_t upper) {
  return (uint32_t)min(max((int)(upper >> 20) - (1023 - 127), 0), 254) << 23;
}

// The scale of a block whose largest magnitude has these bits: its exponent (that of
// subnormals counts as the least) less the largest element's, 8 (448 = 1.75 2^8) or 2
// (6 = 1.5 2^2), at least 2^-127.
template <int KIND>
__device__ __forceinline__ uint32_t scale_byte(uint32_t mag) {
  constexpr int EMAX = KIND == kToE4m3 ? 8 : 2;
  const int e = (int)(mag >> 23);
  return e == 255 ? 255u : (uint32_t)max(e - EMAX, 0);
}
// 1 / scale, exact (the byte is at most 252); a NaN block's is 0.
__device__ __forceinline__ float inverse_scale(uint32_t byte) {
  return byte == 255 ? 0.0f : __uint_as_float((254u - byte) << 23);
}
// 2^(byte - 127) and NaN for 255, as a bf16's bits in the high half (exact).
__device__ __forceinline__ float scale_of(uint32_t byte) {
  return byte == 255 ? __builtin_nanf("") : __uint_as_float(byte == 0 ? 0x00400000u : byte << 23);
}

// Two or four elements' bits from scaled entries, to nearest even by the conversions, which
// take Inf and NaN to no element: a block with one (bad) has NaN (e4m3) or 0 (e2m1).
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d, bool bad) {
  // (above 464 the conversion gives NaN)
  auto lim = [](float v) { return __builtin_amdgcn_fmed3f(v, -448.0f, 448.0f); };
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(lim(a), lim(b), 0, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(lim(c), lim(d), r, true);
  return bad ? 0x7f7f7f7fu : (uint32_t)r;
}
__device__ __forceinline__ uint32_t pack_e2m1(const float (&y)[8], float inv, bool bad) {
  // (saturates at 6)
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[0] * inv, y[1] * inv, 1.0f, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[2] * inv, y[3] * inv, 1.0f, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[4] * inv, y[5] * inv, 1.0f, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[6] * inv, y[7] * inv, 1.0f, 3);
  return bad ? 0u : r;
}
__device__ __forceinline__ uint2 pack_e4m3x8(const float (&y)[8], float inv, bool bad) {
  return make_uint2(pack_e4m3(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv, bad),
                    pack_e4m3(y[4] * inv, y[5] * inv, y[6] * inv, y[7] * inv, bad));
}

// What eight elements stand for, in f32.
__device__ __forceinline__ void values_e2m1(uint32_t q, float s, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t c = q >> (4 * e) & 15u, m = c & 7u;
    // magnitudes by halves, two bits of four: 0 1 2 3 4 6 8 12
    const float h = (float)(m < 4 ? m : (m & 1 ? 3u : 2u) << ((m >> 1) - 1));
    v[e] = __uint_as_float(__float_as_uint(h * 0.5f) | (c & 8u) << 28) * s;
  }
}
__device__ __forceinline__ void values_e4m3(uint2 q, float s, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int a = (int)(q.x >> (8 * e)), b = (int)(q.y >> (8 * e));
    v[e] = __builtin_amdgcn_cvt_f32_fp8(a, 0) * s;
    v[4 + e] = __builtin_amdgcn_cvt_f32_fp8(b, 0) * s;
  }
}
__device__ __forceinline__ u32x4 pack_bf16x8(const float (&v)[8]) {
  return u32x4{cvt_pk_bf16(v[0], v[1]), cvt_pk_bf16(v[2], v[3]), cvt_pk_bf16(v[4], v[5]), cvt_pk_bf16(v[6], v[7])};
}
__device__ __forceinline__ void unpack_bf16x8(u32x4 u, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(u[i] << 16);
    v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  }
}

}  // namespace npu
