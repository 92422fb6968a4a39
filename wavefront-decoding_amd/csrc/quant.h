// The 8-bit slot cache: a row of Dh values of one kv head is Dh codes and one
// exponent byte b, value = code * 2^(b - 127); b = 255 marks a row that held an
// infinity or NaN, which reads as NaN. Codes are e4m3 (OCP, |code| <= 448) or
// int8 (|code| <= 127), and 2^(b - 127) is the smallest power of two, at least
// 2^-126, with max|x| <= 448 (127) times it.
//
// A power of two rather than max|x| / 448 itself: x * 2^-e is exact, so a code
// is one rounding of x whatever the arithmetic around it; reading is exact in
// bf16 (4 or 7 significant bits); a score or a probability is scaled without
// error; and the scale takes 1 byte of the row instead of 4. It costs e4m3
// nothing (a floating format) and int8 at most one bit of the row's range.
#pragma once

#include "wfd_common.h"

namespace wfd {

constexpr uint32_t kExpNaN = 255;
constexpr int kMaxHeads = 65535;

__device__ __forceinline__ float code_scale(uint32_t b) {  // 2^(b - 127); NaN for the marked rows
  return b == kExpNaN ? __uint_as_float(0x7fc00000u) : __uint_as_float(b << 23);
}

// Exponent byte of a row whose largest |x| has the bits amax (as integers the
// bits of |x| order like the values, infinity and NaN last).
template <int CODE>
__device__ __forceinline__ uint32_t exp_byte(uint32_t amax) {
  if (amax >= 0x7f800000u) return kExpNaN;
  // 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6
  constexpr int kBits = CODE == WFD_E4M3 ? 8 : 6;
  constexpr uint32_t kTop = CODE == WFD_E4M3 ? 0x600000u : 0x7e0000u;
  const int b = (int)(amax >> 23) - kBits + ((amax & 0x7fffffu) > kTop ? 1 : 0);
  return (uint32_t)(b < 1 ? 1 : b);
}

// Eight values -> eight codes under exponent byte b (two dwords).
template <int CODE>
__device__ __forceinline__ uint2 encode8(const float (&x)[8], uint32_t b) {
  if (b == kExpNaN) return uint2{0u, 0u};
  const float inv = __uint_as_float((254u - b) << 23);  // 2^-(b - 127); b <= 249
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = x[e] * inv;
  uint2 w;
  if constexpr (CODE == WFD_E4M3) {
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
    int hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], hi, true);
    w.x = (uint32_t)lo;
    w.y = (uint32_t)hi;
  } else {
    uint32_t c[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = (uint32_t)(int)rintf(y[e]) & 0xffu;
    w.x = c[0] | (c[1] << 8) | (c[2] << 16) | (c[3] << 24);
    w.y = c[4] | (c[5] << 8) | (c[6] << 16) | (c[7] << 24);
  }
  return w;
}

// Four codes -> four floats, unscaled (exact).
template <int CODE>
__device__ __forceinline__ void decode4(uint32_t w, float* o) {
  if constexpr (CODE == WFD_E4M3) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
    const f32x2 c = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    o[0] = a[0];
    o[1] = a[1];
    o[2] = c[0];
    o[3] = c[1];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = (float)(int8_t)(w >> (8 * e));
  }
}

// The host's checks of a cache's code type, heads and layout; 0 or a status.
inline int check_qcache(const char* what, int n, int Hkv, int Dh, int code, int64_t block_rows) {
  if (n < 0 || Hkv <= 0 || Hkv > kMaxHeads || block_rows < 0) {
    set_error("%s: bad shape n=%d Hkv=%d kv_block_rows=%lld", what, n, Hkv, (long long)block_rows);
    return kBadArg;
  }
  if ((Dh != 64 && Dh != 128) || (code != WFD_E4M3 && code != WFD_INT8)) {
    set_error("%s: unsupported Dh=%d code=%d (Dh 64/128; WFD_E4M3, WFD_INT8)", what, Dh, code);
    return kUnsupported;
  }
  return kOk;
}

}  // namespace wfd
