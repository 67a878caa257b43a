// Codes and scales of the 8-bit KV cache: int8 (-127 .. 127) or e4m3 (|value| <= 448, finite); a wave's prefix sum.
#pragma once
#include "common.cuh"

namespace iek {

IEK_DEV uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// Inclusive prefix sum over the wave's lanes.
template <int CTRL, int ROWS = 0xF>
IEK_DEV int dpp_up(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
IEK_DEV int wave_scan(int v) {
  v += dpp_up<0x111>(v);  // row_shr 1, 2, 4, 8
  v += dpp_up<0x112>(v);
  v += dpp_up<0x114>(v);
  v += dpp_up<0x118>(v);
  v += dpp_up<DPP_BCAST15, 0xA>(v);
  return v + dpp_up<DPP_BCAST31, 0xC>(v);
}

// The smallest power of two s >= 2^-100 with amax <= M * s (M = 127 or 448) for the bits of a
// non-negative amax; NaN for infinities and NaN. With amax = (1 + f) 2^x: M = (1 + F) 2^X, so
// s = 2^(x - X), doubled when f > F.
template <bool E4M3>
IEK_DEV float kv8_scale(uint32_t amax_bits) {
  if (amax_bits >= 0x7F800000u) return __uint_as_float(0x7FC00000u);
  constexpr uint32_t F = E4M3 ? 0x600000u : 0x7E0000u;  // 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6
  constexpr int X = E4M3 ? 8 : 6;
  int e = (int)(amax_bits >> 23) - X + ((amax_bits & 0x7FFFFFu) > F ? 1 : 0);  // biased
  return __uint_as_float((uint32_t)max(e, 27) << 23);
}

// Four values times f (a power of two), each rounded to its code (to nearest, ties to even).
template <bool E4M3>
IEK_DEV uint32_t kv8_pack(float4 x, float f) {
  if constexpr (E4M3) {
    // |x f| <= 448 by the choice of the scale: nothing saturates
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(x.x * f, x.y * f, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x.z * f, x.w * f, w, true);
  } else {
    const int a = (int)rintf(x.x * f), b = (int)rintf(x.y * f), c = (int)rintf(x.z * f), d = (int)rintf(x.w * f);
    return (uint32_t)(a & 255) | (uint32_t)(b & 255) << 8 | (uint32_t)(c & 255) << 16 | (uint32_t)d << 24;
  }
}

template <bool E4M3>
IEK_DEV float4 kv8_unpack(uint32_t w) {
  if constexpr (E4M3) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    return make_float4(lo[0], lo[1], hi[0], hi[1]);
  } else {
    return make_float4((float)(int8_t)(w & 255), (float)(int8_t)(w >> 8 & 255), (float)(int8_t)(w >> 16 & 255),
                       (float)((int32_t)w >> 24));
  }
}

}  // namespace iek
