// A paged cache held in 8 bits: e4m3 with one power of two as the scale of each page of
// 16 tokens and key head.
//
//   k_cache   [blocks, n_kv, D/16, 16, 16]   chunk of 16 channels, token, channel
//   v_cache   [blocks, n_kv, D, 16]          channel, token
//   kv_scale  [blocks, n_kv, 2] fp32         of the page's keys and of its values
//
// 16 neighbouring bytes are what a lane of a matrix instruction takes: 16 channels of a
// key, 16 keys of a channel. Pages so laid out go to registers as they are, in loads
// whose lanes are neighbours; rows of tokens would need their values turned in LDS.
//
// Powers of two: an e4m3 value times one is exact in bf16 and 32 bits, the conversion
// applies it in the same instruction, and a page whose scale grows keeps its values
// but for the subnormal ones, which are rounded once more. A finer scale would gain
// e4m3 nothing: its step is relative to the value, 2^-4 at most, whatever the scale.
// The largest scale is 2^120, of which finite values are 240 at most: 256 of it is not
// finite in bf16 and 32 bits.
#pragma once
#include "mfma_rows.h"

namespace xllm {

constexpr int KV8_PAGE = 16;               // tokens of a page

// What a kernel that also takes pages of 16 bits is told of these
struct Kv8Pages {
  const float2* scale = nullptr;           // [blocks, n_kv]: of keys, of values
  int blocks = 0;
};

// The exponent of a page whose largest value is `big`: the least e >= -126 with
// big <= 448 * 2^e. 448 is 1.75 * 2^8: a mantissa above 1.75 carries into the exponent.
XLLM_DEV int kv8_exponent(float big) {
  return max((int)((__float_as_uint(big) + 0x1fffffu) >> 23) - 135, -126);
}
XLLM_DEV float kv8_power(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }

// four values to e4m3, the first in the low byte; what is not finite becomes a NaN
XLLM_DEV unsigned kv8_pack(float a, float b, float c, float d) {
  int u = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, u, true);
}
// four e4m3 values times `by`, rounded to e4m3 again
XLLM_DEV unsigned kv8_again(unsigned u, float by) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)u, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)u, true);
  return kv8_pack(lo[0] * by, lo[1] * by, hi[0] * by, hi[1] * by);
}
// eight e4m3 values times a power of two, in bf16
XLLM_DEV bf16x8 kv8_wide(unsigned lo, unsigned hi, float scale) {
  const bfx2 x[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false),
                     __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true),
                     __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false),
                     __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true)};
  bf16x8 y;
  __builtin_memcpy(&y, x, 16);
  return y;
}
// l and both of a pair of bf16 weights
XLLM_DEV float kv8_add(unsigned u, float l) {
  typedef __attribute__((ext_vector_type(2))) __bf16 pair;
  return __builtin_amdgcn_fdot2_f32_bf16(
      __builtin_bit_cast(pair, u), __builtin_bit_cast(pair, 0x3f803f80u), l, false);
}
// the top bits of those of four e4m3 values that are NaNs (0x7f but for the sign)
XLLM_DEV unsigned kv8_nan(unsigned u) {
  return ~((~u & 0x7f7f7f7fu) + 0x7f7f7f7fu) & 0x80808080u;
}
// NaNs of 16 values become zeros; one bit each
XLLM_DEV unsigned short kv8_drop_nan(uint4& u) {
  unsigned bits = 0;
  auto word = [&](unsigned& w, int at) {
    const unsigned n = kv8_nan(w) >> 7;
    w &= ~(n * 0xffu);
    bits |= ((n & 1) | (n >> 7 & 2) | (n >> 14 & 4) | (n >> 21 & 8)) << at;
  };
  word(u.x, 0), word(u.y, 4), word(u.z, 8), word(u.w, 12);
  return (unsigned short)bits;
}
// the first n of 16 bytes, zeros behind them
XLLM_DEV uint4 kv8_first(uint4 u, int n) {
  auto word = [&](unsigned w, int at) {
    const int k = min(max(n - at, 0), 4);
    return k == 4 ? w : w & ((1u << (8 * k)) - 1u);
  };
  return make_uint4(word(u.x, 0), word(u.y, 4), word(u.z, 8), word(u.w, 12));
}

}  // namespace xllm
