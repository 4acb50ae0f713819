// 8-bit codes of a quantised cache: a row of one token and head is whole
// numbers -127 .. 127 or e4m3 floats up to 448, times the row's fp32 scale.
#pragma once

#include "common.hpp"

namespace gptq {
namespace {

template <int kCode>
constexpr float kTop = kCode == GPTQ_CODE_I8 ? 127.0f : 448.0f;

// Rows whose largest value is not above this have code and scale 0.
constexpr float kLeast = 0x1p-120f;

// Rows whose largest value is below this are made kRaise as large, which is exact,
// before they are divided by it: 448 over values up to 1.75 2^-120 is past fp32.
constexpr float kSmall = 0x1p-64f, kRaise = 0x1p64f;

// The largest scale whose product with the last code is a number of fp32 (the
// largest value over top may round past it).
template <int kCode>
constexpr float kMostScale = kCode == GPTQ_CODE_I8 ? 0x1.020406p+121f : 0x1.249248p+119f;

// Four values, each times inv and rounded to the nearest code (ties to even).  inv
// is the top code over the largest of them, so that no product is more than two
// roundings past the top: both types round that back to it.
template <int kCode>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d, float inv) {
  if constexpr (kCode == GPTQ_CODE_I8) {
    auto code = [&](float x) { return static_cast<uint32_t>(static_cast<int>(rintf(x * inv))) & 0xFFu; };
    return code(a) | code(b) << 8 | code(c) << 16 | code(d) << 24;
  } else {
    const int low = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, low, true));
  }
}

// Four codes as floats.
template <int kCode>
__device__ __forceinline__ f32x4 decode4(uint32_t w) {
  if constexpr (kCode == GPTQ_CODE_I8) {
    return f32x4{static_cast<float>(static_cast<int8_t>(w)), static_cast<float>(static_cast<int8_t>(w >> 8)),
                 static_cast<float>(static_cast<int8_t>(w >> 16)), static_cast<float>(static_cast<int8_t>(w >> 24))};
  } else {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
    const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
    return f32x4{a[0], a[1], b[0], b[1]};
  }
}

// Four codes as 16-bit values, which hold every code exactly: two registers.
// One instruction a pair for e4m3; for whole numbers in fp16 a byte permute to
// 1024 + (code + 128) and one packed subtraction a pair; in bf16, whose
// integers end at 256, a conversion a code and a permute a pair.
template <bool kBF16, int kCode>
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (kCode == GPTQ_CODE_E4M3) {
    if constexpr (kBF16) {
      lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
      hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true));
    } else {
      lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
      hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
    }
  } else if constexpr (kBF16) {
    const f32x4 f = decode4<kCode>(w);
    auto top = [&](float a, float b) {  // the high halves hold all of these values
      return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
    };
    lo = top(f[0], f[1]);
    hi = top(f[2], f[3]);
  } else {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const uint32_t u = w ^ 0x80808080u;
    const f16x2 less = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
    auto pair = [&](uint32_t bits) { return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, bits) + less); };
    lo = pair(__builtin_amdgcn_perm(0x64646464u, u, 0x04010400u));
    hi = pair(__builtin_amdgcn_perm(0x64646464u, u, 0x04030402u));
  }
}

}  // namespace
}  // namespace gptq
