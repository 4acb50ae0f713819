// Runs of fp32, fp16 or bf16 values as floats in registers, and back.
#pragma once

#include "common.hpp"

namespace gptq {
namespace {

// N values as floats, and back; the addresses are multiples of N values' bytes
// (or 16)
template <int N, int kType>
__device__ __forceinline__ void load_values(float (&x)[N], const void* p, int64_t at) {
  if constexpr (kType == GPTQ_F32) {
    const float* f = static_cast<const float*>(p) + at;
#pragma unroll
    for (int i = 0; i < N; i += N < 4 ? N : 4) {
      typedef float vec __attribute__((ext_vector_type(N < 4 ? N : 4)));
      const vec v = *reinterpret_cast<const vec*>(f + i);
#pragma unroll
      for (int e = 0; e < (N < 4 ? N : 4); ++e) x[i + e] = v[e];
    }
  } else {
    typedef uint16_t vec __attribute__((ext_vector_type(N)));
    const vec v = *reinterpret_cast<const vec*>(static_cast<const uint16_t*>(p) + at);
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = kType == GPTQ_BF16 ? bf16_bits_to_f32(v[e]) : f16_bits_to_f32(v[e]);
  }
}
template <int N, int kType>
__device__ __forceinline__ void store_values(void* p, int64_t at, const float (&x)[N]) {
  if constexpr (kType == GPTQ_F32) {
    float* f = static_cast<float*>(p) + at;
#pragma unroll
    for (int i = 0; i < N; i += N < 4 ? N : 4) {
      typedef float vec __attribute__((ext_vector_type(N < 4 ? N : 4)));
      vec v;
#pragma unroll
      for (int e = 0; e < (N < 4 ? N : 4); ++e) v[e] = x[i + e];
      *reinterpret_cast<vec*>(f + i) = v;
    }
  } else {
    typedef uint16_t vec __attribute__((ext_vector_type(N)));
    vec v;
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = kType == GPTQ_BF16 ? f32_to_bf16_bits(x[e]) : f32_to_f16_bits(x[e]);
    *reinterpret_cast<vec*>(static_cast<uint16_t*>(p) + at) = v;
  }
}

// store_values by the conversions of a pair at a time (a NaN stays one, with other
// bits than store_values gives it)
template <int N, int kType>
__device__ __forceinline__ void store_pairs(void* p, int64_t at, const float (&x)[N]) {
  if constexpr (kType == GPTQ_F32) {
    store_values<N, kType>(p, at, x);
  } else {
    constexpr int kWide = N / 2 < 4 ? N / 2 : 4;
    typedef uint32_t vec __attribute__((ext_vector_type(kWide)));
    vec* to = reinterpret_cast<vec*>(static_cast<uint16_t*>(p) + at);
#pragma unroll
    for (int i = 0; i < N / 2; i += kWide) {
      vec w;
#pragma unroll
      for (int e = 0; e < kWide; ++e) {
        const float lo = x[2 * (i + e)], hi = x[2 * (i + e) + 1];
        w[e] = kType == GPTQ_BF16 ? pack_bf16(lo, hi) : pack_f16(lo, hi);
      }
      to[i / kWide] = w;
    }
  }
}

}  // namespace
}  // namespace gptq
