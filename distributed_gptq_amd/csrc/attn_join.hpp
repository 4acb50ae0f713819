// The joining of the sums that an attention's parts of a row's keys leave.
#pragma once

#include "attn_index.hpp"
#include "attn_tile.hpp"

namespace gptq {
namespace {

// The splits' sums of a row: o = sum_s o_s 2^(m_s - m) / sum_s l_s 2^(m_s - m),
// m the largest maximum; a row that no split has a key for is zero.  A group of
// 32 lanes, 4 channels a lane, takes every kGroups-th split of a row, and the
// groups of a row are joined through LDS.  With one group for 128 splits the
// loads of a row waited for each other: 27 us, now 3.2 for 32 rows of 64 splits.
// All weights are 2^-kJoinRoom of that: up to 128 sums that end at fp32's end do
// not pass it together.
constexpr float kJoinRoom = 8.0f;
template <bool kBF16, int kGroups>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a) {
  __shared__ float sm[8], sl[8];
  __shared__ __attribute__((aligned(16))) float so[8][128];
  const int64_t rows = static_cast<int64_t>(a.T) * a.H;
  const int group = threadIdx.x >> 5, d = 4 * (threadIdx.x & 31);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (8 / kGroups) + group / kGroups;
  const bool inside = row < rows;
  const float* mm = a.part + a.splits * rows * a.D;
  float m = -INFINITY, l = 0.0f;
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  // 8 splits at a time, all their loads together
  for (int s0 = group % kGroups; inside && s0 < a.splits; s0 += 8 * kGroups) {
    float ms[8], ls[8];
    f32x4 x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int sp = s0 + i * kGroups;
      const bool is = sp < a.splits;
      const int64_t at = (is ? sp : s0) * rows + row;
      ms[i] = is ? mm[at] : -INFINITY;
      ls[i] = mm[a.splits * rows + at];
      x[i] = *reinterpret_cast<const f32x4*>(a.part + at * a.D + (d < a.D ? d : 0));
      if (!is) x[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};  // (a part may hold infinities)
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, ms[i]);
    const float m0 = top == -INFINITY ? 0.0f : top;
    const float keep = __builtin_amdgcn_exp2f(m - m0);
    m = top;
    l *= keep;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= keep;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float w = __builtin_amdgcn_exp2f(ms[i] - m0 - kJoinRoom);  // 0 without keys
      l = fmaf(w, ls[i], l);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(w, x[i][e], o[e]);
    }
  }
  if constexpr (kGroups > 1) {
    *reinterpret_cast<f32x4*>(&so[group][d]) = o;
    if (d == 0) sm[group] = m, sl[group] = l;
    __syncthreads();
    if (group % kGroups) return;
    for (int g = 1; g < kGroups; ++g) m = fmaxf(m, sm[group + g]);
    const float m0 = m == -INFINITY ? 0.0f : m;
    l = 0.0f;
    o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const float w = exp2f(sm[group + g] - m0);
      l = fmaf(w, sl[group + g], l);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(w, so[group + g][d + e], o[e]);
    }
  }
  if (!inside || d >= a.D) return;
  const bool none = m == -INFINITY;
  const float r = 1.0f / l;
  *reinterpret_cast<u32x2*>(a.out + row * a.D + d) =
      none ? u32x2{0, 0} : u32x2{pack16<kBF16>(o[0] * r, o[1] * r), pack16<kBF16>(o[2] * r, o[3] * r)};
}

template <bool kBF16>
int launch_join(const AttnArgs& a, hipStream_t st) {
  const int64_t rows = static_cast<int64_t>(a.T) * a.H;
  if (a.splits > 8)
    attn_join_kernel<kBF16, 8><<<static_cast<uint32_t>(rows), 256, 0, st>>>(a);
  else
    attn_join_kernel<kBF16, 1><<<static_cast<uint32_t>((rows + 7) / 8), 256, 0, st>>>(a);
  return check_launch("attention (join)");
}

}  // namespace
}  // namespace gptq
