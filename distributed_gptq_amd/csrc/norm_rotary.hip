// Norms of query and key heads with the rotation in the same pass, y = R(pos)
// (w x r), r = (mean x^2 + eps)^-1/2, their gradients, and keys and values
// written into the pages of a cache on the way, quantised where it holds codes.
#include "attn_index.hpp"
#include "codes.hpp"
#include "values.hpp"

namespace gptq {
namespace {

struct HeadRows {  // rows of (token, head)
  const void* p;
  int64_t token, head;  // strides, in elements
};
struct CacheRows {  // rows of (page, token, head), and their scales
  void* p;
  int64_t page, token, head;
  float* scale;
  int64_t s_page, s_token, s_head;
};

struct NormArgs {
  HeadRows q, k, v;                  // v.p null without a cache
  const void *q_weight, *k_weight;   // null: nothing is normed
  int weight_type;
  float eps;
  const float* table;                // (P, 2, R / 2): cosines, then sines; null: nothing turns
  const int32_t* positions;          // (T)
  int64_t P;
  const int32_t* slots;              // (T) places in the cache, or null: k_out (T, Hk, D)
  int64_t capacity;
  FastDiv page;
  void *q_out, *k_out;               // (T, heads, D)
  CacheRows kc, vc;
  int T, H, Hk, D, R;
  float inv_d;                       // 1 / D
  int interleaved;
  // a thread's work: `per` heads of one kind of a token
  int per, gq, gk;
  FastDiv groups, tokens;
  // the gradient
  HeadRows grad_q, grad_k;
  void *dq, *dk;                     // (T, heads, D)
  float* part;                       // (blocks, 2, D) sums of the weights' gradients, or null
};

// A row's channels are in `lanes` (a power of two) neighbouring lanes, 2 N each;
// those past the last unit hold nothing.  Sums and maxima over them by moves inside
// the vector unit: halves of a quad, quads, eights and rows mirrored, rows and
// halves of the wave swapped.
template <int kCtrl>
__device__ __forceinline__ float moved(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), kCtrl, 0xF, 0xF, true));
}
template <class Op>
__device__ __forceinline__ float over_row(float v, int lanes, Op&& op) {
  if (lanes > 1) v = op(v, moved<0xB1>(v));
  if (lanes > 2) v = op(v, moved<0x4E>(v));
  if (lanes > 4) v = op(v, moved<0x141>(v));
  if (lanes > 8) v = op(v, moved<0x140>(v));
  if (lanes > 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  if (lanes > 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  return v;
}
__device__ __forceinline__ float row_sum(float v, int lanes) {
  return over_row(v, lanes, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float row_max(float v, int lanes) {
  return over_row(v, lanes, [](float a, float b) { return __builtin_elementwise_maximum(a, b); });
}

// Where a lane's 2 N channels are, and its angles.
template <int N>
struct Unit {
  int first, second;  // N channels each
  bool some, turns;
};
template <int N>
__device__ __forceinline__ Unit<N> unit_at(const NormArgs& a, int u) {
  const int half = a.table ? a.R / 2 : 0;
  Unit<N> at;
  at.some = 2 * u * N < a.D;
  at.turns = u * N < half;
  at.first = at.turns && !a.interleaved ? u * N : 2 * u * N;
  at.second = at.turns && !a.interleaved ? half + u * N : at.first + N;
  return at;
}
template <int N>
__device__ __forceinline__ void load_angles(const NormArgs& a, int t, int u, float sign, float (&c)[N], float (&s)[N]) {
  const int pos = a.positions[t];
  const int64_t row = pos < 0 ? 0 : pos >= a.P ? a.P - 1 : pos;
  const float* p = a.table + row * a.R + u * N;
  load_values<N, GPTQ_F32>(c, p, 0);
  load_values<N, GPTQ_F32>(s, p, a.R / 2);
#pragma unroll
  for (int e = 0; e < N; ++e) s[e] *= sign;
}
// x, y: the channels first .. and second ..; pairs are (x[e], y[e]), or
// neighbours among the 2 N
template <int N>
__device__ __forceinline__ void turn(float (&x)[N], float (&y)[N], const float (&c)[N], const float (&s)[N],
                                     int interleaved) {
  float xy[2 * N];
#pragma unroll
  for (int e = 0; e < N; ++e) xy[e] = x[e], xy[N + e] = y[e];
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float p = interleaved ? xy[2 * e] : x[e], r = interleaved ? xy[2 * e + 1] : y[e];
    const float v = p * c[e] - r * s[e], w = r * c[e] + p * s[e];
    if (interleaved)
      xy[2 * e] = v, xy[2 * e + 1] = w;
    else
      xy[e] = v, xy[N + e] = w;
  }
#pragma unroll
  for (int e = 0; e < N; ++e) x[e] = xy[e], y[e] = xy[N + e];
}

template <int N>
__device__ __forceinline__ void load_weights(const void* w, int type, const Unit<N>& at, float (&x)[N], float (&y)[N]) {
#pragma unroll
  for (int e = 0; e < N; ++e) x[e] = y[e] = 0.0f;
  if (!at.some) return;
  if (type == GPTQ_F32)
    load_values<N, GPTQ_F32>(x, w, at.first), load_values<N, GPTQ_F32>(y, w, at.second);
  else if (type == GPTQ_BF16)
    load_values<N, GPTQ_BF16>(x, w, at.first), load_values<N, GPTQ_BF16>(y, w, at.second);
  else
    load_values<N, GPTQ_F16>(x, w, at.first), load_values<N, GPTQ_F16>(y, w, at.second);
}

// 1 / sqrt(mean of squares + eps) of a row (the hardware's, to a unit of the last
// place).  Squares of values past 2^64 leave fp32: the row's sum is made again of
// values 2^-80 as large, beside whose squares eps is nothing.
template <int N>
__device__ __forceinline__ float rms_inverse(const float (&x)[N], const float (&y)[N], const NormArgs& a, int lanes) {
  float ss = 0.0f;
#pragma unroll
  for (int e = 0; e < N; ++e) ss = fmaf(x[e], x[e], fmaf(y[e], y[e], ss));
  ss = row_sum(ss, lanes);
  if (__builtin_expect(ss == INFINITY, 0)) {
    float s2 = 0.0f;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float p = x[e] * 0x1p-80f, r = y[e] * 0x1p-80f;
      s2 = fmaf(p, p, fmaf(r, r, s2));
    }
    return 0x1p-80f * __builtin_amdgcn_rsqf(row_sum(s2, lanes) * a.inv_d);
  }
  return __builtin_amdgcn_rsqf(fmaf(ss, a.inv_d, a.eps));
}

// A row into the cache: as it is, or as codes and their scale.  A row with a
// value that is not finite reads back as NaN: its scale is one.
template <int N, int kType, int kStore>
__device__ __forceinline__ void store_cached(const CacheRows& r, int64_t page, int64_t at, int h, const Unit<N>& unit,
                                             const float (&x)[N], const float (&y)[N], int lanes, int u) {
  const int64_t o = page * r.page + at * r.token + h * r.head;
  if constexpr (kStore == 0) {
    if (!unit.some) return;
    store_pairs<N, kType>(r.p, o + unit.first, x);
    store_pairs<N, kType>(r.p, o + unit.second, y);
  } else {
    float most = 0.0f;
#pragma unroll
    for (int e = 0; e < N; ++e)
      most = __builtin_elementwise_maximum(__builtin_elementwise_maximum(most, fabsf(x[e])), fabsf(y[e]));
    most = row_max(most, lanes);
    constexpr float top = kTop<kStore>;
    const bool finite = most < INFINITY;
    const bool some = finite && most > kLeast;
    const float raise = most < kSmall ? kRaise : 1.0f;
    const float inv = some ? top / (most * raise) : 0.0f;
    if (!unit.some) return;
    uint8_t* to = static_cast<uint8_t*>(r.p) + o;
    typedef uint32_t words __attribute__((ext_vector_type(N / 4)));
    words w0, w1;
#pragma unroll
    for (int e = 0; e < N; e += 4) {
      auto code = [&](const float (&z)[N]) {
        return encode4<kStore>(z[e] * raise, z[e + 1] * raise, z[e + 2] * raise, z[e + 3] * raise, inv);
      };
      w0[e / 4] = finite ? code(x) : 0u;
      w1[e / 4] = finite ? code(y) : 0u;
    }
    *reinterpret_cast<words*>(to + unit.first) = w0;
    *reinterpret_cast<words*>(to + unit.second) = w1;
    if (u == 0)
      r.scale[page * r.s_page + at * r.s_token + h * r.s_head] =
          some ? fminf(most / top, kMostScale<kStore>) : finite ? 0.0f : __builtin_nanf("");
  }
}

// A thread has 2 N channels of `per` heads of a token, all queries, all keys or
// all values, whose angles and weights it reads once.  Bound by memory: each value
// is read and written once, and 16 waves of a CU (128 registers) hide the loads
// better than fewer with the next heads' loads ahead.  16384 tokens of 32 + 8 heads
// of 128 bf16 values (336 MB): 66 us, 5.1 TB/s, 71 us with two heads at once, 83 us
// with a head per thread.  2048 tokens of 40 + 40 + 40 heads of 128 fp16 values into
// e4m3 (106 MB): 33 us, 3.2 TB/s, the tokens of a head in neighbouring rows so that
// their scales and codes fill lines (38 us by tokens).  One token: 4.4 us, the launch.
template <int N, int kType, int kStore>
__global__ __launch_bounds__(256, 4) void norm_rotary_kernel(NormArgs a, int lanes) {
  const int rows = 256 / lanes;
  const int u = threadIdx.x & (lanes - 1);
  const int64_t id = static_cast<int64_t>(blockIdx.x) * rows + threadIdx.x / lanes;
  if (id >= static_cast<int64_t>(a.T) * a.groups.d) return;
  // a token's groups lie next to each other, but in a cache a head's tokens do
  int t = div_by(static_cast<int>(id), a.groups);
  int g = static_cast<int>(id) - t * static_cast<int>(a.groups.d);
  if (a.slots) {
    g = div_by(static_cast<int>(id), a.tokens);
    t = static_cast<int>(id) - g * a.T;
  }
  const int kind = g < a.gq ? 0 : g < a.gq + a.gk ? 1 : 2;
  g -= kind == 0 ? 0 : kind == 1 ? a.gq : a.gq + a.gk;
  const int heads = kind == 0 ? a.H : a.Hk;
  const int h0 = g * a.per, h1 = h0 + a.per < heads ? h0 + a.per : heads;
  const HeadRows from = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
  int64_t page = 0, at = t;
  if (kind != 0 && a.slots) {
    const int slot = a.slots[t];
    if (slot < 0 || slot >= a.capacity) return;
    page = div_by(slot, a.page);
    at = slot - page * static_cast<int64_t>(a.page.d);
  }
  const Unit<N> unit = unit_at<N>(a, u);
  const bool turns = unit.turns && kind != 2;
  const void* weight = kind == 0 ? a.q_weight : kind == 1 ? a.k_weight : nullptr;
  float c[N], s[N], wx[N], wy[N];
  if (turns) load_angles<N>(a, t, u, 1.0f, c, s);
  if (weight) load_weights<N>(weight, a.weight_type, unit, wx, wy);
  for (int h = h0; h < h1; ++h) {
    float x[N], y[N];
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = y[e] = 0.0f;
    if (unit.some) {
      const int64_t i = t * from.token + h * from.head;
      load_values<N, kType>(x, from.p, i + unit.first);
      load_values<N, kType>(y, from.p, i + unit.second);
    }
    if (weight) {
      const float r = rms_inverse<N>(x, y, a, lanes);
#pragma unroll
      for (int e = 0; e < N; ++e) x[e] = x[e] * r * wx[e], y[e] = y[e] * r * wy[e];  // (r w may leave fp32 where x r w does not)
    }
    if (turns) turn<N>(x, y, c, s, a.interleaved);
    if (kind == 0 || !a.slots) {
      void* to = kind == 0 ? a.q_out : a.k_out;
      const int64_t o = (static_cast<int64_t>(t) * heads + h) * a.D;
      if (unit.some) {
        store_pairs<N, kType>(to, o + unit.first, x);
        store_pairs<N, kType>(to, o + unit.second, y);
      }
    } else {
      store_cached<N, kType, kStore>(kind == 1 ? a.kc : a.vc, page, at, h, unit, x, y, lanes, u);
    }
  }
}

// The gradient.  With g = R^T dy: dw = sum over the rows of g x r, and
// dx = r (g w - x r mean(g w x r)); r is made again.  A workgroup takes tokens'
// groups of heads blockIdx.x * rows + ..., first of the queries, then of the
// keys, and leaves its sums for dw, in the order of its rows.  Bound by memory, with
// the workgroups of back_blocks all on the GPU at once: 8192 tokens of 32 + 8 heads
// of 128 bf16 values (252 MB): 52 us, 4.8 TB/s, 62 us with 3 waves on a SIMD.
template <int N, int kType>
__global__ __launch_bounds__(256, 4) void norm_rotary_back_kernel(NormArgs a, int lanes) {
  __shared__ float sums[512 * N];
  const int rows = 256 / lanes;
  const int row0 = threadIdx.x / lanes;
  const int u = threadIdx.x & (lanes - 1);
  const Unit<N> unit = unit_at<N>(a, u);
#pragma unroll 1
  for (int kind = 0; kind < 2; ++kind) {
    const HeadRows from = kind == 0 ? a.q : a.k, grad = kind == 0 ? a.grad_q : a.grad_k;
    void* to = kind == 0 ? a.dq : a.dk;
    const int heads = kind == 0 ? a.H : a.Hk;
    const int groups = kind == 0 ? a.gq : a.gk;
    const int64_t items = static_cast<int64_t>(a.T) * groups;
    float wx[N], wy[N], dwx[N], dwy[N];
    load_weights<N>(kind == 0 ? a.q_weight : a.k_weight, a.weight_type, unit, wx, wy);
#pragma unroll
    for (int e = 0; e < N; ++e) dwx[e] = dwy[e] = 0.0f;
    for (int64_t id = static_cast<int64_t>(blockIdx.x) * rows + row0; id < items;
         id += static_cast<int64_t>(gridDim.x) * rows) {
      const int t = static_cast<int>(static_cast<uint32_t>(id) / static_cast<uint32_t>(groups));
      const int h0 = (static_cast<int>(id) - t * groups) * a.per;
      const int h1 = h0 + a.per < heads ? h0 + a.per : heads;
      float c[N], s[N];
      if (unit.turns) load_angles<N>(a, t, u, -1.0f, c, s);
      for (int h = h0; h < h1; ++h) {
        float x[N], y[N], gx[N], gy[N];
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = y[e] = gx[e] = gy[e] = 0.0f;
        if (unit.some) {
          const int64_t i = t * from.token + h * from.head, j = t * grad.token + h * grad.head;
          load_values<N, kType>(x, from.p, i + unit.first);
          load_values<N, kType>(y, from.p, i + unit.second);
          load_values<N, kType>(gx, grad.p, j + unit.first);
          load_values<N, kType>(gy, grad.p, j + unit.second);
        }
        const float r = rms_inverse<N>(x, y, a, lanes);
        if (unit.turns) turn<N>(gx, gy, c, s, a.interleaved);
        float dot = 0.0f;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          x[e] *= r, y[e] *= r;
          dwx[e] = fmaf(gx[e], x[e], dwx[e]);
          dwy[e] = fmaf(gy[e], y[e], dwy[e]);
          gx[e] *= wx[e], gy[e] *= wy[e];
          dot = fmaf(gx[e], x[e], fmaf(gy[e], y[e], dot));
        }
        dot = row_sum(dot, lanes) * a.inv_d;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          gx[e] = r * (gx[e] - x[e] * dot);
          gy[e] = r * (gy[e] - y[e] * dot);
        }
        if (unit.some) {
          const int64_t o = (static_cast<int64_t>(t) * heads + h) * a.D;
          store_pairs<N, kType>(to, o + unit.first, gx);
          store_pairs<N, kType>(to, o + unit.second, gy);
        }
      }
    }
    if (!a.part) continue;
    __syncthreads();
    if (unit.some) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        sums[row0 * a.D + unit.first + e] = dwx[e];
        sums[row0 * a.D + unit.second + e] = dwy[e];
      }
    }
    __syncthreads();
    for (int d = threadIdx.x; d < a.D; d += 256) {
      float v = 0.0f;
      for (int i = 0; i < rows; ++i) v += sums[i * a.D + d];
      a.part[(static_cast<int64_t>(blockIdx.x) * 2 + kind) * a.D + d] = v;
    }
  }
}

// The workgroups' sums of 4 channels of one weight: a thread adds every 256th, and
// the threads' are added in the order of a tree.  1024 workgroups of 128 channels: 4.7
// us (11.3 with a thread for each channel).
__global__ __launch_bounds__(256) void norm_weight_sum_kernel(const float* part, int blocks, int D, int type, void* dq_weight,
                                                              void* dk_weight) {
  __shared__ f32x4 sums[256];
  const int kind = blockIdx.y, d = blockIdx.x * 4;
  f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int b = threadIdx.x; b < blocks; b += 256)
    v += *reinterpret_cast<const f32x4*>(part + (static_cast<int64_t>(b) * 2 + kind) * D + d);
  sums[threadIdx.x] = v;
  for (int n = 128; n > 0; n >>= 1) {
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < n) sums[threadIdx.x] = v = v + sums[threadIdx.x + n];
  }
  if (threadIdx.x == 0)
#pragma unroll
    for (int e = 0; e < 4; ++e) store_elem(kind == 0 ? dq_weight : dk_weight, d + e, type, v[e]);
}

// --------------------------------------------------------------- launching ----

// channels of a lane's half: whole units in the head and in its turned part
int unit_of(const NormArgs& a) {
  const int half = a.table ? a.R / 2 : a.D / 2;
  return a.D % 16 == 0 && half % 8 == 0 ? 8 : half % 4 == 0 ? 4 : 2;
}
int lanes_of(int D, int n) {
  int lanes = 1;
  while (lanes * 2 * n < D) lanes *= 2;
  return lanes;
}

template <int N, int kType, int kStore>
int launch(NormArgs a, const char* fn, hipStream_t st) {
  const int lanes = lanes_of(a.D, N);
  const int heads = a.H + a.Hk + (a.v.p ? a.Hk : 0);
  // enough threads for the GPU first, then heads that share a thread's angles
  const int64_t threads = static_cast<int64_t>(a.T) * lanes * heads;
  const int64_t per = threads / (256 * 2048);
  a.per = static_cast<int>(per < 1 ? 1 : per > 8 ? 8 : per);
  a.gq = (a.H + a.per - 1) / a.per;
  a.gk = (a.Hk + a.per - 1) / a.per;
  a.groups = fast_div(static_cast<uint32_t>(a.gq + (a.v.p ? 2 : 1) * a.gk));
  a.tokens = fast_div(static_cast<uint32_t>(a.T));
  const int64_t items = static_cast<int64_t>(a.T) * a.groups.d;
  GPTQ_REQUIRE(items < (int64_t{1} << 31), GPTQ_ERR_SHAPE, "%s: too many tokens", fn);
  norm_rotary_kernel<N, kType, kStore><<<static_cast<uint32_t>(cdiv(items, 256 / lanes)), 256, 0, st>>>(a, lanes);
  return check_launch(fn);
}
template <int N, int kStore>
int launch_type(const NormArgs& a, int dtype, const char* fn, hipStream_t st) {
  if (dtype == GPTQ_F32) return launch<N, GPTQ_F32, kStore>(a, fn, st);
  if (dtype == GPTQ_BF16) return launch<N, GPTQ_BF16, kStore>(a, fn, st);
  return launch<N, GPTQ_F16, kStore>(a, fn, st);
}
template <int kStore>
int launch_unit(const NormArgs& a, int dtype, const char* fn, hipStream_t st) {
  const int n = unit_of(a);
  if (n == 8) return launch_type<8, kStore>(a, dtype, fn, st);
  if constexpr (kStore != 0) {  // (codes are stored in whole words)
    GPTQ_REQUIRE(n == 4, GPTQ_ERR_SHAPE, "%s: the rotated channels of a head that is quantised have to be a multiple of 8",
                 fn);
    return launch_type<4, kStore>(a, dtype, fn, st);
  } else {
    if (n == 4) return launch_type<4, kStore>(a, dtype, fn, st);
    return launch_type<2, kStore>(a, dtype, fn, st);
  }
}

// workgroups of the gradient: as many as 256 CUs hold, four of 4 waves each, and
// no more than there are rows for
int64_t back_blocks(int64_t T, int64_t H, int64_t Hk) {
  const int64_t rows = T * (H > Hk ? H : Hk);
  const int64_t blocks = cdiv(rows, 32);
  return blocks < 1 ? 1 : blocks < 1024 ? blocks : 1024;
}

template <int N, int kType>
int launch_back(NormArgs a, hipStream_t st) {
  const int lanes = lanes_of(a.D, N);
  const int64_t blocks = back_blocks(a.T, a.H, a.Hk);
  const int64_t per = static_cast<int64_t>(a.T) * a.H * lanes / (256 * blocks);
  a.per = static_cast<int>(per < 1 ? 1 : per > 4 ? 4 : per);
  a.gq = (a.H + a.per - 1) / a.per;
  a.gk = (a.Hk + a.per - 1) / a.per;
  GPTQ_REQUIRE(static_cast<int64_t>(a.T) * (a.gq > a.gk ? a.gq : a.gk) < (int64_t{1} << 31), GPTQ_ERR_SHAPE,
               "gptq_norm_rotary_backward: too many tokens");
  norm_rotary_back_kernel<N, kType><<<static_cast<uint32_t>(blocks), 256, 0, st>>>(a, lanes);
  return check_launch("gptq_norm_rotary_backward");
}
template <int N>
int launch_back_type(const NormArgs& a, int dtype, hipStream_t st) {
  if (dtype == GPTQ_F32) return launch_back<N, GPTQ_F32>(a, st);
  if (dtype == GPTQ_BF16) return launch_back<N, GPTQ_BF16>(a, st);
  return launch_back<N, GPTQ_F16>(a, st);
}

int check_sizes(const char* fn, int dtype, int weight_type, bool norm, float eps, const float* table, int64_t P, int64_t R,
                int64_t T, int64_t H, int64_t Hk, int64_t D) {
  GPTQ_REQUIRE(valid_dtype(dtype) && (!norm || valid_dtype(weight_type)), GPTQ_ERR_DTYPE, "%s: expected fp32, fp16 or bf16",
               fn);
  GPTQ_REQUIRE(T >= 0 && T < (int64_t{1} << 31) && H >= 1 && H <= 65536 && Hk >= 1 && Hk <= 65536, GPTQ_ERR_SHAPE,
               "%s: %lld tokens, %lld and %lld heads", fn, static_cast<long long>(T), static_cast<long long>(H),
               static_cast<long long>(Hk));
  GPTQ_REQUIRE(D >= 8 && D <= 256 && D % 8 == 0, GPTQ_ERR_SHAPE,
               "%s: heads of %lld values (multiples of 8 up to 256 are supported)", fn, static_cast<long long>(D));
  GPTQ_REQUIRE(!table || (R >= 4 && R % 4 == 0 && R <= D && P >= 1), GPTQ_ERR_SHAPE,
               "%s: a table of %lld positions for %lld of %lld values (multiples of 4 are supported)", fn,
               static_cast<long long>(P), static_cast<long long>(R), static_cast<long long>(D));
  GPTQ_REQUIRE(!norm || (eps >= 1e-12f && eps <= 1.0f), GPTQ_ERR_ARG, "%s: eps %g (it has to lie in [1e-12, 1])", fn, eps);
  return GPTQ_OK;
}
// rows that vector accesses can take: 16-byte aligned, whole 8s of elements
// (codes: 16s) apart
int check_rows(const char* fn, std::initializer_list<const void*> ps, std::initializer_list<int64_t> strides, int unit) {
  uintptr_t bits = 0;
  for (const void* p : ps) bits |= reinterpret_cast<uintptr_t>(p);
  GPTQ_REQUIRE(bits % 16 == 0, GPTQ_ERR_ARG, "%s: rows and tables have to be 16-byte aligned", fn);
  for (int64_t s : strides)
    GPTQ_REQUIRE(s >= 0 && s % unit == 0, GPTQ_ERR_SHAPE, "%s: strides have to be multiples of %d elements (got %lld)", fn,
                 unit, static_cast<long long>(s));
  return GPTQ_OK;
}

NormArgs common_args(const void* q_weight, const void* k_weight, int weight_type, float eps, const float* table, int64_t P,
                     int64_t R, const int32_t* positions, int interleaved, int64_t T, int64_t H, int64_t Hk, int64_t D) {
  NormArgs a{};
  a.q_weight = q_weight, a.k_weight = k_weight, a.weight_type = weight_type, a.eps = eps;
  a.table = table, a.P = P, a.R = static_cast<int>(R), a.positions = positions;
  a.interleaved = interleaved != 0;
  a.T = static_cast<int>(T), a.H = static_cast<int>(H), a.Hk = static_cast<int>(Hk), a.D = static_cast<int>(D);
  a.inv_d = 1.0f / static_cast<float>(D);
  a.page = fast_div(1);
  return a;
}

}  // namespace
}  // namespace gptq

using namespace gptq;

extern "C" int gptq_norm_rotary(const void* q, const void* k, int dtype, int64_t q_token, int64_t q_head, int64_t k_token,
                                int64_t k_head, const void* q_weight, const void* k_weight, int weight_dtype, float eps,
                                const float* table, int64_t table_rows, int64_t rotary_dim, const int32_t* positions,
                                int interleaved, int64_t T, int64_t H, int64_t Hk, int64_t D, void* q_out, void* k_out,
                                gptq_stream_t stream) {
  const char* fn = "gptq_norm_rotary";
  clear_error();
  int rc = check_sizes(fn, dtype, weight_dtype, true, eps, table, table_rows, rotary_dim, T, H, Hk, D);
  if (rc != GPTQ_OK || T == 0) return rc;
  GPTQ_REQUIRE(q && k && q_weight && k_weight && q_out && k_out && (!table || positions), GPTQ_ERR_ARG, "%s: null pointer",
               fn);
  rc = check_rows(fn, {q, k, q_weight, k_weight, table, q_out, k_out}, {q_token, q_head, k_token, k_head}, 8);
  if (rc != GPTQ_OK) return rc;
  NormArgs a = common_args(q_weight, k_weight, weight_dtype, eps, table, table_rows, rotary_dim, positions, interleaved, T,
                           H, Hk, D);
  a.q = {q, q_token, q_head}, a.k = {k, k_token, k_head};
  a.q_out = q_out, a.k_out = k_out;
  return launch_unit<0>(a, dtype, fn, as_hip(stream));
}

extern "C" size_t gptq_norm_rotary_backward_workspace_size(int64_t T, int64_t H, int64_t Hk, int64_t D) {
  if (T < 0 || T >= (int64_t{1} << 31) || H < 1 || H > 65536 || Hk < 1 || Hk > 65536 || D < 8 || D > 256) return 0;
  return static_cast<size_t>(back_blocks(T, H, Hk) * 2 * D) * sizeof(float);
}

extern "C" int gptq_norm_rotary_backward(const void* grad_q, const void* grad_k, const void* q, const void* k, int dtype,
                                         int64_t gq_token, int64_t gq_head, int64_t gk_token, int64_t gk_head,
                                         int64_t q_token, int64_t q_head, int64_t k_token, int64_t k_head,
                                         const void* q_weight, const void* k_weight, int weight_dtype, float eps,
                                         const float* table, int64_t table_rows, int64_t rotary_dim,
                                         const int32_t* positions, int interleaved, int64_t T, int64_t H, int64_t Hk,
                                         int64_t D, void* dq, void* dk, void* dq_weight, void* dk_weight, void* workspace,
                                         size_t workspace_bytes, gptq_stream_t stream) {
  const char* fn = "gptq_norm_rotary_backward";
  clear_error();
  int rc = check_sizes(fn, dtype, weight_dtype, true, eps, table, table_rows, rotary_dim, T, H, Hk, D);
  if (rc != GPTQ_OK) return rc;
  GPTQ_REQUIRE(q_weight && k_weight && (T == 0 || (grad_q && grad_k && q && k && dq && dk && (!table || positions))) &&
                   !dq_weight == !dk_weight,
               GPTQ_ERR_ARG, "%s: null pointer", fn);
  rc = check_rows(fn, {grad_q, grad_k, q, k, q_weight, k_weight, table, dq, dk, workspace},
                  {gq_token, gq_head, gk_token, gk_head, q_token, q_head, k_token, k_head}, 8);
  if (rc != GPTQ_OK) return rc;
  const size_t need = dq_weight ? gptq_norm_rotary_backward_workspace_size(T, H, Hk, D) : 0;
  GPTQ_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), GPTQ_ERR_WORKSPACE,
               "%s: workspace of %zu bytes, needs %zu", fn, workspace_bytes, need);
  if (T == 0 && !dq_weight) return GPTQ_OK;
  NormArgs a = common_args(q_weight, k_weight, weight_dtype, eps, table, table_rows, rotary_dim, positions, interleaved, T,
                           H, Hk, D);
  a.q = {q, q_token, q_head}, a.k = {k, k_token, k_head};
  a.grad_q = {grad_q, gq_token, gq_head}, a.grad_k = {grad_k, gk_token, gk_head};
  a.dq = dq, a.dk = dk;
  a.part = dq_weight ? static_cast<float*>(workspace) : nullptr;
  const hipStream_t st = as_hip(stream);
  const int n = unit_of(a);
  rc = n == 8 ? launch_back_type<8>(a, dtype, st) : n == 4 ? launch_back_type<4>(a, dtype, st) : launch_back_type<2>(a, dtype, st);
  if (rc != GPTQ_OK || !dq_weight) return rc;
  norm_weight_sum_kernel<<<dim3(static_cast<uint32_t>(D / 4), 2), 256, 0, st>>>(
      a.part, static_cast<int>(back_blocks(T, H, Hk)), a.D, weight_dtype, dq_weight, dk_weight);
  return check_launch(fn);
}

extern "C" int gptq_norm_rotary_append(
    const void* q, const void* k, const void* v, int dtype, int64_t q_token, int64_t q_head, int64_t k_token,
    int64_t k_head, int64_t v_token, int64_t v_head, const void* q_weight, const void* k_weight, int weight_dtype, float eps,
    const float* table, int64_t table_rows, int64_t rotary_dim, const int32_t* positions, int interleaved,
    const int32_t* slots, int64_t page_size, int64_t pages, int64_t T, int64_t H, int64_t Hk, int64_t D, void* q_out,
    int code, void* k_cache, int64_t k_page, int64_t kc_token, int64_t kc_head, void* v_cache, int64_t v_page,
    int64_t vc_token, int64_t vc_head, float* k_scale, int64_t ks_page, int64_t ks_token, int64_t ks_head, float* v_scale,
    int64_t vs_page, int64_t vs_token, int64_t vs_head, gptq_stream_t stream) {
  const char* fn = "gptq_norm_rotary_append";
  clear_error();
  const bool norm = q_weight || k_weight;
  int rc = check_sizes(fn, dtype, weight_dtype, norm, eps, table, table_rows, rotary_dim, T, H, Hk, D);
  if (rc != GPTQ_OK) return rc;
  GPTQ_REQUIRE(code == GPTQ_CODE_NONE || code == GPTQ_CODE_I8 || code == GPTQ_CODE_E4M3, GPTQ_ERR_DTYPE,
               "%s: unknown codes %d", fn, code);
  GPTQ_REQUIRE(code == GPTQ_CODE_NONE || D % 16 == 0, GPTQ_ERR_SHAPE,
               "%s: heads of %lld values (codes take multiples of 16)", fn, static_cast<long long>(D));
  GPTQ_REQUIRE(page_size >= 1 && page_size < (int64_t{1} << 31) && pages >= 0 && pages < (int64_t{1} << 31), GPTQ_ERR_ARG,
               "%s: bad cache (%lld pages of %lld tokens)", fn, static_cast<long long>(pages),
               static_cast<long long>(page_size));
  if (T == 0) return GPTQ_OK;
  GPTQ_REQUIRE(q && k && v && slots && q_out && (pages == 0 || (k_cache && v_cache)) && !q_weight == !k_weight &&
                   (!table || positions) && (code == GPTQ_CODE_NONE || pages == 0 || (k_scale && v_scale)),
               GPTQ_ERR_ARG, "%s: null pointer", fn);
  rc = check_rows(fn, {q, k, v, q_weight, k_weight, table, q_out, k_cache, v_cache},
                  {q_token, q_head, k_token, k_head, v_token, v_head}, 8);
  if (rc != GPTQ_OK) return rc;
  rc = check_rows(fn, {}, {k_page, kc_token, kc_head, v_page, vc_token, vc_head}, code == GPTQ_CODE_NONE ? 8 : 16);
  if (rc != GPTQ_OK) return rc;
  NormArgs a = common_args(q_weight, k_weight, weight_dtype, eps, table, table_rows, rotary_dim, positions, interleaved, T,
                           H, Hk, D);
  a.q = {q, q_token, q_head}, a.k = {k, k_token, k_head}, a.v = {v, v_token, v_head};
  a.slots = slots, a.page = fast_div(static_cast<uint32_t>(page_size)), a.capacity = pages * page_size;
  a.q_out = q_out;
  a.kc = {k_cache, k_page, kc_token, kc_head, k_scale, ks_page, ks_token, ks_head};
  a.vc = {v_cache, v_page, vc_token, vc_head, v_scale, vs_page, vs_token, vs_head};
  const hipStream_t st = as_hip(stream);
  if (code == GPTQ_CODE_I8) return launch_unit<GPTQ_CODE_I8>(a, dtype, fn, st);
  if (code == GPTQ_CODE_E4M3) return launch_unit<GPTQ_CODE_E4M3>(a, dtype, fn, st);
  return launch_unit<0>(a, dtype, fn, st);
}
