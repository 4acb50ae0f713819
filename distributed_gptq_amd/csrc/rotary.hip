// Rotary positions: channels pairs (a, b) of each head of a token turned by the
// token's angles, a' = a cos - b sin, b' = b cos + a sin, and keys and values
// written into the pages of a cache on the way.
#include "values.hpp"

namespace gptq {
namespace {

struct RotaryArgs {
  const void *q, *k, *v;            // (T, heads, D) by strides; v null without a cache
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;
  const float* table;               // (P, 2, R / 2): cosines, then sines; null: nothing turns
  const int32_t* positions;         // (T)
  const int32_t* slots;             // (T) places in the cache, or null: k_out by strides
  void *q_out, *k_out, *v_out;
  int64_t qo_token, qo_head, ko_page, ko_token, ko_head, vo_page, vo_token, vo_head;
  int64_t T, P, capacity;           // tokens, table rows, places of the cache
  int page_size;
  int H, Hk, D, R;
  int interleaved;
  float sign;                       // -1 turns back (the gradient)
};

// A thread has N pairs of channels of a token (unit u: channels u N .. and
// R / 2 + u N .., or 2 u N .. with neighbours as pairs; past R / 2 pairs, 2 N
// channels that are copied) and kPerThread heads, whose angles it reads once.
// Bound by memory: every value is read and written once, with 16-byte accesses
// where the layout allows them (N = 8 of 16 bits).  16384 tokens, 32 over 8 heads
// of 128: 69 us, 5.0 TB/s, the rate of a large copy; 2048 tokens of 40 heads
// stored into a cache on the way 26.6 us.
template <int N, int kType>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a, int units, int groups, int per) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t tg = id / units;
  const int u = static_cast<int>(id - tg * units);
  const int64_t t = tg / groups;
  const int g = static_cast<int>(tg - t * groups);
  if (t >= a.T) return;
  const int half = a.table ? a.R / 2 : 0;
  const bool turns = u * N < half;
  float c[N], s[N];
  if (turns) {
    int64_t pos = a.positions[t];
    pos = pos < 0 ? 0 : pos >= a.P ? a.P - 1 : pos;
    const float* row = a.table + pos * a.R + u * N;
    load_values<N, GPTQ_F32>(c, row, 0);
    load_values<N, GPTQ_F32>(s, row, half);
#pragma unroll
    for (int e = 0; e < N; ++e) s[e] *= a.sign;
  }
  const int first = turns && !a.interleaved ? u * N : 2 * u * N;
  const int second = turns && !a.interleaved ? half + u * N : first + N;
  int64_t page = 0, at = t;
  bool kept = true;
  if (a.slots) {
    const int64_t slot = a.slots[t];
    kept = slot >= 0 && slot < a.capacity;
    page = slot / a.page_size;
    at = slot - page * a.page_size;
  }
  const int heads = a.H + a.Hk + (a.v ? a.Hk : 0);
  for (int h = g * per; h < (g + 1) * per && h < heads; ++h) {
    const void* from;
    void* to;
    int64_t i, o;
    const bool values = h >= a.H + a.Hk;
    if (h < a.H) {
      from = a.q, i = t * a.q_token + h * a.q_head;
      to = a.q_out, o = t * a.qo_token + h * a.qo_head;
    } else if (!values) {
      from = a.k, i = t * a.k_token + (h - a.H) * a.k_head;
      to = a.k_out, o = page * a.ko_page + at * a.ko_token + (h - a.H) * a.ko_head;
    } else {
      from = a.v, i = t * a.v_token + (h - a.H - a.Hk) * a.v_head;
      to = a.v_out, o = page * a.vo_page + at * a.vo_token + (h - a.H - a.Hk) * a.vo_head;
    }
    if (h >= a.H && !kept) continue;
    float x[N], y[N];
    load_values<N, kType>(x, from, i + first);
    load_values<N, kType>(y, from, i + second);
    if (turns && !values) {
      if (a.interleaved) {
        float xy[2 * N];
#pragma unroll
        for (int e = 0; e < N; ++e) xy[e] = x[e], xy[N + e] = y[e];
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float p = xy[2 * e], r = xy[2 * e + 1];
          xy[2 * e] = p * c[e] - r * s[e];
          xy[2 * e + 1] = r * c[e] + p * s[e];
        }
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = xy[e], y[e] = xy[N + e];
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float p = x[e], r = y[e];
          x[e] = p * c[e] - r * s[e];
          y[e] = r * c[e] + p * s[e];
        }
      }
    }
    store_values<N, kType>(to, o + first, x);
    store_values<N, kType>(to, o + second, y);
  }
}

template <int N, int kType>
int launch(const RotaryArgs& a, hipStream_t st) {
  const int units = a.D / 2 / N;
  const int heads = a.H + a.Hk + (a.v ? a.Hk : 0);
  // enough threads for the GPU first, then heads that share a thread's angles
  const int64_t threads = a.T * units * heads;
  int per = static_cast<int>(threads / (256 * 2048));
  per = per < 1 ? 1 : per > 8 ? 8 : per;
  const int groups = (heads + per - 1) / per;
  const int64_t blocks = cdiv(a.T * groups * units, 256);
  GPTQ_REQUIRE(blocks < (int64_t{1} << 31), GPTQ_ERR_SHAPE, "gptq_rotary: too many tokens");
  rotary_kernel<N, kType><<<static_cast<uint32_t>(blocks), 256, 0, st>>>(a, units, groups, per);
  return check_launch("gptq_rotary");
}

template <int N>
int launch_type(const RotaryArgs& a, int dtype, hipStream_t st) {
  if (dtype == GPTQ_F32) return launch<N, GPTQ_F32>(a, st);
  if (dtype == GPTQ_BF16) return launch<N, GPTQ_BF16>(a, st);
  return launch<N, GPTQ_F16>(a, st);
}

// the widest N that every address allows
int run(const RotaryArgs& a, int dtype, const char* fn, hipStream_t st) {
  GPTQ_REQUIRE(valid_dtype(dtype), GPTQ_ERR_DTYPE, "%s: expected fp32, fp16 or bf16", fn);
  GPTQ_REQUIRE(a.T >= 0 && a.H >= 0 && a.Hk >= 0 && a.H <= 65536 && a.Hk <= 65536 && a.D >= 2 && a.D % 2 == 0 &&
                   a.D <= 65536 && a.T < (int64_t{1} << 31),
               GPTQ_ERR_SHAPE, "%s: %lld tokens, %d and %d heads of %d values", fn, static_cast<long long>(a.T), a.H,
               a.Hk, a.D);
  GPTQ_REQUIRE(!a.table || (a.R >= 2 && a.R % 2 == 0 && a.R <= a.D && a.P >= 1), GPTQ_ERR_SHAPE,
               "%s: a table of %lld positions for %d of %d values", fn, static_cast<long long>(a.P), a.R, a.D);
  if (a.T == 0 || a.H + a.Hk == 0) return GPTQ_OK;
  GPTQ_REQUIRE((a.H == 0 || (a.q && a.q_out)) && (a.Hk == 0 || (a.k && a.k_out)) && (!a.v || a.v_out) &&
                   (!a.table || a.positions),
               GPTQ_ERR_ARG, "%s: null pointer", fn);
  const int size = dtype_size(dtype);
  const int half = a.table ? a.R / 2 : 0;
  auto fits = [&](int n) {
    const int64_t bytes = n * size < 16 ? n * size : 16;
    if (half % n || (a.D / 2) % n || (a.table && reinterpret_cast<uintptr_t>(a.table) % (n < 4 ? 4 * n : 16))) return false;
    const void* ps[] = {a.q, a.k, a.v, a.q_out, a.k_out, a.v_out};
    for (const void* p : ps)
      if (reinterpret_cast<uintptr_t>(p) % bytes) return false;
    const int64_t strides[] = {a.q_token, a.q_head,   a.k_token, a.k_head,   a.v_token, a.v_head,   a.qo_token,
                               a.qo_head, a.ko_page, a.ko_token, a.ko_head, a.vo_page,  a.vo_token, a.vo_head};
    for (int64_t s : strides)
      if (s * size % bytes) return false;
    return true;
  };
  if (fits(8)) return launch_type<8>(a, dtype, st);
  if (fits(2)) return launch_type<2>(a, dtype, st);
  return launch_type<1>(a, dtype, st);
}

}  // namespace
}  // namespace gptq

using namespace gptq;

extern "C" int gptq_rotary(const void* q, const void* k, int dtype, int64_t q_token, int64_t q_head, int64_t k_token,
                           int64_t k_head, const float* table, int64_t table_rows, int64_t rotary_dim,
                           const int32_t* positions, int interleaved, int inverse, int64_t T, int64_t H, int64_t Hk,
                           int64_t D, void* q_out, void* k_out, gptq_stream_t stream) {
  clear_error();
  GPTQ_REQUIRE(table, GPTQ_ERR_ARG, "gptq_rotary: null pointer");
  GPTQ_REQUIRE(H >= 0 && H <= 65536 && Hk >= 0 && Hk <= 65536 && D >= 0 && D <= 65536 && rotary_dim >= 0 &&
                   rotary_dim <= 65536,
               GPTQ_ERR_SHAPE, "gptq_rotary: sizes out of range");
  RotaryArgs a{};
  a.q = q, a.k = k;
  a.q_token = q_token, a.q_head = q_head, a.k_token = k_token, a.k_head = k_head;
  a.table = table, a.P = table_rows, a.R = static_cast<int>(rotary_dim), a.positions = positions;
  a.q_out = q_out, a.k_out = k_out;
  a.qo_token = H * D, a.qo_head = D, a.ko_token = Hk * D, a.ko_head = D;
  a.T = T, a.H = static_cast<int>(H), a.Hk = static_cast<int>(Hk), a.D = static_cast<int>(D);
  a.page_size = 1;
  a.interleaved = interleaved != 0;
  a.sign = inverse ? -1.0f : 1.0f;
  return run(a, dtype, "gptq_rotary", as_hip(stream));
}

extern "C" int gptq_rotary_append(const void* q, const void* k, const void* v, int dtype, int64_t q_token,
                                  int64_t q_head, int64_t k_token, int64_t k_head, int64_t v_token, int64_t v_head,
                                  const float* table, int64_t table_rows, int64_t rotary_dim, const int32_t* positions,
                                  int interleaved, const int32_t* slots, int64_t page_size, int64_t pages, int64_t T,
                                  int64_t H, int64_t Hk, int64_t D, void* q_out, void* k_cache, int64_t k_page,
                                  int64_t kc_token, int64_t kc_head, void* v_cache, int64_t v_page, int64_t vc_token,
                                  int64_t vc_head, gptq_stream_t stream) {
  clear_error();
  GPTQ_REQUIRE(H >= 0 && H <= 65536 && Hk >= 1 && Hk <= 65536 && D >= 0 && D <= 65536 && rotary_dim >= 0 &&
                   rotary_dim <= 65536,
               GPTQ_ERR_SHAPE, "gptq_rotary_append: sizes out of range");
  GPTQ_REQUIRE(page_size >= 1 && page_size < (int64_t{1} << 31) && pages >= 0 && pages < (int64_t{1} << 31), GPTQ_ERR_ARG,
               "gptq_rotary_append: bad cache (%lld pages of %lld tokens)", static_cast<long long>(pages),
               static_cast<long long>(page_size));
  GPTQ_REQUIRE(T == 0 || (slots && v && v_cache), GPTQ_ERR_ARG, "gptq_rotary_append: null pointer");
  RotaryArgs a{};
  a.q = q, a.k = k, a.v = v;
  a.q_token = q_token, a.q_head = q_head, a.k_token = k_token, a.k_head = k_head, a.v_token = v_token, a.v_head = v_head;
  a.table = table, a.P = table_rows, a.R = static_cast<int>(rotary_dim), a.positions = positions;
  a.slots = slots, a.page_size = static_cast<int>(page_size), a.capacity = pages * page_size;
  a.q_out = q_out, a.k_out = k_cache, a.v_out = v_cache;
  a.qo_token = H * D, a.qo_head = D;
  a.ko_page = k_page, a.ko_token = kc_token, a.ko_head = kc_head;
  a.vo_page = v_page, a.vo_token = vc_token, a.vo_head = vc_head;
  a.T = T, a.H = static_cast<int>(H), a.Hk = static_cast<int>(Hk), a.D = static_cast<int>(D);
  a.interleaved = interleaved != 0;
  a.sign = 1.0f;
  return run(a, dtype, "gptq_rotary_append", as_hip(stream));
}
