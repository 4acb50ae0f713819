// The rows of a paged cache read back as packed rows: copied, or code * scale
// where it holds codes.
#include "attn_index.hpp"
#include "codes.hpp"
#include "values.hpp"

#include <type_traits>

namespace gptq {
namespace {

struct ReadRows {
  const uint8_t* p;
  int64_t page, token, head;        // strides, in bytes
  const float* scale;
  int64_t s_page, s_token, s_head;  // in elements
};

struct CachedArgs {
  ReadRows k, v;
  void *k_out, *v_out;              // (T, Hk, D)
  const int32_t* table;             // (B, width) page numbers
  const int32_t* context;           // (B) cached tokens
  const int32_t* cu;                // (B + 1) offsets of the rows
  int64_t table_stride;
  FastDiv page, groups, chunks;     // tokens of a page; groups of heads; chunks of a row
  int most, pages, B, T, heads, D;
};

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// 8 codes as kType values, or 16 bytes as they are.
template <int kCode>
using Chunk = std::conditional_t<kCode == GPTQ_CODE_NONE, u32x4, u32x2>;

template <int kType, int kCode>
__device__ __forceinline__ void put_chunk(void* out, int64_t row, int D, int c, const Chunk<kCode>& w, float scale) {
  if constexpr (kCode == GPTQ_CODE_NONE) {
    *reinterpret_cast<u32x4*>(static_cast<uint8_t*>(out) + row * D * (kType == GPTQ_F32 ? 4 : 2) + 16 * c) = w;
  } else {
    float x[8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const f32x4 f = decode4<kCode>(w[i]);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * i + e] = f[e] * scale;
    }
    store_values<8, kType>(out, row * D + 8 * c, x);
  }
}

// A thread has a chunk of the keys and values of kHeads heads of a token, whose
// sequence and page it looks up once and whose loads go together.  Packed row t of
// sequence b is its cached token context - (cu[b + 1] - t).  Bound by memory: 46k
// rows of 8 heads of 128 int8 codes into bf16 (286 MB) take 62 us, 4.6 TB/s; with 2
// heads 67 us, with 8 65 us, with one 99 us, with 16 codes of one head 67 us (half
// of each line per store).
constexpr int kHeads = 4;
template <int kType, int kCode>
__global__ __launch_bounds__(256) void cached_rows_kernel(CachedArgs a) {
  using C = Chunk<kCode>;
  const int per = 256 / static_cast<int>(a.chunks.d);  // items of a workgroup
  const int r = div_by(static_cast<int>(threadIdx.x), a.chunks);
  const int c = static_cast<int>(threadIdx.x) - r * static_cast<int>(a.chunks.d);
  const int64_t item = static_cast<int64_t>(blockIdx.x) * per + r;
  if (r >= per || item >= static_cast<int64_t>(a.T) * a.groups.d) return;
  const int t = div_by(static_cast<int>(item), a.groups);
  const int h0 = (static_cast<int>(item) - t * static_cast<int>(a.groups.d)) * kHeads;
  int b;
  const int key = cached_token(a.cu, a.context, a.B, a.most, t, &b);
  C kw[kHeads], vw[kHeads];
  float ks[kHeads], vs[kHeads];
  if (key >= 0) {
    const int n = div_by(key, a.page);
    const int64_t page = clamp_int(a.table[b * a.table_stride + n], 0, a.pages - 1);
    const int64_t at = key - n * static_cast<int>(a.page.d);
    const uint8_t* kp = a.k.p + page * a.k.page + at * a.k.token + sizeof(C) * c;
    const uint8_t* vp = a.v.p + page * a.v.page + at * a.v.token + sizeof(C) * c;
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      const int64_t h = h0 + i < a.heads ? h0 + i : a.heads - 1;
      kw[i] = *reinterpret_cast<const C*>(kp + h * a.k.head);
      vw[i] = *reinterpret_cast<const C*>(vp + h * a.v.head);
      if constexpr (kCode != GPTQ_CODE_NONE) {
        ks[i] = a.k.scale[page * a.k.s_page + at * a.k.s_token + h * a.k.s_head];
        vs[i] = a.v.scale[page * a.v.s_page + at * a.v.s_token + h * a.v.s_head];
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kHeads; ++i) kw[i] = vw[i] = C{}, ks[i] = vs[i] = 0.0f;
  }
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    if (h0 + i >= a.heads) break;
    const int64_t row = static_cast<int64_t>(t) * a.heads + h0 + i;
    put_chunk<kType, kCode>(a.k_out, row, a.D, c, kw[i], ks[i]);
    put_chunk<kType, kCode>(a.v_out, row, a.D, c, vw[i], vs[i]);
  }
}

template <int kType, int kCode>
int launch(CachedArgs a, hipStream_t st) {
  a.groups = fast_div(static_cast<uint32_t>(cdiv(a.heads, kHeads)));
  a.chunks = fast_div(static_cast<uint32_t>(kCode == GPTQ_CODE_NONE ? a.D * (kType == GPTQ_F32 ? 4 : 2) / 16 : a.D / 8));
  const int64_t items = static_cast<int64_t>(a.T) * a.groups.d;
  const uint32_t blocks = static_cast<uint32_t>(cdiv(items, 256 / a.chunks.d));
  cached_rows_kernel<kType, kCode><<<blocks, 256, 0, st>>>(a);
  return check_launch("gptq_cached_rows");
}
template <int kType>
int launch_code(const CachedArgs& a, int code, hipStream_t st) {
  if (code == GPTQ_CODE_I8) return launch<kType, GPTQ_CODE_I8>(a, st);
  if (code == GPTQ_CODE_E4M3) return launch<kType, GPTQ_CODE_E4M3>(a, st);
  return launch<kType, GPTQ_CODE_NONE>(a, st);
}

}  // namespace
}  // namespace gptq

using namespace gptq;

extern "C" int gptq_cached_rows(int code, const void* k_cache, int64_t k_page, int64_t k_token, int64_t k_head,
                                const void* v_cache, int64_t v_page, int64_t v_token, int64_t v_head, const float* k_scale,
                                int64_t ks_page, int64_t ks_token, int64_t ks_head, const float* v_scale, int64_t vs_page,
                                int64_t vs_token, int64_t vs_head, const int32_t* block_table, int64_t table_stride,
                                int64_t width, int64_t page_size, int64_t pages, const int32_t* context,
                                const int32_t* cu_rows, int64_t B, int64_t T, int64_t Hk, int64_t D, void* k_out,
                                void* v_out, int out_dtype, gptq_stream_t stream) {
  const char* fn = "gptq_cached_rows";
  clear_error();
  GPTQ_REQUIRE(valid_dtype(out_dtype) && (code == GPTQ_CODE_NONE || code == GPTQ_CODE_I8 || code == GPTQ_CODE_E4M3),
               GPTQ_ERR_DTYPE, "%s: expected fp32, fp16 or bf16 rows of values or codes", fn);
  constexpr int64_t kMost = (int64_t{1} << 31) - 4096;
  GPTQ_REQUIRE(B >= 1 && B < kMost && T >= 0 && Hk >= 1 && Hk <= 65536 && T < kMost / Hk, GPTQ_ERR_SHAPE,
               "%s: %lld sequences, %lld rows of %lld heads", fn, static_cast<long long>(B), static_cast<long long>(T),
               static_cast<long long>(Hk));
  const int size = code == GPTQ_CODE_NONE ? dtype_size(out_dtype) : 1;  // of a cached value
  GPTQ_REQUIRE(D >= 8 && D <= 256 && D * size % 16 == 0, GPTQ_ERR_SHAPE,
               "%s: heads of %lld values (multiples of 16 bytes of up to 256 are supported)", fn, static_cast<long long>(D));
  GPTQ_REQUIRE(page_size >= 1 && page_size < (int64_t{1} << 31) && pages >= 1 && pages < (int64_t{1} << 31) && width >= 0,
               GPTQ_ERR_ARG, "%s: bad cache (%lld pages of %lld tokens, table of %lld)", fn, static_cast<long long>(pages),
               static_cast<long long>(page_size), static_cast<long long>(width));
  if (T == 0) return GPTQ_OK;
  GPTQ_REQUIRE(k_cache && v_cache && k_out && v_out && context && cu_rows && (block_table || width == 0) &&
                   (code == GPTQ_CODE_NONE || (k_scale && v_scale)),
               GPTQ_ERR_ARG, "%s: null pointer", fn);
  for (const void* p : {k_cache, v_cache, static_cast<const void*>(k_out), static_cast<const void*>(v_out)})
    GPTQ_REQUIRE(reinterpret_cast<uintptr_t>(p) % 16 == 0, GPTQ_ERR_ARG, "%s: rows have to be 16-byte aligned", fn);
  for (int64_t s : {k_page, k_token, k_head, v_page, v_token, v_head})
    GPTQ_REQUIRE(s >= 0 && s * size % 16 == 0, GPTQ_ERR_SHAPE, "%s: strides have to be multiples of 16 bytes (got %lld)", fn,
                 static_cast<long long>(s));
  CachedArgs a{};
  a.k = {static_cast<const uint8_t*>(k_cache), k_page * size, k_token * size, k_head * size, k_scale, ks_page, ks_token, ks_head};
  a.v = {static_cast<const uint8_t*>(v_cache), v_page * size, v_token * size, v_head * size, v_scale, vs_page, vs_token, vs_head};
  a.k_out = k_out, a.v_out = v_out;
  a.table = block_table, a.context = context, a.cu = cu_rows, a.table_stride = table_stride;
  a.page = fast_div(static_cast<uint32_t>(page_size));
  a.most = static_cast<int>(plan::cached_most(width, page_size));
  a.pages = static_cast<int>(pages);
  a.B = static_cast<int>(B), a.T = static_cast<int>(T), a.heads = static_cast<int>(Hk), a.D = static_cast<int>(D);
  const hipStream_t st = as_hip(stream);
  if (out_dtype == GPTQ_F32) return launch_code<GPTQ_F32>(a, code, st);
  if (out_dtype == GPTQ_BF16) return launch_code<GPTQ_BF16>(a, code, st);
  return launch_code<GPTQ_F16>(a, code, st);
}
