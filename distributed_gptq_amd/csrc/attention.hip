// Attention of packed sequences (keys as rows or in the pages of a cache) on
// gfx950 MFMA: o_i = sum_j p_ij v_j, p_ij = 2^(c q_i k_j) / sum_j 2^(c q_i k_j)
// over the keys j that query i sees, c = scale log2(e).
#include "attn_join.hpp"
#include "attn_tile.hpp"

namespace gptq {
namespace {

constexpr int kKeys = 64;  // keys of a tile

// What one wave carries for its 32 columns: the running maximum m (in log2
// units; for fp16 less kBias, see below), this lane's part of the sum of
// weights, and the sum of weighted values.
//
// Weights are rounded to the values' type before they are multiplied: their
// product then runs on the 16-bit MFMA, and the error (half a unit of each
// weight's last place, independent) stays below the rounding of the result.
// Their sum is of the unrounded weights in fp32.  fp16 weights are kept 2^kBias
// times larger than exp2(s - max): fp16 ends at 2^-24, which would drop the
// tail of a long row; the largest is 2^(kBias + kSlack) < 65504.
//
// The maximum is only raised when a score passes it by kSlack (log2): the sums
// then are rescaled for few tiles, and weights stay below 2^kSlack (2^(kBias +
// kSlack) in fp16), which costs no precision in a floating type.
constexpr float kSlack = 8.0f;
template <bool kBF16>
constexpr float kBias = kBF16 ? 0.0f : 7.0f;

template <int DT>
struct Column {
  float m, l;
  f32x16 o[DT / 32];
};

// Adds NK x 32 keys with scores s (raw q k) to the column's sums.  `value`
// gives the operand of value rows 16 ks .. of the tile, channels 32 db ...
// kRest: what the rounding of the weights left is multiplied too.  For few rows
// over a cache, whose bytes take longer than both products; and where the
// gradient follows, which subtracts delta = g o from every g v of a row, so that
// an error of o reaches all its keys alike and adds up in dq and dk where errors
// of single weights cancel (2 x 2048 tokens, bf16: error of dq against 64 bits
// 1.55 times that of its rounding alone with the rounded weights and output, 1.45
// so).
template <bool kBF16, int DT, int NK, bool kRest, class Value>
__device__ __forceinline__ void softmax_step(Column<DT>& col, f32x16 (&s)[NK], float c, Value&& value) {
  float t = s[0][0];
#pragma unroll
  for (int kt = 0; kt < NK; ++kt)
#pragma unroll
    for (int i = 0; i < 16; ++i) t = __builtin_elementwise_maximum(t, s[kt][i]);  // (fmaxf quiets its arguments first)
  t = half_max(t) * c - kBias<kBF16>;
  if (__builtin_expect(__ballot(t > col.m + kSlack) != 0, 0)) {
    const float m = fmaxf(col.m, t);
    const float alpha = __builtin_amdgcn_exp2f(col.m - m);
    col.m = m;
    col.l *= alpha;
#pragma unroll
    for (int db = 0; db < DT / 32; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) col.o[db][i] *= alpha;
  }
  float sum = 0.0f;
#pragma unroll
  for (int kt = 0; kt < NK; ++kt)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[kt][i] = __builtin_amdgcn_exp2f(fmaf(s[kt][i], c, -col.m));
      sum += s[kt][i];
    }
  col.l += sum;
#pragma unroll
  for (int ks = 0; ks < 2 * NK; ++ks) {
    const u32x4 p = operand_of<kBF16>(s[ks / 2], 8 * (ks % 2));
#pragma unroll
    for (int db = 0; db < DT / 32; ++db) {
      const u32x4 v = value(ks, db);
      col.o[db] = mma32<kBF16>(v, p, col.o[db]);
      if constexpr (kRest) col.o[db] = mma32<kBF16>(v, operand_rest<kBF16>(s[ks / 2], 8 * (ks % 2), p), col.o[db]);
    }
  }
}

// Writes a column's result: the output (and lse), or this split's sums.  kExact:
// of sums that may hold infinities (whose rounding leaves nothing).
template <bool kBF16, int DT, bool kTrain, bool kExact>
__device__ __forceinline__ void store_column(const AttnArgs& a, const Column<DT>& col, float l, int64_t row, bool none,
                                             int split, int half) {
  if (a.splits > 1) {
    float* part = a.part + (split * (static_cast<int64_t>(a.T) * a.H) + row) * a.D;
#pragma unroll
    for (int db = 0; db < DT / 32; ++db)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int d = 32 * db + acc_row(i, half);
        if (d < a.D)
          *reinterpret_cast<f32x4*>(part + d) =
              none ? f32x4{0.0f, 0.0f, 0.0f, 0.0f}
                   : f32x4{col.o[db][i], col.o[db][i + 1], col.o[db][i + 2], col.o[db][i + 3]};
      }
    return;
  }
  const float r = none ? 0.0f : 1.0f / l;
  uint16_t* out = a.out + row * a.D;
#pragma unroll
  for (int db = 0; db < DT / 32; ++db)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int d = 32 * db + acc_row(i, half);
      if (d >= a.D) continue;
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = none ? 0.0f : col.o[db][i + e] * r;
      const u32x2 w = {pack16<kBF16>(y[0], y[1]), pack16<kBF16>(y[2], y[3])};
      *reinterpret_cast<u32x2*>(out + d) = w;
      if constexpr (kTrain) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float rest = y[e] - value16<kBF16>(static_cast<uint16_t>(w[e / 2] >> (16 * (e % 2))));
          y[e] = !kExact || fabsf(y[e]) < INFINITY ? rest : 0.0f;
        }
        *reinterpret_cast<u32x2*>(a.out_rest + row * a.D + d) = u32x2{pack16<kBF16>(y[0], y[1]), pack16<kBF16>(y[2], y[3])};
      }
    }
}

// The e of a sum of weights l that 2^-e brings to [1/2, 1) in bf16 (see
// exact_columns; fp16's values are far from fp32's end).
template <bool kBF16>
__device__ __forceinline__ int down_bits(float l) {
  return kBF16 && l > 0.0f ? ilogbf(l) + 1 : 0;
}

// The row's statistics: lse, or this split's maximum and sum.  A row that sees
// no key (of the split) has maximum -infinity there.
__device__ __forceinline__ void store_stats(const AttnArgs& a, float m, float l, int64_t row, bool none, int split) {
  const int64_t rows = static_cast<int64_t>(a.T) * a.H;
  if (a.splits > 1) {
    float* mm = a.part + a.splits * rows * a.D;
    mm[split * rows + row] = none ? -INFINITY : m;
    mm[(a.splits + split) * rows + row] = none ? 0.0f : l;
  } else if (a.lse) {
    a.lse[row] = none ? -INFINITY : m + log2f(l);
  }
}

// The columns again where the sums are not finite, by one wave, col.m and l of
// all the keys known: tiles of 32 keys t0, t0 + step, ... below t1 through `room`
// in LDS (two tiles), their values added row by row.  Slower than the products
// of tiles by the vector instructions: 64 for a row of 128 values instead of 4
// MFMAs for 32 of them.
//
// A key that is seen has a weight, however small, so that an infinite value of
// it gives an infinity.  `down` (bf16) brings the sum of weights to at most 1:
// sums of bf16's largest values, which end at fp32's end, pass it with weights of
// up to 2^kSlack.
template <bool kBF16, int DT, bool kPaged>
__device__ __forceinline__ void exact_columns(Column<DT>& col, const AttnArgs& a, const Seq& s, int hk,
                                              const u32x4 (&q)[DT / 16], float down, int limit, int t0, int t1, int step,
                                              uint8_t* room, int lane) {
  uint8_t* vroom = room + 32 * DT * 2;
  const lds_u8 *kt = (const lds_u8*)room, *vt = (const lds_u8*)vroom;
  const LaneAt<DT> where = lane_at<DT>(lane, 0);
#pragma unroll
  for (int db = 0; db < DT / 32; ++db) col.o[db] = zero16();
#pragma unroll 1
  for (int t = t0; t < t1; t += step) {
    const int key0 = 32 * t;
    fetch_rows<DT, 32, kPaged>(a, s, hk, kv_at_clamped<kPaged>(a, s, key0 + (lane & 31)), key0, 0, room, vroom, lane);
    landed();
    f32x16 w = zero16();
#pragma unroll
    for (int d = 0; d < DT / 16; ++d) w = mma32<kBF16>(row_operand<DT>(kt, 0, d, where), q[d], w);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float x = __builtin_amdgcn_exp2f(fmaf(w[i], a.c, -col.m)) * down;
      w[i] = x < 0x1p-126f && w[i] > -INFINITY ? 0x1p-126f : x;
    }
    wave_sync();
    store_weights((lds_f32*)room, w, lane);  // (the keys are done with)
    landed();
    add_seen_rows<kBF16, DT>(col.o, (const lds_f32*)room, vt, lane, [&](int r) { return key0 + r <= limit; });
    landed();
  }
}

template <int DT>
__device__ __forceinline__ bool finite_column(const Column<DT>& col) {
  float worst = 0.0f;
#pragma unroll
  for (int db = 0; db < DT / 32; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) worst = fmaf(col.o[db][i], 0.0f, worst);  // 0, or NaN
  return worst == 0.0f;
}

// ------------------------------------------------------------ many rows ----
// A workgroup of 4 waves has 128 packed rows (query token and head of one key
// head, a token's heads next to each other, so that a tile of keys serves all
// heads of the group): 32 rows a wave, one a lane pair.  Tiles of 64 keys and
// values pass through two LDS buffers, the next one's copies in flight while
// one is used.
//
// Bound by the waits between a wave's steps: its scores, maximum, exponentials
// and weighted values of a tile follow from one another, and all waves meet at
// every tile's barrier.  The MFMAs are busy 46% of the cycles (37% with heads of
// 64), where the issue of the instructions alone would allow 79%: so busy are they
// in a loop of 8 MFMAs (32 cycles each), 40 multiply-adds and 8 exponentials (8
// cycles each), a tile's mix, that do not depend on each other, in one or two waves
// a SIMD.  Measured (us; TFLOP/s of the products that the mask leaves): 8192 tokens
// in four prompts, 32 over 8 heads of 128, 209-224 (840-900); 16 x 2048 tokens, 12
// heads of 64, 158-166 (620-650); 512 tokens over 16384 cached ones, 32 over 8
// heads, 157-170 (820-890).  Tiles of 32 keys with 3 workgroups a CU: 3% faster on
// the prompts, 8% slower with gradients, 50% over a cache.
template <int DT>
__shared__ __attribute__((aligned(1024))) uint8_t g_rows_k0[kKeys * DT * 2];
template <int DT>
__shared__ __attribute__((aligned(1024))) uint8_t g_rows_k1[kKeys * DT * 2];
template <int DT>
__shared__ __attribute__((aligned(1024))) uint8_t g_rows_v0[kKeys * DT * 2];
template <int DT>
__shared__ __attribute__((aligned(1024))) uint8_t g_rows_v1[kKeys * DT * 2];

template <bool kBF16, int DT, bool kPaged, bool kTrain>
__global__ __launch_bounds__(256, 2) void attn_rows_kernel(AttnArgs a, int slots) {
  constexpr int R = 128;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  // heads fastest: with 8 key heads each has an XCD of its own, whose cache
  // keeps the head's keys; the last tiles, with the most keys, first
  const int hk = blockIdx.x % a.Hk;
  const int rest = blockIdx.x / a.Hk;
  const int split = rest % a.splits;
  int tile;
  const int b = find_seq(a.cu_q, a.B, a.T, static_cast<int>(a.G.d), R, slots - 1 - rest / a.splits, &tile);
  const Seq s = seq_of<kPaged>(a, b);
  const int rows = s.Lq * static_cast<int>(a.G.d);
  if (tile * R >= rows) return;

  const int r = tile * R + wave * 32 + (lane & 31);
  const bool inside = r < rows;
  const int tok = div_by(inside ? r : rows - 1, a.G);
  const int head = hk * static_cast<int>(a.G.d) + ((inside ? r : rows - 1) - tok * static_cast<int>(a.G.d));
  const uint16_t* qrow = a.q.p + (s.q0 + tok) * a.q.st + head * a.q.sh;
  const int limit = last_key(a, s, tok);
  // the wave's first and the workgroup's last token bound the keys
  const int first_r = tile * R + wave * 32;
  const int full = last_key(a, s, div_by(first_r < rows ? first_r : rows - 1, a.G));  // keys all its rows see
  const int last_r = (tile + 1) * R < rows ? (tile + 1) * R - 1 : rows - 1;
  const int wave_r = first_r + 31 < rows ? first_r + 31 : rows - 1;
  const int wave_end = first_r < rows ? last_key(a, s, div_by(wave_r, a.G)) + 1 : 0;
  const int last = last_key(a, s, div_by(last_r, a.G));
  const int end = last < 0 ? 0 : last + 1;
  const int tiles = (end + kKeys - 1) / kKeys;
  const int per = (tiles + a.splits - 1) / a.splits;
  const int t0 = split * per, t1 = t0 + per < tiles ? t0 + per : tiles;

  u32x4 q[DT / 16];
  load_query<DT>(q, qrow, inside, a.D, half);

  Column<DT> col;
  col.m = kLowest;
  col.l = 0.0f;
#pragma unroll
  for (int db = 0; db < DT / 32; ++db) col.o[db] = zero16();

  const LaneAt<DT> where = lane_at<DT>(lane, 0);
  auto use = [&](int t, const lds_u8* kt, const lds_u8* vt) {
    const int key0 = t * kKeys;
    if (key0 >= wave_end) return;
    f32x16 sc[2] = {zero16(), zero16()};
#pragma unroll
    for (int d = 0; d < DT / 16; ++d)
#pragma unroll
      for (int n = 0; n < 2; ++n) sc[n] = mma32<kBF16>(row_operand<DT>(kt, 32 * n, d, where), q[d], sc[n]);
    reads_ahead<DT / 8, 8>();
    if (key0 + kKeys - 1 > full) {
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (key0 + 32 * n + acc_row(i, half) > limit) sc[n][i] = -INFINITY;
    }
    softmax_step<kBF16, DT, 2, kTrain>(col, sc, a.c, [&](int ks, int db) { return column_operand<DT>(vt, 16 * ks, db, where); });
  };

  // the rows that this wave copies of a tile, and where the next tile's are
  constexpr int W = kKeys / 4;
  KvAt at = kv_at_clamped<kPaged>(a, s, t0 * kKeys + wave * W + lane % W);
  auto fetch = [&](int t, uint8_t* kt, uint8_t* vt) {
    fetch_rows<DT, W, kPaged>(a, s, hk, at, t * kKeys, wave * W, kt, vt, lane);
    at = kv_at_clamped<kPaged>(a, s, (t + 1) * kKeys + wave * W + lane % W);
  };
  if (t0 < t1) {
    fetch(t0, g_rows_k0<DT>, g_rows_v0<DT>);
    __syncthreads();
    for (int t = t0; t < t1; t += 2) {
      if (t + 1 < t1) fetch(t + 1, g_rows_k1<DT>, g_rows_v1<DT>);
      use(t, (const lds_u8*)&g_rows_k0<DT>[0], (const lds_u8*)&g_rows_v0<DT>[0]);
      __syncthreads();
      if (t + 1 >= t1) break;
      if (t + 2 < t1) fetch(t + 2, g_rows_k0<DT>, g_rows_v0<DT>);
      use(t + 1, (const lds_u8*)&g_rows_k1<DT>[0], (const lds_u8*)&g_rows_v1<DT>[0]);
      __syncthreads();
    }
  }

  const int k0 = t0 * kKeys;
  const int k1 = t1 * kKeys < limit + 1 ? t1 * kKeys : limit + 1;
  const bool none = k1 <= k0;
  const float l = half_sum(col.l);
  const int64_t row = static_cast<int64_t>(s.q0 + tok) * a.H + head;
  const bool fine = finite_column(col);
  // (a NaN among the weights, whose sum then is one, makes all of the row one)
  const bool bad = inside && !none && l == l && half_sum(fine ? 0.0f : 1.0f) != 0.0f;
  if (inside && !bad) {
    store_column<kBF16, DT, kTrain, false>(a, col, l, row, none, split, half);
    if (half == 0) store_stats(a, col.m, l, row, none, split);
  }
  if (__builtin_expect(__ballot(bad) != 0, 0)) {
    const int e = down_bits<kBF16>(l);
    uint8_t* const room = wave == 0 ? g_rows_k0<DT> : wave == 1 ? g_rows_k1<DT> : wave == 2 ? g_rows_v0<DT> : g_rows_v1<DT>;
    const int last_tile = (wave_end + 31) / 32;
    exact_columns<kBF16, DT, kPaged>(col, a, s, hk, q, exp2f(static_cast<float>(-e)), limit, 2 * t0,
                                     2 * t1 < last_tile ? 2 * t1 : last_tile, 1, room, late_lane());
    if (bad) {
      const float le = ldexpf(l, -e);
      store_column<kBF16, DT, kTrain, true>(a, col, le, row, none, split, half);
      if (half == 0) store_stats(a, col.m + e, le, row, none, split);
    }
  }
}

// -------------------------------------------------------------- few rows ----
// A workgroup has up to 32 packed rows and its 4 waves share the keys, every
// wave tiles of 32 of its own (t0 + wave, + 4, ...) through an LDS buffer of its
// own, so that no wave waits for another before the end, where the four sums are
// joined.  For one token a sequence: bound by the cache's bytes.  Two workgroups
// run on a CU, so that of 8 waves with 16 KB each (heads of 128) most have their
// copies in flight at any time, and one's start and end hide behind the other.
// Measured (us with the join, 8 key heads of 128): one token over 8192 14.3 (2.3
// TB/s: start, end and the join), over 131072 103 (5.2 TB/s); 24 tokens over
// 77000 70 (4.5 TB/s).  With one workgroup of two buffers a wave: 16.9, 135, 99.
constexpr int kFew = 32;
template <int DT>
__shared__ __attribute__((aligned(1024))) uint8_t g_few[4][2][kFew * DT * 2];

template <bool kBF16, int DT>
__global__ __launch_bounds__(256, 2) void attn_few_kernel(AttnArgs a, int slots) {
  constexpr int R = 32;
  __shared__ float stats[2][4][R];
  __shared__ int redo[R];
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int hk = blockIdx.x % a.Hk;
  const int rest = blockIdx.x / a.Hk;
  const int split = rest % a.splits;
  int tile;
  const int G = static_cast<int>(a.G.d);
  const int b = find_seq(a.cu_q, a.B, a.T, G, R, slots - 1 - rest / a.splits, &tile);
  const Seq s = seq_of<true>(a, b);
  const int rows = s.Lq * G;
  if (tile * R >= rows) return;

  const int r = tile * R + (lane & 31);
  const bool inside = r < rows;
  const int tok = div_by(inside ? r : rows - 1, a.G);
  const int head = hk * G + ((inside ? r : rows - 1) - tok * G);
  const int limit = last_key(a, s, tok);
  const int full = last_key(a, s, div_by(tile * R, a.G));
  const int last_r = (tile + 1) * R < rows ? (tile + 1) * R - 1 : rows - 1;
  const int last = last_key(a, s, div_by(last_r, a.G));
  const int end = last < 0 ? 0 : last + 1;
  const int tiles = (end + kFew - 1) / kFew;
  int per = (tiles + a.splits - 1) / a.splits;
  per = per < 4 ? 4 : per;  // (a tile for each wave)
  const int t0 = split * per, t1 = t0 + per < tiles ? t0 + per : tiles;

  u32x4 q[DT / 16];
  load_query<DT>(q, a.q.p + (s.q0 + tok) * a.q.st + head * a.q.sh, inside, a.D, half);

  Column<DT> col;
  col.m = kLowest;
  col.l = 0.0f;
#pragma unroll
  for (int db = 0; db < DT / 32; ++db) col.o[db] = zero16();

  KvAt at = kv_at_clamped<true>(a, s, (t0 + wave) * kFew + (lane & 31));
  auto fetch = [&](int t, uint8_t* kt, uint8_t* vt) {
    fetch_rows<DT, kFew, true>(a, s, hk, at, t * kFew, 0, kt, vt, lane);
    at = kv_at_clamped<true>(a, s, (t + 4) * kFew + (lane & 31));
  };
  const LaneAt<DT> where = lane_at<DT>(lane, 0);
  auto use = [&](int t, const lds_u8* kt, const lds_u8* vt) {
    const int key0 = t * kFew;
    f32x16 sc[1] = {zero16()};
#pragma unroll
    for (int d = 0; d < DT / 16; ++d) sc[0] = mma32<kBF16>(row_operand<DT>(kt, 0, d, where), q[d], sc[0]);
    if (key0 + kFew - 1 > full) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (key0 + acc_row(i, half) > limit) sc[0][i] = -INFINITY;
    }
    softmax_step<kBF16, DT, 1, true>(col, sc, a.c, [&](int ks, int db) { return column_operand<DT>(vt, 16 * ks, db, where); });
  };
  // one wave's copies are only its own: they have to have landed before its
  // reads, and its reads of a buffer to be done before the next copies into it
  for (int t = t0 + wave; t < t1; t += 4) {
    fetch(t, &g_few<DT>[wave][0][0], &g_few<DT>[wave][1][0]);
    landed();
    use(t, (const lds_u8*)&g_few<DT>[wave][0][0], (const lds_u8*)&g_few<DT>[wave][1][0]);
    landed();
  }
  const float l1 = half_sum(col.l);
  if (half == 0) {
    stats[0][wave][lane] = col.m;
    stats[1][wave][lane] = l1;
  }
  if (threadIdx.x < R) redo[threadIdx.x] = 0;
  __syncthreads();

  // joined: the waves' sums at the largest maximum, each wave's of channel d
  // and column c at (wave * DT + d) * 32 + c of the buffers
  const int c = lane & 31;
  const float m = fmaxf(fmaxf(stats[0][0][c], stats[0][1][c]), fmaxf(stats[0][2][c], stats[0][3][c]));
  float l = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; ++w) l += stats[1][w][c] * exp2f(stats[0][w][c] - m);
  lds_f32* sums = (lds_f32*)&g_few<DT>[0][0][0];
  auto give = [&](float scale) {
#pragma unroll
    for (int db = 0; db < DT / 32; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) sums[(wave * DT + 32 * db + acc_row(i, half)) * 32 + c] = col.o[db][i] * scale;
  };
  give(exp2f(col.m - m));
  __syncthreads();

  const int k0 = t0 * kFew;
  const int k1 = t1 * kFew < limit + 1 ? t1 * kFew : limit + 1;
  const bool none = k1 <= k0;
  const int64_t row = static_cast<int64_t>(s.q0 + tok) * a.H + head;
  constexpr int N = DT / 8;  // channels of a thread
  const int d0 = (threadIdx.x >> 5) * N;
  float o[N];
  auto take = [&]() {
    bool fine = true;
#pragma unroll
    for (int x = 0; x < N; ++x) {
      o[x] = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) o[x] += sums[(w * DT + d0 + x) * 32 + c];
      fine = fine && fabsf(o[x]) < INFINITY;
    }
    return fine;
  };
  auto store = [&](float m, float l) {
    if (threadIdx.x < R) store_stats(a, m, l, row, none, split);
    if (a.splits > 1) {
      float* part = a.part + (split * (static_cast<int64_t>(a.T) * a.H) + row) * a.D;
#pragma unroll
      for (int x = 0; x < N; x += 4)
        if (d0 + x < a.D)
          *reinterpret_cast<f32x4*>(part + d0 + x) =
              none ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : f32x4{o[x], o[x + 1], o[x + 2], o[x + 3]};
    } else {
      const float rl = none ? 0.0f : 1.0f / l;
#pragma unroll
      for (int x = 0; x < N; x += 4)
        if (d0 + x < a.D)
          *reinterpret_cast<u32x2*>(a.out + row * a.D + d0 + x) =
              none ? u32x2{0, 0}
                   : u32x2{pack16<kBF16>(o[x] * rl, o[x + 1] * rl), pack16<kBF16>(o[x + 2] * rl, o[x + 3] * rl)};
    }
  };
  // (a NaN among the weights, whose sum then is one, makes all of the row one)
  if (!take() && inside && !none && l == l) redo[c] = 1;
  if (inside) store(m, l);
  __syncthreads();
  if (__builtin_expect(__ballot(redo[c] != 0) == 0, 1)) return;  // (the same in all waves)
  const int e = down_bits<kBF16>(l);
  col.m = m;
  exact_columns<kBF16, DT, true>(col, a, s, hk, q, exp2f(static_cast<float>(-e)), limit, t0 + wave, t1, 4,
                                 &g_few<DT>[wave][0][0], late_lane());
  __syncthreads();
  give(1.0f);
  __syncthreads();
  take();
  if (inside && redo[c] != 0) store(m + e, ldexpf(l, -e));
}

template <bool kBF16, int DT, bool kPaged>
int launch(const AttnArgs& a, bool few, hipStream_t st) {
  const int R = few ? 32 : 128;
  const int64_t slots = slots_of(a.cu_q, a.B, a.T, a.G.d, R);
  const int64_t grid = slots * a.Hk * a.splits;
  GPTQ_REQUIRE(grid < (int64_t{1} << 31), GPTQ_ERR_SHAPE, "attention: too many rows (%lld workgroups)",
               static_cast<long long>(grid));
  const uint32_t n = static_cast<uint32_t>(grid);
  if constexpr (kPaged) {
    if (few)
      attn_few_kernel<kBF16, DT><<<n, 256, 0, st>>>(a, static_cast<int>(slots));
    else
      attn_rows_kernel<kBF16, DT, true, false><<<n, 256, 0, st>>>(a, static_cast<int>(slots));
  } else if (a.out_rest) {
    attn_rows_kernel<kBF16, DT, false, true><<<n, 256, 0, st>>>(a, static_cast<int>(slots));
  } else {
    attn_rows_kernel<kBF16, DT, false, false><<<n, 256, 0, st>>>(a, static_cast<int>(slots));
  }
  int rc = check_launch("attention");
  if (rc != GPTQ_OK || a.splits == 1) return rc;
  return launch_join<kBF16>(a, st);
}

template <bool kPaged>
int dispatch(const AttnArgs& a, int dtype, bool few, hipStream_t st) {
  const bool wide = a.D > 64;
  if (dtype == GPTQ_BF16)
    return wide ? launch<true, 128, kPaged>(a, few, st) : launch<true, 64, kPaged>(a, few, st);
  return wide ? launch<false, 128, kPaged>(a, few, st) : launch<false, 64, kPaged>(a, few, st);
}

}  // namespace
}  // namespace gptq

using namespace gptq;

extern "C" int gptq_attention(const void* q, const void* k, const void* v, int dtype, int64_t q_token, int64_t q_head,
                              int64_t k_token, int64_t k_head, int64_t v_token, int64_t v_head, const int32_t* cu_q,
                              const int32_t* cu_k, int64_t B, int64_t T, int64_t S, int64_t H, int64_t Hk, int64_t D,
                              int causal, float scale, void* out, void* out_rest, float* lse,
                              gptq_stream_t stream) {
  clear_error();
  int rc = plan::check_attention_args("gptq_attention", dtype, B, T, S, H, Hk, D, scale);
  if (rc != GPTQ_OK) return rc;
  if (T == 0) return GPTQ_OK;
  GPTQ_REQUIRE(q && out && (S == 0 || (k && v)), GPTQ_ERR_ARG, "gptq_attention: null pointer");
  GPTQ_REQUIRE(B == 1 || (cu_q && cu_k), GPTQ_ERR_ARG, "gptq_attention: %lld sequences without their offsets",
               static_cast<long long>(B));
  const int64_t strides[] = {q_token, k_token, v_token, q_head, k_head, v_head};
  rc = plan::check_attention_layout("gptq_attention", q, k, v, strides, 3, 6);
  if (rc != GPTQ_OK) return rc;
  AttnArgs a{};
  a.q = {static_cast<const uint16_t*>(q), q_token, q_head};
  a.k = {static_cast<const uint16_t*>(k), k_token, k_head};
  a.v = {static_cast<const uint16_t*>(v), v_token, v_head};
  a.cu_q = cu_q;
  a.cu_k = cu_k;
  a.B = static_cast<int>(B), a.T = static_cast<int>(T), a.S = static_cast<int>(S);
  a.H = static_cast<int>(H), a.Hk = static_cast<int>(Hk), a.D = static_cast<int>(D);
  a.G = fast_div(static_cast<uint32_t>(H / Hk));
  a.causal = causal != 0;
  a.c = scale * kLog2e;
  a.out = static_cast<uint16_t*>(out);
  a.out_rest = static_cast<uint16_t*>(out_rest);
  a.lse = lse;
  a.splits = 1;
  return dispatch<false>(a, dtype, false, as_hip(stream));
}

extern "C" size_t gptq_paged_attention_workspace_size(int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t D,
                                                      int64_t max_context) {
  return plan::paged_workspace(B, T, H, Hk, D, max_context);
}

extern "C" int gptq_paged_attention(const void* q, const void* k_cache, const void* v_cache, int dtype, int64_t q_token,
                                    int64_t q_head, int64_t k_page, int64_t k_token, int64_t k_head, int64_t v_page,
                                    int64_t v_token, int64_t v_head, const int32_t* block_table, int64_t table_stride,
                                    int64_t width, int64_t page_size, int64_t pages, const int32_t* context,
                                    const int32_t* cu_q, int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t D,
                                    float scale, int64_t max_context, void* out, void* workspace,
                                    size_t workspace_bytes, gptq_stream_t stream) {
  clear_error();
  int rc = plan::check_attention_args("gptq_paged_attention", dtype, B, T, 0, H, Hk, D, scale);
  if (rc != GPTQ_OK) return rc;
  GPTQ_REQUIRE(page_size >= 1 && page_size < (int64_t{1} << 31) && pages >= 1 && pages < (int64_t{1} << 31) && width >= 0,
               GPTQ_ERR_ARG, "gptq_paged_attention: bad cache (%lld pages of %lld tokens, table of %lld)",
               static_cast<long long>(pages), static_cast<long long>(page_size), static_cast<long long>(width));
  if (T == 0) return GPTQ_OK;
  GPTQ_REQUIRE(q && k_cache && v_cache && out && context && (block_table || width == 0), GPTQ_ERR_ARG,
               "gptq_paged_attention: null pointer");
  GPTQ_REQUIRE(cu_q || T == B, GPTQ_ERR_SHAPE,
               "gptq_paged_attention: %lld new tokens of %lld sequences without their offsets", static_cast<long long>(T),
               static_cast<long long>(B));
  const int64_t strides[] = {q_token, k_token, v_token, q_head, k_page, k_head, v_page, v_head};
  rc = plan::check_attention_layout("gptq_paged_attention", q, k_cache, v_cache, strides, 3, 8);
  if (rc != GPTQ_OK) return rc;
  const plan::PagedPlan p = plan::paged_plan(B, T, H, Hk, max_context);
  const size_t need = plan::paged_workspace(B, T, H, Hk, D, max_context);
  GPTQ_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), GPTQ_ERR_WORKSPACE,
               "gptq_paged_attention: workspace of %zu bytes, needs %zu", workspace_bytes, need);
  AttnArgs a{};
  a.q = {static_cast<const uint16_t*>(q), q_token, q_head};
  a.k = {static_cast<const uint16_t*>(k_cache), k_token, k_head};
  a.v = {static_cast<const uint16_t*>(v_cache), v_token, v_head};
  a.paged.table = block_table;
  a.paged.context = context;
  a.paged.table_stride = table_stride;
  a.paged.k_page = k_page, a.paged.v_page = v_page;
  a.paged.most = static_cast<int>(plan::cached_most(width, page_size));
  a.paged.pages = static_cast<int>(pages);
  a.paged.page = fast_div(static_cast<uint32_t>(page_size));
  a.paged.whole = page_size % 16 == 0;
  a.cu_q = cu_q;
  a.B = static_cast<int>(B), a.T = static_cast<int>(T);
  a.H = static_cast<int>(H), a.Hk = static_cast<int>(Hk), a.D = static_cast<int>(D);
  a.G = fast_div(static_cast<uint32_t>(H / Hk));
  a.causal = 1;
  a.c = scale * kLog2e;
  a.out = static_cast<uint16_t*>(out);
  a.part = static_cast<float*>(workspace);
  a.splits = p.splits;
  return dispatch<true>(a, dtype, p.few, as_hip(stream));
}
