// Attention of new tokens over a paged cache of 8-bit codes: scores s_ij =
// (scale log2 e ks_j) (q_i kc_j), o_i = sum_j p_ij vs_j vc_j / sum_j p_ij, p_ij =
// 2^(s_ij - m_i), with kc, vc the codes and ks, vs the scales of key j's rows.
//
// The 16-bit types hold every code exactly, so both products run on their MFMA
// with the codes as they are, and the scales, one a key, go into the scores and
// into the weights.  The weights times scales are rounded to the queries' type;
// their unrounded sum divides.  Of few rows what that leaves is multiplied too (a
// decode step waits for the cache's bytes); of many rows it is not, as over a cache of
// 16-bit values: each weight is off by no more than the output's own rounding, and the
// second product takes a quarter more time (512 tokens over 16896, bf16: 193 us, error
// against 64 bits 0.0016; without it 152 us, 0.0023; the output's rounding 0.0016).
//
// Both sums are kept 2^-e as large, with e a wave's own that follows the scales: it
// is added to m, and leaves the quotient.  The sums of values of any size then stay
// inside fp32, and fp16 weights inside their 16 bits; what is lost below is small beside
// the largest scale so far.
#include "attn_join.hpp"
#include "attn_tile.hpp"
#include "codes.hpp"

namespace gptq {
namespace {

struct CodeRows {
  const uint8_t* p;
  int64_t page, token, head;        // strides, in bytes
  const float* scale;
  int64_t s_page, s_token, s_head;  // in elements
};
struct CodeArgs {
  AttnArgs a;                       // (its k and v are not used)
  CodeRows k, v;
};

// fp16 weights are kept 2^7 times larger than 2^(s - m), which is at most
// 2^kSlack (of many rows their sums of 32 are): above their smallest and below their largest value (attention.hip).
constexpr float kSlack = 8.0f;
template <bool kBF16>
constexpr float kBias = kBF16 ? 0.0f : 7.0f;
// how far a scale may pass 2^e before e is raised, and the largest e: fp32 ends at
// 2^-126, and 2^-26 of the largest weight is still above it (in fp16, whose outputs
// end at 2^16, scales of more than 2^100 need not be exact)
template <bool kBF16>
constexpr int kScaleRoom = kBF16 ? 24 : 0;
template <bool kBF16>
constexpr int kMostE = kBF16 ? 100 : 120;
constexpr int kLeastE = -80;  // (2^31 weights of 2^(kSlack + 7 + 80) are inside fp32)

// A wave's e, and the largest scale that it allows.
struct ScaleRoom {
  int e = 0;
  float cap = -1.0f;
};
__device__ __forceinline__ float uniform_float(float v) { return __int_as_float(uniform_int(__float_as_int(v))); }
// `vs`: a scale of each lane's (0 for none); those that are not finite are no
// reason for another e.
__device__ __forceinline__ bool lacks_room(const ScaleRoom& r, float vs) { return __ballot(vs > r.cap && vs < INFINITY) != 0; }
// Raises e, by how much it returns.  That is up to 200: the sums are made so much
// smaller by ldexpf, since no factor of fp32 is (2^-149 is the last), while a sum of
// weights, 2^-e and more, stays one.
template <bool kBF16>
__device__ __forceinline__ int make_room(ScaleRoom& r, float vs) {
  float top = vs > 0.0f && vs < INFINITY ? vs : 0.0f;
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor(top, s));
  if (top == 0.0f) return 0;  // (scales of 0 need no e)
  const int e = uniform_int(clamp_int(ilogbf(top) + 1, kLeastE, kMostE<kBF16>));
  const int more = e - r.e;
  r.e = e;
  r.cap = uniform_float(e == kMostE<kBF16> ? INFINITY : ldexpf(1.0f, e + kScaleRoom<kBF16>));
  return more;
}

template <int DT>
struct CodeColumn {
  float m, l;  // the running maximum and e, and this lane's part of the sum of weights
  f32x16 o[DT / 32];
};

// Makes the products s of NK x 32 keys into operands p of weights times scales;
// `ahead` is e less kBias.  `key_scale` and `value_scale` give the scales of keys 32 kt
// + 8 g + 4 (lane / 32) .. + 3, those of keys times c; `hide` sets what belongs to keys
// that the column does not see, where the tile has any.
//
// s ks - m is one instruction, with the m so far, and the sum of the weights that it
// gives is made in any case: where that is small enough for each of them, m stays.
// Otherwise, and where no key was seen before, the largest score is looked for and m
// raised to it.
template <bool kBF16, int DT, int NK, class KeyScale, class ValueScale, class Hide>
__device__ __forceinline__ void code_weights(CodeColumn<DT>& col, f32x16 (&s)[NK], u32x4 (&p)[2 * NK], float ahead,
                                             KeyScale&& key_scale, ValueScale&& value_scale, Hide&& hide) {
  const float m0 = col.m == kLowest ? 0.0f : col.m;  // (kLowest: no key seen)
#pragma unroll
  for (int kt = 0; kt < NK; ++kt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 ks = key_scale(kt, g);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[kt][4 * g + e] = fmaf(s[kt][4 * g + e], ks[e], -m0);
    }
  hide(s, -INFINITY);
  f32x16 w[NK];
  float sum;
  auto weigh = [&]() {
    sum = 0.0f;
#pragma unroll
    for (int kt = 0; kt < NK; ++kt)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        w[kt][i] = __builtin_amdgcn_exp2f(s[kt][i]);
        sum += w[kt][i];
      }
  };
  weigh();
  if (__builtin_expect(__ballot(col.m == kLowest || sum > __builtin_amdgcn_exp2f(kSlack - ahead)) != 0, 0)) {
    float t = s[0][0];
#pragma unroll
    for (int kt = 0; kt < NK; ++kt)
#pragma unroll
      for (int i = 0; i < 16; ++i) t = __builtin_elementwise_maximum(t, s[kt][i]);
    t = half_max(t) + ahead;
    const float m = col.m == kLowest ? fmaxf(kLowest, t) : col.m + fmaxf(0.0f, t);
    const float alpha = __builtin_amdgcn_exp2f(col.m - m);
    const float more = (m == kLowest ? 0.0f : m) - m0;
    col.m = m;
    col.l *= alpha;
#pragma unroll
    for (int db = 0; db < DT / 32; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) col.o[db][i] *= alpha;
#pragma unroll
    for (int kt = 0; kt < NK; ++kt)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[kt][i] -= more;
    weigh();
  }
  col.l += sum;
#pragma unroll
  for (int kt = 0; kt < NK; ++kt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 vs = value_scale(kt, g);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[kt][4 * g + e] *= vs[e];
    }
  hide(w, 0.0f);  // (a scale there may be NaN)
#pragma unroll
  for (int ks = 0; ks < 2 * NK; ++ks) p[ks] = operand_of<kBF16>(w[ks / 2], 8 * (ks % 2));
}

// 16 codes as two operands of 8 values.
template <bool kBF16, int kCode>
__device__ __forceinline__ void widen16(const u32x4& w, u32x4& lo, u32x4& hi) {
  uint32_t x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) widen4<kBF16, kCode>(w[i], x[2 * i], x[2 * i + 1]);
  lo = u32x4{x[0], x[1], x[2], x[3]};
  hi = u32x4{x[4], x[5], x[6], x[7]};
}

// A part's statistics of a row, whose sums are divided already: a weight of 1 at
// the maximum m + log2 l.  Of a sum l that is 0 (all its scores -infinity) or NaN (m may
// be too) that is the weight, at the lowest maximum: the join adds the first to other
// parts without a trace and makes NaN of a row that has no others, and it passes over a
// maximum that is no number, and takes a row without any for one that sees no key.
__device__ __forceinline__ void store_part_stats(const AttnArgs& a, float m, float l, int64_t row, bool none, int split) {
  const int64_t rows = static_cast<int64_t>(a.T) * a.H;
  float* mm = a.part + a.splits * rows * a.D;
  const bool some = l > 0.0f;
  mm[split * rows + row] = none ? -INFINITY : some ? m + log2f(l) : kLowest;
  mm[(a.splits + split) * rows + row] = none ? 0.0f : some ? 1.0f : l;
}
// What a row's sums of values are divided by, as a factor; a part whose weights are all
// 0 leaves zeros.
__device__ __forceinline__ float inverse_sum(const AttnArgs& a, float l, bool none) {
  return none || (l == 0.0f && a.splits > 1) ? 0.0f : 1.0f / l;
}

// -------------------------------------------------------------- few rows ----
// A workgroup has up to 16 NQ packed rows (query token and head of one key head)
// and its 4 waves share the keys, every wave tiles of 32 of its own (t0 + wave, +
// 4, ...), whose sums are joined at the end.  The products are 16 x 16: of a row of
// 16 keys a lane ends with keys 4 (lane / 16) + i of query lane % 16, and the
// weights of a tile's two such rows are the next product's operand as they are.
//
// A lane loads 16-byte pieces of rows lane % 16 of a tile's halves: of keys they
// are operands as they come (the contraction's order is free, the queries are
// loaded in the same one), values go through LDS to be read transposed.  The next
// tile's loads are in flight while one is used.
//
// Bound by memory where the rows are many and alike: one token over 131072 (heads 32
// over 8 of 128, e4m3, 277 MB) 51 us and 4 for the join, 5.4 TB/s; 48 sequences of
// 200 to 1939 tokens over 40 heads (int8) 99.5 us, 5.5 TB/s.  24 sequences of 1 to
// 8192 (int8, 163 MB) 43 us, 3.8 TB/s: their parts differ, and the longest end last.
// One over 8192 takes 12.8 us, of which three dependent loads (lengths, block table,
// rows), two joins and two launches are the larger part.
constexpr int kFew = 32;

// 16-byte chunk c of a row of values is at slot c ^ this in LDS: the writes of 8
// neighbouring rows' chunks (128 bytes at a time), and the transposing reads of 16
// rows by 32 lanes (256 bytes), meet each bank once.
template <int DT>
__device__ __forceinline__ int code_slot(int row) {
  if constexpr (DT == 128)
    return ((row >> 1) & 3) | (((row >> 4) ^ row) & 1) << 2;
  else
    return ((row >> 2) & 1) | (((row >> 4) ^ (row >> 1)) & 1) << 1;
}

template <bool kBF16>
__device__ __forceinline__ f32x4 mma16(const u32x4& a, const u32x4& b, const f32x4& c) {
  if constexpr (kBF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// over a column's four lanes, l % 16 alike: in all of them
__device__ __forceinline__ void both_rows(float v, float& even, float& odd) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  even = __uint_as_float(r[0]);
  odd = __uint_as_float(r[1]);
}
__device__ __forceinline__ float quarter_max(float v) {
  float a, b;
  both_rows(v, a, b);
  return half_max(__builtin_elementwise_maximum(a, b));
}
__device__ __forceinline__ float quarter_sum(float v) {
  float a, b;
  both_rows(v, a, b);
  return half_sum(a + b);
}

// what tiles past the last one read
__device__ __attribute__((aligned(16))) const uint32_t g_no_codes[4] = {};

typedef __attribute__((address_space(1))) const u32x4 gbl_u32x4;
typedef __attribute__((address_space(1))) const float gbl_f32;
typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
typedef __attribute__((address_space(3))) const f32x4 lds_cf32x4;

// the join's sums, and before it the waves' tiles of values
template <int DT, int R>
__shared__ __attribute__((aligned(1024))) uint8_t g_code_few[4 * DT * R * 4];

// kWhole: pages hold whole 16s of tokens, so that each half of a tile is in one
// page and its addresses are scalar.
template <bool kBF16, int DT, int kCode, int NQ, bool kWhole>
__global__ __launch_bounds__(256, NQ == 1 ? 3 : 2) void code_few_kernel(CodeArgs c, int slots) {
  constexpr int R = 16 * NQ, NX = DT / 64, NB = DT / 16;
  const AttnArgs& a = c.a;
  __shared__ float stats[4][R];
  __shared__ __attribute__((aligned(16))) float scales[4][64];
  const int lane = threadIdx.x & 63, row = lane & 15, quarter = lane >> 4;
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

  // this lane's columns: their queries (in LDS where the registers do not suffice)
  // and the last key that they see
  constexpr bool kHeld = NQ == 1 || DT == 64;
  __shared__ __attribute__((aligned(16))) u32x4 queries[kHeld ? 1 : NQ * 2 * NX][64];
  int limit[NQ];
  u32x4 q[NQ][2 * NX];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int r = tile * R + 16 * n + row;
    const bool inside = r < rows;
    const int tok = div_by(inside ? r : rows - 1, a.G);
    const int head = hk * G + ((inside ? r : rows - 1) - tok * G);
    limit[n] = last_key(a, s, tok);
    const uint16_t* qrow = a.q.p + (s.q0 + tok) * a.q.st + head * a.q.sh;
#pragma unroll
    for (int x = 0; x < 2 * NX; ++x) {
      const int d = 64 * (x / 2) + 16 * quarter + 8 * (x % 2);
      q[n][x] = inside && d < a.D ? *reinterpret_cast<const u32x4*>(qrow + d) : u32x4{0, 0, 0, 0};
    }
  }
  auto query = [&](int n, int x) {
    if constexpr (kHeld) return q[n][x];
    return queries[2 * NX * n + x][lane];
  };
  const int full = last_key(a, s, div_by(tile * R, a.G));  // keys that all rows see
  const int last_r = (tile + 1) * R < rows ? (tile + 1) * R - 1 : rows - 1;
  const int last = last_key(a, s, div_by(last_r, a.G));
  const int end = last < 0 ? 0 : last + 1;
  const int tiles = (end + kFew - 1) / kFew;
  int per = (tiles + a.splits - 1) / a.splits;
  per = per < 4 ? 4 : per;  // (a tile for each wave)
  const int t0 = split * per, t1 = t0 + per < tiles ? t0 + per : tiles;

  float m[NQ], l[NQ];
  f32x4 o[NQ][NB];
  ScaleRoom room;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    m[n] = kLowest, l[n] = 0.0f;
#pragma unroll
    for (int x = 0; x < NB; ++x) o[n][x] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  lds_u8* const vt = (lds_u8*)&g_code_few<DT, R>[wave * (kFew * DT)];
  lds_f32* const sc_lds = (lds_f32*)&scales[wave][0];
  // where a lane's chunks are in a row (one past the head: its first chunk, which
  // meets zeros of the queries and channels that are not stored), and where they
  // go; of a row 16 further the slot's high bit is turned
  uint32_t chunk[NX];
  int put[NX];
#pragma unroll
  for (int x = 0; x < NX; ++x) {
    chunk[x] = 64 * x + 16 * quarter;
    if (chunk[x] >= static_cast<uint32_t>(a.D)) chunk[x] = 0;
    put[x] = row * DT + (((4 * x + quarter) ^ code_slot<DT>(row)) << 4);
  }
  constexpr int kTurn = DT == 128 ? 64 : 32;
  // A transposing read takes from 16 lanes the addresses of 8 rows x 16 codes, 8
  // codes a lane, and gives lane i the 8 rows' code i: the rows 16 (i / 8) + 4
  // quarter + (i / 2) % 4 here, chunk 0; chunk c is at the address ^ 16 c.
  const int from = 16 * (row >> 3) + 4 * quarter + ((row >> 1) & 3);
  const int get = from * DT + (code_slot<DT>(from) << 4) + ((row & 1) << 3);

  // kWhole: a lane of quarter i has of half i % 2 of a tile the keys (i < 2) or the
  // values, and makes the address of their codes, for all lanes, and of its row's
  // scale.  What it needs, base and strides of pages and tokens, is in LDS where the
  // registers do not suffice.
  constexpr bool kBasesHeld = NQ > 1;
  __shared__ __attribute__((aligned(16))) u32x4 bases[kWhole && !kBasesHeld ? 512 : 1];
  u32x4 base0, base1;
  if constexpr (kWhole) {
    const CodeRows& from = quarter >= 2 ? c.v : c.k;
    const uint64_t codes = reinterpret_cast<uint64_t>(from.p) + hk * from.head;
    const uint64_t first = reinterpret_cast<uint64_t>(from.scale) + 4 * (hk * from.s_head + row * from.s_token);
    base0 = u32x4{static_cast<uint32_t>(codes), static_cast<uint32_t>(codes >> 32), static_cast<uint32_t>(from.page),
                  static_cast<uint32_t>(from.token)};
    base1 = u32x4{static_cast<uint32_t>(first), static_cast<uint32_t>(first >> 32), static_cast<uint32_t>(4 * from.s_page),
                  static_cast<uint32_t>(4 * from.s_token)};
    if constexpr (!kBasesHeld) bases[threadIdx.x] = base0, bases[256 + threadIdx.x] = base1;
  }
  auto base_of = [&](int i) {
    if constexpr (kBasesHeld) return i ? base1 : base0;
    return bases[256 * i + threadIdx.x];
  };

  // The block table's entries of a tile: of the lane's half, or of its two rows.  They
  // are loaded a tile before the rows are, and before the rows of the tile between:
  // loads return in order, so that a wait for an entry does not wait for rows.
  constexpr int NP = kWhole ? 1 : 2;
  struct Pages {
    int p[NP];
  };
  auto key_of = [&](int t, int n) {  // a half's first key, or the lane's: one of the sequence in any case
    if constexpr (kWhole) return clamp_int(t * kFew + 16 * (quarter & 1), 0, (s.Lk - 1) & ~15);
    return clamp_int(t * kFew + 16 * n + row, 0, s.Lk - 1);
  };
  auto pages_of = [&](int t) {
    Pages r;
#pragma unroll
    for (int n = 0; n < NP; ++n) r.p[n] = a.paged.table[s.b * a.paged.table_stride + div_by(key_of(t, n), a.paged.page)];
    return r;
  };
  // A tile's rows.  Every lane loads in any case, of tiles past the last one the
  // same few bytes: with loads under a branch the compiler waits for all of them
  // where it could wait for the older ones.
  auto load = [&](u32x4 (&k)[2][NX], u32x4 (&v)[2][NX], float& scale, int t, const Pages& pages) {
    const bool some = t < t1;
    const uint32_t keep = some ? ~0u : 0u;
    const uint64_t none = reinterpret_cast<uint64_t>(&g_no_codes[0]);
    uint64_t kp[2], vp[2], sp;
    uint32_t krow = 0, vrow = 0;
    if constexpr (kWhole) {
      const int key = key_of(t, 0);
      const uint32_t at = key - div_by(key, a.paged.page) * static_cast<int>(a.paged.page.d);
      const uint32_t page = clamp_int(pages.p[0], 0, a.paged.pages - 1);
      auto address = [&](int i) {
        const u32x4 x = base_of(i);
        const uint64_t to = (static_cast<uint64_t>(x[1]) << 32 | x[0]) + static_cast<uint64_t>(page) * x[2] +
                            static_cast<uint64_t>(at) * x[3];
        return some ? to : none;
      };
      const uint64_t codes = address(0);
      sp = address(1);
      auto from = [&](int i) {
        const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(codes), 16 * i);
        const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(codes >> 32), 16 * i);
        return static_cast<uint64_t>(hi) << 32 | lo;
      };
#pragma unroll
      for (int n = 0; n < 2; ++n) kp[n] = from(n), vp[n] = from(2 + n);
      krow = row * static_cast<uint32_t>(c.k.token), vrow = row * static_cast<uint32_t>(c.v.token);
    } else {
      int page[2], at[2];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int key = key_of(t, n);
        at[n] = key - div_by(key, a.paged.page) * static_cast<int>(a.paged.page.d);
        page[n] = clamp_int(pages.p[n], 0, a.paged.pages - 1);
        kp[n] = reinterpret_cast<uint64_t>(c.k.p) + page[n] * c.k.page + at[n] * c.k.token + hk * c.k.head;
        vp[n] = reinterpret_cast<uint64_t>(c.v.p) + page[n] * c.v.page + at[n] * c.v.token + hk * c.v.head;
        kp[n] = some ? kp[n] : none;
        vp[n] = some ? vp[n] : none;
      }
      // quarters 0 and 1: the keys' scales of the two halves, 2 and 3: the values'
      const int pg = quarter & 1 ? page[1] : page[0], to = quarter & 1 ? at[1] : at[0];
      const bool values = quarter >= 2;
      const int64_t i = pg * (values ? c.v.s_page : c.k.s_page) + to * (values ? c.v.s_token : c.k.s_token) +
                        hk * (values ? c.v.s_head : c.k.s_head);
      sp = some ? reinterpret_cast<uint64_t>(values ? c.v.scale : c.k.scale) + 4 * i : none;
    }
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int x = 0; x < NX; ++x) k[n][x] = *(gbl_u32x4*)(kp[n] + ((krow + chunk[x]) & keep));
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int x = 0; x < NX; ++x) v[n][x] = *(gbl_u32x4*)(vp[n] + ((vrow + chunk[x]) & keep));
    scale = *(gbl_f32*)sp;
  };
  // Uses a tile's rows, and has the next one's loaded into their registers as soon
  // as these are free: the loads are in flight for the larger part of a tile's time.
  u32x4 k[2][NX], v[2][NX];
  float scale;
  auto use = [&](int t, const Pages& next) {
    const int key0 = t * kFew;
    if (key0 + kFew > s.Lk) {  // rows past the end hold anything
#pragma unroll
      for (int n = 0; n < 2; ++n)
        if (key0 + 16 * n + row >= s.Lk)
#pragma unroll
          for (int x = 0; x < NX; ++x) v[n][x] = u32x4{0, 0, 0, 0};
      if (key0 + 16 * (quarter & 1) + row >= s.Lk) scale = 0.0f;
    }
#pragma unroll
    for (int x = 0; x < NX; ++x) {
      *(lds_u32x4*)(vt + put[x]) = v[0][x];
      *(lds_u32x4*)(vt + (put[x] ^ kTurn) + 16 * DT) = v[1][x];
    }
    sc_lds[lane] = quarter >= 2 ? scale : scale * a.c;
    const float vs = quarter >= 2 ? scale : 0.0f;
    if (__builtin_expect(lacks_room(room, vs), 0)) {
      const int more = make_room<kBF16>(room, vs);
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        m[n] += static_cast<float>(more);
        l[n] = __builtin_amdgcn_ldexpf(l[n], -more);
#pragma unroll
        for (int x = 0; x < NB; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][x][e] = __builtin_amdgcn_ldexpf(o[n][x][e], -more);
      }
    }

    f32x4 sc[NQ][2];
#pragma unroll
    for (int n = 0; n < NQ; ++n) sc[n][0] = sc[n][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int x = 0; x < NX; ++x)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        u32x4 lo, hi;
        widen16<kBF16, kCode>(k[y][x], lo, hi);
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          sc[n][y] = mma16<kBF16>(lo, query(n, 2 * x), sc[n][y]);
          sc[n][y] = mma16<kBF16>(hi, query(n, 2 * x + 1), sc[n][y]);
        }
      }
    __builtin_amdgcn_sched_barrier(0);
    load(k, v, scale, t + 4, next);
    __builtin_amdgcn_sched_barrier(0);
    wave_sync();
    f32x4 ks[2], vs4[2];
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      ks[y] = *(lds_cf32x4*)(sc_lds + 16 * y + 4 * quarter);
      vs4[y] = *(lds_cf32x4*)(sc_lds + 32 + 16 * y + 4 * quarter);
    }
    const bool cut = key0 + kFew - 1 > full;
    u32x4 p[NQ], pr[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float top = -INFINITY;
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[n][y][e] *= ks[y][e];
      auto mask = [&](float (&x)[2][4], float with) {
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (key0 + 16 * y + 4 * quarter + e > limit[n]) x[y][e] = with;
      };
      float w[2][4], left[2][4];
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int e = 0; e < 4; ++e) w[y][e] = sc[n][y][e];
      if (cut) mask(w, -INFINITY);
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = __builtin_elementwise_maximum(top, w[y][e]);
      top = quarter_max(top) + (static_cast<float>(room.e) - kBias<kBF16>);
      if (__builtin_expect(__ballot(top > m[n] + kSlack) != 0, 0)) {
        const float now = fmaxf(m[n], top);
        const float alpha = __builtin_amdgcn_exp2f(m[n] - now);
        m[n] = now;
        l[n] *= alpha;
#pragma unroll
        for (int x = 0; x < NB; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][x][e] *= alpha;
      }
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = __builtin_amdgcn_exp2f(w[y][e] - m[n]);
          l[n] += x;
          w[y][e] = x * vs4[y][e];
        }
      if (cut) mask(w, 0.0f);  // (a scale there may be NaN)
      p[n] = u32x4{pack16<kBF16>(w[0][0], w[0][1]), pack16<kBF16>(w[0][2], w[0][3]), pack16<kBF16>(w[1][0], w[1][1]),
                   pack16<kBF16>(w[1][2], w[1][3])};
      // what the rounding of the weights left is multiplied too: the cache's bytes
      // take longer than both products
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          left[y][e] = w[y][e] - value16<kBF16>(static_cast<uint16_t>(p[n][2 * y + e / 2] >> (16 * (e % 2))));
      pr[n] = u32x4{pack16<kBF16>(left[0][0], left[0][1]), pack16<kBF16>(left[0][2], left[0][3]),
                    pack16<kBF16>(left[1][0], left[1][1]), pack16<kBF16>(left[1][2], left[1][3])};
    }
#pragma unroll
    for (int x = 0; x < NB; ++x) {
      typedef int i32x2 __attribute__((ext_vector_type(2)));
      typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
      const i32x2 z = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)(vt + (get ^ (x << 4))));
      uint32_t y[4];
      widen4<kBF16, kCode>(static_cast<uint32_t>(z[0]), y[0], y[1]);
      widen4<kBF16, kCode>(static_cast<uint32_t>(z[1]), y[2], y[3]);
      const u32x4 value = {y[0], y[1], y[2], y[3]};
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        o[n][x] = mma16<kBF16>(value, p[n], o[n][x]);
        o[n][x] = mma16<kBF16>(value, pr[n], o[n][x]);
      }
    }
    wait_lgkm<0>();  // (this tile's reads, before the next one's writes)
    wave_sync();
  };
  const int first = t0 + wave;
  Pages p0, p1;
  if (first < t1) {
    p0 = pages_of(first), p1 = pages_of(first + 4);
    load(k, v, scale, first, p0);
  }
  if constexpr (!kHeld) {  // (while the first rows are on their way)
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int x = 0; x < 2 * NX; ++x)
        if (wave == x % 4) queries[2 * NX * n + x][lane] = q[n][x];  // (the waves' are the same)
    __syncthreads();
  }
  for (int t = first; t < t1; t += 4) {
    p0 = p1;
    p1 = pages_of(t + 8);
    use(t, p0);
  }
  // a column's sums of this wave as a weighted mean, and the log2 of its weights
  float lse[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    l[n] = quarter_sum(l[n]);
    lse[n] = l[n] == 0.0f ? -INFINITY : m[n] + log2f(l[n]);
    if (quarter == 0) stats[wave][16 * n + row] = lse[n];
  }
  __syncthreads();

  // The waves' means are joined.  Wave w's channels 4 d .. 4 d + 3 of column x are at
  // chunk d ^ (x % (DT / 4)) of row (w, x): neither side's accesses meet in a bank.
  lds_u8* const sums = (lds_u8*)&g_code_few<DT, R>[0];
  auto sum_at = [&](int w, int x, int d) { return ((w * R + x) * (DT / 4) + (d ^ (x & (DT / 4 - 1)))) * 16; };
  auto top_of = [&](int x) {
    float top = stats[0][x];
#pragma unroll
    for (int w = 1; w < 4; ++w) top = __builtin_elementwise_maximum(top, stats[w][x]);
    return top == -INFINITY ? 0.0f : top;  // (no wave has a key)
  };
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int x = 16 * n + row;
    if (tile * R + x >= rows) continue;
    const float f = l[n] == 0.0f ? 0.0f : exp2f(lse[n] - top_of(x)) / l[n];
#pragma unroll
    for (int d = 0; d < NB; ++d)
      *(lds_f32x4*)(sums + sum_at(wave, x, 4 * d + quarter)) =
          f32x4{o[n][d][0] * f, o[n][d][1] * f, o[n][d][2] * f, o[n][d][3] * f};
  }
  __syncthreads();

  const int x = threadIdx.x % R;
  const int r = tile * R + x;
  if (r >= rows) return;
  const int tok = div_by(r, a.G);
  const float top = top_of(x);
  float sum = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; ++w) sum += exp2f(stats[w][x] - top);
  const int seen = last_key(a, s, tok) + 1;
  const int k0 = t0 * kFew;
  const int k1 = t1 * kFew < seen ? t1 * kFew : seen;
  const bool none = k1 <= k0;
  const int64_t out_row = static_cast<int64_t>(s.q0 + tok) * a.H + hk * G + (r - tok * G);
  constexpr int N = DT * R / 256;  // channels of a thread
  const int d0 = (threadIdx.x / R) * N;
  if (threadIdx.x < R && a.splits > 1) store_part_stats(a, top, sum, out_row, none, split);
  const float inv = inverse_sum(a, sum, none);
#pragma unroll
  for (int d = 0; d < N; d += 4) {
    if (d0 + d >= a.D) break;
    f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < 4; ++w) y += *(lds_cf32x4*)(sums + sum_at(w, x, (d0 + d) / 4));
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = none ? 0.0f : y[e] * inv;
    if (a.splits > 1)
      *reinterpret_cast<f32x4*>(a.part + (split * (static_cast<int64_t>(a.T) * a.H) + out_row) * a.D + d0 + d) = y;
    else
      *reinterpret_cast<u32x2*>(a.out + out_row * a.D + d0 + d) = u32x2{pack16<kBF16>(y[0], y[1]), pack16<kBF16>(y[2], y[3])};
  }
}

// ------------------------------------------------------------- many rows ----
// A workgroup of NW waves has 32 NW packed rows, 32 a wave.  Tiles of 64 keys are
// loaded as codes by all threads, widened once and left in LDS as 16-bit values, in
// one of two buffers while the other one is used.
//
// A tile's 16-byte chunk c (8 channels) of row r is at c kChunk + 16 r: one address
// and constants reach all operands of a lane.  kChunk is 64 bytes past a multiple of
// all banks' 256, so that the transposing reads of 4 rows x 4 chunks by 32 lanes,
// the reads of 16 rows, and the writes of 4 rows x 2 chunks by 8 lanes (128 bytes)
// meet each bank once.
//
// Bound by issue: of a tile of 32 queries and 64 keys the products hold the matrix
// unit for 1024 cycles and, for about half of these, the vector unit's port; the
// weights take it for 1200 (32 exponentials a lane are 512 of them).  Measured, 512
// new tokens over 16896, heads 32 over 8 of 128, bf16 over e4m3 (140 GFLOP): 144 us
// and 8 us for the join, 915 TFLOP/s; with the join 177 us with 128 rows and all waves
// in step, 161 us with 256 rows in step, 154.6 us with the largest score looked for in
// every tile.  Cycles of a tile: 1880 for its weights, 1720 for its products and
// staging, 420 at both barriers.
constexpr int kKeys = 64;
constexpr int kChunk = kKeys * 16 + 64;
template <int DT>
__shared__ __attribute__((aligned(1024))) uint8_t g_code_tiles[2][2][DT / 8 * kChunk];  // buffer; keys, values

template <bool kBF16, int DT, int kCode, int NW, bool kWhole>
__global__ __launch_bounds__(64 * NW, 2) void code_rows_kernel(CodeArgs c, int slots) {
  constexpr int R = 32 * NW;
  constexpr int CH = DT / 16, RPI = 64 * NW / CH, NX = kKeys / RPI;  // chunks of a row of codes, rows at a time
  const AttnArgs& a = c.a;
  __shared__ __attribute__((aligned(16))) float scales[4][2 * kKeys + 32];  // of tile t at t % 4: keys', times c; then values'
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int hk = blockIdx.x % a.Hk;
  const int rest = blockIdx.x / a.Hk;
  const int split = rest % a.splits;
  int tile;
  const int b = find_seq(a.cu_q, a.B, a.T, static_cast<int>(a.G.d), R, slots - 1 - rest / a.splits, &tile);
  const Seq s = seq_of<true>(a, b);
  const int rows = s.Lq * static_cast<int>(a.G.d);
  if (tile * R >= rows) return;

  u32x4 q[DT / 16];
  int limit;
  {
    const int r = tile * R + wave * 32 + (lane & 31);
    const bool inside = r < rows;
    const int tok = div_by(inside ? r : rows - 1, a.G);
    const int head = hk * static_cast<int>(a.G.d) + ((inside ? r : rows - 1) - tok * static_cast<int>(a.G.d));
    load_query<DT>(q, a.q.p + (s.q0 + tok) * a.q.st + head * a.q.sh, inside, a.D, half);
    limit = last_key(a, s, tok);
  }
  const int first_r = tile * R + wave * 32;
  const int full = last_key(a, s, div_by(first_r < rows ? first_r : rows - 1, a.G));  // keys all its rows see
  const int last_r = (tile + 1) * R < rows ? (tile + 1) * R - 1 : rows - 1;
  const int last = last_key(a, s, div_by(last_r, a.G));
  const int end = last < 0 ? 0 : last + 1;
  const int tiles = (end + kKeys - 1) / kKeys;
  const int per = (tiles + a.splits - 1) / a.splits;
  const int t0 = split * per, t1 = t0 + per < tiles ? t0 + per : tiles;

  CodeColumn<DT> col;
  ScaleRoom room;
  col.m = kLowest;
  col.l = 0.0f;
#pragma unroll
  for (int db = 0; db < DT / 32; ++db) col.o[db] = zero16();

  // This thread's chunk of rows row0 + RPI x of a tile.  Chunks past the head are its
  // first one, which meets zeros of the queries and channels that are not stored.
  // 8 neighbouring lanes have 2 chunks of 4 rows.
  const int ch = (lane & 1) | ((lane >> 3) & (CH / 2 - 1)) << 1;
  const int own_row = ((lane >> 1) & 3) | (lane >> (CH == 8 ? 5 : 4)) << 2;
  const int wave_row = wave * (64 / CH);
  const int row0 = wave_row + own_row;
  const uint32_t chunk = 16 * ch < a.D ? 16 * ch : 0;
  u32x4 nk[NX], nv[NX];
  float nks[NX], nvs[NX];  // (kWhole: the lane's one scale in nks[0])

  // kWhole: the W rows of a wave for each x are in one page.  Lane i < 2 NX makes the
  // address of the first one's codes, for x = i % NX, of keys or values by i / NX, for
  // all lanes; lanes from 32 on those of their scale, of row lane % W for x = lane / W
  // % NX.  (As scalar arithmetic, twenty times as many instructions, it took a fifth
  // of the time.)
  constexpr int W = 64 / CH;
  const int x_of = half ? lane / W % NX : lane % NX;
  const int values_of = (half ? (lane - 32) / (W * NX) : lane / NX) % 2;
  // in the tile, or for codes of values in the tile before it
  const int my_key = RPI * x_of + wave_row + (half ? lane % W : values_of ? -kKeys : 0);
  __shared__ __attribute__((aligned(16))) u32x4 bases[kWhole ? 64 * NW : 1];  // address; strides of pages and tokens
  if constexpr (kWhole) {
    const CodeRows& from = values_of ? c.v : c.k;
    const uint64_t base = half ? reinterpret_cast<uint64_t>(from.scale) + 4 * (hk * from.s_head + lane % W * from.s_token)
                               : reinterpret_cast<uint64_t>(from.p) + hk * from.head;
    bases[threadIdx.x] = u32x4{static_cast<uint32_t>(base), static_cast<uint32_t>(base >> 32),
                               static_cast<uint32_t>(half ? 4 * from.s_page : from.page),
                               static_cast<uint32_t>(half ? 4 * from.s_token : from.token)};
  }
  const uint32_t k_off = own_row * static_cast<uint32_t>(c.k.token) + chunk;
  const uint32_t v_off = own_row * static_cast<uint32_t>(c.v.token) + chunk;
  constexpr int NP = kWhole ? 1 : 2 * NX;
  auto key_of = [&](int t, int x) {  // one of the sequence in any case
    if constexpr (kWhole) return clamp_int(t * kKeys + (my_key & ~(W - 1)), 0, (s.Lk - 1) & ~(W - 1));
    return clamp_int((t - x / NX) * kKeys + RPI * (x % NX) + row0, 0, s.Lk - 1);
  };
  struct Pages {
    int p[NP];
  };
  auto pages_of = [&](int t) {
    Pages r;
#pragma unroll
    for (int x = 0; x < NP; ++x) r.p[x] = a.paged.table[s.b * a.paged.table_stride + div_by(key_of(t, x), a.paged.page)];
    return r;
  };
  auto address_of = [&](int t, const Pages& pages) {  // kWhole: the lane's
    if constexpr (!kWhole) return uint64_t{0};
    const int key = key_of(t, 0);
    const uint32_t at = key - div_by(key, a.paged.page) * static_cast<int>(a.paged.page.d);
    const uint32_t page = clamp_int(pages.p[0], 0, a.paged.pages - 1);
    const u32x4 base = bases[threadIdx.x];
    return (static_cast<uint64_t>(base[1]) << 32 | base[0]) + static_cast<uint64_t>(page) * base[2] +
           static_cast<uint64_t>(at) * base[3];
  };
  // the keys of tile t and the values of tile t - 1, and the scales of tile t
  auto load = [&](int t, const Pages& pages, uint64_t mine) {
    if constexpr (kWhole) {
      auto from = [&](int i) {
        const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(mine), i);
        const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(mine >> 32), i);
        return static_cast<uint64_t>(hi) << 32 | lo;
      };
#pragma unroll
      for (int x = 0; x < NX; ++x) {
        nk[x] = *(gbl_u32x4*)(from(x) + k_off);
        nv[x] = *(gbl_u32x4*)(from(NX + x) + v_off);
      }
      nks[0] = *(gbl_f32*)(mine);  // (of lanes below 32 the first of the codes)
    } else {
#pragma unroll
      for (int x = 0; x < NX; ++x) {
        auto place = [&](int i, int64_t& page, int64_t& at) {
          const int key = key_of(t, i);
          at = key - div_by(key, a.paged.page) * static_cast<int>(a.paged.page.d);
          page = clamp_int(pages.p[i], 0, a.paged.pages - 1);
        };
        int64_t page, at, v_page, v_at;
        place(x, page, at);
        place(NX + x, v_page, v_at);
        nk[x] = *reinterpret_cast<const u32x4*>(c.k.p + page * c.k.page + at * c.k.token + hk * c.k.head + chunk);
        nv[x] = *reinterpret_cast<const u32x4*>(c.v.p + v_page * c.v.page + v_at * c.v.token + hk * c.v.head + chunk);
        nks[x] = c.k.scale[page * c.k.s_page + at * c.k.s_token + hk * c.k.s_head];  // (the same for a row's threads)
        nvs[x] = c.v.scale[page * c.v.s_page + at * c.v.s_token + hk * c.v.s_head];
      }
    }
  };
  // (the order of a thread's two chunks takes turns: two lanes' first ones would meet)
  const bool turn = ch & 1;
  const int put0 = (2 * ch + (turn ? 1 : 0)) * kChunk + 16 * row0;
  const int put1 = (2 * ch + (turn ? 0 : 1)) * kChunk + 16 * row0;
  auto put = [&](lds_u8* to, const u32x4& w, int x) {
    u32x4 lo, hi;
    widen16<kBF16, kCode>(turn ? u32x4{w[2], w[3], w[0], w[1]} : w, lo, hi);
    *(lds_u32x4*)(to + put0 + 16 * RPI * x) = lo;
    *(lds_u32x4*)(to + put1 + 16 * RPI * x) = hi;
  };
  // (of lanes without a scale to a place that nothing reads)
  const int scale_at = kWhole && !half ? 2 * kKeys + lane : kKeys * values_of + my_key;
  const float scale_by = values_of ? 1.0f : a.c;
  auto put_scales = [&](int t) {  // those past the end are zeros
    if constexpr (kWhole) {
      scales[t & 3][scale_at] = t * kKeys + my_key < s.Lk ? nks[0] * scale_by : 0.0f;
    } else {
#pragma unroll
      for (int x = 0; x < NX; ++x) {
        const bool some = t * kKeys + RPI * x + row0 < s.Lk;
        scales[t & 3][row0 + RPI * x] = some ? nks[x] * a.c : 0.0f;
        scales[t & 3][kKeys + row0 + RPI * x] = some ? nvs[x] : 0.0f;
      }
    }
  };
  auto clear_values = [&](int t) {  // rows past the end hold anything
    if (__builtin_expect((t + 1) * kKeys > s.Lk, 0)) {
#pragma unroll
      for (int x = 0; x < NX; ++x)
        if (t * kKeys + RPI * x + row0 >= s.Lk) nv[x] = u32x4{0, 0, 0, 0};
    }
  };
  auto put_rows = [&](int t) {  // the keys of tile t, the values of tile t - 1
#pragma unroll
    for (int x = 0; x < NX; ++x) {
      put((lds_u8*)&g_code_tiles<DT>[t & 1][0][0], nk[x], x);
      put((lds_u8*)&g_code_tiles<DT>[(t & 1) ^ 1][1][0], nv[x], x);
    }
  };

  // where a lane reads: row lane % 32, channels 8 (lane / 32) .. of a product over
  // channels; for one over rows, by 16 lanes, 4 rows x 16 channels (attn_tile.hpp)
  int krow = half * kChunk + 16 * (lane & 31);
  int vrow = (2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) * kChunk + 16 * (4 * half + ((lane & 15) >> 2)) + 8 * (lane & 1);
  asm volatile("" : "+v"(krow), "+v"(vrow));  // (so that the constant parts go into the instructions)
  f32x16 sc[2];
  u32x4 p[4];
  auto keys_times_queries = [&](int t) {
    const lds_u8* const kt = (const lds_u8*)&g_code_tiles<DT>[t & 1][0][0] + krow;
    sc[0] = sc[1] = zero16();
#pragma unroll
    for (int d = 0; d < DT / 16; ++d)
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const u32x4 k = *(const lds_u32x4*)(kt + 2 * d * kChunk + 512 * n);
        sc[n] = mma32<kBF16>(k, q[d], sc[n]);
      }
  };
  f32x4 ks[8];  // the scales of a tile's keys, and of values one a lane
  float vs;
  auto read_scales = [&](int t) {
    const lds_f32* const sl = (const lds_f32*)&scales[t & 3][0];
    vs = sl[kKeys + lane];
#pragma unroll
    for (int i = 0; i < 8; ++i) ks[i] = *(lds_cf32x4*)(sl + 8 * i + 4 * half);
  };
  auto weights = [&](int t) {
    const int key0 = t * kKeys;
    const lds_f32* const sl = (const lds_f32*)&scales[t & 3][0];
    if (__builtin_expect(lacks_room(room, vs), 0)) {
      const int more = make_room<kBF16>(room, vs);
      col.m += static_cast<float>(more);
      col.l = __builtin_amdgcn_ldexpf(col.l, -more);
#pragma unroll
      for (int db = 0; db < DT / 32; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) col.o[db][i] = __builtin_amdgcn_ldexpf(col.o[db][i], -more);
    }
    const bool cut = key0 + kKeys - 1 > full;
    auto hide = [&](f32x16 (&x)[2], float with) {
      if (!cut) return;
      int last_seen = limit - key0 - 4 * half;
      asm volatile("" : "+v"(last_seen));  // (so that the comparisons stay behind the branch)
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (32 * n + acc_row(i, 0) > last_seen) x[n][i] = with;
    };
    code_weights<kBF16, DT, 2>(
        col, sc, p, static_cast<float>(room.e) - kBias<kBF16>,
        [&](int n, int g) { return ks[4 * n + g]; },
        [&](int n, int g) { return *(lds_cf32x4*)(sl + kKeys + 32 * n + 8 * g + 4 * half); }, hide);
  };
  auto weights_times_values = [&](int t) {
    const lds_u8* const vt = (const lds_u8*)&g_code_tiles<DT>[t & 1][1][0] + vrow;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
      for (int db = 0; db < DT / 32; ++db) {
        s16x4 v[2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
          v[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vt + 4 * db * kChunk + 256 * ks + 128 * j));
        const u32x4 value = __builtin_bit_cast(u32x4, __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7));
        col.o[db] = mma32<kBF16>(value, p[ks], col.o[db]);
      }
  };

  // Phases between barriers: a wave makes a tile's weights (vector instructions), then
  // multiplies them with the values and the next keys with the queries (matrix
  // instructions) and stages its part of later tiles meanwhile.  Of 8 waves the second
  // four, each of which shares a SIMD with one of the first, are a phase behind: one of
  // both has the matrix unit while the other one has the vector unit.
  //
  // Keys of tile t are read in phases 2 t and 2 t + 1 and written in 2 t - 2 and 2 t -
  // 1, values read in 2 t + 2 and 2 t + 3 and written in 2 t and 2 t + 1 (by the first
  // four, then by the others), each over what was read last a phase before.  Scales of
  // tile t, written like its keys, are read until 2 t + 2.
  //
  // A tile's entries of the block table are loaded before the rows of the tile before
  // it: loads return in order.
  if (t0 < t1) {
    const bool late = NW == 8 && wave >= 4;
    Pages p0 = pages_of(t0), p1 = pages_of(t0 + 1);
    auto stage = [&](int t) {  // tile t's keys, tile t - 1's values, and the loads of the next ones
      clear_values(t - 1);
      put_scales(t);
      put_rows(t);
      p0 = p1;
      p1 = pages_of(t + 2);
      load(t + 1, p0, address_of(t + 1, p0));
    };
    load(t0, p0, address_of(t0, p0));
    stage(t0);
    stage(t0 + 1);
    __syncthreads();
    if (late) __syncthreads();
    keys_times_queries(t0);
    read_scales(t0);
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
      weights(t);
      p0 = p1;
      p1 = pages_of(t + 4);
      uint64_t next = address_of(t + 3, p0);
      asm volatile("" : "+v"(p[0]), "+v"(p[1]), "+v"(p[2]), "+v"(p[3]), "+v"(col.l), "+v"(next));  // (all in this phase)
      __syncthreads();
      clear_values(t + 1);
      put_scales(t + 2);
      __builtin_amdgcn_s_setprio(1);
      // reads ahead of the products, so that none waits for one just issued; the writes,
      // which pass no read, between both products
      constexpr int kAhead = 12;
      weights_times_values(t);
      __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
      sfor<0, DT / 8 - kAhead / 2>([](auto) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      });
      __builtin_amdgcn_sched_group_barrier(0x008, kAhead / 2, 0);
      __builtin_amdgcn_sched_barrier(0);
      put_rows(t + 2);
      load(t + 3, p0, next);
      __builtin_amdgcn_sched_barrier(0);
      keys_times_queries(t + 1);
      read_scales(t + 1);
      __builtin_amdgcn_sched_group_barrier(0x100, kAhead / 2, 0);
      sfor<0, DT / 8 - kAhead / 2>([](auto) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      });
      sfor<0, kAhead / 2>([](auto) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      });
      __builtin_amdgcn_s_setprio(0);
      __syncthreads();
    }
    if (NW == 8 && !late) __syncthreads();
  }

  int again = threadIdx.x;
  asm volatile("" : "+v"(again));  // (what stores need is made again: nothing of it is held over the loop)
  const int r = tile * R + wave * 32 + (again & 31);
  if (r >= rows) return;
  const int tok = div_by(r, a.G);
  const int head = hk * static_cast<int>(a.G.d) + (r - tok * static_cast<int>(a.G.d));
  const int seen = last_key(a, s, tok) + 1;
  const int k0 = t0 * kKeys;
  const int k1 = t1 * kKeys < seen ? t1 * kKeys : seen;
  const bool none = k1 <= k0;
  const float l = half_sum(col.l);
  const int64_t row = static_cast<int64_t>(s.q0 + tok) * a.H + head;
  if (half == 0 && a.splits > 1) store_part_stats(a, col.m, l, row, none, split);
  const float rl = inverse_sum(a, l, none);
#pragma unroll
  for (int db = 0; db < DT / 32; ++db)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int d = 32 * db + acc_row(i, half);
      if (d >= a.D) continue;
      f32x4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = none ? 0.0f : col.o[db][i + e] * rl;
      if (a.splits > 1)
        *reinterpret_cast<f32x4*>(a.part + (split * (static_cast<int64_t>(a.T) * a.H) + row) * a.D + d) = y;
      else
        *reinterpret_cast<u32x2*>(a.out + row * a.D + d) = u32x2{pack16<kBF16>(y[0], y[1]), pack16<kBF16>(y[2], y[3])};
    }
}

template <bool kBF16, int DT, int kCode, int NQ>
void launch_few(const CodeArgs& c, uint32_t grid, int slots, hipStream_t st) {
  if (c.a.paged.whole)
    code_few_kernel<kBF16, DT, kCode, NQ, true><<<grid, 256, 0, st>>>(c, slots);
  else
    code_few_kernel<kBF16, DT, kCode, NQ, false><<<grid, 256, 0, st>>>(c, slots);
}
template <bool kBF16, int DT, int kCode, int NW>
void launch_rows(const CodeArgs& c, uint32_t grid, int slots, hipStream_t st) {
  if (c.a.paged.whole)
    code_rows_kernel<kBF16, DT, kCode, NW, true><<<grid, 64 * NW, 0, st>>>(c, slots);
  else
    code_rows_kernel<kBF16, DT, kCode, NW, false><<<grid, 64 * NW, 0, st>>>(c, slots);
}
template <bool kBF16, int DT, int kCode>
int launch(const CodeArgs& c, int R, hipStream_t st) {
  const AttnArgs& a = c.a;
  const int64_t slots = slots_of(a.cu_q, a.B, a.T, a.G.d, R);
  const int64_t grid = slots * a.Hk * a.splits;
  GPTQ_REQUIRE(grid < (int64_t{1} << 31), GPTQ_ERR_SHAPE, "attention: too many rows (%lld workgroups)",
               static_cast<long long>(grid));
  if (R == 16)
    launch_few<kBF16, DT, kCode, 1>(c, static_cast<uint32_t>(grid), static_cast<int>(slots), st);
  else if (R == 32)
    launch_few<kBF16, DT, kCode, 2>(c, static_cast<uint32_t>(grid), static_cast<int>(slots), st);
  else if (R == 128)
    launch_rows<kBF16, DT, kCode, 4>(c, static_cast<uint32_t>(grid), static_cast<int>(slots), st);
  else if constexpr (DT == 128)
    launch_rows<kBF16, DT, kCode, 8>(c, static_cast<uint32_t>(grid), static_cast<int>(slots), st);
  const int rc = check_launch("attention");
  if (rc != GPTQ_OK || a.splits == 1) return rc;
  return launch_join<kBF16>(a, st);
}
template <bool kBF16, int DT>
int launch_code(const CodeArgs& c, int code, int R, hipStream_t st) {
  return code == GPTQ_CODE_I8 ? launch<kBF16, DT, GPTQ_CODE_I8>(c, R, st) : launch<kBF16, DT, GPTQ_CODE_E4M3>(c, R, st);
}

}  // namespace
}  // namespace gptq

using namespace gptq;

extern "C" size_t gptq_code_attention_workspace_size(int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t D,
                                                     int64_t max_context) {
  return plan::code_workspace(B, T, H, Hk, D, max_context);
}

extern "C" int gptq_code_attention(const void* q, int dtype, int64_t q_token, int64_t q_head, int code, const void* k_cache,
                                   int64_t k_page, int64_t k_token, int64_t k_head, const void* v_cache, int64_t v_page,
                                   int64_t v_token, int64_t v_head, const float* k_scale, int64_t ks_page, int64_t ks_token,
                                   int64_t ks_head, const float* v_scale, int64_t vs_page, int64_t vs_token,
                                   int64_t vs_head, const int32_t* block_table, int64_t table_stride, int64_t width,
                                   int64_t page_size, int64_t pages, const int32_t* context, const int32_t* cu_q, int64_t B,
                                   int64_t T, int64_t H, int64_t Hk, int64_t D, float scale, int64_t max_context, void* out,
                                   void* workspace, size_t workspace_bytes, gptq_stream_t stream) {
  const char* fn = "gptq_code_attention";
  clear_error();
  int rc = plan::check_attention_args(fn, dtype, B, T, 0, H, Hk, D, scale);
  if (rc != GPTQ_OK) return rc;
  GPTQ_REQUIRE(code == GPTQ_CODE_I8 || code == GPTQ_CODE_E4M3, GPTQ_ERR_DTYPE, "%s: unknown codes %d", fn, code);
  GPTQ_REQUIRE(D % 16 == 0, GPTQ_ERR_SHAPE, "%s: heads of %lld values (codes take multiples of 16)", fn,
               static_cast<long long>(D));
  GPTQ_REQUIRE(page_size >= 1 && page_size < (int64_t{1} << 31) && pages >= 1 && pages < (int64_t{1} << 31) && width >= 0,
               GPTQ_ERR_ARG, "%s: bad cache (%lld pages of %lld tokens, table of %lld)", fn, static_cast<long long>(pages),
               static_cast<long long>(page_size), static_cast<long long>(width));
  if (T == 0) return GPTQ_OK;
  GPTQ_REQUIRE(q && k_cache && v_cache && k_scale && v_scale && out && context && (block_table || width == 0), GPTQ_ERR_ARG,
               "%s: null pointer", fn);
  GPTQ_REQUIRE(cu_q || T == B, GPTQ_ERR_SHAPE, "%s: %lld new tokens of %lld sequences without their offsets", fn,
               static_cast<long long>(T), static_cast<long long>(B));
  const int64_t q_strides[] = {q_token, q_head}, code_strides[] = {k_page, k_token, k_head, v_page, v_token, v_head};
  rc = plan::check_attention_layout(fn, q, k_cache, v_cache, q_strides, 1, 2);
  if (rc != GPTQ_OK) return rc;
  for (int64_t x : code_strides)
    GPTQ_REQUIRE(x >= 0 && x % 16 == 0, GPTQ_ERR_SHAPE, "%s: strides of codes have to be multiples of 16 (got %lld)", fn,
                 static_cast<long long>(x));
  for (int64_t x : {k_token, v_token})  // (16 tokens' offsets are 32 bits)
    GPTQ_REQUIRE(x < (int64_t{1} << 27), GPTQ_ERR_SHAPE, "%s: tokens of codes have to be less than 2^27 apart (got %lld)", fn,
                 static_cast<long long>(x));
  const plan::CodePlan p = plan::code_plan(B, T, H, Hk, D, max_context);
  const size_t need = plan::code_workspace(B, T, H, Hk, D, max_context);
  GPTQ_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), GPTQ_ERR_WORKSPACE,
               "%s: workspace of %zu bytes, needs %zu", fn, workspace_bytes, need);
  CodeArgs c{};
  AttnArgs& a = c.a;
  a.q = {static_cast<const uint16_t*>(q), q_token, q_head};
  c.k = {static_cast<const uint8_t*>(k_cache), k_page, k_token, k_head, k_scale, ks_page, ks_token, ks_head};
  c.v = {static_cast<const uint8_t*>(v_cache), v_page, v_token, v_head, v_scale, vs_page, vs_token, vs_head};
  a.paged.table = block_table;
  a.paged.context = context;
  a.paged.table_stride = table_stride;
  a.paged.most = static_cast<int>(plan::cached_most(width, page_size));
  a.paged.pages = static_cast<int>(pages);
  a.paged.page = fast_div(static_cast<uint32_t>(page_size));
  // Pages of whole 16s of tokens, and strides whose products with 32 bits are 64:
  // addresses by lanes.  Pages of 16 / 24 tokens (us): 512 tokens over 16896 152 / 162,
  // one over 131072 55.3 / 56.8.
  a.paged.whole = page_size % 16 == 0;
  for (int64_t x : {k_page / 4, v_page / 4, ks_page, vs_page}) a.paged.whole &= x >= 0 && x < (int64_t{1} << 30);
  for (int64_t x : {ks_token, vs_token}) a.paged.whole &= x >= 0 && x < (int64_t{1} << 25);
  a.cu_q = cu_q;
  a.B = static_cast<int>(B), a.T = static_cast<int>(T);
  a.H = static_cast<int>(H), a.Hk = static_cast<int>(Hk), a.D = static_cast<int>(D);
  a.G = fast_div(static_cast<uint32_t>(H / Hk));
  a.causal = 1;
  a.c = scale * kLog2e;
  a.out = static_cast<uint16_t*>(out);
  a.part = static_cast<float*>(workspace);
  a.splits = p.splits;
  const hipStream_t st = as_hip(stream);
  const bool wide = D > 64;
  if (dtype == GPTQ_BF16)
    return wide ? launch_code<true, 128>(c, code, p.rows, st) : launch_code<true, 64>(c, code, p.rows, st);
  return wide ? launch_code<false, 128>(c, code, p.rows, st) : launch_code<false, 64>(c, code, p.rows, st);
}
