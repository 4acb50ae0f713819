// Attention of new tokens over a paged cache of 8-bit codes: scores s_ij =
// (scale log2 e ks_j) (q_i kc_j), o_i = sum_j p_ij vs_j vc_j / sum_j p_ij, p_ij =
// 2^(s_ij - m_i), with kc, vc the codes and ks, vs the scales of key j's rows.
//
// The 16-bit types hold every code exactly, so both products run on their MFMA
// with the codes as they are, and the scales, one a key, go into the scores and
// into the weights.  The weights times scales are rounded to the queries' type;
// their unrounded sum divides.
//
// The scales are taken relative to 2^e, with e a wave's own: the sums of values
// of any size then stay inside fp32, and fp16 weights inside their 16 bits.
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
// 2^kSlack: above their smallest and below their largest value (attention.hip).
constexpr float kSlack = 8.0f;
template <bool kBF16>
constexpr float kBias = kBF16 ? 0.0f : 7.0f;
// how far a scale may pass 2^e before e is raised
template <bool kBF16>
constexpr int kScaleRoom = kBF16 ? 24 : 0;

template <int DT>
struct CodeColumn {
  float m, l;       // the running maximum, and this lane's part of the sum of weights
  f32x16 o[DT / 32];
  float down, cap;  // 2^-e, and the largest scale that it allows (the same in the wave's lanes)
};

template <int DT>
__device__ __forceinline__ void start_column(CodeColumn<DT>& col) {
  col.m = kLowest;
  col.l = 0.0f;
  col.down = 1.0f;
  col.cap = -1.0f;
#pragma unroll
  for (int db = 0; db < DT / 32; ++db) col.o[db] = zero16();
}

// Raises e where a tile's scales pass what it allows.  `vs`: a scale of each
// lane's (0 for none); those that are not finite are no reason.
template <bool kBF16, int DT>
__device__ __forceinline__ void allow_scales(CodeColumn<DT>& col, float vs) {
  if (__builtin_expect(__ballot(vs > col.cap && vs < INFINITY) == 0, 1)) return;
  float top = vs > 0.0f && vs < INFINITY ? vs : 0.0f;
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor(top, s));
  if (top == 0.0f) return;  // (scales of 0 need no e)
  int e = ilogbf(top) + 1;
  e = clamp_int(e, -100, 126);
  const float down = ldexpf(1.0f, -e);
  const float less = down / col.down;
  col.down = down;
  col.cap = ldexpf(1.0f, clamp_int(e + kScaleRoom<kBF16>, -126, 127));
  if (less == 1.0f) return;
#pragma unroll
  for (int db = 0; db < DT / 32; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) col.o[db][i] *= less;
}

// Adds NK x 32 keys with scores s (scaled, -infinity where not seen) and scales
// vs (0 where not seen) of their values to the column's sums.  `value` gives the
// operand of value rows 16 ks .. of the tile, channels 32 db ..  kRest: what the
// rounding of the weights left is multiplied too.
template <bool kBF16, int DT, int NK, bool kRest, class Value>
__device__ __forceinline__ void code_step(CodeColumn<DT>& col, f32x16 (&s)[NK], const f32x16 (&vs)[NK], Value&& value) {
  float t = s[0][0];
#pragma unroll
  for (int kt = 0; kt < NK; ++kt)
#pragma unroll
    for (int i = 0; i < 16; ++i) t = __builtin_elementwise_maximum(t, s[kt][i]);
  t = half_max(t) - kBias<kBF16>;
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
      const float p = __builtin_amdgcn_exp2f(s[kt][i] - col.m);
      sum += p;
      s[kt][i] = p * vs[kt][i];
    }
  col.l += sum;
#pragma unroll
  for (int ks = 0; ks < 2 * NK; ++ks) {
    const u32x4 p = operand_of<kBF16>(s[ks / 2], 8 * (ks % 2));
    u32x4 rest;
    if constexpr (kRest) rest = operand_rest<kBF16>(s[ks / 2], 8 * (ks % 2), p);
#pragma unroll
    for (int db = 0; db < DT / 32; ++db) {
      const u32x4 v = value(ks, db);
      col.o[db] = mma32<kBF16>(v, p, col.o[db]);
      if constexpr (kRest) col.o[db] = mma32<kBF16>(v, rest, col.o[db]);
    }
  }
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

// The row's statistics as a part's: the maximum, and a sum of weights of 1
// beside values that are divided by theirs already.  A sum that is NaN stays one.
__device__ __forceinline__ void store_part_stats(const AttnArgs& a, float m, float l, int64_t row, bool none, int split) {
  const int64_t rows = static_cast<int64_t>(a.T) * a.H;
  float* mm = a.part + a.splits * rows * a.D;
  const bool number = l == l;
  mm[split * rows + row] = none ? -INFINITY : number ? m + log2f(l) : m;
  mm[(a.splits + split) * rows + row] = none ? 0.0f : number ? 1.0f : l;
}

// -------------------------------------------------------------- few rows ----
// A workgroup has up to 32 packed rows (query token and head of one key head) and
// its 4 waves share the keys, every wave tiles of 32 of its own (t0 + wave, + 4,
// ...), whose sums are joined at the end.  A lane loads 16-byte pieces of one
// row: of a key they are operands as they come (the contraction's order is free,
// the queries are loaded in the same one), a value's go through LDS to be read
// transposed.  The next tile's loads are in flight while one is used.
constexpr int kFew = 32;

template <int DT>
__device__ __forceinline__ int code_slot(int row) {  // 16-byte chunk c of a row of codes is at slot c ^ this
  if constexpr (DT == 128)
    return ((row >> 3) & 1) << 2 | ((row >> 1) & 1) << 1 | ((row >> 2) & 1);
  else
    return (row >> 2) & 3;
}

template <int DT>
struct FewTile {
  u32x4 k[DT / 32], v[DT / 32];  // chunks 2 j + lane / 32 of row lane % 32
  float scale;                   // of that row's key (lanes below 32) or value
};

template <int DT>
__device__ __forceinline__ void load_few(FewTile<DT>& x, const CodeArgs& c, const Seq& s, int hk, KvAt at, int key0, int lane) {
  const int half = lane >> 5;
  const bool in = key0 + (lane & 31) < s.Lk;
  const uint8_t* kp = c.k.p + at.page * c.k.page + at.at * c.k.token + hk * c.k.head + 16 * half;
  const uint8_t* vp = c.v.p + at.page * c.v.page + at.at * c.v.token + hk * c.v.head + 16 * half;
#pragma unroll
  for (int j = 0; j < DT / 32; ++j) {
    x.k[j] = x.v[j] = u32x4{0, 0, 0, 0};
    if (in && 32 * j + 16 * half < c.a.D) {
      x.k[j] = *reinterpret_cast<const u32x4*>(kp + 32 * j);
      x.v[j] = *reinterpret_cast<const u32x4*>(vp + 32 * j);
    }
  }
  const CodeRows& r = half ? c.v : c.k;
  x.scale = in ? r.scale[at.page * r.s_page + at.at * r.s_token + hk * r.s_head] : 0.0f;
}

template <int DT>
__shared__ __attribute__((aligned(1024))) uint8_t g_code_few[4 * DT * 32 * 4];  // the join's, and before it the waves' tiles

template <bool kBF16, int DT, int kCode>
__global__ __launch_bounds__(256, 2) void code_few_kernel(CodeArgs c, int slots) {
  constexpr int R = 32;
  const AttnArgs& a = c.a;
  __shared__ float stats[3][4][R];
  __shared__ __attribute__((aligned(16))) float scales[4][64];
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

  // channels 32 j + 16 half + 8 e .. + 7: the order of a key's pieces
  u32x4 q[DT / 16];
  const uint16_t* qrow = a.q.p + (s.q0 + tok) * a.q.st + head * a.q.sh;
#pragma unroll
  for (int j = 0; j < DT / 16; ++j) {
    const int d = 32 * (j / 2) + 16 * half + 8 * (j % 2);
    q[j] = inside && d < a.D ? *reinterpret_cast<const u32x4*>(qrow + d) : u32x4{0, 0, 0, 0};
  }

  CodeColumn<DT> col;
  start_column(col);

  uint8_t* const vroom = &g_code_few<DT>[wave * (kFew * DT)];
  lds_u8* const vt = (lds_u8*)vroom;
  lds_f32* const sc_lds = (lds_f32*)&scales[wave][0];
  int put[DT / 32], get[DT / 32];
#pragma unroll
  for (int j = 0; j < DT / 32; ++j) {
    const int row = lane & 31;
    put[j] = row * DT + (((2 * j + half) ^ code_slot<DT>(row)) << 4);
    // a transposing read takes from 16 lanes the addresses of 8 rows x 16 codes,
    // 8 codes a lane, and gives lane i the 8 rows' code i: here the rows 8 (i / 8)
    // + 4 half + (i / 2) % 4 (+ 16 ks, which leaves their slots)
    const int i = lane & 15;
    const int from = 8 * (i >> 3) + 4 * half + ((i >> 1) & 3);
    get[j] = from * DT + (((2 * j + ((lane >> 4) & 1)) ^ code_slot<DT>(from)) << 4) + ((i & 1) << 3);
  }

  FewTile<DT> now;
  KvAt at = kv_at_clamped<true>(a, s, (t0 + wave) * kFew + (lane & 31));
  if (t0 + wave < t1) load_few(now, c, s, hk, at, (t0 + wave) * kFew, lane);
  at = kv_at_clamped<true>(a, s, (t0 + wave + 4) * kFew + (lane & 31));
  for (int t = t0 + wave; t < t1; t += 4) {
    FewTile<DT> next = now;
    if (t + 4 < t1) {
      load_few(next, c, s, hk, at, (t + 4) * kFew, lane);
      at = kv_at_clamped<true>(a, s, (t + 8) * kFew + (lane & 31));
    }
    const int key0 = t * kFew;
#pragma unroll
    for (int j = 0; j < DT / 32; ++j) *(lds_u32x4*)(vt + put[j]) = now.v[j];
    sc_lds[lane] = half ? now.scale : now.scale * a.c;
    allow_scales<kBF16>(col, half ? now.scale : 0.0f);

    f32x16 sc[1] = {zero16()};
#pragma unroll
    for (int j = 0; j < DT / 32; ++j) {
      u32x4 lo, hi;
      widen16<kBF16, kCode>(now.k[j], lo, hi);
      sc[0] = mma32<kBF16>(lo, q[2 * j], sc[0]);
      sc[0] = mma32<kBF16>(hi, q[2 * j + 1], sc[0]);
    }
    wave_sync();
    f32x16 vs[1];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 ks4 = *(const __attribute__((address_space(3))) f32x4*)(sc_lds + 8 * g + 4 * half);
      const f32x4 vs4 = *(const __attribute__((address_space(3))) f32x4*)(sc_lds + 32 + 8 * g + 4 * half);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sc[0][4 * g + e] *= ks4[e];
        vs[0][4 * g + e] = vs4[e] * col.down;
      }
    }
    if (key0 + kFew - 1 > full) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (key0 + acc_row(i, half) > limit) sc[0][i] = -INFINITY, vs[0][i] = 0.0f;
    }
    code_step<kBF16, DT, 1, true>(col, sc, vs, [&](int ks, int db) {
      typedef int i32x2 __attribute__((ext_vector_type(2)));
      typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
      const i32x2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)(vt + get[db] + 16 * ks * DT));
      u32x4 v;
      uint32_t x[4];
      widen4<kBF16, kCode>(static_cast<uint32_t>(w[0]), x[0], x[1]);
      widen4<kBF16, kCode>(static_cast<uint32_t>(w[1]), x[2], x[3]);
      v = u32x4{x[0], x[1], x[2], x[3]};
      return v;
    });
    wait_lgkm<0>();  // (this tile's reads, before the next one's writes)
    wave_sync();
    now = next;
  }
  const float l1 = half_sum(col.l);
  if (half == 0) {
    stats[0][wave][lane] = col.m;
    stats[1][wave][lane] = l1;
    stats[2][wave][lane] = col.down;
  }
  __syncthreads();

  // joined: the waves' sums at the largest maximum and the smallest 2^-e.  Wave
  // w's channels d .. d + 3 of column x are at chunk (d / 4) ^ (x % (DT / 4)) of row
  // (w, x), so that neither side's accesses meet in a bank.
  const int x = lane & 31;
  float m = stats[0][0][x], down = stats[2][0][x];
#pragma unroll
  for (int w = 1; w < 4; ++w) m = fmaxf(m, stats[0][w][x]), down = fminf(down, stats[2][w][x]);
  float l = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; ++w) l += stats[1][w][x] * exp2f(stats[0][w][x] - m);
  lds_u8* const sums = (lds_u8*)&g_code_few<DT>[0];
  auto chunk = [&](int w, int d4) { return ((w * 32 + x) * (DT / 4) + (d4 ^ (x & (DT / 4 - 1)))) * 16; };
  typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
  if (inside) {
    const float scale = exp2f(col.m - m) * (down / col.down);
#pragma unroll
    for (int db = 0; db < DT / 32; ++db)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *(lds_f32x4*)(sums + chunk(wave, (32 * db + acc_row(i, half)) / 4)) =
            f32x4{col.o[db][i] * scale, col.o[db][i + 1] * scale, col.o[db][i + 2] * scale, col.o[db][i + 3] * scale};
  }
  __syncthreads();
  if (!inside) return;

  const int k0 = t0 * kFew;
  const int k1 = t1 * kFew < limit + 1 ? t1 * kFew : limit + 1;
  const bool none = k1 <= k0;
  const int64_t row = static_cast<int64_t>(s.q0 + tok) * a.H + head;
  constexpr int N = DT / 8;  // channels of a thread
  const int d0 = (threadIdx.x >> 5) * N;
  if (threadIdx.x < R && a.splits > 1) store_part_stats(a, m, l, row, none, split);
  const float rl = none ? 0.0f : 1.0f / l;
  const float up = 1.0f / down;
#pragma unroll
  for (int d = 0; d < N; d += 4) {
    if (d0 + d >= a.D) break;
    f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < 4; ++w) y += *(const lds_f32x4*)(sums + chunk(w, (d0 + d) / 4));
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = none ? 0.0f : y[e] * rl * up;
    if (a.splits > 1)
      *reinterpret_cast<f32x4*>(a.part + (split * (static_cast<int64_t>(a.T) * a.H) + row) * a.D + d0 + d) = y;
    else
      *reinterpret_cast<u32x2*>(a.out + row * a.D + d0 + d) = u32x2{pack16<kBF16>(y[0], y[1]), pack16<kBF16>(y[2], y[3])};
  }
}

// ------------------------------------------------------------- many rows ----
// A workgroup of 4 waves has 128 packed rows, 32 a wave.  Tiles of 64 keys are
// loaded as codes by all threads, widened once and left in LDS as 16-bit rows,
// in one of two buffers while the other one is used.
constexpr int kKeys = 64;
template <int DT>
__shared__ __attribute__((aligned(1024))) uint8_t g_code_k[2][kKeys * DT * 2];
template <int DT>
__shared__ __attribute__((aligned(1024))) uint8_t g_code_v[2][kKeys * DT * 2];

template <int DT>
struct ManyTile {
  static constexpr int CH = DT / 16, RPI = 256 / CH, NX = kKeys / RPI;  // chunks of a row, rows at a time
  u32x4 k[NX], v[NX];
  float scale;
};

template <bool kBF16, int DT, int kCode>
__global__ __launch_bounds__(256, 2) void code_rows_kernel(CodeArgs c, int slots) {
  constexpr int R = 128;
  using Tile = ManyTile<DT>;
  const AttnArgs& a = c.a;
  __shared__ __attribute__((aligned(16))) float scales[2][2 * kKeys];  // keys', times c; then values'
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

  const int r = tile * R + wave * 32 + (lane & 31);
  const bool inside = r < rows;
  const int tok = div_by(inside ? r : rows - 1, a.G);
  const int head = hk * static_cast<int>(a.G.d) + ((inside ? r : rows - 1) - tok * static_cast<int>(a.G.d));
  const uint16_t* qrow = a.q.p + (s.q0 + tok) * a.q.st + head * a.q.sh;
  const int limit = last_key(a, s, tok);
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
#pragma unroll
  for (int d = 0; d < DT / 16; ++d) {
    const int at = 16 * d + 8 * half;
    q[d] = inside && at < a.D ? *reinterpret_cast<const u32x4*>(qrow + at) : u32x4{0, 0, 0, 0};
  }

  CodeColumn<DT> col;
  start_column(col);

  // this thread's chunk of rows row0, row0 + RPI, ..; and one of the tile's scales
  const int ch = threadIdx.x % Tile::CH, row0 = threadIdx.x / Tile::CH;
  const int srow = threadIdx.x & 63;
  KvAt at[Tile::NX], sat;
  auto find = [&](int t) {
#pragma unroll
    for (int x = 0; x < Tile::NX; ++x) at[x] = kv_at_clamped<true>(a, s, t * kKeys + row0 + x * Tile::RPI);
    sat = kv_at_clamped<true>(a, s, t * kKeys + srow);
  };
  Tile next;
  auto load = [&](int t) {
#pragma unroll
    for (int x = 0; x < Tile::NX; ++x) {
      next.k[x] = next.v[x] = u32x4{0, 0, 0, 0};
      if (t * kKeys + row0 + x * Tile::RPI < s.Lk && 16 * ch < a.D) {
        next.k[x] = *reinterpret_cast<const u32x4*>(c.k.p + at[x].page * c.k.page + at[x].at * c.k.token + hk * c.k.head + 16 * ch);
        next.v[x] = *reinterpret_cast<const u32x4*>(c.v.p + at[x].page * c.v.page + at[x].at * c.v.token + hk * c.v.head + 16 * ch);
      }
    }
    next.scale = 0.0f;
    if (threadIdx.x < 2 * kKeys && t * kKeys + srow < s.Lk) {
      const CodeRows& rr = wave == 0 ? c.k : c.v;
      next.scale = rr.scale[sat.page * rr.s_page + sat.at * rr.s_token + hk * rr.s_head];
    }
    find(t + 1);
  };
  auto put = [&](int buf) {
#pragma unroll
    for (int x = 0; x < Tile::NX; ++x) {
      const int row = row0 + x * Tile::RPI;
      u32x4 lo, hi;
      const int o0 = row * (DT * 2) + (((2 * ch) ^ row_slot<DT>(row)) << 4);
      const int o1 = row * (DT * 2) + (((2 * ch + 1) ^ row_slot<DT>(row)) << 4);
      widen16<kBF16, kCode>(next.k[x], lo, hi);
      *(lds_u32x4*)((lds_u8*)&g_code_k<DT>[buf][0] + o0) = lo;
      *(lds_u32x4*)((lds_u8*)&g_code_k<DT>[buf][0] + o1) = hi;
      widen16<kBF16, kCode>(next.v[x], lo, hi);
      *(lds_u32x4*)((lds_u8*)&g_code_v<DT>[buf][0] + o0) = lo;
      *(lds_u32x4*)((lds_u8*)&g_code_v<DT>[buf][0] + o1) = hi;
    }
    if (threadIdx.x < 2 * kKeys) scales[buf][threadIdx.x] = wave == 0 ? next.scale * a.c : next.scale;
  };

  const LaneAt<DT> where = lane_at<DT>(lane, 0);
  auto use = [&](int t, int buf) {
    const int key0 = t * kKeys;
    if (key0 >= wave_end) return;
    const lds_u8 *kt = (const lds_u8*)&g_code_k<DT>[buf][0], *vt = (const lds_u8*)&g_code_v<DT>[buf][0];
    const lds_f32* sl = (const lds_f32*)&scales[buf][0];
    allow_scales<kBF16>(col, sl[kKeys + lane]);
    f32x16 sc[2] = {zero16(), zero16()}, vs[2];
#pragma unroll
    for (int d = 0; d < DT / 16; ++d)
#pragma unroll
      for (int n = 0; n < 2; ++n) sc[n] = mma32<kBF16>(row_operand<DT>(kt, 32 * n, d, where), q[d], sc[n]);
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        typedef __attribute__((address_space(3))) const f32x4 lds_cf32x4;
        const f32x4 ks4 = *(lds_cf32x4*)(sl + 32 * n + 8 * g + 4 * half);
        const f32x4 vs4 = *(lds_cf32x4*)(sl + kKeys + 32 * n + 8 * g + 4 * half);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sc[n][4 * g + e] *= ks4[e];
          vs[n][4 * g + e] = vs4[e] * col.down;
        }
      }
    if (key0 + kKeys - 1 > full) {
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (key0 + 32 * n + acc_row(i, half) > limit) sc[n][i] = -INFINITY, vs[n][i] = 0.0f;
    }
    code_step<kBF16, DT, 2, false>(col, sc, vs, [&](int ks, int db) { return column_operand<DT>(vt, 16 * ks, db, where); });
  };

  if (t0 < t1) {
    find(t0);
    load(t0);
    put(0);
    if (t0 + 1 < t1) load(t0 + 1);
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
      const int buf = (t - t0) & 1;
      if (t + 1 < t1) put(buf ^ 1);
      if (t + 2 < t1) load(t + 2);
      use(t, buf);
      __syncthreads();
    }
  }

  const int k0 = t0 * kKeys;
  const int k1 = t1 * kKeys < limit + 1 ? t1 * kKeys : limit + 1;
  const bool none = k1 <= k0;
  const float l = half_sum(col.l);
  const int64_t row = static_cast<int64_t>(s.q0 + tok) * a.H + head;
  if (!inside) return;
  if (half == 0 && a.splits > 1) store_part_stats(a, col.m, l, row, none, split);
  const float rl = none ? 0.0f : 1.0f / l;
  const float up = 1.0f / col.down;
#pragma unroll
  for (int db = 0; db < DT / 32; ++db)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int d = 32 * db + acc_row(i, half);
      if (d >= a.D) continue;
      f32x4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = none ? 0.0f : col.o[db][i + e] * rl * up;
      if (a.splits > 1)
        *reinterpret_cast<f32x4*>(a.part + (split * (static_cast<int64_t>(a.T) * a.H) + row) * a.D + d) = y;
      else
        *reinterpret_cast<u32x2*>(a.out + row * a.D + d) = u32x2{pack16<kBF16>(y[0], y[1]), pack16<kBF16>(y[2], y[3])};
    }
}

template <bool kBF16, int DT, int kCode>
int launch(const CodeArgs& c, bool few, hipStream_t st) {
  const AttnArgs& a = c.a;
  const int64_t slots = slots_of(a.cu_q, a.B, a.T, a.G.d, few ? 32 : 128);
  const int64_t grid = slots * a.Hk * a.splits;
  GPTQ_REQUIRE(grid < (int64_t{1} << 31), GPTQ_ERR_SHAPE, "attention: too many rows (%lld workgroups)",
               static_cast<long long>(grid));
  if (few)
    code_few_kernel<kBF16, DT, kCode><<<static_cast<uint32_t>(grid), 256, 0, st>>>(c, static_cast<int>(slots));
  else
    code_rows_kernel<kBF16, DT, kCode><<<static_cast<uint32_t>(grid), 256, 0, st>>>(c, static_cast<int>(slots));
  const int rc = check_launch("attention");
  if (rc != GPTQ_OK || a.splits == 1) return rc;
  return launch_join<kBF16>(a, st);
}
template <bool kBF16, int DT>
int launch_code(const CodeArgs& c, int code, bool few, hipStream_t st) {
  return code == GPTQ_CODE_I8 ? launch<kBF16, DT, GPTQ_CODE_I8>(c, few, st) : launch<kBF16, DT, GPTQ_CODE_E4M3>(c, few, st);
}

}  // namespace
}  // namespace gptq

using namespace gptq;

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
  const plan::PagedPlan p = plan::paged_plan(B, T, H, Hk, max_context);
  const size_t need = plan::paged_workspace(B, T, H, Hk, D, max_context);
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
    return wide ? launch_code<true, 128>(c, code, p.few, st) : launch_code<true, 64>(c, code, p.few, st);
  return wide ? launch_code<false, 128>(c, code, p.few, st) : launch_code<false, 64>(c, code, p.few, st);
}
