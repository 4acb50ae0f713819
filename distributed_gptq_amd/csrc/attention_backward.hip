// Gradients of the attention of packed sequences on gfx950 MFMA.  With the
// forward pass' weights p_ij = 2^(c q_i k_j - lse_i) and g = dL/do:
//   delta_i = g_i o_i (o to about 16 bits),  ds_ij = p_ij (g_i v_j - delta_i),
//   dv_j = sum_i p_ij g_i,  dk_j = scale sum_i ds_ij q_i,  dq_i = scale sum_j ds_ij k_j,
// sums over the query heads of a key head included.  The weights are computed
// again from the scores, in one kernel per key (dk, dv) and one per query (dq):
// seven products of tiles instead of five, but every sum is made in one place
// and in one order, so that the gradients are the same from call to call.
#include "attn_tile.hpp"

namespace gptq {
namespace {

constexpr int kRows = 64;        // packed query rows, or keys, of a tile
constexpr int kMaxima = plan::kBackMaxima;  // workgroups of the first kernel

struct BackArgs {
  AttnArgs f;                    // q, k, v, offsets, sizes; lse as input
  Rows16 g;                      // dL/do
  const uint16_t *o, *o_rest;    // (T, H, D): the output, and what its rounding left
  float* delta;                  // (T, H)
  float* maxima;                 // 2 x kMaxima: largest finite |g_i|^2 and |v_j|^2 of each workgroup (fp16)
  float* part;                   // with splits > 1: dk and dv of each split (S, Hk, D) each
  int splits;                    // parts of the rows of each 64 keys
  float scale;
  uint16_t *dq, *dk, *dv;        // contiguous
};

// fp16 ends at 2^-24, far above the ds of a long row (p alone is 1 / length):
// ds is multiplied by 2^e before it is rounded, and the sum by 2^-e.  With
// |ds_ij| <= 2 max |g_i| max |v_j|, e is the largest that keeps ds below 2^14.
// p is multiplied by 2^14.  bf16 has fp32's exponents and needs neither.
constexpr float kWeightShift = 14.0f;

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v = fmaxf(v, __shfl_xor(v, m));
  return v;
}

// e for all of a kernel's ds, by the 256 threads of a workgroup (one barrier)
__device__ __forceinline__ float ds_shift(const BackArgs& a, float (*room)[4]) {
  float g = 0.0f, v = 0.0f;
#pragma unroll
  for (int x = 0; x < kMaxima / 256; ++x) {
    g = fmaxf(g, a.maxima[256 * x + threadIdx.x]);
    v = fmaxf(v, a.maxima[kMaxima + 256 * x + threadIdx.x]);
  }
  g = wave_max(g);
  v = wave_max(v);
  if ((threadIdx.x & 63) == 0) room[0][threadIdx.x >> 6] = g, room[1][threadIdx.x >> 6] = v;
  __syncthreads();
  g = fmaxf(fmaxf(room[0][0], room[0][1]), fmaxf(room[0][2], room[0][3]));
  v = fmaxf(fmaxf(room[1][0], room[1][1]), fmaxf(room[1][2], room[1][3]));
  const float bound = 2.0f * sqrtf(g) * sqrtf(v);
  if (!(bound > 0.0f && bound < 1e30f)) return 0.0f;
  const float e = floorf(14.0f - log2f(bound));
  return e < -100.0f ? -100.0f : e > 100.0f ? 100.0f : e;
}

// For fp16, whose ds need their scale first: delta and the maxima, 16 lanes a row,
// 8 values a lane.  Bound by memory: 12 us for 4096 tokens of 32 heads of 128 (101
// MB, in part cached).  In bf16 the dq kernel, which runs first, gives delta.
__global__ __launch_bounds__(256) void attn_delta_kernel(BackArgs a) {
  const int sub = threadIdx.x & 15, d = 8 * sub;
  // (rows past the offsets have no gradient, and may hold anything)
  const int64_t rows = static_cast<int64_t>(first_row(a.f.cu_q, a.f.B, a.f.B, a.f.T)) * a.f.H;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 16;
  float most[2] = {0.0f, 0.0f};
  auto values = [&](const uint16_t* p, float (&x)[8]) {
    const u32x4 w = d < a.f.D ? *reinterpret_cast<const u32x4*>(p + d) : u32x4{0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = value16<false>(static_cast<uint16_t>(w[e / 2] >> (16 * (e % 2))));
  };
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * 16 + (threadIdx.x >> 4); row < rows; row += step) {
    const int64_t t = row / a.f.H;
    const int h = static_cast<int>(row - t * a.f.H);
    float g[8], o[8], rest[8];
    values(a.g.p + t * a.g.st + h * a.g.sh, g);
    values(a.o + row * a.f.D, o);
    values(a.o_rest + row * a.f.D, rest);
    float dot = 0.0f, sq = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) dot = fmaf(g[e], o[e] + rest[e], dot), sq = fmaf(g[e], g[e], sq);
#pragma unroll
    for (int m = 8; m; m >>= 1) dot += __shfl_xor(dot, m), sq += __shfl_xor(sq, m);
    if (sub == 0) a.delta[row] = dot;
    if (sq < INFINITY) most[0] = fmaxf(most[0], sq);  // (an infinity makes its ds infinite at any scale)
  }
  const int64_t vrows = static_cast<int64_t>(first_row(a.f.cu_k, a.f.B, a.f.B, a.f.S)) * a.f.Hk;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * 16 + (threadIdx.x >> 4); row < vrows; row += step) {
    const int64_t t = row / a.f.Hk;
    float v[8], sq = 0.0f;
    values(a.f.v.p + t * a.f.v.st + (row - t * a.f.Hk) * a.f.v.sh, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) sq = fmaf(v[e], v[e], sq);
#pragma unroll
    for (int m = 8; m; m >>= 1) sq += __shfl_xor(sq, m);
    if (sq < INFINITY) most[1] = fmaxf(most[1], sq);
  }
  __shared__ float room[2][4];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const float w = wave_max(most[x]);
    if ((threadIdx.x & 63) == 0) room[x][threadIdx.x >> 6] = w;
  }
  __syncthreads();
  if (threadIdx.x < 2)
    a.maxima[threadIdx.x * kMaxima + blockIdx.x] =
        fmaxf(fmaxf(room[threadIdx.x][0], room[threadIdx.x][1]), fmaxf(room[threadIdx.x][2], room[threadIdx.x][3]));
}

// 32 columns' channels to memory: y = x * r, rounded
template <bool kBF16, int DT>
__device__ __forceinline__ void store_rows(uint16_t* row, const f32x16 (&x)[DT / 32], float r, int D, int half) {
#pragma unroll
  for (int db = 0; db < DT / 32; ++db)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int d = 32 * db + acc_row(i, half);
      if (d < D)
        *reinterpret_cast<u32x2*>(row + d) =
            u32x2{pack16<kBF16>(x[db][i] * r, x[db][i + 1] * r), pack16<kBF16>(x[db][i + 2] * r, x[db][i + 3] * r)};
    }
}

template <int DT>
__device__ __forceinline__ void load_operand(u32x4 (&x)[DT / 16], const uint16_t* row, bool inside, int D, int half) {
#pragma unroll
  for (int s = 0; s < DT / 16; ++s) {
    const int d = 16 * s + 8 * half;
    x[s] = inside && d < D ? *reinterpret_cast<const u32x4*>(row + d) : u32x4{0, 0, 0, 0};
  }
}

template <int DT>
__shared__ __attribute__((aligned(1024))) uint8_t g_back_a0[kRows * DT * 2];
template <int DT>
__shared__ __attribute__((aligned(1024))) uint8_t g_back_a1[kRows * DT * 2];
template <int DT>
__shared__ __attribute__((aligned(1024))) uint8_t g_back_b0[kRows * DT * 2];
template <int DT>
__shared__ __attribute__((aligned(1024))) uint8_t g_back_b1[kRows * DT * 2];

template <int DT>
__device__ __forceinline__ bool all_finite(const f32x16 (&x)[DT / 32]) {
  float worst = 0.0f;
#pragma unroll
  for (int db = 0; db < DT / 32; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) worst = fmaf(x[db][i], 0.0f, worst);  // 0, or NaN
  return worst == 0.0f;
}

// The weight of a score that is seen, however small: an infinity that it
// multiplies gives one.
__device__ __forceinline__ float seen_weight(float score, float c, float lse) {
  const float p = __builtin_amdgcn_exp2f(fmaf(score, c, -lse));
  return p < 0x1p-126f && score > -INFINITY ? 0x1p-126f : p;
}

// A wave's columns of dq again where the product of tiles is not finite: tiles of
// 32 keys below t1 through `room` in LDS (two tiles), the keys added row by row.
template <bool kBF16, int DT>
__device__ __forceinline__ void exact_dq(f32x16 (&acc)[DT / 32], const AttnArgs& a, const Seq& s, int hk,
                                         const u32x4 (&q)[DT / 16], const u32x4 (&g)[DT / 16], float lse, float delta,
                                         int limit, int t1, uint8_t* room, int lane) {
  uint8_t* vroom = room + 32 * DT * 2;
  const lds_u8 *kt = (const lds_u8*)room, *vt = (const lds_u8*)vroom;
  const LaneAt<DT> where = lane_at<DT>(lane, 0);
#pragma unroll
  for (int db = 0; db < DT / 32; ++db) acc[db] = zero16();
#pragma unroll 1
  for (int t = 0; t < t1; ++t) {
    const int key0 = 32 * t;
    fetch_rows<DT, 32, false>(a, s, hk, kv_at<false>(a, s, key0 + (lane & 31)), key0, 0, room, vroom, lane);
    landed();
    f32x16 sc = zero16(), dp = zero16();
#pragma unroll
    for (int d = 0; d < DT / 16; ++d) {
      sc = mma32<kBF16>(row_operand<DT>(kt, 0, d, where), q[d], sc);
      dp = mma32<kBF16>(row_operand<DT>(vt, 0, d, where), g[d], dp);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) sc[i] = seen_weight(sc[i], a.c, lse) * (dp[i] - delta);
    wave_sync();
    store_weights((lds_f32*)vroom, sc, lane);  // (the values are done with)
    landed();
    add_seen_rows<kBF16, DT>(acc, (const lds_f32*)vroom, kt, lane, [&](int r) { return key0 + r <= limit; });
    landed();
  }
}

// dq: as the forward pass, 32 packed rows a wave (a lane's column), tiles of 64
// keys and values in LDS.
//
// ds is multiplied as its rounded value and what the rounding left.  The ds of a
// row sum to zero, so the part of the keys that those with weight have in common
// (along q) cancels in dq, but not in the errors of rounded ds: with them alone
// the error of dq against 64 bits is 1.45 times that of its own rounding for 2048
// tokens and heads of 128, 1.50 for 3400 and heads of 64, and grows on.
//
// Bound by the waits between a wave's steps (MFMAs busy 50% of the cycles): 152-159
// us for 2 x 2048 tokens, 32 over 8 heads of 128, of which the rests take 29 and
// delta 8 (bf16; a kernel of its own took 17 with its launch).
template <bool kBF16, int DT>
__global__ __launch_bounds__(256, 2) void attn_dq_kernel(BackArgs args, int slots) {
  constexpr int R = 128, W = kRows / 4;
  __shared__ float room[2][4];
  const AttnArgs& a = args.f;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int G = static_cast<int>(a.G.d);
  const int hk = blockIdx.x % a.Hk;
  int tile;
  const int b = find_seq(a.cu_q, a.B, a.T, G, R, slots - 1 - static_cast<int>(blockIdx.x / a.Hk), &tile);
  const Seq s = seq_of<false>(a, b);
  const int rows = s.Lq * G;
  if (tile * R >= rows) return;
  float shift = 0.0f;
  if constexpr (!kBF16) shift = ds_shift(args, room);
  const float up = exp2f(shift);

  const int r = tile * R + wave * 32 + (lane & 31);
  const bool inside = r < rows;
  const int tok = div_by(inside ? r : rows - 1, a.G);
  const int head = hk * G + ((inside ? r : rows - 1) - tok * G);
  const int limit = last_key(a, s, tok);
  const int first_r = tile * R + wave * 32;
  const int full = last_key(a, s, div_by(first_r < rows ? first_r : rows - 1, a.G));
  const int last_r = (tile + 1) * R < rows ? (tile + 1) * R - 1 : rows - 1;
  const int wave_r = first_r + 31 < rows ? first_r + 31 : rows - 1;
  const int wave_end = first_r < rows ? last_key(a, s, div_by(wave_r, a.G)) + 1 : 0;
  const int last = last_key(a, s, div_by(last_r, a.G));
  const int tiles = last < 0 ? 0 : last / kRows + 1;

  const int64_t row = static_cast<int64_t>(s.q0 + tok) * a.H + head;
  u32x4 q[DT / 16], g[DT / 16];
  load_operand<DT>(q, a.q.p + (s.q0 + tok) * a.q.st + head * a.q.sh, inside, a.D, half);
  load_operand<DT>(g, args.g.p + (s.q0 + tok) * args.g.st + head * args.g.sh, inside, a.D, half);
  const float lse = a.lse[row];
  float delta;
  if constexpr (kBF16) {
    float dot = 0.0f;
#pragma unroll
    for (int x = 0; x < DT / 16; ++x) {
      const int d = 16 * x + 8 * half;
      if (!inside || d >= a.D) continue;
      const u32x4 o = *reinterpret_cast<const u32x4*>(args.o + row * a.D + d);
      const u32x4 rest = *reinterpret_cast<const u32x4*>(args.o_rest + row * a.D + d);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int to = 16 * (e % 2);
        dot = fmaf(value16<true>(static_cast<uint16_t>(g[x][e / 2] >> to)),
                   value16<true>(static_cast<uint16_t>(o[e / 2] >> to)) + value16<true>(static_cast<uint16_t>(rest[e / 2] >> to)),
                   dot);
      }
    }
    delta = half_sum(dot);
    if (inside && half == 0) args.delta[row] = delta;
  } else {
    delta = args.delta[row];
  }

  f32x16 acc[DT / 32];
#pragma unroll
  for (int db = 0; db < DT / 32; ++db) acc[db] = zero16();

  KvAt at = kv_at<false>(a, s, wave * W + lane % W);
  auto fetch = [&](int t, uint8_t* kt, uint8_t* vt) {
    at.at = s.k0 + t * kRows + wave * W + lane % W;
    fetch_rows<DT, W, false>(a, s, hk, at, t * kRows, wave * W, kt, vt, lane);
  };
  const LaneAt<DT> where = lane_at<DT>(lane, 0);
  auto use = [&](int t, const lds_u8* kt, const lds_u8* vt) {
    const int key0 = t * kRows;
    if (key0 >= wave_end) return;
    const bool masked = key0 + kRows - 1 > full;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      f32x16 sc = zero16(), dp = zero16();
#pragma unroll
      for (int d = 0; d < DT / 16; ++d) {
        sc = mma32<kBF16>(row_operand<DT>(kt, 32 * n, d, where), q[d], sc);
        dp = mma32<kBF16>(row_operand<DT>(vt, 32 * n, d, where), g[d], dp);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float p = __builtin_amdgcn_exp2f(fmaf(sc[i], a.c, -lse));
        sc[i] = p * (dp[i] - delta) * up;
      }
      if (masked) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (key0 + 32 * n + acc_row(i, half) > limit) sc[i] = 0.0f;
      }
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        const u32x4 x = operand_of<kBF16>(sc, 8 * ks), rest = operand_rest<kBF16>(sc, 8 * ks, x);
#pragma unroll
        for (int db = 0; db < DT / 32; ++db) {
          const u32x4 k = column_operand<DT>(kt, 32 * n + 16 * ks, db, where);
          acc[db] = mma32<kBF16>(k, x, acc[db]);
          acc[db] = mma32<kBF16>(k, rest, acc[db]);
        }
      }
    }
  };
  if (tiles > 0) {
    fetch(0, g_back_a0<DT>, g_back_b0<DT>);
    __syncthreads();
    for (int t = 0; t < tiles; t += 2) {
      if (t + 1 < tiles) fetch(t + 1, g_back_a1<DT>, g_back_b1<DT>);
      use(t, (const lds_u8*)&g_back_a0<DT>[0], (const lds_u8*)&g_back_b0<DT>[0]);
      __syncthreads();
      if (t + 1 >= tiles) break;
      if (t + 2 < tiles) fetch(t + 2, g_back_a0<DT>, g_back_b0<DT>);
      use(t + 1, (const lds_u8*)&g_back_a1<DT>[0], (const lds_u8*)&g_back_b1<DT>[0]);
      __syncthreads();
    }
  }
  const bool fine = all_finite<DT>(acc);
  // (with a NaN for delta or lse all of the row is, from its own keys)
  const bool bad = inside && half_sum(fine ? 0.0f : 1.0f) != 0.0f && lse == lse && delta == delta;
  if (inside && !bad) store_rows<kBF16, DT>(args.dq + row * a.D, acc, args.scale * exp2f(-shift), a.D, half);
  if (__builtin_expect(__ballot(bad) != 0, 0)) {
    uint8_t* const room = wave == 0 ? g_back_a0<DT> : wave == 1 ? g_back_a1<DT> : wave == 2 ? g_back_b0<DT> : g_back_b1<DT>;
    exact_dq<kBF16, DT>(acc, a, s, hk, q, g, lse, delta, limit, (wave_end + 31) / 32, room, late_lane());
    if (bad) store_rows<kBF16, DT>(args.dq + row * a.D, acc, args.scale, a.D, half);
  }
}

// dk and dv: a workgroup of 4 waves has 64 keys, whose value rows stay in LDS,
// and passes tiles of 64 query rows (of one head) and their gradients through
// two LDS buffers.  Wave w has keys 32 (w % 2) .. (a lane's column) and each
// tile's rows 32 (w / 2) ..; the two waves of a key are joined at the end.
//
// Two workgroups run on a CU, the vector work of one beside the MFMAs of the
// other, which takes all registers (256 a lane) and all of LDS (80 KB each): the
// rows' lse and delta have no place in either, and are added by one MFMA more
// each, as 16 further channels of q and g (their parts, below) and of k and v
// (the parts' units).
//
// 175-182 us and 13 of the join for 2 x 2048 tokens, 32 over 8 heads of 128 (MFMAs
// busy 43% of the cycles, no LDS conflicts); one workgroup of 8 waves a CU, lse
// and delta in registers: 218.
constexpr int kBackRows = 64;
template <int DT>
__shared__ __attribute__((aligned(1024))) uint8_t g_dkv_q0[kBackRows * DT * 2];
template <int DT>
__shared__ __attribute__((aligned(1024))) uint8_t g_dkv_q1[kBackRows * DT * 2];
template <int DT>
__shared__ __attribute__((aligned(1024))) uint8_t g_dkv_g0[kBackRows * DT * 2];
template <int DT>
__shared__ __attribute__((aligned(1024))) uint8_t g_dkv_g1[kBackRows * DT * 2];
template <int DT>
__shared__ __attribute__((aligned(1024))) uint8_t g_dkv_v[64 * DT * 2];

// A float x as values of 16 bits, x = sum of part i times unit i: in bf16, which
// has fp32's range, three parts of unit 1; in fp16 four of 2^15, 2^4, 2^-7 and
// 2^-14, the rest of each within the next one's range, for |x| < 2^31 to 2^-33 of
// it or to 2^-39.  (fp16 queries, keys and gradients of a few hundred already give
// scores and deltas beyond fp16's 65504.)
template <bool kBF16>
__device__ __forceinline__ u32x2 parts_of(float x) {
  if constexpr (kBF16) {
    const uint32_t hi = pack16<true>(x, 0.0f) & 0xFFFFu;
    const float r1 = x - bf16_bits_to_f32(static_cast<uint16_t>(hi));
    const uint32_t mid = pack16<true>(r1, 0.0f) & 0xFFFFu;
    return u32x2{hi | mid << 16, pack16<true>(r1 - bf16_bits_to_f32(static_cast<uint16_t>(mid)), 0.0f)};
  } else {
    constexpr float kUnit[4] = {0x1p15f, 0x1p4f, 0x1p-7f, 0x1p-14f}, kInverse[4] = {0x1p-15f, 0x1p-4f, 0x1p7f, 0x1p14f};
    uint32_t part[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      part[i] = pack16<false>(x * kInverse[i], 0.0f) & 0xFFFFu;
      x = fmaf(-f16_bits_to_f32(static_cast<uint16_t>(part[i])), kUnit[i], x);
    }
    return u32x2{part[0] | part[1] << 16, part[2] | part[3] << 16};
  }
}
template <bool kBF16>
__device__ __forceinline__ u32x4 units() {
  return kBF16 ? u32x4{0x3F803F80u, 0x3F80u, 0, 0} : u32x4{0x4C007800u, 0x04002000u, 0, 0};
}

// A wave's 32 keys' dv, or dk, again where the products of tiles are not finite
// (as exact_dq): tiles first .. last - 1 of 64 query rows, 32 at a time through
// the wave's halves of the tiles' buffers, the rows' weights in another half.
template <bool kBF16, int DT, bool kKeyGrad>
__device__ __forceinline__ void exact_dkv(f32x16 (&sums)[DT / 32], const BackArgs& args, const Seq& s, int hk,
                                          const u32x4 (&kf)[DT / 16], int kw, bool bad, int t0, int nt, int first, int last,
                                          const lds_u8* vt, uint8_t* qroom, uint8_t* groom, int lane) {
  constexpr int CH = DT / 8, RPI = 64 / CH;
  const AttnArgs& a = args.f;
  const int half = lane >> 5, G = static_cast<int>(a.G.d), key = kw + (lane & 31), off = s.Lk - s.Lq;
  const lds_u8 *qt = (const lds_u8*)qroom, *gt = (const lds_u8*)groom;
  lds_f32* weights = (lds_f32*)(qroom + 32 * DT * 2);
  const LaneAt<DT> where = lane_at<DT>(lane, 0);
#pragma unroll
  for (int db = 0; db < DT / 32; ++db) sums[db] = zero16();
#pragma unroll 1
  for (int x = 2 * first; x < 2 * last; ++x) {
    const int head = hk * G + x / 2 / nt, r0 = (t0 + nt - 1 - x / 2 % nt) * kBackRows + 32 * (x & 1);
    if (r0 >= s.Lq || last_key(a, s, r0 + 31 < s.Lq ? r0 + 31 : s.Lq - 1) < kw) continue;
    const uint16_t* qp = a.q.p + s.q0 * a.q.st + head * a.q.sh;
    const uint16_t* gp = args.g.p + s.q0 * args.g.st + head * args.g.sh;
#pragma unroll
    for (int y = 0; y < 32 / RPI; ++y) {
      const int i = y * RPI + lane / CH;
      const int64_t tok = r0 + i;
      const int ch = (lane % CH) ^ row_slot<DT>(i);
      const bool in = tok < s.Lq && ch * 8 < a.D;
      copy16_to_lds(in ? static_cast<const void*>(qp + tok * a.q.st + ch * 8) : g_attn_zeros, qroom + y * 1024);
      copy16_to_lds(in ? static_cast<const void*>(gp + tok * args.g.st + ch * 8) : g_attn_zeros, groom + y * 1024);
    }
    const int tok = r0 + (lane & 31) < s.Lq ? r0 + (lane & 31) : s.Lq - 1;
    const int64_t row = static_cast<int64_t>(s.q0 + tok) * a.H + head;
    const float lse = a.lse[row], delta = args.delta[row];
    landed();
    f32x16 w = zero16();
#pragma unroll
    for (int d = 0; d < DT / 16; ++d) w = mma32<kBF16>(row_operand<DT>(qt, 0, d, where), kf[d], w);
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = seen_weight(w[i], a.c, __shfl(lse, acc_row(i, half)));
    if constexpr (kKeyGrad) {
      f32x16 dp = zero16();
#pragma unroll
      for (int d = 0; d < DT / 16; ++d) dp = mma32<kBF16>(row_operand<DT>(gt, 0, d, where), row_operand<DT>(vt, 0, d, where), dp);
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] *= dp[i] - __shfl(delta, acc_row(i, half));
    }
    store_weights(weights, w, lane);
    landed();
    const int seen = a.causal ? key - off - r0 : 0, rows = s.Lq - r0;
    add_seen_rows<kBF16, DT>(sums, weights, kKeyGrad ? qt : gt, lane, [&](int r) { return r >= seen && r < rows; });
    landed();
    bool open = false;
#pragma unroll
    for (int db = 0; db < DT / 32; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) open = open || sums[db][i] == sums[db][i];
    if (__ballot(bad && open) == 0) break;  // (all NaN, whatever follows)
  }
}

template <bool kBF16, int DT>
__global__ __launch_bounds__(256, 2) void attn_dkv_kernel(BackArgs args) {
  constexpr int R = 64, W = kBackRows / 4, CH = DT / 8, RPI = 64 / CH;
  const AttnArgs& a = args.f;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int G = static_cast<int>(a.G.d);
  const int hk = blockIdx.x % a.Hk;
  // (causal: the first keys' workgroups, with the most rows, go first)
  const int rest = static_cast<int>(blockIdx.x / a.Hk), split = rest % args.splits;
  int tile;
  const int b = find_seq(a.cu_k, a.B, a.S, 1, R, rest / args.splits, &tile);
  Seq s = seq_of<false>(a, b);
  if (b == a.B) {  // rows past the offsets
    s.Lk = a.S - s.k0;
    s.Lq = 0;
  }
  if (tile * R >= s.Lk) return;
  float shift = 0.0f;
  if constexpr (!kBF16) {
    shift = ds_shift(args, reinterpret_cast<float(*)[4]>(&g_dkv_q0<DT>[0]));
    __syncthreads();
  }
  const float up = exp2f(kBF16 ? 0.0f : shift - kWeightShift);

  const int key0 = tile * R, kw = key0 + 32 * (wave & 1), n = wave >> 1;
  const int key = kw + (lane & 31);
  const bool inside = key < s.Lk;
  const int off = s.Lk - s.Lq;
  // tiles of 64 tokens of one query head after the other, from the first token
  // that sees the workgroup's first key on
  const int i0 = a.causal && key0 > off ? key0 - off : 0;
  const int t0 = (i0 < s.Lq ? i0 : s.Lq) / kBackRows, nt = (s.Lq + kBackRows - 1) / kBackRows - t0;

  u32x4 kf[DT / 16];
  load_operand<DT>(kf, a.k.p + static_cast<int64_t>(s.k0 + (inside ? key : 0)) * a.k.st + hk * a.k.sh, inside, a.D, half);
#pragma unroll
  for (int x = 0; x < W / RPI; ++x) {  // 16 of the values' rows a wave
    const int i = wave * W + x * RPI + lane / CH;
    const int ch = (lane % CH) ^ row_slot<DT>(i);
    const bool in = key0 + i < s.Lk && ch * 8 < a.D;
    const uint16_t* vp = a.v.p + static_cast<int64_t>(s.k0 + (in ? key0 + i : 0)) * a.v.st + hk * a.v.sh + ch * 8;
    copy16_to_lds(in ? static_cast<const void*>(vp) : g_attn_zeros, g_dkv_v<DT> + (wave * (W / RPI) + x) * 1024);
  }
  f32x16 dk[DT / 32], dv[DT / 32];
#pragma unroll
  for (int db = 0; db < DT / 32; ++db) dk[db] = zero16(), dv[db] = zero16();

  const float inv_c = -1.0f / a.c;
  float n_lse = 0.0f, n_delta = 0.0f;  // of the next tile's row n 32 + lane % 32
  // a lane's part of the copies' offsets and of those of lse and delta; opaque in
  // the loop, where what follows from them is cheaper than registers
  const uint32_t q_step = (lane / CH) * static_cast<uint32_t>(a.q.st * 2);
  const uint32_t g_step = (lane / CH) * static_cast<uint32_t>(args.g.st * 2);
  uint32_t chunk = ((lane % CH) ^ row_slot<DT>(lane / CH)) << 4;
  // tile x: of head x / nt, from the last tokens (which see all keys) on, so that
  // the workgroups of a key head read the same rows at the same time
  auto fetch = [&](int x, uint8_t* qt, uint8_t* gt) {
    const int g = x / nt, head = hk * G + g, tok0 = (t0 + nt - 1 - (x - g * nt)) * kBackRows;
    const uint16_t* qp = a.q.p + s.q0 * a.q.st + head * a.q.sh;
    const uint16_t* gp = args.g.p + s.q0 * args.g.st + head * args.g.sh;
    const int first = tok0 + wave * W;
    asm volatile("" : "+v"(chunk));
    {
      const int row = tok0 + 32 * n < s.Lq ? tok0 + 32 * n : s.Lq - 1, left = s.Lq - 1 - row;
      const int64_t at = static_cast<int64_t>(s.q0 + row) * a.H + head;
      const int more = ((lane & 31) < left ? lane & 31 : left) * a.H;  // (rows past the last are masked)
      n_lse = a.lse[at + more];
      n_delta = args.delta[at + more];
    }
    if (first + W <= s.Lq && a.D == DT) {
      auto copy = [&](const uint16_t* p, int64_t st, uint32_t step, uint8_t* tile) {
        const uint8_t* base = reinterpret_cast<const uint8_t*>(uniform_u64(reinterpret_cast<uint64_t>(p + first * st)));
#pragma unroll
        for (int y = 0; y < W / RPI; ++y)  // (row_slot of rows y RPI apart: its other bits)
          copy16_to_lds(base + static_cast<int64_t>(y * RPI) * (st * 2) + (step + (chunk ^ (row_slot<DT>(y * RPI) << 4))),
                        tile + (wave * (W / RPI) + y) * 1024);
      };
      copy(qp, a.q.st, q_step, qt);
      copy(gp, args.g.st, g_step, gt);
    } else {
#pragma unroll
      for (int y = 0; y < W / RPI; ++y) {
        const int i = wave * W + y * RPI + lane / CH;
        const int64_t tok = tok0 + i;
        const int ch = (lane % CH) ^ row_slot<DT>(i);
        const bool in = tok < s.Lq && ch * 8 < a.D;
        copy16_to_lds(in ? static_cast<const void*>(qp + tok * a.q.st + ch * 8) : g_attn_zeros,
                      qt + (wave * (W / RPI) + y) * 1024);
        copy16_to_lds(in ? static_cast<const void*>(gp + tok * args.g.st + ch * 8) : g_attn_zeros,
                      gt + (wave * (W / RPI) + y) * 1024);
      }
    }
  };
  const LaneAt<DT> where = lane_at<DT>(lane, 32 * n * (DT * 2));  // of the wave's rows of a tile
  auto use = [&](int x, float lse, float delta, const lds_u8* qt, const lds_u8* gt) {
    const int r0 = (t0 + nt - 1 - x % nt) * kBackRows + 32 * n;
    if (r0 >= s.Lq) return;
    if (last_key(a, s, r0 + 31 < s.Lq ? r0 + 31 : s.Lq - 1) < kw) return;  // no row of these sees a key of the wave
    const bool masked = r0 + 31 >= s.Lq || last_key(a, s, r0) < kw + 31;
    const lds_u8* vt = (const lds_u8*)&g_dkv_v<DT>[0] + (32 * (wave & 1) - 32 * n) * (DT * 2);
    f32x16 sc = zero16(), dp = zero16();
    {
      const u32x2 l = parts_of<kBF16>(half ? 0.0f : lse * inv_c), d = parts_of<kBF16>(half ? 0.0f : -delta);
      sc = mma32<kBF16>(u32x4{l[0], l[1], 0, 0}, units<kBF16>(), sc);
      dp = mma32<kBF16>(u32x4{d[0], d[1], 0, 0}, units<kBF16>(), dp);
    }
#pragma unroll
    for (int d = 0; d < DT / 16; ++d) {
      sc = mma32<kBF16>(row_operand<DT>(qt, 0, d, where), kf[d], sc);
      dp = mma32<kBF16>(row_operand<DT>(gt, 0, d, where), row_operand<DT>(vt, 0, d, where), dp);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      sc[i] = __builtin_amdgcn_exp2f(kBF16 ? sc[i] * a.c : fmaf(sc[i], a.c, kWeightShift));
      dp[i] = sc[i] * dp[i] * up;
    }
    if (masked) {
      // row r0 + 4 half + i sees the key where i >= seen, and is one where i < rows
      const int seen = a.causal ? key - off - r0 - 4 * half : 0, rows = s.Lq - r0 - 4 * half;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (acc_row(i, 0) < seen || acc_row(i, 0) >= rows) sc[i] = 0.0f, dp[i] = 0.0f;
    }
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const u32x4 p = operand_of<kBF16>(sc, 8 * ks), w = operand_of<kBF16>(dp, 8 * ks);
#pragma unroll
      for (int db = 0; db < DT / 32; ++db) {
        dv[db] = mma32<kBF16>(column_operand<DT>(gt, 16 * ks, db, where), p, dv[db]);
        dk[db] = mma32<kBF16>(column_operand<DT>(qt, 16 * ks, db, where), w, dk[db]);
      }
    }
  };
  const int per = (nt * G + args.splits - 1) / args.splits;
  const int first = split * per, last = first + per < nt * G ? first + per : nt * G;
  if (first < last) {
    fetch(first, g_dkv_q0<DT>, g_dkv_g0<DT>);
    __syncthreads();
    for (int t = first; t < last; t += 2) {
      float lse = n_lse, delta = n_delta;
      if (t + 1 < last) fetch(t + 1, g_dkv_q1<DT>, g_dkv_g1<DT>);
      use(t, lse, delta, (const lds_u8*)&g_dkv_q0<DT>[0], (const lds_u8*)&g_dkv_g0<DT>[0]);
      __syncthreads();
      if (t + 1 >= last) break;
      lse = n_lse, delta = n_delta;
      if (t + 2 < last) fetch(t + 2, g_dkv_q0<DT>, g_dkv_g0<DT>);
      use(t + 1, lse, delta, (const lds_u8*)&g_dkv_q1<DT>[0], (const lds_u8*)&g_dkv_g1<DT>[0]);
      __syncthreads();
    }
  }
  // (the tiles are done with: the last barrier is behind every wave's reads)
  lds_f32* sum_k = (lds_f32*)((wave & 1) ? &g_dkv_q1<DT>[0] : &g_dkv_q0<DT>[0]);
  lds_f32* sum_v = (lds_f32*)((wave & 1) ? &g_dkv_g1<DT>[0] : &g_dkv_g0<DT>[0]);
  if (n == 1) {
#pragma unroll
    for (int db = 0; db < DT / 32; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        sum_k[(16 * db + i) * 64 + lane] = dk[db][i];
        sum_v[(16 * db + i) * 64 + lane] = dv[db][i];
      }
  }
  __syncthreads();
  if (n == 1) return;
#pragma unroll
  for (int db = 0; db < DT / 32; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      dk[db][i] += sum_k[(16 * db + i) * 64 + lane];
      dv[db][i] += sum_v[(16 * db + i) * 64 + lane];
    }
  const int64_t row = (static_cast<int64_t>(s.k0 + key) * a.Hk + hk) * a.D;
  const bool fine = all_finite<DT>(dk) && all_finite<DT>(dv);
  const bool bad = inside && half_sum(fine ? 0.0f : 1.0f) != 0.0f;
  const int64_t all = static_cast<int64_t>(a.S) * a.Hk * a.D;
  float* part = args.part + 2 * split * all + row;
  auto store = [&](const f32x16 (&x)[DT / 32], float* to_part, uint16_t* to, float r) {
    if (args.splits == 1) {
      store_rows<kBF16, DT>(to + row, x, r, a.D, half);
      return;
    }
#pragma unroll
    for (int db = 0; db < DT / 32; ++db)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int d = 32 * db + acc_row(i, half);
        if (d < a.D) *reinterpret_cast<f32x4*>(to_part + d) = f32x4{x[db][i], x[db][i + 1], x[db][i + 2], x[db][i + 3]} * r;
      }
  };
  if (inside && !bad) {
    store(dk, part, args.dk, args.scale * exp2f(-shift));
    store(dv, part + all, args.dv, exp2f(kBF16 ? 0.0f : -kWeightShift));
  }
  if (__builtin_expect(__ballot(bad) == 0, 1)) return;
  // (the other wave of these keys is done, and this one with its sums)
  landed();
  const lds_u8* vt = (const lds_u8*)&g_dkv_v<DT>[0] + 32 * (wave & 1) * (DT * 2);
  uint8_t *const qroom = (wave & 1) ? g_dkv_q1<DT> : g_dkv_q0<DT>, *const groom = (wave & 1) ? g_dkv_g1<DT> : g_dkv_g0<DT>;
  exact_dkv<kBF16, DT, false>(dv, args, s, hk, kf, kw, bad, t0, nt, first, last, vt, qroom, groom, late_lane());
  if (bad) store(dv, part + all, args.dv, 1.0f);
  exact_dkv<kBF16, DT, true>(dk, args, s, hk, kf, kw, bad, t0, nt, first, last, vt, qroom, groom, late_lane());
  if (bad) store(dk, part, args.dk, args.scale);
}

// The splits' sums of dk and dv, 4 values a thread.
template <bool kBF16>
__global__ __launch_bounds__(256) void attn_dkv_join_kernel(BackArgs args, int64_t all) {
  const int64_t at = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
  if (at >= 2 * all) return;
  f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int split = 0; split < args.splits; ++split) x += *reinterpret_cast<const f32x4*>(args.part + 2 * split * all + at);
  *reinterpret_cast<u32x2*>((at < all ? args.dk + at : args.dv + (at - all))) =
      u32x2{pack16<kBF16>(x[0], x[1]), pack16<kBF16>(x[2], x[3])};
}

template <bool kBF16, int DT>
int launch(const BackArgs& a, hipStream_t st) {
  const int64_t qs = slots_of(a.f.cu_q, a.f.B, a.f.T, a.f.G.d, 128), ks = slots_of(a.f.cu_k, a.f.B, a.f.S, 1, 64);
  GPTQ_REQUIRE(qs * a.f.Hk < (int64_t{1} << 31) && ks * a.f.Hk * a.splits < (int64_t{1} << 31), GPTQ_ERR_SHAPE,
               "gptq_attention_backward: too many rows");
  if constexpr (!kBF16) {
    attn_delta_kernel<<<kMaxima, 256, 0, st>>>(a);
    const int rc = check_launch("gptq_attention_backward");
    if (rc != GPTQ_OK) return rc;
  }
  if (a.f.T > 0)
    attn_dq_kernel<kBF16, DT><<<static_cast<uint32_t>(qs * a.f.Hk), 256, 0, st>>>(a, static_cast<int>(qs));
  int rc = check_launch("gptq_attention_backward");
  if (rc != GPTQ_OK) return rc;
  if (a.f.S > 0) {
    attn_dkv_kernel<kBF16, DT><<<static_cast<uint32_t>(ks * a.f.Hk * a.splits), 256, 0, st>>>(a);
    if (a.splits > 1) {
      rc = check_launch("gptq_attention_backward");
      if (rc != GPTQ_OK) return rc;
      const int64_t all = static_cast<int64_t>(a.f.S) * a.f.Hk * a.f.D;
      attn_dkv_join_kernel<kBF16><<<static_cast<uint32_t>(cdiv(2 * all, 1024)), 256, 0, st>>>(a, all);
    }
  }
  return check_launch("gptq_attention_backward");
}

}  // namespace
}  // namespace gptq

using namespace gptq;

extern "C" size_t gptq_attention_backward_workspace_size(int64_t B, int64_t T, int64_t S, int64_t H, int64_t Hk,
                                                         int64_t D) {
  return plan::backward_workspace(B, T, S, H, Hk, D);
}

extern "C" int gptq_attention_backward(const void* grad, const void* q, const void* k, const void* v, const void* out,
                                       const void* out_rest, const float* lse, int dtype, int64_t g_token, int64_t g_head, int64_t q_token,
                                       int64_t q_head, int64_t k_token, int64_t k_head, int64_t v_token, int64_t v_head,
                                       const int32_t* cu_q, const int32_t* cu_k, int64_t B, int64_t T, int64_t S,
                                       int64_t H, int64_t Hk, int64_t D, int causal, float scale, void* dq, void* dk,
                                       void* dv, void* workspace, size_t workspace_bytes, gptq_stream_t stream) {
  clear_error();
  int rc = plan::check_attention_args("gptq_attention_backward", dtype, B, T, S, H, Hk, D, scale);
  if (rc != GPTQ_OK) return rc;
  if (T == 0 && S == 0) return GPTQ_OK;
  GPTQ_REQUIRE((T == 0 || (grad && q && out && out_rest && lse && dq)) && (S == 0 || (k && v && dk && dv)), GPTQ_ERR_ARG,
               "gptq_attention_backward: null pointer");
  GPTQ_REQUIRE(B == 1 || (cu_q && cu_k), GPTQ_ERR_ARG,
               "gptq_attention_backward: %lld sequences without their offsets", static_cast<long long>(B));
  const int64_t strides[] = {g_token, q_token, k_token, v_token, g_head, q_head, k_head, v_head};
  rc = plan::check_attention_layout("gptq_attention_backward", q, k, v, strides, 4, 8);
  if (rc != GPTQ_OK) return rc;
  rc = plan::check_attention_layout("gptq_attention_backward", grad, out, out_rest, nullptr, 0, 0);
  if (rc != GPTQ_OK) return rc;
  const size_t need = plan::backward_workspace(B, T, S, H, Hk, D);
  GPTQ_REQUIRE(workspace && workspace_bytes >= need, GPTQ_ERR_WORKSPACE,
               "gptq_attention_backward: workspace of %zu bytes, needs %zu", workspace_bytes, need);
  BackArgs a{};
  a.f.q = {static_cast<const uint16_t*>(q), q_token, q_head};
  a.f.k = {static_cast<const uint16_t*>(k), k_token, k_head};
  a.f.v = {static_cast<const uint16_t*>(v), v_token, v_head};
  a.g = {static_cast<const uint16_t*>(grad), g_token, g_head};
  a.o = static_cast<const uint16_t*>(out);
  a.o_rest = static_cast<const uint16_t*>(out_rest);
  a.f.lse = const_cast<float*>(lse);
  a.f.cu_q = cu_q;
  a.f.cu_k = cu_k;
  a.f.B = static_cast<int>(B), a.f.T = static_cast<int>(T), a.f.S = static_cast<int>(S);
  a.f.H = static_cast<int>(H), a.f.Hk = static_cast<int>(Hk), a.f.D = static_cast<int>(D);
  a.f.G = fast_div(static_cast<uint32_t>(H / Hk));
  a.f.causal = causal != 0;
  a.f.c = scale * kLog2e;
  a.scale = scale;
  a.f.splits = 1;
  a.maxima = static_cast<float*>(workspace);
  a.delta = a.maxima + 2 * kMaxima;
  a.part = a.delta + plan::ceil_div(T * H, 4) * 4;
  a.splits = plan::backward_splits(B, S, Hk);
  a.dq = static_cast<uint16_t*>(dq);
  a.dk = static_cast<uint16_t*>(dk);
  a.dv = static_cast<uint16_t*>(dv);
  const bool wide = D > 64;
  const hipStream_t st = as_hip(stream);
  if (dtype == GPTQ_BF16) return wide ? launch<true, 128>(a, st) : launch<true, 64>(a, st);
  return wide ? launch<false, 128>(a, st) : launch<false, 64>(a, st);
}
