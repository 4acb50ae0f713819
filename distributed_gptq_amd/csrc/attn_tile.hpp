// What the attention kernels share: 32x32 MFMA tiles fed from swizzled LDS
// rows and direct-to-LDS copies of key and value rows.
//
// Every product is laid out so that a lane's accumulators belong to one column
// (lane % 32), a query in the forward and dQ kernels, a key in the dK/dV
// kernel: softmax statistics then are one value a lane, and the weights that
// one product leaves in a lane's registers are the next product's operand
// without moving between lanes.  With a 32x32x16 MFMA a lane ends with rows
// 8 (i / 4) + 4 (lane / 32) + i % 4 of its column (i < 16), and as an operand
// it gives 8 values of the contraction; both operands of the second product
// take the contraction in that same order, so the order needs no shuffle.
#pragma once

#include "attn_index.hpp"
#include "common.hpp"
#include "mfma_lds.hpp"

namespace gptq {
namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) uint8_t lds_u8;
typedef __attribute__((address_space(3))) u32x2 lds_u32x2;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) float lds_f32;
typedef __attribute__((address_space(1))) const void gbl_void;

constexpr float kLog2e = 1.4426950408889634f;
// what a running maximum starts from: finite, so that differences with it are
// never NaN, and below every score
constexpr float kLowest = -3.0e38f;

// ---------------------------------------------------------- element types ----
template <bool kBF16>
__device__ __forceinline__ f32x16 mma32(const u32x4& a, const u32x4& b, const f32x16& c) {
  if constexpr (kBF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
}
template <bool kBF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  return kBF16 ? pack_bf16(lo, hi) : pack_f16(lo, hi);
}
template <bool kBF16>
__device__ __forceinline__ float value16(uint16_t b) {
  return kBF16 ? bf16_bits_to_f32(b) : f16_bits_to_f32(b);
}
// the 8 values i0 .. i0 + 7 of a lane's accumulators as an operand
template <bool kBF16>
__device__ __forceinline__ u32x4 operand_of(const f32x16& p, int i0) {
  return u32x4{pack16<kBF16>(p[i0], p[i0 + 1]), pack16<kBF16>(p[i0 + 2], p[i0 + 3]),
               pack16<kBF16>(p[i0 + 4], p[i0 + 5]), pack16<kBF16>(p[i0 + 6], p[i0 + 7])};
}
// and what its rounding left, as an operand too
template <bool kBF16>
__device__ __forceinline__ u32x4 operand_rest(const f32x16& p, int i0, const u32x4& x) {
  u32x4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    r[j] = pack16<kBF16>(p[i0 + 2 * j] - value16<kBF16>(static_cast<uint16_t>(x[j])),
                         p[i0 + 2 * j + 1] - value16<kBF16>(static_cast<uint16_t>(x[j] >> 16)));
  return r;
}
// row of the 32 x 32 result that register i of this lane holds
__device__ __forceinline__ int acc_row(int i, int half) { return 8 * (i >> 2) + 4 * half + (i & 3); }

__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.0f;
  return z;
}

// a column's two lanes, l and l + 32: their values, in both
__device__ __forceinline__ void both_halves(float v, float& low, float& high) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  low = __uint_as_float(r[0]);
  high = __uint_as_float(r[1]);
}
__device__ __forceinline__ float half_max(float v) {
  float a, b;
  both_halves(v, a, b);
  return __builtin_elementwise_maximum(a, b);
}
__device__ __forceinline__ float half_sum(float v) {
  float a, b;
  both_halves(v, a, b);
  return a + b;
}

// ------------------------------------------------------------------- LDS ----
// A tile row holds DT 16-bit values in 16-byte chunks, chunk c at slot
// c ^ row_slot(row).  A 128-bit read of 32 rows at one chunk then meets 16
// distinct quads of banks 16 lanes at a time, and a transposing read of 4 rows
// x 32 values 4 distinct rows of quads (the low two bits of the row are the
// slot's high bits).
template <int DT>
__device__ __forceinline__ int row_slot(int row) {
  if constexpr (DT == 128)
    return ((row & 3) << 2) | ((row >> 2) & 3);
  else
    return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
}

// Where a lane reads its operands of a tile.  The offsets are opaque to the
// compiler, so that a read's constant part (the tile and its rows) goes into
// the instruction instead of an addition each.
template <int DT>
struct LaneAt {
  int row[DT / 16];     // values 16 s + 8 (l / 32) .. of row l % 32
  int col[DT / 32][2];  // the rows 8 j + 4 (l / 32) .., for a transposing read
};
template <int DT>
__device__ __forceinline__ LaneAt<DT> lane_at(int lane, int more) {
  LaneAt<DT> at;
  const int h = lane >> 5, r = lane & 31;
#pragma unroll
  for (int s = 0; s < DT / 16; ++s) {
    at.row[s] = more + r * (DT * 2) + (((2 * s + h) ^ row_slot<DT>(r)) << 4);
    asm volatile("" : "+v"(at.row[s]));
  }
  const int i = lane & 15;
#pragma unroll
  for (int db = 0; db < DT / 32; ++db)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int chunk = 4 * db + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
      const int row = 8 * j + 4 * h + (i >> 2);
      at.col[db][j] = more + row * (DT * 2) + ((chunk ^ row_slot<DT>(row)) << 4) + ((i & 1) << 3);
      asm volatile("" : "+v"(at.col[db][j]));
    }
  return at;
}

// Operand of a product over the row's values: lane l gives row l % 32 (+ row0,
// a multiple of 16), values 16 s + 8 (l / 32) .. + 7.
template <int DT>
__device__ __forceinline__ u32x4 row_operand(const lds_u8* tile, int row0, int s, const LaneAt<DT>& at) {
  return *(const lds_u32x4*)(tile + at.row[s] + row0 * (DT * 2));
}

// Operand of a product over the rows (the transposed tile): lane l gives value
// 32 db + l % 32 of the rows row0 + 8 j + 4 (l / 32) + 0 .. 3, j = 0, 1.  A
// transposing read takes from 16 lanes the addresses of 4 rows x 16 values, 4
// values a lane, and gives lane i the 4 rows' value i.
template <int DT>
__device__ __forceinline__ u32x4 column_operand(const lds_u8* tile, int row0, int db, const LaneAt<DT>& at) {
  s16x4 v[2];
#pragma unroll
  for (int j = 0; j < 2; ++j)
    v[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tile + at.col[db][j] + row0 * (DT * 2)));
  return __builtin_bit_cast(u32x4, __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7));
}

// The lane's query row as an operand over its channels: zeros past D and for
// rows outside the tile.
template <int DT>
__device__ __forceinline__ void load_query(u32x4 (&q)[DT / 16], const uint16_t* row, bool inside, int D, int half) {
#pragma unroll
  for (int s = 0; s < DT / 16; ++s) {
    const int d = 16 * s + 8 * half;
    q[s] = inside && d < D ? *reinterpret_cast<const u32x4*>(row + d) : u32x4{0, 0, 0, 0};
  }
}

// The lane for a path taken seldom: what follows from it is computed there, and
// not kept in registers until then.
__device__ __forceinline__ int late_lane() {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));
  return lane;
}

// One wave's own copies into LDS have landed, and its reads of LDS are done.
__device__ __forceinline__ void landed() {
  wait_vm<0>();
  wait_lgkm<0>();
  wave_sync();
}

// sums += weights x rows of a tile of 32 rows, row by row and only those that
// the lane's column sees: a product of the tile multiplies the zero weights of
// the others with what they hold, and zero times an infinity is no term of a
// sum.  weights: 32 floats for each row, in LDS.
template <bool kBF16, int DT, class Sees>
__device__ __forceinline__ void add_seen_rows(f32x16 (&sums)[DT / 32], const lds_f32* weights, const lds_u8* tile, int lane,
                                              Sees&& sees) {
  const int half = lane >> 5;
#pragma unroll 1
  for (int r = 0; r < 32; ++r) {
    const float w = weights[r * 32 + (lane & 31)];
    const bool in = sees(r);
#pragma unroll
    for (int db = 0; db < DT / 32; ++db) {
      __builtin_amdgcn_sched_barrier(0);  // (all values at once would take as many registers as the sums)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const u32x2 x = *(const lds_u32x2*)(tile + r * (DT * 2) + (((4 * db + j) ^ row_slot<DT>(r)) << 4) + 8 * half);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float sum = sums[db][4 * j + e];
          const float y = fmaf(w, value16<kBF16>(static_cast<uint16_t>(x[e / 2] >> (16 * (e % 2)))), sum);
          sums[db][4 * j + e] = in ? y : sum;
        }
      }
    }
  }
}
// a column's 16 values of a lane as such weights
__device__ __forceinline__ void store_weights(lds_f32* weights, const f32x16& w, int lane) {
#pragma unroll
  for (int i = 0; i < 16; ++i) weights[acc_row(i, lane >> 5) * 32 + (lane & 31)] = w[i];
}

// The order of a run of N pairs of an LDS read and an MFMA (two pairs of them at
// a time): kAhead reads first, so that no MFMA waits for a read just issued.
template <int N, int kAhead>
__device__ __forceinline__ void reads_ahead() {
  __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
  sfor<0, (N - kAhead) / 2>([](auto) {
    __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
  });
  __builtin_amdgcn_sched_group_barrier(0x008, kAhead, 0);
}

// 16 bytes per lane from memory to LDS, lane l's at lds + 16 l.
__device__ __forceinline__ void copy16_to_lds(const void* from, uint8_t* lds) {
  __builtin_amdgcn_global_load_lds((gbl_void*)from, (lds_void*)lds, 16, 0, 0);
}

// what the copies of rows and channels outside the tensors read
__device__ const uint32_t g_attn_zeros[4] = {0, 0, 0, 0};

// ----------------------------------------------------------------- copies ----
// Copies N consecutive rows of DT values, all of them valid and the first at
// the (wave-uniform) `row`, to rows slot0 .. of a tile.  The lanes differ by 32
// bits of offset only: the address arithmetic of a tile is scalar.
template <int DT, int N>
__device__ __forceinline__ void copy_rows(const uint16_t* row, int64_t st, uint8_t* tile, int slot0, int lane) {
  constexpr int CH = DT / 8, RPI = 64 / CH;
  const uint8_t* base = reinterpret_cast<const uint8_t*>(uniform_u64(reinterpret_cast<uint64_t>(row)));
  const uint32_t step = static_cast<uint32_t>(st * 2);
#pragma unroll
  for (int x = 0; x < N / RPI; ++x) {
    const int i = x * RPI + lane / CH;
    const uint32_t off = (lane / CH) * step + (((lane % CH) ^ row_slot<DT>(i)) << 4);
    copy16_to_lds(base + static_cast<int64_t>(x * RPI) * (st * 2) + off, tile + (slot0 / RPI + x) * 1024);
  }
}

// Copies a wave's W consecutive rows of a tile (the first of them row `row0` of
// the tile, a multiple of 16) into LDS: keys and values, zeros past the
// sequence's end and past D.  `mine` is where the row of lane % W is.
template <int DT, int W, bool kPaged>
__device__ __forceinline__ void fetch_rows(const AttnArgs& a, const Seq& s, int hk, KvAt mine, int key0, int row0,
                                           uint8_t* kt, uint8_t* vt, int lane) {
  constexpr int CH = DT / 8, RPI = 64 / CH;
  const int first = key0 + row0;
  if (first + W <= s.Lk && a.D == DT && (!kPaged || a.paged.whole)) {
    constexpr int N = kPaged ? 16 : W;  // 16 rows from a multiple of 16 on are in one page
#pragma unroll
    for (int h = 0; h < W; h += N) {
      KvAt u{0, s.k0 + first};
      if constexpr (kPaged) u = KvAt{__builtin_amdgcn_readlane(mine.page, h), __builtin_amdgcn_readlane(mine.at, h)};
      copy_rows<DT, N>(kv_row<kPaged>(a.k, a.paged.k_page, hk, u), a.k.st, kt, row0 + h, lane);
      copy_rows<DT, N>(kv_row<kPaged>(a.v, a.paged.v_page, hk, u), a.v.st, vt, row0 + h, lane);
    }
    return;
  }
#pragma unroll
  for (int x = 0; x < W / RPI; ++x) {
    const int i = x * RPI + lane / CH, row = row0 + i;
    KvAt at = mine;
    if constexpr (kPaged) {
      at.page = __shfl(mine.page, i);
      at.at = __shfl(mine.at, i);
    } else {
      at.at = mine.at - lane % W + i;
    }
    const int ch = (lane % CH) ^ row_slot<DT>(row);
    const bool in = key0 + row < s.Lk && ch * 8 < a.D;
    const uint16_t* kp = kv_row<kPaged>(a.k, a.paged.k_page, hk, at) + ch * 8;
    const uint16_t* vp = kv_row<kPaged>(a.v, a.paged.v_page, hk, at) + ch * 8;
    copy16_to_lds(in ? static_cast<const void*>(kp) : g_attn_zeros, kt + (row0 / RPI + x) * 1024);
    copy16_to_lds(in ? static_cast<const void*>(vp) : g_attn_zeros, vt + (row0 / RPI + x) * 1024);
  }
}

// kv_at of a key that may lie past the end (in a cache then the last one's)
template <bool kPaged>
__device__ __forceinline__ KvAt kv_at_clamped(const AttnArgs& a, const Seq& s, int key) {
  if constexpr (!kPaged) return kv_at<kPaged>(a, s, key);
  if (s.Lk == 0) return KvAt{0, 0};  // (no copy uses it)
  return kv_at<kPaged>(a, s, clamp_int(key, 0, s.Lk - 1));
}

}  // namespace
}  // namespace gptq
