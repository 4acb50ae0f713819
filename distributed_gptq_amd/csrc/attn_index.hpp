// Which rows the attention kernels' workgroups have, and where keys are: the
// sequences of packed rows, the slots of the grid, the causal mask's bounds and
// the pages of a cache.  Integer functions only, so that a CPU build checks them
// with whatever the device arrays may hold.
#pragma once

#include <cstdint>

#ifdef __HIP__
#include <hip/hip_runtime.h>
#define GPTQ_INDEX __device__ __forceinline__
#else
#define GPTQ_INDEX inline
#endif

namespace gptq {
namespace {

// v of a wave's lanes that all have the same, as a scalar
GPTQ_INDEX int uniform_int(int v) {
#ifdef __HIP_DEVICE_COMPILE__
  v = __builtin_amdgcn_readfirstlane(v);
#endif
  return v;
}

// ------------------------------------------------------------ division ----
// n / d for 0 <= n < 2^31 by a product: m = ceil(2^(31 + s) / d) with
// s = ceil(log2 d) (Granlund and Montgomery, "Division by invariant integers
// using multiplication")
struct FastDiv {
  uint32_t d, m, shift;
};
inline FastDiv fast_div(uint32_t d) {
  uint32_t s = 0;
  while ((uint64_t{1} << s) < d) ++s;
  return FastDiv{d, static_cast<uint32_t>(((uint64_t{1} << (31 + s)) + d - 1) / d), 31 + s};
}
GPTQ_INDEX int div_by(int n, const FastDiv& f) {
  return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * f.m) >> f.shift);
}

// ------------------------------------------------------------ the problem ----
struct Rows16 {            // 16-bit rows of (token, head)
  const uint16_t* p;
  int64_t st, sh;          // strides of a token and of a head, in elements
};

struct Paged {
  const int32_t* table;    // (B, width) page numbers
  const int32_t* context;  // (B) cached tokens of each sequence
  int64_t table_stride, k_page, v_page;  // elements
  int most, pages;         // tokens that a table row reaches; pages of the cache
  FastDiv page;            // tokens of a page
  int whole;               // whether pages hold whole 16s of tokens
};

struct AttnArgs {
  Rows16 q, k, v;
  Paged paged;
  const int32_t* cu_q;     // (B + 1) offsets, or null: B equal lengths
  const int32_t* cu_k;
  int B, T, S;             // sequences, packed queries, packed keys
  int H, Hk, D;
  FastDiv G;               // query heads of a key head
  int causal;
  float c;                 // scale * log2(e)
  uint16_t* out;           // (T, H, D)
  uint16_t* out_rest;      // (T, H, D): what the rounding of out left, for the gradient (or null)
  float* lse;              // (T, H) or null: log2 of the sum of 2^(c q k)
  float* part;             // with splits > 1: sums (splits, T H, D), then maxima, then sums of weights (splits, T H)
  int splits;
};

// One sequence: its queries and keys.
struct Seq {
  int b, q0, Lq, k0, Lk;
};

GPTQ_INDEX int clamp_int(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

// The first of sequence b's rows among `total`, those of B sequences.  Without
// offsets the sequences are equally long (one sequence, or one token each).
// With them the first is 0, rows past the last one are a sequence B of their
// own (whose outputs are zeros), and offsets outside the tensor are clamped:
// the kernels stay inside it.
GPTQ_INDEX int first_row(const int32_t* cu, int b, int B, int total) {
  if (b == 0) return 0;
  if (!cu) return b * (total / B);
  return b > B ? total : clamp_int(uniform_int(cu[b]), 0, total);
}

// The sequence and tile of a slot, when a sequence of rows [r0, r1) takes the
// slots from r0 / R + b on: at least ceil((r1 - r0) / R) of them, whatever the
// lengths, so the host needs no lengths for the grid.  Rows are `per` to a
// token.
GPTQ_INDEX int find_seq(const int32_t* cu, int B, int total, int per, int R, int slot, int* tile) {
  int lo = 0, hi = B + (cu ? 1 : 0), start = 0;
  while (hi - lo > 1) {
    const int mid = lo + ((hi - lo) >> 1);
    const int at = static_cast<int>(static_cast<int64_t>(first_row(cu, mid, B, total)) * per / R) + mid;
    if (at <= slot) {
      lo = mid;
      start = at;
    } else {
      hi = mid;
    }
  }
  *tile = slot - start;
  return lo;
}
// what find_seq's grid needs
inline int64_t slots_of(const int32_t* cu, int64_t B, int64_t total, int64_t per, int64_t R) {
  return total * per / R + B + (cu ? 1 : 0);
}

template <bool kPaged>
GPTQ_INDEX Seq seq_of(const AttnArgs& a, int b) {
  Seq s;
  s.b = b;
  s.q0 = first_row(a.cu_q, b, a.B, a.T);
  const int qe = first_row(a.cu_q, b + 1, a.B, a.T);
  s.Lq = qe > s.q0 ? qe - s.q0 : 0;
  if constexpr (kPaged) {
    s.k0 = 0;
    s.Lk = b == a.B ? 0 : clamp_int(uniform_int(a.paged.context[b]), 0, a.paged.most);
  } else {
    s.k0 = first_row(a.cu_k, b, a.B, a.S);
    const int ke = first_row(a.cu_k, b + 1, a.B, a.S);
    s.Lk = ke > s.k0 ? ke - s.k0 : 0;
    if (b == a.B) s.Lk = 0;
  }
  return s;
}

// the last key that query token i of the sequence sees (-1: none)
GPTQ_INDEX int last_key(const AttnArgs& a, const Seq& s, int i) {
  const int last = a.causal ? i - s.Lq + s.Lk : s.Lk - 1;
  return last < s.Lk ? last : s.Lk - 1;
}

// Where row `key` of a sequence's keys and values is: in the pages of a cache
// (page number and place in it) or in the packed rows.  Page numbers outside
// the cache are clamped.
struct KvAt {
  int page, at;
};
template <bool kPaged>
GPTQ_INDEX KvAt kv_at(const AttnArgs& a, const Seq& s, int key) {
  if constexpr (kPaged) {
    const int n = div_by(key, a.paged.page);
    return KvAt{clamp_int(a.paged.table[s.b * a.paged.table_stride + n], 0, a.paged.pages - 1),
                key - n * static_cast<int>(a.paged.page.d)};
  } else {
    return KvAt{0, s.k0 + key};
  }
}
// The sequence of packed row t of B sequences by their offsets, each thread's own
// row: the last whose offset is not past it, or B for rows behind the last one.
// Offsets that do not ascend give some sequence.
GPTQ_INDEX int sequence_of(const int32_t* cu, int B, int t) {
  if (t >= cu[B]) return B;
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = lo + ((hi - lo) >> 1);
    if (cu[mid] <= t)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}
// Which cached token packed row t is, when a sequence's rows are its last ones:
// -1 where it has none.
GPTQ_INDEX int cached_token(const int32_t* cu, const int32_t* context, int B, int most, int t, int* b) {
  *b = sequence_of(cu, B, t);
  if (*b >= B) return -1;
  const int have = clamp_int(context[*b], 0, most);
  const int64_t key = static_cast<int64_t>(have) - cu[*b + 1] + t;
  return key >= 0 && key < have ? static_cast<int>(key) : -1;
}

template <bool kPaged>
GPTQ_INDEX const uint16_t* kv_row(const Rows16& r, int64_t page_stride, int hk, KvAt k) {
  const uint16_t* p = r.p + hk * r.sh + k.at * r.st;
  if constexpr (kPaged) p += k.page * page_stride;
  return p;
}

}  // namespace
}  // namespace gptq
