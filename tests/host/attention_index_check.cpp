// Host-side checks of the attention kernels' index arithmetic
// (csrc/attn_index.hpp), built with g++ under AddressSanitizer and
// UndefinedBehaviorSanitizer by tests/test_attention_plan.py.  No GPU, no HIP.
// Offsets, lengths and page numbers of every kind, those that no caller should
// give too: no row outside the tensors is named, and with proper offsets every
// row is in one workgroup.  Exit status 0 = every check held.
#include <cinttypes>
#include <cstdio>
#include <initializer_list>
#include <random>
#include <vector>

#include "../../distributed_gptq_amd/csrc/attn_index.hpp"

using namespace gptq;

static int g_fail = 0;
static int64_t g_done = 0;
#define CHECK(cond, ...)                                                            \
  do {                                                                              \
    ++g_done;                                                                       \
    if (!(cond) && ++g_fail < 20) {                                                 \
      std::fprintf(stderr, "FAIL %s:%d: ", __FILE__, __LINE__);                     \
      std::fprintf(stderr, __VA_ARGS__);                                            \
      std::fprintf(stderr, "\n");                                                   \
    }                                                                               \
  } while (0)

constexpr int kInt = INT32_MAX;

// what the kernels do with one slot of a grid over the queries (per rows a
// token) or, with per = 0, over the keys
template <bool kPaged>
static void slot_checks(const AttnArgs& a, int per, int R, int64_t slot, std::vector<int>* seen) {
  int tile;
  const bool keys = per == 0;
  const int total = keys ? a.S : a.T, rows_a_token = keys ? 1 : per;
  const int b = find_seq(keys ? a.cu_k : a.cu_q, a.B, total, rows_a_token, R, static_cast<int>(slot), &tile);
  CHECK(b >= 0 && b <= a.B && (b < a.B || (keys ? a.cu_k : a.cu_q)), "sequence %d", b);
  CHECK(tile >= 0 && static_cast<int64_t>(tile) * R <= static_cast<int64_t>(total) * rows_a_token, "tile %d of %d", tile, R);
  Seq s = seq_of<kPaged>(a, b);
  CHECK(s.q0 >= 0 && s.Lq >= 0 && static_cast<int64_t>(s.q0) + s.Lq <= a.T, "queries %d + %d of %d", s.q0, s.Lq, a.T);
  CHECK(s.Lk >= 0 && s.k0 >= 0, "keys %d + %d", s.k0, s.Lk);
  if (kPaged)
    CHECK(s.Lk <= a.paged.most, "context %d of %d", s.Lk, a.paged.most);
  else
    CHECK(static_cast<int64_t>(s.k0) + s.Lk <= a.S, "keys %d + %d of %d", s.k0, s.Lk, a.S);
  if (keys && b == a.B) s.Lk = a.S - s.k0, s.Lq = 0;
  const int rows = keys ? s.Lk : s.Lq * rows_a_token;
  if (tile * R >= rows) return;
  for (int r = tile * R; r < tile * R + R; ++r) {
    const bool inside = r < rows;
    if (keys) {
      if (inside && seen) ++(*seen)[s.k0 + r];
      continue;
    }
    const int tok = div_by(inside ? r : rows - 1, a.G);
    CHECK(tok == (inside ? r : rows - 1) / static_cast<int>(a.G.d) && tok < s.Lq, "token %d of %d", tok, s.Lq);
    if (inside && seen) ++(*seen)[(static_cast<int64_t>(s.q0) + tok) * per + r % per];
    const int limit = last_key(a, s, tok);
    CHECK(limit < s.Lk, "last key %d of %d", limit, s.Lk);
    CHECK(static_cast<int64_t>(limit) == (a.causal ? static_cast<int64_t>(tok) + s.Lk - s.Lq : static_cast<int64_t>(s.Lk) - 1) ||
              s.Lk == 0, "last key %d", limit);
    if (kPaged && seen == nullptr) continue;
    for (int key : {0, limit / 2, limit}) {
      if (key < 0 || key > limit) continue;
      const KvAt at = kv_at<kPaged>(a, s, key);  // (reads the table, under the sanitizer)
      if (kPaged)
        CHECK(at.page >= 0 && at.page < a.paged.pages && at.at == key % static_cast<int>(a.paged.page.d), "page %d", at.page);
      else
        CHECK(at.at >= 0 && at.at < a.S, "row %d of %d", at.at, a.S);
    }
  }
}

static AttnArgs sizes(int B, int T, int S, int G) {
  AttnArgs a{};
  a.B = B, a.T = T, a.S = S, a.G = fast_div(G), a.causal = 1;
  a.splits = 1;
  return a;
}

static void proper_checks() {
  std::mt19937 rng(1);
  for (int round = 0; round < 300; ++round) {
    const int B = 1 + rng() % 6, G = 1 + rng() % 5, R = std::initializer_list<int>{32, 64, 128}.begin()[rng() % 3];
    std::vector<int32_t> cq{0}, ck{0};
    for (int b = 0; b < B; ++b) {
      cq.push_back(cq.back() + (rng() % 4 ? rng() % 300 : 0));
      ck.push_back(ck.back() + (rng() % 4 ? rng() % 300 : 0));
    }
    AttnArgs a = sizes(B, cq.back() + rng() % 3 * 70, ck.back() + rng() % 3 * 70, G);
    a.cu_q = cq.data(), a.cu_k = ck.data();
    a.causal = rng() % 2;
    std::vector<int> seen(static_cast<size_t>(a.T) * G);
    for (int64_t slot = 0; slot < slots_of(a.cu_q, B, a.T, G, R); ++slot) slot_checks<false>(a, G, R, slot, &seen);
    for (int n : seen) CHECK(n == 1, "a row in %d workgroups", n);
    std::vector<int> keys(a.S);
    for (int64_t slot = 0; slot < slots_of(a.cu_k, B, a.S, 1, 64); ++slot) slot_checks<false>(a, 0, 64, slot, &keys);
    for (int n : keys) CHECK(n == 1, "a key in %d workgroups", n);
  }
}

static void hostile_checks() {
  const int32_t odd[] = {INT32_MIN, -1, 0, 5, 70, 129, 130, kInt};
  std::vector<int32_t> cq(4), ck(4);
  for (int B = 1; B <= 3; ++B)
    for (int x = 0; x < 8 * 8 * 8 * 8; ++x) {
      cq.assign(B + 1, 0), ck.assign(B + 1, 0);  // (exact sizes: reads past them are seen)
      for (int b = 0; b <= B; ++b) cq[b] = odd[x >> (3 * b) & 7], ck[b] = odd[x >> (3 * ((b + 1) % 4)) & 7];
      AttnArgs a = sizes(B, 129, 130, 3);
      a.cu_q = cq.data(), a.cu_k = ck.data();
      std::vector<int> seen(129 * 3), keys(130);
      for (int64_t slot = 0; slot < slots_of(a.cu_q, B, 129, 3, 32); ++slot) slot_checks<false>(a, 3, 32, slot, &seen);
      for (int64_t slot = 0; slot < slots_of(a.cu_k, B, 130, 1, 64); ++slot) slot_checks<false>(a, 0, 64, slot, &keys);
      // the same offsets with contexts and page numbers of the kind, pages of 24
      std::vector<int32_t> context(B), table(B * 3);
      for (int b = 0; b < B; ++b) context[b] = odd[x >> (3 * b) & 7];
      for (size_t i = 0; i < table.size(); ++i) table[i] = odd[(x + i) & 7];
      a.cu_k = nullptr;
      a.paged.table = table.data(), a.paged.context = context.data(), a.paged.table_stride = 3;
      a.paged.most = 72, a.paged.pages = 7, a.paged.page = fast_div(24);
      for (int R : {32, 128})
        for (int64_t slot = 0; slot < slots_of(a.cu_q, B, 129, 3, R); ++slot) slot_checks<true>(a, 3, R, slot, &seen);
    }
}

static void largest_checks() {
  constexpr int kMost = kInt - 4096;
  std::mt19937 rng(2);
  for (const std::vector<int32_t>& cu : std::initializer_list<std::vector<int32_t>>{
           {0, kMost}, {0, kInt, kInt, kInt}, {0, kMost, 0, kMost}, {0, 1 << 30, 5, INT32_MIN, kMost}, {7, 3, 1 << 29}}) {
    AttnArgs a = sizes(static_cast<int>(cu.size()) - 1, kMost, kMost, 1);
    a.cu_q = a.cu_k = cu.data();
    for (int causal : {0, 1})
      for (int R : {32, 64, 128}) {
        a.causal = causal;
        const int64_t n = slots_of(a.cu_q, a.B, a.T, 1, R);
        for (int i = 0; i < 300; ++i) {
          const int64_t slot = i < 20 ? i : i < 40 ? n - 1 - (i - 20) : static_cast<int64_t>(rng()) % n;
          slot_checks<false>(a, 1, R, slot, nullptr);
          slot_checks<false>(a, 0, R, slot, nullptr);
        }
      }
  }
  // one token for each of so many sequences that twice their number passes 31 bits, long contexts
  for (int B : {1 << 30, 1200000000, 2000000000}) {
    AttnArgs a = sizes(B, B, 0, 1);
    const std::vector<int32_t> context(1, kMost);
    a.paged.most = kMost, a.paged.pages = 1, a.paged.page = fast_div(16);
    for (int R : {32, 128}) {
      const int64_t n = slots_of(nullptr, B, B, 1, R);
      for (int i = 0; i < 300; ++i) {
        const int64_t slot = i < 20 ? i : i < 40 ? n - 1 - (i - 20) : static_cast<int64_t>(rng()) % n;
        int tile;
        if (slot >= kInt) continue;
        const int b = find_seq(nullptr, B, B, 1, R, static_cast<int>(slot), &tile);
        CHECK(b >= 0 && b < B && first_row(nullptr, b, B, B) == b && tile >= 0, "sequence %d of %d", b, B);
      }
    }
    // a new token's last key, of the longest context
    for (int i : {0, 1, 4095}) {
      const Seq s{0, 0, 4096, 0, kMost};
      CHECK(last_key(a, s, i) == kMost - 4096 + i, "last key");
    }
  }
  for (uint32_t d : {1u, 2u, 3u, 7u, 24u, 65536u, 0x7FFFFFFFu})
    for (int n : {0, 1, 23, 65535, 1 << 30, kInt})
      CHECK(div_by(n, fast_div(d)) == n / static_cast<int64_t>(d), "%d / %u", n, d);
}

int main() {
  proper_checks();
  hostile_checks();
  largest_checks();
  std::fprintf(stderr, "%" PRId64 " checks, %d check(s) failed\n", g_done, g_fail);
  return g_fail ? 1 : 0;
}
