// Host-side checks of which cached token a packed row reads back
// (csrc/attn_index.hpp), built with g++ under AddressSanitizer and
// UndefinedBehaviorSanitizer by tests/test_code_host.py.  No GPU, no HIP.
// Offsets and lengths of every kind, those that no caller should give too.
// Exit status 0 = every check held.
#include <cinttypes>
#include <cstdio>
#include <random>
#include <vector>

#include "../../distributed_gptq_amd/csrc/attn_index.hpp"

using namespace gptq;

static int g_fail = 0;
static int64_t g_done = 0;
#define CHECK(cond, ...)                                        \
  do {                                                          \
    ++g_done;                                                   \
    if (!(cond) && ++g_fail < 20) {                             \
      std::fprintf(stderr, "FAIL %s:%d: ", __FILE__, __LINE__); \
      std::fprintf(stderr, __VA_ARGS__);                        \
      std::fprintf(stderr, "\n");                               \
    }                                                           \
  } while (0)

static void proper() {
  std::mt19937 rng(3);
  for (int round = 0; round < 400; ++round) {
    const int B = 1 + rng() % 9;
    std::vector<int32_t> cu{0}, context;
    for (int b = 0; b < B; ++b) {
      const int n = rng() % 3 ? rng() % 40 : 0;
      cu.push_back(cu.back() + n);
      context.push_back(rng() % 4 ? n + rng() % 50 : rng() % 20);  // (fewer cached than rows, too)
    }
    const int T = cu.back() + rng() % 5;
    for (int t = 0; t < T; ++t) {
      int want_b = B;
      for (int b = 0; b < B; ++b)
        if (t >= cu[b] && t < cu[b + 1]) want_b = b;
      int want = -1;
      if (want_b < B) want = context[want_b] - (cu[want_b + 1] - t);
      if (want < 0) want = -1;
      int b;
      const int key = cached_token(cu.data(), context.data(), B, 1 << 20, t, &b);
      CHECK(key == want && (key < 0 || b == want_b), "row %d: token %d of %d, not %d of %d", t, key, b, want, want_b);
    }
  }
}

static void hostile() {
  const int32_t odd[] = {INT32_MIN, -1, 0, 5, 70, 129, 130, INT32_MAX};
  for (int B = 1; B <= 3; ++B)
    for (int x = 0; x < 8 * 8 * 8 * 8; ++x)
      for (int most : {0, 1, 72, INT32_MAX - 4095}) {
        std::vector<int32_t> cu(B + 1), context(B);  // (exact sizes: reads past them are seen)
        for (int b = 0; b <= B; ++b) cu[b] = odd[x >> (3 * b) & 7];
        for (int b = 0; b < B; ++b) context[b] = odd[x >> (3 * ((b + 2) % 4)) & 7];
        for (int t : {0, 1, 69, 70, 128, 129, INT32_MAX - 1}) {
          int b;
          const int key = cached_token(cu.data(), context.data(), B, most, t, &b);
          CHECK(b >= 0 && b <= B && (key == -1 || (b < B && key >= 0 && key < most)), "token %d of sequence %d", key, b);
        }
      }
}

int main() {
  proper();
  hostile();
  std::fprintf(stderr, "%" PRId64 " checks, %d check(s) failed\n", g_done, g_fail);
  return g_fail != 0;
}
