// Host-side checks of the attention calls' planning code (csrc/plan.cpp), built
// with g++ under AddressSanitizer and UndefinedBehaviorSanitizer by
// tests/test_attention_plan.py.  No GPU, no HIP.  It walks the plans, workspace
// queries and argument checks over zero, the smallest and the largest sizes,
// checks the properties each must have, and prints every query's result as
// "name args = value".  Exit status 0 = every check held.
#include <cinttypes>
#include <cmath>
#include <cstdio>
#include <initializer_list>

#include "../../distributed_gptq_amd/csrc/plan.hpp"

using namespace gptq;

static int g_fail = 0;
#define CHECK(cond, ...)                                  \
  do {                                                    \
    if (!(cond)) {                                        \
      std::fprintf(stderr, "FAIL %s:%d: ", __FILE__, __LINE__); \
      std::fprintf(stderr, __VA_ARGS__);                  \
      std::fprintf(stderr, "\n");                         \
      ++g_fail;                                           \
    }                                                     \
  } while (0)

static const int64_t kTokens[] = {0, 1, 2, 31, 32, 33, 513, 4096, 100000, (int64_t{1} << 31) - 4097, int64_t{1} << 31,
                                  int64_t{1} << 62, INT64_MAX, -1};
static const int64_t kBatches[] = {0, 1, 2, 24, 4096, (int64_t{1} << 31) - 4097, int64_t{1} << 40, INT64_MAX, -1};
static const int64_t kHeads[][2] = {{1, 1}, {32, 8}, {40, 40}, {65536, 1}, {65536, 65536}, {4, 3}, {0, 1}, {1, 0}};
static const int64_t kDims[] = {8, 64, 128, 0, 12, 136};
static const int64_t kContext[] = {0, 1, 127, 128, 8192, int64_t{1} << 31, INT64_MAX, -5};

static void paged_checks() {
  for (int64_t B : kBatches)
    for (int64_t T : kTokens)
      for (const auto& h : kHeads)
        for (int64_t n : kContext) {
          const plan::PagedPlan p = plan::paged_plan(B, T, h[0], h[1], n);
          CHECK(p.splits >= 1 && p.splits <= 128, "splits(B=%" PRId64 ", T=%" PRId64 ") = %d", B, T, p.splits);
          CHECK(n > 128 || p.splits == 1, "a context of %" PRId64 " in %d parts", n, p.splits);
          for (int64_t D : kDims) {
            const size_t ws = gptq_paged_attention_workspace_size(B, T, h[0], h[1], D, n);
            std::printf("gptq_paged_attention_workspace_size %" PRId64 " %" PRId64 " %" PRId64 " %" PRId64 " %" PRId64
                        " %" PRId64 " = %zu\n", B, T, h[0], h[1], D, n, ws);
            const bool sized = plan::check_attention_args("check", GPTQ_F16, B, T, 0, h[0], h[1], D, 1.0f) == GPTQ_OK;
            CHECK(ws == (sized && p.splits > 1 ? static_cast<size_t>(T * h[0]) * (D + 2) * 4 * p.splits : 0),
                  "workspace(B=%" PRId64 ", T=%" PRId64 ", D=%" PRId64 ") = %zu", B, T, D, ws);
            CHECK(T != 0 || ws == 0, "a workspace for no tokens");
          }
        }
}

static void backward_checks() {
  for (int64_t B : kBatches)
    for (int64_t T : kTokens)
      for (int64_t S : kTokens)
        for (const auto& h : kHeads)
          for (int64_t D : kDims) {
            const size_t ws = gptq_attention_backward_workspace_size(B, T, S, h[0], h[1], D);
            std::printf("gptq_attention_backward_workspace_size %" PRId64 " %" PRId64 " %" PRId64 " %" PRId64 " %" PRId64
                        " %" PRId64 " = %zu\n", B, T, S, h[0], h[1], D, ws);
            if (plan::check_attention_args("check", GPTQ_F16, B, T, S, h[0], h[1], D, 1.0f) != GPTQ_OK) {
              CHECK(ws == 0, "a workspace for refused sizes");
              continue;
            }
            const int splits = plan::backward_splits(B, S, h[1]);
            CHECK(splits >= 1 && splits <= 8, "backward_splits(%" PRId64 ", %" PRId64 ") = %d", B, S, splits);
            const size_t part = splits > 1 ? static_cast<size_t>(2 * splits) * S * h[1] * D : 0;
            CHECK(ws == 4 * (static_cast<size_t>((T * h[0] + 3) / 4 * 4) + part + 2 * plan::kBackMaxima),
                  "backward workspace(B=%" PRId64 ", T=%" PRId64 ", S=%" PRId64 ") = %zu", B, T, S, ws);
          }
}

static void argument_checks() {
  for (int64_t width : kTokens)
    for (int64_t page : kTokens) {
      const int64_t most = plan::cached_most(width, page);
      CHECK(most >= 0 && most <= (int64_t{1} << 31) - 4096, "cached_most(%" PRId64 ", %" PRId64 ") = %" PRId64, width, page,
            most);
      if (width > 0 && width < 1000000 && page > 0 && page < 1000)
        CHECK(most == width * page, "cached_most(%" PRId64 ", %" PRId64 ") = %" PRId64, width, page, most);
    }
  for (float scale : {0.0f, -1.0f, 1e-8f, 1e8f, static_cast<float>(NAN), static_cast<float>(INFINITY)})
    CHECK(plan::check_attention_args("check", GPTQ_F16, 1, 1, 1, 1, 1, 64, scale) == GPTQ_ERR_ARG, "scale %g", scale);
  CHECK(plan::check_attention_args("check", GPTQ_F32, 1, 1, 1, 1, 1, 64, 1.0f) == GPTQ_ERR_DTYPE, "fp32 passes");
  const void* at = reinterpret_cast<const void*>(uintptr_t{64});
  const void* odd = reinterpret_cast<const void*>(uintptr_t{72});
  for (int64_t st : {int64_t{0}, int64_t{8}, (int64_t{1} << 28) - 8, int64_t{4}, int64_t{-8}, int64_t{1} << 28}) {
    const bool token = st >= 0 && st % 8 == 0 && st < (int64_t{1} << 28), head = st >= 0 && st % 8 == 0;
    const int64_t first[] = {st, 64}, second[] = {64, st};
    CHECK((plan::check_attention_layout("check", at, at, at, first, 1, 2) == GPTQ_OK) == token, "token stride %" PRId64, st);
    CHECK((plan::check_attention_layout("check", at, at, at, second, 1, 2) == GPTQ_OK) == head, "head stride %" PRId64, st);
  }
  CHECK(plan::check_attention_layout("check", at, odd, at, nullptr, 0, 0) == GPTQ_ERR_ARG, "odd pointer passes");
}

// (the entry points of the workspace queries are in the kernels' files)
extern "C" size_t gptq_paged_attention_workspace_size(int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t D,
                                                      int64_t max_context) {
  return plan::paged_workspace(B, T, H, Hk, D, max_context);
}
extern "C" size_t gptq_attention_backward_workspace_size(int64_t B, int64_t T, int64_t S, int64_t H, int64_t Hk,
                                                         int64_t D) {
  return plan::backward_workspace(B, T, S, H, Hk, D);
}

int main() {
  paged_checks();
  backward_checks();
  argument_checks();
  std::fprintf(stderr, "%d check(s) failed\n", g_fail);
  return g_fail ? 1 : 0;
}
