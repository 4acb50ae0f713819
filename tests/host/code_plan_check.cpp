// The plan and workspace of attention over codes, and of the norms' gradient, at
// zero, ordinary, odd and the largest sizes.  Prints what the shipped library has
// to answer too: B T H Hk D context bytes.
#include <cstdint>
#include <cstdio>
#include <initializer_list>

#include "../../distributed_gptq_amd/csrc/plan.hpp"

int main() {
  using namespace gptq::plan;
  int64_t failed = 0, checks = 0;
  auto check = [&](bool ok, const char* what, int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t D, int64_t n) {
    ++checks;
    if (ok) return;
    if (++failed < 20)
      std::fprintf(stderr, "%s: B %lld T %lld H %lld Hk %lld D %lld context %lld\n", what, static_cast<long long>(B),
                   static_cast<long long>(T), static_cast<long long>(H), static_cast<long long>(Hk),
                   static_cast<long long>(D), static_cast<long long>(n));
  };
  const int64_t most = INT64_MAX;
  const int64_t heads[][2] = {{1, 1}, {8, 2}, {32, 8}, {7, 1}, {65536, 1}, {65536, 65536}, {3, 2}, {0, 1}, {1, 0}, {-4, -2}};
  for (const auto& h : heads)
    for (int64_t B : {int64_t{-1}, int64_t{0}, int64_t{1}, int64_t{8}, int64_t{9}, int64_t{100000}, (int64_t{1} << 31) - 5000, most})
      for (int64_t T : {int64_t{-1}, int64_t{0}, int64_t{1}, int64_t{8}, int64_t{9}, int64_t{40}, int64_t{64}, int64_t{65}, int64_t{5000},
                        (int64_t{1} << 31) - 5000, most})
        for (int64_t D : {int64_t{0}, int64_t{16}, int64_t{64}, int64_t{80}, int64_t{128}, int64_t{144}, most})
          for (int64_t n : {-most, int64_t{0}, int64_t{1}, int64_t{129}, int64_t{8192}, int64_t{1} << 31, most}) {
            const int64_t H = h[0], Hk = h[1];
            const CodePlan p = code_plan(B, T, H, Hk, D, n);
            const size_t w = code_workspace(B, T, H, Hk, D, n);
            check(p.rows == 16 || p.rows == 32 || p.rows == 128 || (p.rows == 256 && D > 64), "rows", B, T, H, Hk, D, n);
            check(p.splits >= 1 && p.splits <= 128, "splits", B, T, H, Hk, D, n);
            check(n > 1 || p.splits == 1, "a short context is cut", B, T, H, Hk, D, n);
            check(p.splits > 1 || w == 0, "bytes for nothing", B, T, H, Hk, D, n);
            if (p.splits > 1)
              check(w == static_cast<size_t>(T) * H * (D + 2) * 4 * p.splits, "bytes", B, T, H, Hk, D, n);
            std::printf("%lld %lld %lld %lld %lld %lld %zu\n", static_cast<long long>(B), static_cast<long long>(T),
                        static_cast<long long>(H), static_cast<long long>(Hk), static_cast<long long>(D),
                        static_cast<long long>(n), w);
          }
  std::fprintf(stderr, "%lld checks, %lld check(s) failed\n", static_cast<long long>(checks), static_cast<long long>(failed));
  return failed != 0;
}
