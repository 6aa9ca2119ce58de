// How the norm and rotation lay a call's rows over lanes and workgroups.  Host arithmetic alone: a test compiles it without a GPU.
#pragma once

#include <cstdint>

namespace si {

constexpr int kRotThreads = 256;
constexpr int64_t kRotMostD = 1024;
constexpr int kRotTable = 40 * 1024;  // bytes of LDS for cosines and sines at most

// How a call's rows are laid over lanes and workgroups.
struct RotPlan {
  int vec, cpl, lpr, log_lpr, iters, per, tokens;
  int64_t blocks;
};

inline RotPlan rot_plan(int64_t rows, int64_t H, int64_t D, int64_t pairs, int vec, bool bwd) {
  RotPlan p{};
  p.vec = vec;
  const int64_t n = (D + vec - 1) / vec;  // pieces of a row
  // The fewest lanes of a row that 9 pieces each reach, 5 in the backward (16 from 64 lanes on): longer runs of independent loads.
  // 4,096 tokens, 64 heads, D = 576: forward 112.7 us (5 pieces 117, 3 120), training step 307 (9 pieces 340, 3 331).
  p.log_lpr = 0;
  while ((int64_t{bwd ? 5 : 9} << p.log_lpr) < n && p.log_lpr < 6) ++p.log_lpr;
  while (p.log_lpr < 3 && (int64_t{1} << p.log_lpr) < n) ++p.log_lpr;  // (128 bytes of a row at once)
  // few rows: shorter chains, more workgroups (64 tokens of 64 heads, D = 576: kernel 5.7 us, 7.0 without)
  while (p.log_lpr < 6 && (int64_t{1} << p.log_lpr) < n && rows <= int64_t{512} * (kRotThreads >> p.log_lpr) / 2) ++p.log_lpr;
  // Tokens of k rows that follow each other at most: from a multiple of k rows on, and from any row on (k >= 2).
  auto from_any = [&](int64_t k) { return (k - 2) / H + 2; };
  auto tokens = [&](int64_t k) { return k % H == 0 || H % k == 0 ? (k + H - 1) / H : from_any(k); };
  while (p.log_lpr < 6 && tokens(kRotThreads >> p.log_lpr) * pairs * 8 > kRotTable) ++p.log_lpr;  // (4 rows of 512 pairs fit)
  p.lpr = 1 << p.log_lpr;
  const int64_t cpl = (n + p.lpr - 1) / p.lpr;
  p.cpl = cpl <= 1 ? 1 : cpl <= 2 ? 2 : cpl <= 4 ? 4 : cpl <= 5 ? 5 : cpl <= 9 ? 9 : 16;
  const int64_t groups = kRotThreads / p.lpr, all = (rows + groups - 1) / groups;
  // Backward: at most 512 workgroups, two a CU, whose sums of dw are joined (training step of 4,096 tokens, 64 heads, D = 576: 311 us,
  // 384 workgroups 337, 256 363).  Forward: two groups of rows, so that a weight and a table serve both; 1 / 2 / 4 groups: 137 / 117 /
  // 120 us with a weight at those sizes, 490 / 427 / 454 at 16,384 tokens; without one 108.5 / 112.8 / 119 and 419 / 424 / 456;
  // rotation alone, 24 heads of 128, 100,003 tokens, 229 / 227 / 231 (8: 249), 64 heads of 64 365 / 334 / 333.  One rule for all: it
  // costs wide rows without a weight 1 to 4 %.  (A launch has fewer than 2^24 workgroups.)
  int64_t iters = bwd ? (all + 511) / 512 : all < 4096 ? 1 : 2 + (all >> 24), per;
  per = iters = iters < 1 ? 1 : iters;
  // A filling begins at a multiple of `groups` rows, and of `per` times as many only where `per` divides `iters`.
  auto filled = [&]() { return iters % per == 0 || groups % H == 0 ? tokens(per * groups) : from_any(per * groups); };
  while (per > 1 && filled() * pairs * 8 > kRotTable / 3) per = (per + 1) / 2;
  p.per = static_cast<int>(per);
  p.tokens = static_cast<int>(filled());
  p.iters = static_cast<int>(iters);
  p.blocks = (all + iters - 1) / iters;
  return p;
}

}  // namespace si
