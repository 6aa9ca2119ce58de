"""The plan of the norm and rotation, as the C++ that the library holds, on the CPU: the table of cosines and sines has every
token that the rows of one of its fillings belong to, at every size.

A workgroup takes ``iters`` groups of ``256 / lanes`` rows, and its table is filled anew every ``per`` of them, so filling j of
workgroup b begins at row ``(b iters + j per) 256 / lanes``, which need not be a token's first one.
"""

from __future__ import annotations

import os
import shutil
import subprocess

import pytest

import streamindex_amd

CSRC = os.path.join(os.path.dirname(streamindex_amd.__file__), "csrc")

PROGRAM = r"""
#include <algorithm>
#include <cstdio>
#include <random>

#include "rotary_plan.h"

using namespace si;
typedef int64_t I;

static int bad = 0;
static I refilled = 0;  // plans whose table is filled more than once

static void check(I T, I H, I D, I pairs, int vec, bool bwd) {
  const I rows = T * H;
  const RotPlan p = rot_plan(rows, H, D, pairs, vec, bwd);
  const I g = kRotThreads / p.lpr;
  const char* what = nullptr;
  I at = 0;
  if (p.lpr != 1 << p.log_lpr || p.lpr > 64 || static_cast<I>(p.lpr) * p.cpl * vec < D) what = "lanes that do not reach a row's end";
  if (p.per < 1 || p.per > p.iters || p.blocks * p.iters * g < rows || (p.blocks - 1) * p.iters * g >= rows) what = "rows left out";
  if (p.blocks > 0xffffffffLL / kRotThreads) what = "too many workgroups";
  if (static_cast<I>(p.tokens) * pairs * 8 > kRotTable) what = "table too large";
  refilled += p.per < p.iters;
  // (a workgroup's first row within its token goes round after H of them at most)
  for (I b = 0; !what && b < std::min(p.blocks, H); ++b)
    for (I j = 0; j < p.iters; j += p.per) {
      const I first = (b * p.iters + j) * g, k = std::min<I>(p.per, p.iters - j) * g;
      const I last = std::min(first + k, rows) - 1;
      if (first < rows && last / H - first / H + 1 > p.tokens) {
        what = "tokens that the table does not hold";
        at = first;
        break;
      }
    }
  // The same of the last workgroups, up to the last row.
  for (I b = std::max<I>(p.blocks - 3, 0); !what && b < p.blocks; ++b)
    for (I j = 0; j < p.iters; j += p.per) {
      const I first = (b * p.iters + j) * g, last = std::min(first + std::min<I>(p.per, p.iters - j) * g, rows) - 1;
      if (first < rows && last / H - first / H + 1 > p.tokens) what = "tokens that the table does not hold";
    }
  if (what && ++bad <= 20)
    std::printf("T %lld H %lld D %lld pairs %lld vec %d bwd %d: %s (row %lld; iters %d per %d tokens %d)\n", (long long)T, (long long)H,
                (long long)D, (long long)pairs, vec, bwd, what, (long long)at, p.iters, p.per, p.tokens);
}

int main() {
  const I known[][4] = {{15000, 64, 128, 64}, {12806, 64, 128, 64}, {27405, 64, 576, 32}, {61300, 64, 576, 32}, {14000, 64, 128, 64},
                        {28500, 64, 576, 32}, {60000, 5, 64, 32}, {11000, 6, 128, 64}};
  for (auto& c : known)
    for (int vec = 1; vec <= 8; vec *= 2)
      for (int bwd = 0; bwd < 2; ++bwd) check(c[0], c[1], c[2], c[3], vec, bwd);
  const I heads[] = {1, 2, 3, 4, 5, 6, 7, 8, 12, 16, 24, 32, 40, 48, 64, 96, 100, 128, 1000};
  const I dims[] = {2, 32, 64, 96, 100, 128, 192, 256, 500, 512, 576, 1024};
  std::mt19937_64 rng(1);
  auto below = [&](I n) { return static_cast<I>(rng() % static_cast<uint64_t>(n)); };
  for (I H : heads)
    for (I D : dims)
      for (int k = 0; k < 60; ++k) {
        const I pairs = k % 3 == 0 ? D / 2 : k % 3 == 1 ? std::min<I>(32, D / 2) : below(D / 2 + 1);
        const int vec = D % 8 == 0 && pairs % 8 == 0 ? 1 << below(4) : 1;
        const I T = 1 + below(I{1} << (1 + below(18)));
        check(T, H, D, pairs, vec, false);
        check(T, H, D, pairs, vec, true);
      }
  // far more rows than one launch's workgroups: several groups each in the forward as well
  for (I H : {1, 3, 24, 64, 128})
    for (I D : {64, 128, 576, 1024})
      for (int k = 0; k < 8; ++k) {
        const I T = ((I{1} << 40) >> below(8)) / H - below(1000);
        check(T, H, D, D / 2, 1, false);
        if (k == 0) check(T >> 8, H, D, D / 2, 1, true);
      }
  std::printf("%lld plans fill their table more than once\n", (long long)refilled);
  return bad != 0 || refilled < 100;
}
"""


def test_every_filling_of_the_table_holds_its_rows_tokens(tmp_path):
    cxx = shutil.which("g++") or shutil.which("clang++")
    if cxx is None:
        pytest.skip("no host compiler")
    (tmp_path / "plan.cpp").write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-O2", "-I", CSRC, str(tmp_path / "plan.cpp"), "-o", str(tmp_path / "plan")], check=True)
    r = subprocess.run([str(tmp_path / "plan")], stdout=subprocess.PIPE, text=True, timeout=120)
    assert r.returncode == 0, r.stdout
