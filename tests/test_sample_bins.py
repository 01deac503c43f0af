"""The sampler's running sums over its histogram (csrc/sample_bins.h) on the host: whichever threads and CTAs hold the
bins, one of them reaches a goal, and none only where the whole sum is below it."""
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "thvm_b200" / "csrc"

HARNESS = r"""
#include "sample_bins.h"
#include <math.h>
#include <stdio.h>
#include <random>
#include <vector>
using namespace sm100;
enum { kBins = 4096, kThreads = 512, kWarps = 16 };

// block_before of the kernel: a warp's inclusive sums, then the warps' totals in the same way
template <typename Sum> void scan(std::vector<Sum> &v, Sum *all) {
  std::vector<Sum> up = v;
  Sum w[32] = {};
  for (int warp = 0; warp < kWarps; warp++) {
    Sum *a = &up[warp * 32], b[32];
    for (int o = 1; o < 32; o <<= 1) {
      for (int i = 0; i < 32; i++) b[i] = i >= o ? a[i] + a[i - o] : a[i];
      for (int i = 0; i < 32; i++) a[i] = b[i];
    }
    w[warp] = a[31];
  }
  for (int o = 1; o < kWarps; o <<= 1) {
    Sum b[32];
    for (int i = 0; i < 32; i++) b[i] = i >= o ? w[i] + w[i - o] : w[i];
    for (int i = 0; i < 32; i++) w[i] = b[i];
  }
  *all = w[kWarps - 1];
  for (int t = 0; t < kThreads; t++) v[t] = (t >= 32 ? w[t / 32 - 1] : Sum(0)) + up[t] - v[t];
}

// goals with another number of owners than they should have
template <typename Sum> int faults(int C, const std::vector<uint32_t> &cnt, const std::vector<Sum> &weight, int goals, std::mt19937 &rng) {
  const int kB = kBins / C / kThreads;
  std::vector<Sum> before(C * kThreads), heavy(C);
  for (int r = 0; r < C; r++) {
    std::vector<Sum> v(kThreads);
    for (int t = 0; t < kThreads; t++) {
      Sum s = 0;
      for (int i = 0; i < kB; i++) s += weight[(r * kThreads + t) * kB + i];
      v[t] = s;
    }
    scan(v, &heavy[r]);
    for (int t = 0; t < kThreads; t++) before[r * kThreads + t] = v[t];
  }
  Sum total = 0;
  for (int r = 0; r < C; r++) total += heavy[r];
  int wrong = 0;
  for (int g = 0; g <= goals; g++) {
    // anywhere, at a thread's own sums (where two threads can disagree), and at nothing
    Sum goal = (Sum)((double)total * std::uniform_real_distribution<>(0, 1.02)(rng));
    if (g % 3 == 1) {
      const int t = (int)(rng() % (C * kThreads));
      goal = before[t];
      for (int r = 0; r < t / kThreads; r++) goal += heavy[r];
    }
    if (g == goals) goal = 0;
    int owners = 0;
    Sum base = 0;
    for (int r = 0; r < C; r++) {
      for (int t = 0; t < kThreads; t++) {
        Sum ww = before[r * kThreads + t] + base;
        for (int i = 0; i < kB; i++) {
          const int b = (r * kThreads + t) * kB + i;
          if (!cnt[b]) continue;
          bool first = true;
          for (int j = b - 1; j >= 0 && first; j--) first = !cnt[j];
          const Sum w1 = ww + weight[b];
          owners += reaches<Sum>(ww, w1, first, goal);
          ww = w1;
        }
      }
      base += heavy[r];
    }
    wrong += owners != (total >= goal ? 1 : 0);
  }
  return wrong;
}

int main() {
  std::mt19937 rng(1);
  int whole = 0, single = 0;
  for (int row = 0; row < 24; row++)
    for (int C = 1; C <= 8; C *= 2) {
      // some strong ids over a wide heap, as logits are
      std::vector<uint32_t> cnt(kBins);
      std::normal_distribution<> heap(900 + 40 * row, 250);
      for (int i = 0; i < 60000; i++) {
        const int b = (int)heap(rng);
        if (b >= 0 && b < kBins) cnt[b]++;
      }
      for (int i = 0; i < 24; i++) cnt[rng() % 1200]++;
      std::vector<BinSum> wi(kBins);
      std::vector<float> wf(kBins);
      for (int b = 0; b < kBins; b++) {
        const float e = expf(-(float)b / 128.0f);
        wi[b] = cnt[b] * (BinSum)llrint((double)e * 1099511627776.0);
        wf[b] = cnt[b] * e;
      }
      whole += faults<BinSum>(C, cnt, wi, 90, rng);
      single += faults<float>(C, cnt, wf, 90, rng);
    }
  printf("%d %d\n", whole, single);
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_each_goal_has_one_owner(tmp_path):
    src = tmp_path / "owners.cpp"
    src.write_text(HARNESS)
    subprocess.run(["g++", "-O2", "-std=c++17", f"-I{CSRC}", "-o", str(tmp_path / "owners"), str(src)], check=True)
    whole, single = map(int, subprocess.run([str(tmp_path / "owners")], check=True, capture_output=True, text=True).stdout.split())
    assert whole == 0
    assert single > 0   # f32 sums leave goals with two owners or none: the harness sees them

