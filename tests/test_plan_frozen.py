"""Launch plans of the gated feed-forward block's backward where only some gradients are asked for:
they are made for the products that run, and the workspace holds nothing for the others."""
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "trainscale_amd" / "csrc"

DRIVER = r"""
#include <cstdio>
#include <initializer_list>
#include "plan.hpp"
using namespace ts_plan;
static int fails = 0;
#define CHECK(c, ...) do { if (!(c)) { if (fails++ < 20) { std::printf(__VA_ARGS__); std::printf("\n"); } } } while (0)
static void split_ok(const KSplit& k, long long K, long long M, long long N, const char* what) {
  CHECK(k.splits >= 1, "%s: slots", what);
  if (k.splits == 1) return;
  CHECK(k.kper > 0 && k.kper % kGemmBlockK == 0, "%s: kper %lld", what, (long long)k.kper);
  CHECK(k.splits * k.kper >= K && (k.splits - 1) * k.kper < K, "%s: slots of K %lld", what, K);
  CHECK(mlp_part_bytes(k, M, N) <= kMlpSlotBytes, "%s: partials", what);
}
int main() {
  for (long long N : {1, 2, 16, 17, 64, 65, 100, 257, 1000, 2045, 8192, 70000})
    for (long long H : {8, 64, 768, 2048, 4096, 8192})
      for (long long F : {8, 40, 2048, 5632, 14336, 28672})
        for (long long O : {0ll, 8ll, H}) {
          const MlpShape s{N, H, F, O};
          split_ok(mlp_fwd_plan(s).down, F, N, O, "down");
          for (int g = 1; g <= kMlpGrads; ++g) {
            const MlpBwdPlan b = mlp_bwd_plan(s, g);
            CHECK((b.da_waves == 8 || b.da_waves == 4) && (b.grad_waves == 8 || b.grad_waves == 4),
                  "waves");
            split_ok(b.dx, 2 * F, N, H, "dx");
            if (g & (kMlpDwGate | kMlpDwUp)) split_ok(b.dw, N, F, H, "dw");
            if ((g & kMlpDwDown) && O > 0) split_ok(b.dw, N, O, F, "dw_down");
            CHECK((g & kMlpDx) || b.dx.splits == 1, "slots of no dx");
            CHECK((g & (kMlpGrads - kMlpDx)) || b.dw.splits == 1, "slots of no weights");
            const MlpBwdWorkspace w = mlp_bwd_workspace(s, b, g);
            const long long at[] = {w.dg, w.du, w.dx, w.dw[0], w.dw[1], w.dw[2], w.total};
            const long long inner = g & kMlpInner ? 2 * N * F : 0, dw = mlp_part_bytes(b.dw, F, H);
            const long long need[] = {inner, inner, mlp_part_bytes(b.dx, N, H),
                                      g & kMlpDwGate ? dw : 0, g & kMlpDwUp ? dw : 0,
                                      (g & kMlpDwDown) && O > 0 ? mlp_part_bytes(b.dw, O, F) : 0};
            for (int i = 0; i < 6; ++i)
              CHECK(at[i] % 256 == 0 && at[i + 1] - at[i] == (need[i] + 255) / 256 * 256,
                    "workspace part %d of gradients %d", i, g);
          }
        }
  // dx alone: 128 tiles of whole K on 256 CUs, or half the K on all of them
  for (long long N : {1024, 2048}) {
    const MlpShape s{N, 4096, 14336, 4096};
    const MlpBwdPlan b = mlp_bwd_plan(s, kMlpDx);
    CHECK(mlp_tiles(N, 4096, b.grad_waves, false) * b.dx.splits >= kCus, "dx of %lld rows", N);
  }
  std::printf("%d failures\n", fails);
  return fails != 0;
}
"""


def test_plans_of_some_gradients(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    src, exe = tmp_path / "frozen.cpp", tmp_path / "frozen"
    src.write_text(DRIVER)
    subprocess.run([gxx, "-O2", "-std=c++17", f"-I{CSRC}", str(src), "-o", str(exe)], check=True)
    proc = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert proc.returncode == 0, proc.stdout + proc.stderr
