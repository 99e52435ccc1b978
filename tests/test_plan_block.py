"""Launch plans of the gated feed-forward block and of dropout with the next norm, swept on the CPU:
slots of a product's K are whole k-blocks, none empty, and cover K; the workspace covers the
partials; a few rows' ring fits the LDS; a row's threads cover its groups, and the backward's
workgroups its rows."""
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
  CHECK(k.splits * k.kper >= K, "%s: K %lld not covered", what, K);
  CHECK((k.splits - 1) * k.kper < K, "%s: empty slot of K %lld", what, K);
  CHECK(mlp_part_bytes(k, M, N) <= 2 * kMlpSlotBytes, "%s: partials", what);
}
int main() {
  for (long long N : {1, 2, 16, 17, 64, 65, 100, 257, 1000, 2045, 8192, 70000})
    for (long long H : {8, 64, 768, 2048, 4096, 8192})
      for (long long F : {8, 40, 2048, 5632, 14336, 28672})
        for (long long O : {0ll, 8ll, H}) {
          const MlpShape s{N, H, F, O};
          const MlpFwdPlan f = mlp_fwd_plan(s);
          CHECK(f.up_waves == 8 || f.up_waves == 4, "up_waves");
          CHECK(f.down_waves == 8 || f.down_waves == 4, "down_waves");
          split_ok(f.down, F, N, O, "down");
          const long long fw = mlp_fwd_workspace(s, f);
          CHECK(fw == (O > 0 && N > kMlpFewRows && f.down.splits > 1 ? f.down.splits * N * O * 4 : 0),
                "forward workspace");
          const MlpBwdPlan b = mlp_bwd_plan(s);
          CHECK(b.da_waves == 8 || b.da_waves == 4, "da_waves");
          CHECK(b.grad_waves == 8 || b.grad_waves == 4, "grad_waves");
          split_ok(b.dx, 2 * F, N, H, "dx");
          split_ok(b.dw, N, F, H, "dw");
          const MlpBwdWorkspace w = mlp_bwd_workspace(s, b);
          const long long at[] = {w.dg, w.du, w.dx, w.dw[0], w.dw[1], w.dw[2], w.total};
          const long long need[] = {2 * N * F, 2 * N * F, mlp_part_bytes(b.dx, N, H),
                                    mlp_part_bytes(b.dw, F, H), mlp_part_bytes(b.dw, F, H),
                                    O > 0 ? mlp_part_bytes(b.dw, O, F) : 0};
          for (int i = 0; i < 6; ++i)
            CHECK(at[i] % 256 == 0 && at[i] + need[i] <= at[i + 1], "workspace part %d", i);
        }
  for (long long K : {1, 31, 64, 65, 200, 4096}) {
    const int waves = mlp_few_waves(K);
    CHECK(waves >= 1 && waves <= kMlpFewWaves, "waves of K %lld", K);
    for (int tiles = 1; tiles <= kMlpFewRows / 16; ++tiles)
      for (int pair = 1; pair <= 2; ++pair) {
        const int d = mlp_few_depth(tiles);
        CHECK(d >= 2 && waves * (pair + tiles) * d * 2048 <= 160 * 1024, "LDS");
        // the waves' sums take the ring's place, and two feature tiles fit too
        CHECK(waves * pair * tiles * 1024 <= waves * (pair + tiles) * d * 2048, "sums");
        CHECK(waves * (2 * pair + tiles) * d * 2048 <= 160 * 1024, "LDS of two");
        CHECK(2 * pair * tiles * 1024 <= (2 * pair + tiles) * d * 2048, "sums of two");
      }
  }
  for (long long F = 1; F <= 40000; F += 7)
    for (long long N : {1, 16, 17, 32, 33, 48, 49, 64})
      for (bool pair : {false, true}) {
        const bool two = mlp_few_two(N, F, pair);
        CHECK(!two || (N > (pair ? 32 : 16) && F > 16 * kCus), "two tiles of %lld rows", N);
      }
  for (long long cols = 1; cols <= kDropNormMaxCols; ++cols) {
    const long long groups = (cols + 7) / 8;
    for (int bytes : {0, 2, 4}) {  // 0: the forward
      const DropNormPlan p = bytes ? drop_norm_bwd_plan(groups, bytes) : drop_norm_plan(groups);
      CHECK((long long)p.tpr * p.kv >= groups, "cols %lld not covered", cols);
      CHECK(p.rows == drop_norm_plan(groups).rows, "rows of cols %lld", cols);
      CHECK(p.tpr * p.rows == (p.tpr > 256 ? 512 : 256), "threads of cols %lld", cols);
      CHECK((p.tpr & (p.tpr - 1)) == 0, "threads a row");
    }
    for (long long rows : {1ll, 32ll, 513ll, 16383ll, 16384ll, 70000ll, 1ll << 33}) {
      const long long grid = drop_norm_bwd_grid(rows, groups), per = drop_norm_plan(groups).rows;
      CHECK(grid >= 1 && grid <= 1024 && (grid - 1) * per < rows, "grid of %lld x %lld", rows, cols);
    }
  }
  CHECK(drop_norm_plan(kDropNormMaxCols / 8 + 1).tpr == 0, "too wide");
  std::printf("%d failures\n", fails);
  return fails != 0;
}
"""


def test_block_plans(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    src, exe = tmp_path / "block.cpp", tmp_path / "block"
    src.write_text(DRIVER)
    subprocess.run([gxx, "-O2", "-std=c++17", f"-I{CSRC}", str(src), "-o", str(exe)], check=True)
    proc = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert proc.returncode == 0, proc.stdout + proc.stderr
