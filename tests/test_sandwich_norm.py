"""Norms before and after a block on the CPU: host checks, refusals, and the plan."""
import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from trainscale_amd import _lib
from trainscale_amd.kernels import FusedSandwichRMSNorm, fused_sandwich_rms_layernorm
from trainscale_amd.kernels.layernorm_kernels import _gate_rows

TS_OK, INVALID, DTYPE, SHAPE, WORKSPACE = 0, -1, -2, -3, -4
CSRC = Path(__file__).resolve().parent.parent / "trainscale_amd" / "csrc"
FAKE = ctypes.c_void_p(0x1000)  # never dereferenced: every call below ends on the host
ODD = ctypes.c_void_p(0x1001)


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def fwd(lib, **k):
    a = dict(y=FAKE, ldy=64, x=FAKE, ldx=64, dt=1, post=FAKE, pre=FAKE, wdt=1, gate=None, gdt=0,
             groups=1, n=FAKE, ldn=64, h=FAKE, ldh=64, ry=FAKE, rh=FAKE, rows=6, cols=64, eps=1e-6)
    a.update(k)
    return lib.ts_sandwich_norm_fwd(a["y"], a["ldy"], a["x"], a["ldx"], a["dt"], a["post"],
                                    a["pre"], a["wdt"], a["gate"], a["gdt"], a["groups"], a["n"],
                                    a["ldn"], a["h"], a["ldh"], a["ry"], a["rh"], a["rows"],
                                    a["cols"], 1.0, 0.0, a["eps"], None)


def test_forward_validation(lib):
    assert fwd(lib, dt=4) == DTYPE and fwd(lib, wdt=2) == DTYPE and fwd(lib, wdt=9) == DTYPE
    assert fwd(lib, rows=-1) == SHAPE and fwd(lib, cols=0) == SHAPE
    big = dict(ldy=1 << 20, ldx=1 << 20, ldn=1 << 20, ldh=1 << 20)
    assert fwd(lib, cols=16385, **big) == SHAPE and b"16384" in lib.ts_last_error()
    assert fwd(lib, cols=8193, dt=0, wdt=0, **big) == SHAPE
    for name in ("ldy", "ldx", "ldn", "ldh"):
        assert fwd(lib, **{name: 63}) == SHAPE
    for name in ("y", "x", "post", "pre", "n", "h", "ry", "rh"):
        assert fwd(lib, **{name: None}) == INVALID
    for name in ("y", "x", "post", "pre", "n", "h", "gate"):
        assert fwd(lib, **{"gdt": 1, name: ODD}) == INVALID
    assert fwd(lib, groups=2) == INVALID  # groups without a gate
    assert fwd(lib, gate=FAKE, gdt=1, groups=4) == SHAPE  # 6 rows
    assert fwd(lib, gate=FAKE, gdt=1, groups=0) == SHAPE
    assert fwd(lib, gate=FAKE, gdt=2) == DTYPE
    assert fwd(lib, eps=-1.0) == INVALID and fwd(lib, eps=float("nan")) == INVALID
    assert fwd(lib, rows=0, y=None, x=None, n=None, h=None, ry=None, rh=None) == TS_OK


def test_backward_validation(lib):
    need = lib.ts_sandwich_norm_bwd_workspace_size(6, 64, 1)
    assert need > 0
    assert lib.ts_sandwich_norm_bwd_workspace_size(0, 64, 1) == 0
    assert lib.ts_sandwich_norm_bwd_workspace_size(6, 64, 7) == 0

    def f(**k):
        a = dict(dn=FAKE, lddn=64, dh=FAKE, lddh=64, y=FAKE, x=FAKE, dt=1, gate=None, gdt=0,
                 groups=1, ry=FAKE, rh=FAKE, dy=FAKE, lddy=64, dx=FAKE, lddx=64, dpost=FAKE,
                 dpre=FAKE, dgate=None, rows=6, ws=FAKE, wsb=need)
        a.update(k)
        return lib.ts_sandwich_norm_bwd(
            a["dn"], a["lddn"], a["dh"], a["lddh"], a["y"], 64, a["x"], 64, a["dt"], FAKE, FAKE, 1,
            a["gate"], a["gdt"], a["groups"], a["ry"], a["rh"], a["dy"], a["lddy"], a["dx"],
            a["lddx"], a["dpost"], a["dpre"], a["dgate"], a["rows"], 64, 1.0, 0.0, a["ws"],
            a["wsb"], None)

    assert f(dt=7) == DTYPE and f(rows=0) == SHAPE
    for name in ("lddn", "lddh", "lddy", "lddx"):
        assert f(**{name: 63}) == SHAPE
    for name in ("dn", "dh", "dy", "dx", "dpost", "dpre"):
        assert f(**{name: ODD}) == INVALID
    assert f(ry=None) == INVALID and f(rh=None) == INVALID and f(y=None) == INVALID
    assert f(dgate=FAKE) == INVALID  # no gate
    assert f(gate=FAKE, gdt=1, dgate=ODD) == INVALID
    assert f(wsb=need - 1) == WORKSPACE and f(ws=None) == WORKSPACE
    assert f(ws=ctypes.c_void_p(0x1008)) == WORKSPACE


def test_python_refusals():
    x, w = torch.zeros(4, 6, 8), torch.ones(8)
    with pytest.raises(RuntimeError, match="GPU"):
        fused_sandwich_rms_layernorm(x, x, w, w)
    with pytest.raises(ValueError, match="residual"):
        fused_sandwich_rms_layernorm(x, x[:3], w, w)
    m = FusedSandwichRMSNorm(8, layer_gate=True, gate_init=0.5, weight_offset=1.0)
    assert not m.post_weight.any() and bool((m.gate == 0.5).all())
    with pytest.raises(ValueError, match="gate of its own"):
        m(x, x, gate=w)


def test_gates():
    x = torch.zeros(4, 6, 8)
    for shape, groups in (((8,), 1), ((4, 1, 8), 4), ((1, 1, 8), 1), ((4, 6, 8), 24)):
        assert _gate_rows(torch.zeros(shape), x).shape == (groups, 8)
    for shape in ((7,), (6, 8), (4, 8), (1, 6, 8), (4, 1, 7), (1, 4, 1, 8), ()):
        with pytest.raises(ValueError, match="gate"):
            _gate_rows(torch.zeros(shape), x)
    assert _gate_rows(torch.zeros(2, 3, 1, 8), torch.zeros(2, 3, 5, 8)).shape == (6, 8)


DRIVER = r"""
#include <cstdio>
#include <initializer_list>
#include <vector>
#include "plan.hpp"
using namespace ts_plan;
static int fails = 0;
#define CHECK(c, ...) do { if (!(c)) { if (fails++ < 20) { std::printf(__VA_ARGS__); std::printf("\n"); } } } while (0)
int main() {
  for (int parts = 1; parts <= kSandwichMaxParts; ++parts) {
    const SandwichPlan p = sandwich_fwd_plan(parts);
    CHECK(p.tpr * p.kv >= parts && p.tpr % 64 == 0 && p.rpb >= 1, "forward of %d parts", parts);
    CHECK(p.rpb * p.tpr == (p.tpr > 256 ? p.tpr : 256), "forward block of %d parts", parts);
  }
  for (int V : {4, 8})
    for (long long cols : {1ll, 3ll, 64ll, 511ll, 512ll, 513ll, 2048ll, 2049ll, 4096ll, 8192ll, 8200ll, 16384ll}) {
      if ((cols + V - 1) / V > kSandwichMaxParts) continue;
      for (long long groups : {1ll, 2ll, 3ll, 64ll, 511ll, 512ll, 513ll, 4000ll})
        for (long long per : {1ll, 2ll, 7ll, 8ll, 9ll, 100ll, 2048ll, 16384ll}) {
          const long long rows = groups * per;
          const SandwichBwdPlan b = sandwich_bwd_plan(rows, groups, cols, V);
          CHECK((long long)b.row.tpr * b.row.kv * V >= cols, "row not covered");
          CHECK(b.row.rpb * b.row.tpr == (b.row.tpr > 512 ? b.row.tpr : 512), "block");
          // every row of a group once, no workgroup without a row
          std::vector<char> seen(per, 0);
          for (long long p = 0; p < b.per_group; ++p) {
            bool some = false;
            for (long long st = 0; st < b.steps; ++st)
              for (int sub = 0; sub < b.row.rpb; ++sub) {
                const long long r = (p + st * b.per_group) * b.row.rpb + sub;
                if (r < per) { CHECK(!seen[r], "row twice"); seen[r] = 1; some = true; }
              }
            CHECK(some, "idle workgroup");
          }
          for (char x : seen) CHECK(x, "row missing");
          const long long ldp = (cols + V - 1) / V * V;
          const long long need = (2 * groups * b.per_group + (groups > 1 ? 2 * groups : 0)) * ldp * 4;
          CHECK(need <= sandwich_workspace(rows, groups, cols), "workspace");
        }
    }
  std::printf("%d failures\n", fails);
  return fails != 0;
}
"""


def test_plan(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    src, exe = tmp_path / "plan.cpp", tmp_path / "plan"
    src.write_text(DRIVER)
    subprocess.run([gxx, "-O2", "-std=c++17", f"-I{CSRC}", str(src), "-o", str(exe)], check=True)
    proc = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert proc.returncode == 0, proc.stdout + proc.stderr
