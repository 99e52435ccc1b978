"""Embedding on the CPU: the C ABI's host checks, the Python refusals, and the plan of the
gradient (sort passes, workspace, runs, rows)."""
import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from trainscale_amd import _lib
from trainscale_amd.kernels import ScaledEmbedding, scaled_embedding

TS_OK, INVALID, DTYPE, SHAPE, WORKSPACE = 0, -1, -2, -3, -4
CSRC = Path(__file__).resolve().parent.parent / "trainscale_amd" / "csrc"
FAKE = ctypes.c_void_p(0x1000)  # never dereferenced: every call below ends on the host


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def test_forward_validation(lib):
    def f(ids=FAKE, N=4, w=FAKE, ldw=64, dt=1, V=10, H=64, out=FAKE, ldo=64):
        return lib.ts_embedding_fwd(ids, N, w, ldw, dt, V, H, 1.0, out, ldo, None)

    assert f(dt=5) == DTYPE
    assert f(N=-1) == SHAPE and f(V=-1) == SHAPE and f(H=-1) == SHAPE
    assert f(ldw=63) == SHAPE and f(ldo=63) == SHAPE
    assert f(V=0) == SHAPE  # tokens, but no rows
    assert f(ids=None) == INVALID and f(w=None) == INVALID and f(out=None) == INVALID
    assert f(ids=ctypes.c_void_p(0x1004)) == INVALID
    assert f(w=ctypes.c_void_p(0x1001)) == INVALID
    assert f(dt=0, out=ctypes.c_void_p(0x1002)) == INVALID
    assert f(N=0, ids=None, out=None) == TS_OK
    assert f(H=0) == TS_OK


def test_backward_validation(lib):
    need = lib.ts_embedding_bwd_workspace_size(100, 50, 64)
    assert need >= 100 * 8 + 100 // 32 * 64 * 4
    assert lib.ts_embedding_bwd_workspace_size(3000, 50, 64) >= 3000 * 16 + 3000 // 32 * 64 * 4
    assert lib.ts_embedding_bwd_workspace_size(-1, 50, 64) == 0
    assert lib.ts_embedding_bwd_workspace_size(1 << 31, 50, 64) == 0

    def f(ids=FAKE, N=100, d=FAKE, ldd=64, dt=1, V=50, H=64, g=FAKE, ws=FAKE, wsb=need):
        return lib.ts_embedding_bwd(ids, N, d, ldd, dt, V, H, 1.0, -1, g, ws, wsb, None)

    assert f(dt=3) == DTYPE
    assert f(N=-1) == SHAPE and f(N=1 << 31) == SHAPE and f(V=1 << 31) == SHAPE
    assert f(ldd=63) == SHAPE
    assert f(ids=None) == INVALID and f(d=None) == INVALID and f(g=None) == INVALID
    assert f(g=ctypes.c_void_p(0x1001)) == INVALID
    assert f(ids=ctypes.c_void_p(0x1004)) == INVALID
    assert f(wsb=need - 1) == WORKSPACE and f(ws=None) == WORKSPACE
    assert f(ws=ctypes.c_void_p(0x1008)) == WORKSPACE
    assert f(V=0) == TS_OK and f(H=0) == TS_OK


def test_python_refusals():
    w, ids = torch.zeros(10, 8), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="GPU"):
        scaled_embedding(ids, w)
    with pytest.raises(ValueError, match="weight must be"):
        scaled_embedding(ids, w[0])
    with pytest.raises(ValueError, match="weight must be"):
        scaled_embedding(ids, w[:, :0])
    with pytest.raises(TypeError, match="ids must be"):
        scaled_embedding(ids.float(), w)
    with pytest.raises(TypeError, match="ids must be"):
        scaled_embedding(ids.bool(), w)
    with pytest.raises(ValueError, match="scale"):
        scaled_embedding(ids, w, scale=float("inf"))
    for bad in (10, -11):
        with pytest.raises(ValueError, match="padding_idx"):
            scaled_embedding(ids, w, padding_idx=bad)
        with pytest.raises(ValueError, match="padding_idx"):
            ScaledEmbedding(10, 8, padding_idx=bad)


def test_module_initialisation():
    m = ScaledEmbedding(20, 8, scale=2.5, padding_idx=-1, dtype=torch.bfloat16)
    # a normal draw in bfloat16 holds exact zeros: a row has some value that is not one
    assert m.padding_idx == 19 and not m.weight[19].any() and m.weight[:19].any(1).all()
    assert m.weight.dtype == torch.bfloat16 and "scale=2.5" in repr(m)


DRIVER = r"""
#include <cstdio>
#include <initializer_list>
#include <vector>
#include "plan.hpp"
using namespace ts_plan;
static int fails = 0;
#define CHECK(c, ...) do { if (!(c)) { if (fails++ < 20) { std::printf(__VA_ARGS__); std::printf("\n"); } } } while (0)
int main() {
  for (long long N : {0ll, 1ll, 31ll, 32ll, 2048ll, 2049ll, 8192ll, 8193ll, 16384ll, 262144ll, 262145ll, 1000003ll, (long long)kEmbedMaxIndex})
    for (long long V : {1ll, 2ll, 1023ll, 1024ll, 50257ll, 128256ll, (1ll << 20) - 1, 1ll << 20, (long long)kEmbedMaxIndex}) {
      const EmbedSort p = embed_sort(N, V);
      CHECK(p.bits >= 1 && p.bits <= kEmbedMaxBits, "bits");
      CHECK(p.passes * p.bits >= 63 - __builtin_clzll(V) + 1, "keys 0 .. V do not fit");
      CHECK((p.passes - 1) * p.bits < 32, "shift");
      CHECK((p.blocks == 0) == (N <= kEmbedSmallTokens), "placed by counting");
      if (p.blocks > 0) {
        CHECK(p.blocks >= 1 && p.blocks <= kEmbedMaxBlocks && p.len % kEmbedTile == 0, "blocks");
        CHECK(p.blocks * p.len >= N && (p.blocks - 1) * p.len < N, "blocks do not cover");
      }
      for (long long H : {1ll, 7ll, 8ll, 768ll, 4097ll}) {
        const EmbedWorkspace w = embed_workspace(N, V, H);
        CHECK(w.keys[0] == 0 && w.vals[0] >= w.keys[0] + 4 * N, "list");
        if (p.blocks > 0) CHECK(w.keys[1] >= w.vals[0] + 4 * N && w.vals[1] >= w.keys[1] + 4 * N &&
                                w.table >= w.vals[1] + 4 * N, "lists");
        else CHECK(w.table >= w.vals[0] + 4 * N, "lists of a small sort");
        CHECK(w.sums1 >= w.table + (p.blocks << p.bits) * 4, "table");
        CHECK(w.ld >= H && w.ld % 8 == 0, "row of sums");
        CHECK(w.sums2 >= w.sums1 + N / kEmbedChunk * w.ld * 4, "sums");
        CHECK(w.bytes >= w.sums2 + N / kEmbedChunk / kEmbedChunk * w.ld * 4 && w.bytes > 0, "bytes");
        for (long long o : {w.vals[0], w.keys[1], w.vals[1], w.table, w.sums1, w.sums2})
          CHECK(o % 16 == 0, "alignment");
      }
    }
  // placing by counting: the groups share the whole list in eights, the last own keys fit
  for (int groups : {8, 16, 32})
    for (int N = 1; N <= kEmbedSmallTokens; ++N) {
      const EmbedRanks r = embed_ranks(N, groups);
      const int own = 256 / groups;
      CHECK(r.len % 8 == 0 && r.len > 0 && r.padded == groups * r.len, "len");
      CHECK(r.padded >= (N + own - 1) / own * own && r.padded <= kEmbedSmallTokens, "padding of %d", N);
    }
  // a run's pieces: every token once, whole chunks and whole chunks of chunks inside the run
  const long long C = kEmbedChunk;
  for (long long s : {0ll, 1ll, 31ll, 32ll, 33ll, 1000ll, 1023ll, 1024ll, 1025ll, 5000ll})
    for (long long n : {1ll, 2ll, 31ll, 32ll, 33ll, 63ll, 64ll, 95ll, 1024ll, 1025ll, 2047ll, 2048ll, 5000ll, 100000ll}) {
      const long long e = s + n;
      const EmbedRun r = embed_run(s, e);
      std::vector<char> seen(n, 0);
      auto take = [&](long long a, long long b) {
        for (long long i = a; i < b; ++i) {
          CHECK(i >= s && i < e, "outside the run");
          if (i >= s && i < e) { CHECK(!seen[i - s], "twice"); seen[i - s] = 1; }
        }
      };
      take(s, r.t0);
      take(r.t1, e);
      for (long long c = r.a0; c < r.a1; ++c) take(c * C, c * C + C);
      for (long long c = r.c0; c < r.c1; ++c) take(c * C, c * C + C);
      for (long long c = r.b0; c < r.b1; ++c) take(c * C * C, c * C * C + C * C);
      for (char x : seen) CHECK(x, "missing");
      CHECK(r.t0 - s < 2 * C && e - r.t1 < C, "too many tokens");
      CHECK(r.a1 - r.a0 < 2 * C && r.c1 - r.c0 < C, "too many sums");
    }
  std::printf("%d failures\n", fails);
  return fails != 0;
}
"""


def test_plan(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    src, exe = tmp_path / "embed.cpp", tmp_path / "embed"
    src.write_text(DRIVER)
    subprocess.run([gxx, "-O2", "-std=c++17", f"-I{CSRC}", str(src), "-o", str(exe)], check=True)
    proc = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert proc.returncode == 0, proc.stdout + proc.stderr
