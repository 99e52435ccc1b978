"""Gradient norm and clipping on the CPU: host checks of the C ABI and of the Python entry
points, and the cutting of tensors into chunks."""
import ctypes
import shutil
import subprocess
import weakref
from pathlib import Path

import pytest
import torch

from trainscale_amd import _lib
from trainscale_amd.kernels import (clip_grad_norm_, clip_grads_with_norm_, clipped_grads,
                                    get_total_norm)
from trainscale_amd.kernels.grad_kernels import (_is_dense, _refuse_overlap,
                                                 _refuse_strided_overlap, _share_memory)
from trainscale_amd.ops import HostList

TS_OK, INVALID, DTYPE, SHAPE, WORKSPACE = 0, -1, -2, -3, -4
CSRC = Path(__file__).resolve().parent.parent / "trainscale_amd" / "csrc"
FAKE = ctypes.c_void_p(0x1000)  # never dereferenced: every call below ends on the host


def _lists(ptrs, numels, dtypes):
    n = len(ptrs)
    return ((ctypes.c_void_p * n)(*ptrs), (ctypes.c_int64 * n)(*numels),
            (ctypes.c_int32 * n)(*dtypes))


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def test_norm_validation(lib):
    need = lib.ts_grad_norm_workspace_size(2)

    def call(ptrs=(0x1000, 0x2000), numels=(5, 7), dtypes=(0, 1), norm=FAKE, ws=FAKE, wsb=need,
             count=2):
        p, n, d = _lists(ptrs, numels, dtypes)
        return lib.ts_grad_norm(p, n, d, count, norm, ws, wsb, None)

    assert call(count=-1) == SHAPE
    assert call(numels=(5, -1)) == SHAPE
    assert call(dtypes=(0, 3)) == DTYPE
    assert call(ptrs=(0x1000, None)) == INVALID
    assert call(ptrs=(0x1002, 0x2000)) == INVALID  # an fp32 tensor off its elements
    assert b"aligned" in lib.ts_last_error()
    assert call(ptrs=(0x1000, 0x2001)) == INVALID
    assert call(norm=None) == INVALID
    assert call(ws=None) == WORKSPACE
    assert call(ws=ctypes.c_void_p(0x1004)) == WORKSPACE
    assert call(wsb=need - 1) == WORKSPACE
    assert call(numels=(5, 1 << 62)) == SHAPE
    assert lib.ts_grad_norm(None, None, None, 2, FAKE, FAKE, need, None) == INVALID


def test_scale_and_clip_validation(lib):
    need = lib.ts_grad_norm_workspace_size(1)

    def scale(ptr=0x1000, out=0x2000, numel=5, dt=1, odt=1, norm=FAKE, max_norm=1.0):
        p, n, d = _lists([ptr], [numel], [dt])
        return lib.ts_grad_scale(p, (ctypes.c_void_p * 1)(out), n, d, (ctypes.c_int32 * 1)(odt), 1,
                                 norm, max_norm, None)

    assert scale(odt=2) == DTYPE  # bf16 into fp16
    assert scale(dt=0, odt=1) == DTYPE  # fp32 into bf16
    assert scale(out=None) == INVALID
    assert scale(out=0x2002, odt=0) == INVALID
    assert scale(norm=None) == INVALID
    assert scale(max_norm=-1.0) == INVALID
    assert scale(max_norm=float("nan")) == INVALID
    assert scale(numel=0, ptr=None, out=None) == TS_OK  # an empty tensor is nothing to do
    p, n, d = _lists([0x1000], [5], [1])
    o, od = (ctypes.c_void_p * 1)(0x2000), (ctypes.c_int32 * 1)(0)
    clip = lambda **k: lib.ts_grad_clip(p, o, n, d, od, 1, k.get("max_norm", 1.0),
                                        k.get("norm", FAKE), k.get("ws", FAKE),
                                        k.get("wsb", need), None)
    assert clip(max_norm=-0.5) == INVALID
    assert clip(norm=None) == INVALID
    assert clip(wsb=8) == WORKSPACE
    assert clip(ws=None) == WORKSPACE


def test_python_refusals():
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.zeros(4)
    with pytest.raises(RuntimeError, match="GPU"):
        clip_grad_norm_([p], 1.0)
    with pytest.raises(ValueError, match="max_norm"):
        clip_grad_norm_([p], -1.0)
    with pytest.raises(ValueError, match="max_norm"):
        clip_grads_with_norm_([p], float("nan"), torch.tensor(1.0))
    with pytest.raises(ValueError, match="2-norm"):
        clip_grad_norm_([p], 1.0, norm_type=1)
    with pytest.raises(ValueError, match="2-norm"):
        get_total_norm([p.grad], float("inf"))
    with pytest.raises(TypeError, match="dtype"):
        get_total_norm([torch.zeros(3, dtype=torch.float64)])
    with pytest.raises(TypeError, match="sparse"):
        get_total_norm([torch.zeros(3, 3).to_sparse()])
    with pytest.raises(TypeError, match="expected tensors"):
        get_total_norm([1.0])
    with pytest.raises(TypeError, match="local tensor"):
        get_total_norm([torch.zeros(3).as_subclass(type("Sharded", (torch.Tensor,), {}))])


def test_nothing_to_clip():
    assert float(clip_grad_norm_([torch.nn.Parameter(torch.zeros(3))], 1.0)) == 0.0
    assert float(get_total_norm([])) == 0.0
    assert float(clipped_grads([], 1.0, [])) == 0.0
    clip_grads_with_norm_([], 1.0, torch.tensor(1.0))


def test_dense_and_overlap():
    t = torch.zeros(4, 6, 5)
    assert _is_dense(t) and _is_dense(t.permute(2, 0, 1)) and _is_dense(t[1])
    assert not _is_dense(t[:, 1:]) and not _is_dense(t[:, :, ::2])
    assert not _is_dense(torch.zeros(1, 5).expand(3, 5))
    flat = torch.zeros(100)
    a, b = flat[:50], flat[50:]

    def check(written, read=None):
        w = HostList(written)
        _refuse_overlap("x", w, w if read is None else HostList(read))

    check([a, b])
    check([a, b], [a, b])
    for written, read in (([a, flat[49:]], None),
                          ([a, a], None),  # the same tensor twice
                          ([a, a], [a, a]),
                          ([b, torch.zeros(50)], [a, flat[20:70]]),  # over another's gradient
                          ([torch.zeros(100), flat[10:12]], [flat, torch.zeros(2)]),
                          ([a.view(torch.bfloat16)[:50]], [a])):
        with pytest.raises(ValueError, match="share memory"):
            check(written, read)
    check([torch.zeros(50), torch.zeros(50)], [a, a])  # read twice
    check([flat[:0], flat])
    check([torch.zeros(40), flat[60:]], [flat[:60].view(torch.bfloat16)[10:50], flat[:40]])


def _strided_refused(grads):
    try:
        _refuse_strided_overlap("x", grads, [not (t.is_contiguous() or _is_dense(t)) for t in grads])
    except ValueError as e:
        assert "share memory" in str(e)
        return True
    return False


def test_strided_gradients_that_share_memory():
    buf = torch.zeros(12, 20)
    for grads in ([buf, buf[:, :4]], [buf[:, :4], buf], [buf[:, :6], buf[:, 3:9]],
                  [buf[2:, 5:], buf[:3, 5:9]], [buf[:, 3], buf[4:6, 2:5]],
                  [buf[:, ::2], buf[:, 1:9]], [buf[:, ::2], buf[:, ::3]],
                  [buf.t()[3:7], buf[:, 6:8]], [buf[:, :4]] * 2,
                  [buf[:, 4:9], buf.view(torch.bfloat16)[3:5, 17:19]],
                  [torch.zeros(5).expand(3, 5)], [torch.zeros(40).as_strided((4, 4), (3, 1))],
                  [torch.zeros(40).as_strided((4, 4), (4, 4))],
                  [torch.zeros(40).as_strided((3, 3, 2), (9, 4, 2))]):
        if grads[-1].stride() == (9, 4, 2):  # odd, but its elements are apart
            assert not _strided_refused(grads)
        else:
            assert _strided_refused(grads), [t.stride() for t in grads]
    for grads in ([buf[:, :6], buf[:, 6:9], buf[:, 9:]], [buf[:, ::2], buf[:, 1::2]],
                  [buf[:5, :6], buf[5:, :6], buf[:, 6:]], [buf[:, 3], buf[:, 4:6], buf[:, 2]],
                  [buf[:, :0], buf[:, :4]], [buf[:, 4:9], buf.view(torch.bfloat16)[:, :7]],
                  [torch.zeros(2, 3, 8, 8)[:, :, 1:, ::3]],
                  [torch.zeros(3, 300)[:, k:290:7] for k in range(7)]):
        assert not _strided_refused(grads), [t.stride() for t in grads]


def test_interleaved_slices_of_wide_rows():
    wide = torch.zeros(6, 12000)
    assert not _strided_refused([wide[:, ::2], wide[:, 1::4], wide[:, 3::4]])
    assert _strided_refused([wide[:, ::2], wide[:, 1::4], wide[:, 3::4], wide[5:, 11999]])
    assert _strided_refused([wide[:, ::2], wide[:, 1::3]])


def test_shared_memory_as_by_addresses():
    # against the bytes written down one by one
    gen = torch.Generator().manual_seed(3)
    r = lambda lo, hi: int(torch.randint(lo, hi, (), generator=gen))
    buf = torch.zeros(8000, dtype=torch.uint8)
    base = buf.data_ptr()
    found = set()
    for _ in range(3000):
        ts, places = [], []
        for _ in range(2):
            dtype = (torch.float32, torch.bfloat16)[r(0, 2)]
            flat = buf.view(dtype)
            shape = [r(1, 5) for _ in range(r(1, 4))]
            strides = [r(1, 30) for _ in shape]
            if r(0, 2):
                strides = [strides[0] * (3, 1, 9)[i] for i in range(len(shape))]
            t = flat.as_strided(shape, strides, r(0, 60))
            at = torch.zeros(shape, dtype=torch.int64) + t.data_ptr() - base
            for k, st in enumerate(strides):
                view = [1] * len(shape)
                view[k] = shape[k]
                at += (torch.arange(shape[k]) * st * t.element_size()).view(view)
            ts.append(t)
            places.append([p + i for p in at.reshape(-1).tolist() for i in range(t.element_size())])
        own = len(set(places[0])) < len(places[0])
        assert _share_memory(ts[0]) == own, (ts[0].shape, ts[0].stride())
        both = not set(places[0]).isdisjoint(places[1])
        assert _share_memory(*ts) == both
        found.add((own, both))
    assert len(found) == 4


def test_list_keeps_its_tensors():
    # the copies of strided gradients have no other owner until the launches are queued
    from trainscale_amd.kernels.grad_kernels import _storage_order
    made = _storage_order([torch.zeros(4, 8)[:, :3]])
    refs = [weakref.ref(t) for t in made]
    held = HostList(made)
    del made
    assert all(r() is not None for r in refs)
    assert [t.data_ptr() for t in held.tensors] == held.ptr.tolist()
    del held
    assert all(r() is None for r in refs)


DRIVER = r"""
#include <cstdio>
#include <initializer_list>
#include <vector>
#include "plan.hpp"
using namespace ts_plan;
int main() {
  int fails = 0;
  unsigned r = 12345;
  for (int elt : {2, 4})
    for (int count : {1, 2, 3, 100, kGradTensors})
      for (int rep = 0; rep < 20; ++rep) {
        std::vector<int64_t> numel(count);
        std::vector<int32_t> end(count);
        int64_t chunks = 0;
        const int64_t per = grad_chunk(elt, rep % 2 ? kGradNormPieces : kGradScalePieces);
        for (int i = 0; i < count; ++i) {
          r = r * 1664525u + 1013904223u;
          const int64_t edge[] = {1, per - 1, per, per + 1, 3 * per, (int64_t)(r >> 12) + 1};
          numel[i] = edge[r % 6];
          chunks += grad_chunks(numel[i], per);
          end[i] = (int32_t)chunks;
        }
        // every chunk belongs to one tensor and holds at least one of its values; together
        // they hold all of them
        std::vector<int64_t> held(count, 0);
        for (int64_t c = 0; c < chunks; ++c) {
          const int t = grad_find_tensor(end, count, (int)c);
          const int64_t first = (c - (t ? end[t - 1] : 0)) * per;
          const int64_t left = numel[t] - first;
          if (t < 0 || t >= count || c >= end[t] || first < 0 || left <= 0) { ++fails; continue; }
          held[t] += left < per ? left : per;
        }
        for (int i = 0; i < count; ++i) fails += held[i] != numel[i];
      }
  // launches of a list: full ones, and at most one that is not full for each of three types
  for (int64_t count = 1; count < 2000; ++count) {
    int64_t most = 0;
    for (int64_t a = 0; a <= 2; ++a)
      for (int64_t b = 0; b <= 2; ++b) {
        const int64_t n1 = count > a ? a : 0, n2 = count - n1 > b ? b : 0, n3 = count - n1 - n2;
        int64_t l = 0;
        for (int64_t n : {n1, n2, n3}) l += (n + kGradTensors - 1) / kGradTensors;
        most = l > most ? l : most;
      }
    fails += most * kGradGrid > grad_norm_parts(count);
  }
  fails += grad_chunks(0, 2048) != 0 || grad_norm_parts(0) < 1;
  std::printf("%d failures\n", fails);
  return fails != 0;
}
"""


def test_chunks(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    src, exe = tmp_path / "chunks.cpp", tmp_path / "chunks"
    src.write_text(DRIVER)
    subprocess.run([gxx, "-O2", "-std=c++17", f"-I{CSRC}", str(src), "-o", str(exe)], check=True)
    proc = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert proc.returncode == 0, proc.stdout + proc.stderr
