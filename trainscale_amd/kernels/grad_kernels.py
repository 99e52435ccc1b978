"""Global gradient norm over many tensors, and clipping.

The trainer clips the global norm between the backward pass and the optimizer's step
(data_pipeline/trainer/trainers/sota_trainer.py:2214-2245, through torch's ``clip_grad_norm_``).
The functions here keep torch's names, arguments and arithmetic for the 2-norm:

    norm = sqrt(sum of x^2 over all gradients),  gradients *= min(1, max_norm / (norm + 1e-6))

A few launches cover every tensor of a model, whatever their number, sizes and types (fp32,
bf16, fp16 mixed); the norm is summed in double in a fixed order and nothing waits for the host.
A norm that is NaN makes every clipped gradient NaN, an infinite one zeros the finite gradients,
as torch's arithmetic does.

``clipped_grads`` writes the clipped gradients elsewhere, for optimizers that keep fp32 main
gradients next to 16-bit ones: one pass instead of a copy and a scaling.
"""
from __future__ import annotations

import math
from typing import Iterable, List, Optional, Sequence, Tuple, Union

import numpy as np
import torch
from torch import Tensor
from torch.autograd.forward_ad import unpack_dual

from .. import _lib, ops

__all__ = ["get_total_norm", "clip_grads_with_norm_", "clip_grad_norm_", "clipped_grads"]


def _is_dense(t: Tensor) -> bool:
    """Whether the elements fill their memory without gaps or overlaps, in any order."""
    want = 1
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if stride != want:
            return False
        want *= size
    return True


def _checked(what: str, tensors: Union[Tensor, Iterable[Tensor]]) -> List[Tensor]:
    """The tensors as a list: dense fp32/bf16/fp16 torch tensors on one GPU."""
    tensors = [tensors] if isinstance(tensors, Tensor) else list(tensors)
    if not tensors:
        return tensors
    # over whole lists (a model has hundreds of tensors): the interpreter's time is the call's
    for cls in {type(t) for t in tensors} - {Tensor, torch.nn.Parameter}:
        if not issubclass(cls, Tensor):
            raise TypeError(f"{what}: expected tensors, got {cls.__name__}")
        raise TypeError(f"{what}: {cls.__name__} is not supported: pass its local tensor")
    if ops.in_forward_ad() and any(unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{what}: forward-mode derivatives are not supported")
    if {t.layout for t in tensors} != {torch.strided}:
        raise TypeError(f"{what}: sparse gradients are not supported")
    for dtype in {t.dtype for t in tensors}:
        if dtype not in _lib.DTYPE_CODE:
            raise TypeError(f"{what}: unsupported dtype {dtype} (float32/bfloat16/float16)")
    if len({t.get_device() for t in tensors}) != 1:
        raise RuntimeError(f"{what}: tensors are on different devices")
    _lib.require_gpu(what, tensors[0])
    return tensors


def _storage_order(tensors: List[Tensor]) -> List[Tensor]:
    """The tensors with their values contiguous, in an order of their own: dense ones themselves,
    a copy of the others."""
    return [t if t.is_contiguous() or _is_dense(t) else t.detach().contiguous() for t in tensors]


def _refuse_overlap(what: str, written: ops.HostList, read: ops.HostList) -> None:
    """Raises if a written tensor shares memory with another tensor of either list. A tensor of
    `read` that is the written one at the same place in the list does not count."""
    start, end = written.ptr, written.end()
    if read is not written:
        rstart, rend = read.ptr, read.end()
        other = (rstart != start) | (rend != end)
        rstart, rend = rstart[other], rend[other]
        # what is read may overlap: as disjoint stretches
        order = np.argsort(rstart, kind="stable")
        rstart, rend = rstart[order], rend[order]
        if rend.size:
            first = np.ones(rstart.size, dtype=bool)
            first[1:] = rstart[1:] >= np.maximum.accumulate(rend)[:-1]
            at = np.flatnonzero(first)
            start = np.concatenate([start, rstart[at]])
            end = np.concatenate([end, np.maximum.reduceat(rend, at)])
    some = end > start
    start, end = start[some], end[some]
    order = np.argsort(start, kind="stable")
    if (start[order][1:] < end[order][:-1]).any():
        raise ValueError(f"{what}: gradients share memory: each must be written once")


def _reaches(distance: int, ranges: List[Tuple[int, int, int]], other: bool) -> Optional[bool]:
    """Whether distance = sum of d * stride with low <= d <= high for every (stride, low, high),
    strides falling; `other`: by other d than 0 everywhere. None if there are too many ways."""
    reach = [(0, 0)]  # what the strides behind k reach at least and at most
    for stride, low, high in reversed(ranges):
        reach.append((reach[-1][0] + stride * low, reach[-1][1] + stride * high))
    reach.reverse()
    tries, todo = 0, [(0, distance, not other)]
    while todo:
        k, left, counts = todo.pop()
        if k == len(ranges):
            if left == 0 and counts:
                return True
            continue
        stride, low, high = ranges[k]
        least, most = reach[k + 1]  # of left - d * stride
        d = range(max(low, -((most - left) // stride)), min(high, (left - least) // stride) + 1)
        tries += len(d)
        if tries > 1 << 16:
            return None
        todo += [(k + 1, left - i * stride, counts or i != 0) for i in d]
    return False


def _share_memory(a: Tensor, b: Optional[Tensor] = None) -> Optional[bool]:
    """Whether a byte belongs to both tensors, or to two elements of a where b is None. Found by
    their strides, one after the other: where strides nest, as those of slices do, each leaves one
    or two ways open. None where there are too many ways to tell."""
    size = a.element_size()
    dims = [(st * size, n) for st, n in zip(a.stride(), a.shape) if n > 1]
    if b is None and len({0, *[st for st, _ in dims]}) <= len(dims):
        return True  # no stride, or two alike
    # address of an element's byte: the tensor's plus those of its indices, bytes of stride 1
    ranges = {}
    for st, n in dims + [(1, size)]:
        low, high = ranges.get(st, (0, 0))
        ranges[st] = (low, high + n - 1)
    other = a if b is None else b
    size = other.element_size()
    for st, n in [(st * size, n) for st, n in zip(other.stride(), other.shape)] + [(1, size)]:
        low, high = ranges.get(st, (0, 0))
        ranges[st] = (low - (n - 1), high)
    return _reaches(other.data_ptr() - a.data_ptr(),
                    sorted([(st, *r) for st, r in ranges.items() if st > 0], reverse=True),
                    b is None)


def _refuse_strided_overlap(what: str, grads: List[Tensor], strided: List[bool]) -> None:
    """Raises if a gradient that is marked strided shares memory with itself or another one. Slices
    of one buffer that lie beside each other do not, though their stretches of addresses meet."""
    spans = []
    for k, t in enumerate(grads):
        if t.numel() > 0:
            last = sum((n - 1) * st for st, n in zip(t.stride(), t.shape))
            spans.append((t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size(), k))
    still = []  # spans that reach behind the next one's start
    for start, end, k in sorted(spans):
        still = [s for s in still if s[1] > start]
        pairs = [(grads[k], grads[s[2]]) for s in still if strided[k] or strided[s[2]]]
        if strided[k]:
            pairs.append((grads[k], None))
        for a, b in pairs:
            shared = _share_memory(a, b)
            if shared is None:
                raise ValueError(f"{what}: gradients of these strides may share memory: pass "
                                 "contiguous ones")
            if shared:
                raise ValueError(f"{what}: gradients share memory: each must be written once")
        still.append((start, end, k))


def _max_norm(what: str, max_norm: float) -> float:
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"{what}: max_norm must be >= 0, got {max_norm}")
    return max_norm


def _check_norm_type(what: str, norm_type: float) -> None:
    if float(norm_type) != 2.0:
        raise ValueError(f"{what}: only the 2-norm is supported, got norm_type {norm_type}")


def _grads(parameters: Union[Tensor, Iterable[Tensor]]) -> List[Tensor]:
    """The gradients of the parameters that have one; a parameter given twice counts once."""
    parameters = [parameters] if isinstance(parameters, Tensor) else list(parameters)
    by_id = dict(zip(map(id, parameters), parameters))
    return [g for g in [p.grad for p in by_id.values()] if g is not None]


def get_total_norm(tensors: Union[Tensor, Iterable[Tensor]], norm_type: float = 2.0,
                   error_if_nonfinite: bool = False, foreach: Optional[bool] = None) -> Tensor:
    """The 2-norm of all values of the tensors as a 0-dim fp32 tensor (torch's
    ``get_total_norm``; foreach is accepted for its signature). Of an empty list 0, on the CPU.
    Tensors are read only: they may share memory, and each counts as often as it is given."""
    del foreach
    _check_norm_type("get_total_norm", norm_type)
    tensors = _checked("get_total_norm", tensors)
    if not tensors:
        return torch.tensor(0.0)
    norm = ops.grad_norm(ops.HostList(_storage_order(tensors)), tensors[0].device)
    if error_if_nonfinite:
        _raise_if_nonfinite(norm)
    return norm


def _raise_if_nonfinite(norm: Tensor) -> None:
    if not math.isfinite(norm.item()):
        raise RuntimeError("the total norm of the gradients is non-finite, so it cannot be "
                           "clipped; pass error_if_nonfinite=False to scale them all the same")


def _scale_in_place(what: str, grads: List[Tensor], launch) -> Optional[Tensor]:
    """Runs launch(list of contiguous tensors) over the gradients; those that are not dense (slices of a
    larger buffer) are scaled in a copy and copied back."""
    held = _storage_order(grads)
    strided = [g is not h for g, h in zip(grads, held)]
    if True in strided:
        _refuse_strided_overlap(what, grads, strided)
    listed = ops.HostList(held)
    _refuse_overlap(what, listed, listed)
    out = launch(listed)
    with torch.no_grad():
        for g, h, copied in zip(grads, held, strided):
            if copied:
                g.copy_(h)
    torch.autograd.graph.increment_version(grads)
    return out


def clip_grads_with_norm_(parameters: Union[Tensor, Iterable[Tensor]], max_norm: float,
                          total_norm: Tensor, foreach: Optional[bool] = None) -> None:
    """Scales the parameters' gradients in place by min(1, max_norm / (total_norm + 1e-6))
    (torch's ``clip_grads_with_norm_``): for a norm formed before, over the ranks of a sharded
    model for instance. total_norm is a tensor of one value on the gradients' device."""
    del foreach
    what = "clip_grads_with_norm_"
    max_norm = _max_norm(what, max_norm)
    grads = _checked(what, _grads(parameters))
    if not grads:
        return
    dev = grads[0].device
    if not isinstance(total_norm, Tensor) or total_norm.numel() != 1:
        raise TypeError(f"{what}: total_norm must be a tensor of one value")
    _lib.require_gpu(what, grads[0], total_norm)
    norm = total_norm.detach().to(torch.float32).reshape(())

    def scale(listed: ops.HostList) -> None:
        at = norm.data_ptr()
        inside = ((listed.ptr <= at) & (at < listed.end())).any()  # one of the values to scale
        ops.grad_scale(listed, listed, norm.clone() if inside else norm, max_norm, dev)

    _scale_in_place(what, grads, scale)


def clip_grad_norm_(parameters: Union[Tensor, Iterable[Tensor]], max_norm: float,
                    norm_type: float = 2.0, error_if_nonfinite: bool = False,
                    foreach: Optional[bool] = None) -> Tensor:
    """Clips the global 2-norm of the parameters' gradients in place and returns the norm before
    clipping, a 0-dim fp32 tensor (torch's ``clip_grad_norm_``; foreach is accepted for its
    signature). Parameters without a gradient are skipped; a parameter given twice counts once.
    Gradients that share memory with one another are refused. error_if_nonfinite waits for the
    norm and raises, with the gradients unscaled, if it is not finite."""
    del foreach
    what = "clip_grad_norm_"
    _check_norm_type(what, norm_type)
    max_norm = _max_norm(what, max_norm)
    grads = _checked(what, _grads(parameters))
    if not grads:
        return torch.tensor(0.0)
    dev = grads[0].device
    if error_if_nonfinite:
        norm = ops.grad_norm(ops.HostList(_storage_order(grads)), dev)
        _raise_if_nonfinite(norm)
        _scale_in_place(what, grads, lambda t: ops.grad_scale(t, t, norm, max_norm, dev))
        return norm
    return _scale_in_place(what, grads, lambda t: ops.grad_clip(t, t, max_norm, dev))


def clipped_grads(grads: Sequence[Tensor], max_norm: float, out: Sequence[Tensor]) -> Tensor:
    """out[i] = grads[i] * min(1, max_norm / (norm + 1e-6)), norm the global 2-norm of grads,
    which is returned (0-dim fp32). out[i] has grads[i]'s shape, is contiguous, and is fp32 or of
    the gradient's dtype: fp32 main gradients of 16-bit ones, for instance. It may be grads[i]
    itself and otherwise shares no memory with any other tensor of the call."""
    what = "clipped_grads"
    max_norm = _max_norm(what, max_norm)
    grads = _checked(what, grads)
    out = _checked(what, out)
    if len(out) != len(grads):
        raise ValueError(f"{what}: {len(out)} outputs for {len(grads)} gradients")
    if not grads:
        return torch.tensor(0.0)
    for g, o in zip(grads, out):
        if o.shape != g.shape:
            raise ValueError(f"{what}: output {tuple(o.shape)} for a gradient {tuple(g.shape)}")
    for got, want in {(o.dtype, g.dtype) for g, o in zip(grads, out)}:
        if got not in (want, torch.float32):
            raise TypeError(f"{what}: output dtype {got} for a gradient of {want}")
    if not all([o.is_contiguous() for o in out]):
        raise ValueError(f"{what}: outputs must be contiguous")
    _lib.require_gpu(what, grads[0], out[0])
    src = [g if g.is_contiguous() else g.detach().contiguous() for g in grads]
    src_list, out_list = ops.HostList(src), ops.HostList(out)
    _refuse_overlap(what, out_list, src_list)
    norm = ops.grad_clip(src_list, out_list, max_norm, grads[0].device)
    torch.autograd.graph.increment_version(out)
    return norm
