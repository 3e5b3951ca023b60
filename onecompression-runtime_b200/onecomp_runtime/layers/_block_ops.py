"""Argument checks shared by the transformer-block operators (rotary positions, attention, dense linear).
They run on every call, in front of kernels of a few microseconds, so they are written for speed."""
from __future__ import annotations

import contextlib

import torch
from torch.autograd import forward_ad

from .. import _lib

MAX_COUNT = 2**30 - 1   # rows, heads and features of a call: the kernels count them, and their sums, in 32 bits
_NOTHING = contextlib.nullcontext()


def inference_only(what: str, *tensors: torch.Tensor | None) -> None:
    """The operators have no derivatives: refuse inputs that autograd would track, backward or forward."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{what} is inference only (no backward pass): call it under torch.no_grad() or "
                                   "detach the inputs")
    if forward_ad._current_level >= 0:   # inside a dual_level block; asking every tensor would cost 4 us a call
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{what} is inference only (no forward-mode derivative): pass the primals "
                                   "(torch.autograd.forward_ad.unpack_dual)")


def one_device(what: str, first: torch.Tensor, *tensors: torch.Tensor | None) -> torch.device:
    """The B200 device all tensors live on."""
    dev = first.device
    for t in tensors:
        if t is not None and t.device != dev:
            raise ValueError(f"{what}: tensors on {dev} and {t.device}")
    _lib.require_b200(dev)
    return dev


def on_device(dev: torch.device):
    """Make ``dev`` current for the launch if it is not."""
    return _NOTHING if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


def span(t: torch.Tensor) -> tuple[int, int]:
    """First byte and one past the last byte that the elements of a tensor, of one at least, touch."""
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _rows_of_pitch(t: torch.Tensor) -> dict[int, int]:
    """Ways to see the tensor as rows: {pitch: row length} in bytes, every element inside a row that begins a multiple
    of the pitch behind the first one, and no row longer than the pitch."""
    e = t.element_size()
    dims = sorted((s * e, n) for n, s in zip(t.shape, t.stride()) if n > 1 and s > 0)
    ways, length = {}, e
    for i, (s, n) in enumerate(dims):
        if length <= s and all(outer % s == 0 for outer, _ in dims[i + 1:]):
            ways[s] = length
        length += (n - 1) * s
    ways[0] = length   # all of it as one row
    return ways


def overlap(a: torch.Tensor, b: torch.Tensor | None) -> bool:
    """Whether two tensors share memory. Where their address ranges meet they do not if both are rows of one pitch that
    lie beside one another (column slices of one buffer); tensors interleaved in other ways count as sharing."""
    if b is None or a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = span(a), span(b)
    if not (a0 < b1 and b0 < a1):
        return False
    ways_a, ways_b = _rows_of_pitch(a), _rows_of_pitch(b)
    for pitch in {*ways_a, *ways_b} - {0}:   # rows of a multiple of the pitch (or one row) are rows of the pitch too
        la = min(n for p, n in ways_a.items() if p % pitch == 0)
        lb = min(n for p, n in ways_b.items() if p % pitch == 0)
        at = (b0 - a0) % pitch
        if la <= at and at + lb <= pitch:
            return False
    return True
