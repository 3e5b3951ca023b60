"""Attention over packed sequences on B200: prompts, parts of prompts and single tokens."""
from __future__ import annotations

import functools
import math

import torch

from .. import _lib
from ._block_ops import inference_only, on_device, one_device, overlap


@functools.lru_cache(maxsize=None)
def _workspace_bytes(device_index: int, head_dim: int) -> int:
    with torch.cuda.device(device_index):
        return _lib.lib().oc_b200_attention_workspace(head_dim)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` [tokens, heads, D] if the kernels can address it (unit stride inside a head, 16-byte aligned
    rows), else a contiguous copy."""
    ok = t.stride(2) == 1 and t.data_ptr() % 16 == 0
    ok = ok and all(n <= 1 or (s > 0 and s % 8 == 0) for n, s in zip(t.shape[:2], t.stride()[:2]))
    if not ok:
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
    return t


def _strides(t: torch.Tensor) -> tuple[int, int]:
    """Token and head strides; a dimension of one row gets the contiguous one (its own may be anything)."""
    head = t.stride(1) if t.shape[1] > 1 else t.shape[2]
    return (t.stride(0) if t.shape[0] > 1 else t.shape[1] * t.shape[2]), head


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor | None = None,
                     cu_seqlens_k: torch.Tensor | None = None, *, kv_lens: torch.Tensor | None = None,
                     causal: bool = True, scale: float | None = None, max_seqlen_q: int | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """``softmax(scale * q @ k.T) @ v`` per sequence and head, fp32 softmax and sums, one rounding.

    ``q`` [Tq, Hq, D]; ``k``, ``v`` [Tk, Hkv, D], fp16 or bf16, Hq a multiple of Hkv (query head h reads key
    head ``h // (Hq // Hkv)``), D a multiple of 8 up to 256. Any token and head strides, so the column slices
    of one qkv projection go in as they are (a last dimension that is not contiguous, rows off 16-byte
    boundaries and expanded dimensions are copied).

    ``cu_seqlens_q`` / ``cu_seqlens_k``: int32 [B + 1] on the device, first row of each sequence (given
    together; without them all rows are one sequence). ``kv_lens``: int32 [B], how many keys from
    ``cu_seqlens_k[b]`` on are in use: a cache with room for more. They are read on the device when the kernel
    runs, so a captured graph follows their values. Values outside the tensors are clamped and set the
    device error word (``_lib.read_device_error``).

    ``causal``: the last query of a sequence sees its last key, query i of nq the keys up to
    ``i + nk - nq``. Rows that see no key give zeros; what lies behind a sequence's keys never reaches a
    result, not even infinities or NaN. ``scale`` defaults to ``D ** -0.5``. ``max_seqlen_q``: the longest
    query run if the host knows it; it only helps to pick the kernel (results are right whatever it says).
    ``out``: [Tq, Hq, D] to write into, sharing no memory with the inputs; rows that no sequence owns stay as
    they were (a new output holds zeros behind the last sequence).
    """
    what = "packed_attention"
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError(f"{what}: q, k, v are [tokens, heads, head size], got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    if k.shape != v.shape or q.shape[2] != k.shape[2]:
        raise ValueError(f"{what}: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} do not fit")
    Tq, Hq, D = q.shape
    Tk, Hkv = k.shape[:2]
    if Hkv == 0 or Hq == 0 or Hq % Hkv:
        raise ValueError(f"{what}: {Hq} query heads over {Hkv} key heads")
    if D == 0 or D % 8 or D > 256:
        raise ValueError(f"{what}: head size {D} (a multiple of 8 up to 256)")
    if q.dtype not in (torch.float16, torch.bfloat16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"{what} takes fp16 or bf16 of one dtype, got {q.dtype}, {k.dtype}, {v.dtype}")
    if (cu_seqlens_q is None) != (cu_seqlens_k is None):
        raise ValueError(f"{what}: cu_seqlens_q and cu_seqlens_k come together")
    tables = (cu_seqlens_q, cu_seqlens_k, kv_lens)
    B = 1 if cu_seqlens_q is None else cu_seqlens_q.numel() - 1
    for name, t, n in zip(("cu_seqlens_q", "cu_seqlens_k", "kv_lens"), tables, (B + 1, B + 1, B)):
        if t is not None and (t.dtype != torch.int32 or t.dim() != 1 or t.numel() != n or n < 1):
            raise ValueError(f"{what}: {name} must be int32 [{max(n, 1)}], got {t.dtype} {tuple(t.shape)}")
    if scale is None:
        scale = D ** -0.5
    if not math.isfinite(scale):
        raise ValueError(f"{what}: scale {scale}")
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype):
        raise ValueError(f"{what}: out is {out.dtype} {tuple(out.shape)}, expected {q.dtype} {tuple(q.shape)}")
    inference_only(what, q, k, v, out)
    dev = one_device(what, q, k, v, out, *tables)
    if out is not None:
        if any(overlap(out, t) for t in (q, k, v)):
            raise ValueError(f"{what}: out shares memory with an input")
        if Tq and _rows(out) is not out:
            raise ValueError(f"{what}: out needs a unit last stride and 16-byte aligned rows")
        target = out
    else:
        target = torch.empty((Tq, Hq, D), dtype=q.dtype, device=dev)
    if Tq == 0:
        return target
    q, k, v = _rows(q), _rows(k), _rows(v)
    cu_q, cu_k, lens = (None if t is None else t.contiguous() for t in tables)
    with on_device(dev):
        ws = torch.empty(_workspace_bytes(dev.index, D), dtype=torch.uint8, device=dev)
        _lib.call("oc_b200_attention", q.data_ptr(), *_strides(q), k.data_ptr(), *_strides(k), v.data_ptr(),
                  *_strides(v), target.data_ptr(), *_strides(target), _lib.DT[q.dtype], Tq, Tk, Hq, Hkv, D,
                  _lib.ptr(cu_q), _lib.ptr(cu_k), _lib.ptr(lens), B, int(causal), float(scale),
                  0 if max_seqlen_q is None else max(0, int(max_seqlen_q)), int(out is None), ws.data_ptr(),
                  ws.numel(), _lib.stream_of(dev))
    return target
