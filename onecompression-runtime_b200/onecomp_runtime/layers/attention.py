"""Attention over packed sequences on B200: prompts, parts of prompts and single tokens."""
from __future__ import annotations

import math

import torch

from .. import _lib
from ._block_ops import MAX_COUNT, inference_only, on_device, one_device, overlap


def _rows(t: torch.Tensor, copy: bool = True) -> tuple[torch.Tensor, int, int, int] | None:
    """``t`` [tokens, heads, D] as the kernels address it: (tensor, pointer, token stride, head stride). A
    layout they cannot address (they need a unit stride inside a head and 16-byte aligned rows) is copied,
    or gives None. A dimension of one row gets the contiguous stride (its own may be anything)."""
    st, sh, sd = t.stride()
    T, H, D = t.shape
    if H <= 1:
        sh = D
    if T <= 1:
        st = H * D
    ptr = t.data_ptr()
    if sd == 1 and ptr % 16 == 0 and st > 0 and sh > 0 and st % 8 == 0 and sh % 8 == 0:
        return t, ptr, st, sh
    if not copy:
        return None
    t = t.contiguous()
    if t.data_ptr() % 16:
        t = t.clone()
    return t, t.data_ptr(), H * D, D


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
    device error word (``_lib.read_device_error``); a ``cu_seqlens_q`` that decreases sets it and runs no sequence
    (a new output is all zeros, a given one stays).

    ``causal``: the last query of a sequence sees its last key, query i of nq the keys up to
    ``i + nk - nq``. Rows that see no key give zeros (rows whose visible scores are all minus infinity give NaN, as
    their softmax does); what lies behind a sequence's keys never reaches a
    result, not even infinities or NaN. ``scale`` defaults to ``D ** -0.5``. ``max_seqlen_q``: the longest
    query run if the host knows it; it only helps to pick the kernel (results are right whatever it says),
    and matters where one batch holds prompts beside single tokens: the mean run counts without it.
    ``out``: [Tq, Hq, D] to write into, sharing no memory with the inputs (columns of the same buffer beside
    theirs are fine); rows that no sequence owns stay as they were (a new output holds zeros there).
    """
    what = "packed_attention"
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError(f"{what}: q, k, v are [tokens, heads, head size], got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    if k.shape != v.shape or q.shape[2] != k.shape[2]:
        raise ValueError(f"{what}: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} do not fit")
    Tq, Hq, D = q.shape
    Tk, Hkv, _ = k.shape
    if max(Tq, Tk, Hq) > MAX_COUNT:
        raise ValueError(f"{what}: {Tq} query rows, {Tk} key rows, {Hq} heads (each below 2**30)")
    if Hkv == 0 or Hq == 0 or Hq % Hkv:
        raise ValueError(f"{what}: {Hq} query heads over {Hkv} key heads")
    if D == 0 or D % 8 or D > 256:
        raise ValueError(f"{what}: head size {D} (a multiple of 8 up to 256)")
    dtype = q.dtype
    if dtype not in (torch.float16, torch.bfloat16) or k.dtype != dtype or v.dtype != dtype:
        raise TypeError(f"{what} takes fp16 or bf16 of one dtype, got {dtype}, {k.dtype}, {v.dtype}")
    if (cu_seqlens_q is None) != (cu_seqlens_k is None):
        raise ValueError(f"{what}: cu_seqlens_q and cu_seqlens_k come together")
    B = 1 if cu_seqlens_q is None else cu_seqlens_q.numel() - 1
    if B < 0:
        raise ValueError(f"{what}: cu_seqlens_q must be int32 [sequences + 1], got an empty tensor")
    for name, t, n in (("cu_seqlens_q", cu_seqlens_q, B + 1), ("cu_seqlens_k", cu_seqlens_k, B + 1),
                       ("kv_lens", kv_lens, B)):
        if t is not None and (t.dtype != torch.int32 or t.dim() != 1 or t.numel() != n):
            raise ValueError(f"{what}: {name} must be int32 [{n}], got {t.dtype} {tuple(t.shape)}")
    scale = D ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"{what}: scale {scale}")
    if out is not None and (out.shape != q.shape or out.dtype != dtype):
        raise ValueError(f"{what}: out is {out.dtype} {tuple(out.shape)}, expected {dtype} {tuple(q.shape)}")
    inference_only(what, q, k, v, out)
    dev = one_device(what, q, k, v, out, cu_seqlens_q, cu_seqlens_k, kv_lens)
    if out is not None:
        if overlap(out, q) or overlap(out, k) or overlap(out, v):
            raise ValueError(f"{what}: out shares memory with an input")
        rows_out = _rows(out, copy=False)
        if rows_out is None:
            raise ValueError(f"{what}: out needs a unit last stride and 16-byte aligned rows")
        target, o_ptr, o_st, o_sh = rows_out
        (s0, n0), (s1, n1) = sorted(((o_st, Tq), (o_sh, Hq)))
        if (n0 > 1 and s0 < D) or (n1 > 1 and s1 < (s0 * (n0 - 1) + D if n0 > 1 else D)):
            raise ValueError(f"{what}: out rows overlap (strides {out.stride()})")
    else:
        target = torch.empty((Tq, Hq, D), dtype=dtype, device=dev)
        o_ptr, o_st, o_sh = target.data_ptr(), Hq * D, D
    if Tq == 0:
        return target
    q, q_ptr, q_st, q_sh = _rows(q)
    k, k_ptr, k_st, k_sh = _rows(k)
    v, v_ptr, v_st, v_sh = _rows(v)
    cu_q = None if cu_seqlens_q is None else cu_seqlens_q.contiguous()
    cu_k = None if cu_seqlens_k is None else cu_seqlens_k.contiguous()
    lens = None if kv_lens is None else kv_lens.contiguous()
    with on_device(dev):
        run = 0 if max_seqlen_q is None else min(max(0, int(max_seqlen_q)), Tq)
        size = _lib.lib().oc_b200_attention_workspace(Tq, Tk, B, Hq, Hkv, D, run)
        ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        _lib.call("oc_b200_attention", q_ptr, q_st, q_sh, k_ptr, k_st, k_sh, v_ptr, v_st, v_sh, o_ptr, o_st, o_sh,
                  _lib.DT[dtype], Tq, Tk, Hq, Hkv, D, _lib.ptr(cu_q), _lib.ptr(cu_k), _lib.ptr(lens), B, causal, scale,
                  run, out is None, _lib.ptr(ws), size, _lib.stream_of(dev))
    return target
