"""Dense 16-bit linear on B200 with bias, activation and residual in its epilogue, for the layers of a
checkpoint that are not packed (or that ``build_eager`` dequantized)."""
from __future__ import annotations

import torch

from .. import _lib
from ._block_ops import MAX_COUNT, inference_only, on_device, one_device, overlap

ACTIVATIONS = {None: 0, "none": 0, "gelu_tanh": 1, "gelu": 2, "silu": 3, "relu": 4}


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """Rows the TMA can read (unit column stride, 16-byte aligned rows), or a contiguous copy."""
    rows = t.shape[0] <= 1 or (t.stride(0) % 8 == 0 and t.stride(0) >= t.shape[1])
    if not rows or t.stride(1) != 1 or t.data_ptr() % 16:
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
    return t


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _output(what: str, out: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None,
            residual: torch.Tensor | None, M: int, N: int) -> tuple[int, int]:
    """Pointer and row stride of a given output."""
    try:
        rows = out.view(M, N)
    except RuntimeError as e:
        raise ValueError(f"{what}: out's leading dimensions must fold into one stride, got {out.stride()}") from e
    if rows.numel() and N > 1 and rows.stride(1) != 1:
        raise ValueError(f"{what}: out needs a unit column stride, got {out.stride()}")
    if M > 1 and rows.stride(0) < N:
        raise ValueError(f"{what}: out rows overlap (strides {out.stride()})")
    if overlap(rows, x) or overlap(rows, weight) or overlap(rows, bias):
        raise ValueError(f"{what}: out shares memory with an input")
    if residual is not None and overlap(rows, residual) and \
            (residual.data_ptr(), _ld(residual), residual.stride(1)) != (rows.data_ptr(), _ld(rows), rows.stride(1)):
        raise ValueError(f"{what}: out overlaps the residual but is not the residual itself")
    return rows.data_ptr(), _ld(rows)


def linear_fused(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                 activation: str | None = None, residual: torch.Tensor | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual`` in one kernel: fp32 accumulation and epilogue, one rounding.

    ``x`` [..., K] and ``weight`` [N, K] fp16 or bf16 of one dtype, K a multiple of 8; ``bias`` [N] fp16, bf16
    or fp32; ``activation`` None, ``"gelu_tanh"``, ``"gelu"``, ``"silu"`` or ``"relu"``; ``residual`` and
    ``out`` [..., N] in ``x``'s dtype, ``out`` may be ``residual`` itself and otherwise shares no memory with
    the inputs (columns of the same buffer beside theirs are fine). Rows of ``x`` and ``weight`` that are not
    contiguous or not 16-byte aligned are copied.
    """
    what = "linear_fused"
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"{what}: x {tuple(x.shape)} and weight {tuple(weight.shape)} do not fit")
    N, K = weight.shape
    M = x.numel() // max(K, 1)
    if max(M, N, K) > MAX_COUNT:
        raise ValueError(f"{what}: {M} rows, {N} x {K} weights (each below 2**30)")
    if K == 0 or K % 8:
        raise ValueError(f"{what}: K={K} must be a multiple of 8")
    if x.dtype not in (torch.float16, torch.bfloat16) or weight.dtype != x.dtype:
        raise TypeError(f"{what} takes fp16 or bf16 of one dtype, got {x.dtype} and {weight.dtype}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"{what}: activation {activation!r}, one of {sorted(a for a in ACTIVATIONS if a)}")
    if bias is not None and (bias.shape != (N,) or bias.dtype not in _lib.DT):
        raise ValueError(f"{what}: bias {bias.dtype} {tuple(bias.shape)}, expected [{N}] fp16, bf16 or fp32")
    shape = (*x.shape[:-1], N)
    for name, t in (("residual", residual), ("out", out)):
        if t is not None and (t.shape != shape or t.dtype != x.dtype):
            raise ValueError(f"{what}: {name} {t.dtype} {tuple(t.shape)}, expected {x.dtype} {shape}")
    inference_only(what, x, weight, bias, residual, out)
    dev = one_device(what, x, weight, bias, residual, out)
    x2 = x if x.dim() == 2 else x.reshape(-1, K)
    res2 = residual if residual is None or residual.dim() == 2 else residual.reshape(M, N)
    if out is None:
        target = torch.empty(shape, dtype=x.dtype, device=dev)
        o_ptr, ldc = target.data_ptr(), N
    else:
        target = out
        o_ptr, ldc = _output(what, out, x, weight, bias, res2, M, N)
    if M == 0 or N == 0:
        return target
    x2, w2 = _aligned(x2), _aligned(weight)
    if res2 is not None and (res2.stride(1) != 1 or (M > 1 and res2.stride(0) < N)):
        res2 = res2.contiguous()
    b = None if bias is None else bias.contiguous()
    with on_device(dev):
        _lib.call("oc_b200_dense_gemm", x2.data_ptr(), _ld(x2), w2.data_ptr(), _ld(w2), _lib.DT[x.dtype], M, N, K,
                  _lib.ptr(b), 0 if b is None else _lib.DT[b.dtype], _lib.ptr(res2), 0 if res2 is None else _ld(res2),
                  ACTIVATIONS[activation], o_ptr, ldc, _lib.stream_of(dev))
    return target


class EagerLinear(torch.nn.Linear):
    """The dense layer ``build_eager`` makes: ``nn.Linear``, with the ``forward_fused`` of the packed layers."""

    def forward_fused(self, x: torch.Tensor, residual: torch.Tensor | None = None,
                      activation: str | None = None) -> torch.Tensor:
        """``act(x @ W.T + bias) + residual`` in one kernel (:func:`linear_fused`, whose dtypes and multiple of 8
        input features it needs), one rounding."""
        bias = None if self.bias is None else self.bias.detach()
        return linear_fused(x, self.weight.detach(), bias, activation=activation, residual=residual)
