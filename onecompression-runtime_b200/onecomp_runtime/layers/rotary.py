"""Rotary positions on B200: half and interleaved layouts, part of the head, several position axes,
frequencies scaled for long contexts."""
from __future__ import annotations

import math

import torch

from .. import _lib
from ._block_ops import MAX_COUNT, inference_only, on_device, one_device, overlap


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: dict | None = None
                       ) -> tuple[list[float], float]:
    """Angle per position of every rotated pair, ``base ** (-2 i / rotary_dim)``, and the gain of the rotated
    values. ``scaling``: None or one of

    * ``{"type": "linear", "factor": s}``: positions divided by s;
    * ``{"type": "ntk", "factor": s}``: base times ``s ** (R / (R - 2))``, which divides the lowest frequency
      by s and keeps the highest;
    * ``{"type": "yarn", "factor": s, "original_max_position": L}``: pairs that turn more than ``beta_fast``
      (32) times over L keep their frequency, pairs that turn less than ``beta_slow`` (1) times are divided
      by s, a linear ramp between; gain ``attention_factor`` (``0.1 ln s + 1``).
    """
    half = rotary_dim // 2
    s = dict(scaling or {})
    kind = s.pop("type", None)
    factor = float(s.pop("factor", 1.0))
    if kind not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"rotary scaling type {kind!r} (linear, ntk or yarn)")
    if kind is not None and not (math.isfinite(factor) and factor >= 1.0):
        raise ValueError(f"rotary scaling factor {factor} (at least 1)")
    if not (math.isfinite(base) and base > 1.0):
        raise ValueError(f"rotary base {base} (above 1)")
    gain = 1.0
    if kind == "ntk":
        if rotary_dim <= 2:
            raise ValueError("ntk scaling needs more than one pair")
        base = base * factor ** (rotary_dim / (rotary_dim - 2.0))
    freq = [base ** (-2.0 * i / rotary_dim) for i in range(half)]
    if kind == "linear":
        freq = [f / factor for f in freq]
    if kind == "yarn":
        length = float(s.pop("original_max_position"))
        fast, slow = float(s.pop("beta_fast", 32.0)), float(s.pop("beta_slow", 1.0))
        if not (length > 0 and fast > 0 and slow > 0):
            raise ValueError("yarn scaling: original_max_position, beta_fast and beta_slow are positive")

        def pair_of(turns: float) -> float:   # the pair that turns this often over the original length
            return rotary_dim * math.log(length / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

        low, high = max(math.floor(pair_of(fast)), 0), min(math.ceil(pair_of(slow)), rotary_dim - 1)
        width = max(high - low, 1e-3)
        keep = [1.0 - min(max((i - low) / width, 0.0), 1.0) for i in range(half)]
        freq = [f * k + f / factor * (1.0 - k) for f, k in zip(freq, keep)]
        given = s.pop("attention_factor", None)
        gain = 0.1 * math.log(factor) + 1.0 if given is None else float(given)
    if s:
        raise ValueError(f"rotary scaling: unknown keys {sorted(s)}")
    return freq, gain


_NO_TENSOR = (None, 0, 0, None, 0, 0, 0)


def _out_of_place(t: torch.Tensor, T: int, D: int, dtype: torch.dtype, dev: torch.device):
    """(what the kernel reads, the new output, kernel arguments) for ``t`` [..., H, D]."""
    out = torch.empty(t.shape, dtype=dtype, device=dev)
    src = t if t.dim() == 3 else t.reshape(T, -1, D) if t.numel() else t.reshape(T, t.shape[-2], D)
    st, sh, sd = src.stride()
    if sd != 1 and D > 1:
        src = src.contiguous()
        st, sh, sd = src.stride()
    H = src.shape[1]
    return src, out, (src.data_ptr(), st, sh, out.data_ptr(), H * D, D, H)


def _in_place(what: str, t: torch.Tensor, T: int) -> tuple:
    """Kernel arguments that rotate ``t`` [..., H, D] where it lies."""
    H, D = t.shape[-2:]
    try:
        x = t if t.dim() == 3 else t.view(T, H, D)
    except RuntimeError as e:
        raise ValueError(f"{what}: in place needs token dimensions that fold into one stride, got strides "
                         f"{t.stride()}") from e
    st, sh, sd = x.stride()
    if t.numel():
        (s0, n0), (s1, n1) = sorted(((st, T), (sh, H)))
        if D > 1 and sd != 1:
            raise ValueError(f"{what}: in place needs a contiguous head, got strides {t.stride()}")
        if (n0 > 1 and s0 < D) or (n1 > 1 and s1 < (max(s0 * (n0 - 1) + D, D) if n0 > 1 else D)):
            raise ValueError(f"{what}: in place on overlapping rows (strides {t.stride()})")
    return x.data_ptr(), st, sh, x.data_ptr(), st, sh, H


def _may_overlap(a: tuple, b: tuple, D: int, size: int) -> bool:
    """False for the kernel arguments of two slices beside one another in one projection's output, the common case,
    without walking their dimensions (:func:`overlap` does for the others)."""
    pitch = a[1]
    if pitch != b[1] or pitch <= 0:
        return True
    at = (b[0] - a[0]) // size % pitch
    return at < (a[6] - 1) * a[2] + D or at + (b[6] - 1) * b[2] + D > pitch


class RotaryEmbedding(torch.nn.Module):
    """Rotates queries and keys by their positions (``oc_b200_rope``, one launch for both).

    ``rotary_dim`` of the ``head_dim`` values are rotated (default all; the rest passes through, and is copied in pairs:
    an odd head size works in place only). ``layout``:
    ``"half"`` pairs value i with i + rotary_dim/2, ``"interleaved"`` pairs neighbours. ``axes``: sizes that
    sum to ``rotary_dim`` for tokens with several coordinates (time, height, width); the pairs of section a
    turn by coordinate a, with the frequencies of a head of that size. ``scaling``: see
    :func:`rotary_frequencies` (not with ``axes``); ``inv_freq``: frequencies of the pairs, instead of base
    and scaling.

    Angles are 64-bit fixed point modulo one turn, for any integer position: off by 2^-25 of a half turn, plus
    position times the table's rounding (2^-52 of the frequency, as doubles have it, and 2^-64 of a half turn).
    The module has no buffers, so it survives a build on the meta device; the table of a device is copied
    there by the first call on it (or by ``device=``), which belongs before a graph capture.
    """

    def __init__(self, head_dim: int, *, rotary_dim: int | None = None, base: float = 10000.0,
                 layout: str = "half", axes: list[int] | None = None, scaling: dict | None = None,
                 inv_freq: torch.Tensor | list[float] | None = None, device=None) -> None:
        super().__init__()
        self.head_dim = int(head_dim)
        self.rotary_dim = self.head_dim if rotary_dim is None else int(rotary_dim)
        R = self.rotary_dim
        if not (0 < R <= self.head_dim <= 1024) or R % 2:
            raise ValueError(f"rotary_dim {R} of head size {head_dim} (even, at most the head; heads up to 1024)")
        if layout not in ("half", "interleaved"):
            raise ValueError(f"rotary layout {layout!r} (half or interleaved)")
        self.layout = layout
        self.axes = None if axes is None else [int(a) for a in axes]
        gain = 1.0
        if inv_freq is not None:
            if scaling is not None:
                raise ValueError("inv_freq already holds the scaled frequencies")
            freq = inv_freq.detach().double().cpu().reshape(-1).tolist() if isinstance(inv_freq, torch.Tensor) \
                else [float(f) for f in inv_freq]
            if len(freq) != R // 2 or not all(math.isfinite(f) for f in freq):
                raise ValueError(f"inv_freq needs {R // 2} finite values")
        if self.axes is not None:
            if not self.axes or any(a <= 0 or a % 2 for a in self.axes) or sum(self.axes) != R or len(self.axes) > 255:
                raise ValueError(f"axes {axes} must be even sizes that sum to rotary_dim {R}")
            if scaling is not None:
                raise ValueError("scaling with axes: give inv_freq")
            if inv_freq is None:
                freq = [f for a in self.axes for f in rotary_frequencies(a, base)[0]]
        elif inv_freq is None:
            freq, gain = rotary_frequencies(R, base, scaling)
        self.inv_freq, self.gain = freq, float(gain)
        self._interleaved = layout == "interleaved"
        # fraction of a turn per position as 0.64 fixed point (two's complement bits in int64)
        turns = [int(round(math.fmod(f / (2.0 * math.pi), 1.0) * 2.0 ** 64)) % 2 ** 64 for f in freq]
        self._turns = [t - 2 ** 64 if t >= 2 ** 63 else t for t in turns]
        self._tables: dict[int, tuple[torch.Tensor, torch.Tensor | None]] = {}
        if device is not None and torch.device(device).type == "cuda":
            dev = torch.device(device)
            self._table(torch.device("cuda", torch.cuda.current_device() if dev.index is None else dev.index))

    def _table(self, dev: torch.device):
        t = self._tables.get(dev.index)
        if t is None:
            axis = None
            if self.axes is not None:
                ids = [i for i, a in enumerate(self.axes) for _ in range(a // 2)]
                axis = torch.tensor(ids, dtype=torch.uint8, device="cpu").to(dev)
            t = self._tables[dev.index] = (torch.tensor(self._turns, dtype=torch.int64, device="cpu").to(dev), axis)
        return t

    def forward(self, q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, inplace: bool = False):
        """``q`` [..., Hq, head_dim] and ``k`` [..., Hk, head_dim] (or None) over the same leading token
        dimensions, fp16, bf16 or fp32 of one dtype, any strides with a contiguous head; ``positions`` int32 or
        int64 [...], with ``axes`` [..., len(axes)]. Returns the rotated ``(q, k)``, rounded once; ``inplace``
        writes into the inputs (which may be slices of one projection's output)."""
        what = "RotaryEmbedding"
        D, dtype = self.head_dim, q.dtype
        q_shape, p_shape = q.shape, positions.shape
        tokens, A = q_shape[:-2], 1
        fits = q.dim() >= 3 and q_shape[-1] == D
        if self.axes is None:
            fits_p = p_shape == tokens
        else:
            A = len(self.axes)
            fits_p = p_shape[:-1] == tokens and positions.dim() > 0 and p_shape[-1] == A
        if not fits or (k is not None and (k.dim() != q.dim() or k.shape[-1] != D or k.shape[:-2] != tokens)):
            raise ValueError(f"{what}: q {tuple(q_shape)}, k {None if k is None else tuple(k.shape)}, expected "
                             f"{(*tokens, 'heads', D)}")
        pos_dtype = positions.dtype
        if not fits_p or (pos_dtype is not torch.int64 and pos_dtype is not torch.int32):
            raise ValueError(f"{what}: positions {pos_dtype} {tuple(p_shape)}, expected int32 or int64 "
                             f"{tuple(tokens) if self.axes is None else (*tokens, A)}")
        if dtype not in _lib.DT or (k is not None and k.dtype is not dtype):
            raise TypeError(f"{what} takes fp16, bf16 or fp32 of one dtype, got {dtype} and "
                            f"{None if k is None else k.dtype}")
        T = q_shape[0] if len(tokens) == 1 else math.prod(tokens)
        if max(T, q_shape[-2], 0 if k is None else k.shape[-2]) > MAX_COUNT:
            raise ValueError(f"{what}: {T} tokens, {q_shape[-2]} query heads (each below 2**30)")
        if D % 2 and not inplace:
            raise ValueError(f"{what}: head size {D} must be even out of place")
        inference_only(what, q, k)
        dev = one_device(what, q, k, positions)
        if inplace:
            q_out, k_out = q, k
            q_args = _in_place(what, q, T)
            k_args = _NO_TENSOR if k is None else _in_place(what, k, T)
            if k is not None and _may_overlap(q_args, k_args, D, q.element_size()) and overlap(q, k):
                raise ValueError(f"{what}: in place on q and k that share memory")
        else:
            q, q_out, q_args = _out_of_place(q, T, D, dtype, dev)
            k_out, k_args = None, _NO_TENSOR
            if k is not None:
                k, k_out, k_args = _out_of_place(k, T, D, dtype, dev)
        if T == 0:
            return q_out, k_out
        turns, axis = self._tables.get(dev.index) or self._table(dev)
        pos_st = 1
        if A > 1 or positions.dim() != 1 or positions.stride(0) != 1:
            positions = positions.reshape(T, A)
            if A > 1 and positions.stride(1) != 1:
                positions = positions.contiguous()
            pos_st = positions.stride(0)
        with on_device(dev):
            _lib.call("oc_b200_rope", *q_args, *k_args, _lib.DT[dtype], T, D, self.rotary_dim, positions.data_ptr(),
                      pos_dtype is torch.int64, pos_st, turns.data_ptr(), None if axis is None else axis.data_ptr(),
                      self.gain, self._interleaved, _lib.stream_of(dev))
        return q_out, k_out

    def extra_repr(self) -> str:
        return (f"head_dim={self.head_dim}, rotary_dim={self.rotary_dim}, layout={self.layout}, axes={self.axes}, "
                f"gain={self.gain}")
