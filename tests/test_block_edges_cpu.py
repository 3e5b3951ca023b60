"""Calls of the transformer-block operators at the edges of what their documentation allows: what the host decides."""
from __future__ import annotations

import random

import pytest
import torch


def zeros(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def test_forward_mode_derivatives_are_refused():
    """An input that carries a tangent would lose it without a word; inputs without one go on inside the same block
    (to the refusal of CPU tensors here), and so does the primal of a dual tensor."""
    from torch.autograd import forward_ad
    from onecomp_runtime.layers import EagerLinear, RotaryEmbedding, linear_fused, packed_attention
    a, x, w, pos = zeros(3, 4, 64), zeros(3, 64), zeros(40, 64), torch.arange(3)
    rope = RotaryEmbedding(64)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        lin = EagerLinear(64, 40, dtype=torch.bfloat16)
        for call in (lambda: packed_attention(dual(a), a, a), lambda: packed_attention(a, dual(a), a),
                     lambda: packed_attention(a, a, dual(a)), lambda: rope(dual(a), a, pos), lambda: rope(a, dual(a), pos),
                     lambda: linear_fused(dual(x), w), lambda: linear_fused(x, dual(w)),
                     lambda: linear_fused(x, w, dual(zeros(40))), lambda: linear_fused(x, w, residual=dual(zeros(3, 40))),
                     lambda: lin.forward_fused(dual(x))):
            for guard in (torch.no_grad(), torch.enable_grad()):
                with guard, pytest.raises(RuntimeError, match="forward-mode"):
                    call()
        primal = forward_ad.unpack_dual(dual(a)).primal
        for call in (lambda: packed_attention(a, a, primal), lambda: rope(a, primal, pos), lambda: linear_fused(x, w)):
            with pytest.raises(RuntimeError, match="CUDA"):
                call()


def pi_by_machin(digits: int):
    """pi as a fraction, from 16 atan(1/5) - 4 atan(1/239), to this many decimals."""
    from fractions import Fraction

    def atan_inverse(n):
        total, k = Fraction(0), 0
        while n ** (2 * k + 1) < 10 ** (digits + 5):
            total += Fraction((-1) ** k, (2 * k + 1) * n ** (2 * k + 1))
            k += 1
        return total

    return 16 * atan_inverse(5) - 4 * atan_inverse(239)


@pytest.mark.parametrize("kw", [{}, dict(base=1e6), dict(scaling={"type": "ntk", "factor": 8.0}),
                                dict(scaling={"type": "yarn", "factor": 16.0, "original_max_position": 32768}),
                                dict(inv_freq=[1.0, 3.0, -1.0, 0.75, 6.25, -1e-9, 123.456, 0.0] * 4)])
def test_rotary_table_against_long_arithmetic(kw):
    """A fraction of a turn is off by 2^-52 of itself before it is taken modulo one turn: division and 2 pi are each
    rounded to a double (2^-53 and 2^-54 relative), and to a unit of 2^-64."""
    from fractions import Fraction
    from onecomp_runtime.layers import RotaryEmbedding
    two_pi = 2 * pi_by_machin(50)
    rope = RotaryEmbedding(64, **kw)
    for f, t in zip(rope.inv_freq, rope._turns):
        exact = Fraction(f) / two_pi
        off = (t - exact * 2**64) % 2**64
        assert min(off, 2**64 - off) <= abs(exact) * 2**12 + 1, (f, float(off))
        assert -2**63 <= t < 2**63


def test_attention_takes_the_lengths_of_an_empty_batch():
    """No sequence: the tables hold one entry and kv_lens none. Past the checks such a call ends here in the refusal
    of CPU tensors; wrong sizes and empty tables are refused before."""
    from onecomp_runtime.layers import packed_attention
    a, one, none = zeros(3, 4, 64), torch.zeros(1, dtype=torch.int32), torch.zeros(0, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        packed_attention(a, a, a, one, one, kv_lens=none)
    with pytest.raises(ValueError, match="kv_lens"):
        packed_attention(a, a, a, one, one, kv_lens=one)
    with pytest.raises(ValueError, match="cu_seqlens_q"):
        packed_attention(a, a, a, none, none)
    with pytest.raises(ValueError, match="cu_seqlens_q"):
        packed_attention(a, a, a, none, one, kv_lens=none)


def addresses(t):
    """The byte addresses of a tensor's elements."""
    if t.numel() == 0:
        return set()
    at = torch.zeros(t.shape, dtype=torch.int64)
    for d, (n, s) in enumerate(zip(t.shape, t.stride())):
        at += (torch.arange(n) * s).view([-1 if i == d else 1 for i in range(t.dim())])
    e = t.element_size()
    return {t.data_ptr() + e * int(x) + i for x in at.flatten() for i in range(e)}


def test_shared_memory_is_seen():
    """Random strided tensors over one buffer: whatever shares a byte is found to share memory."""
    from onecomp_runtime.layers._block_ops import overlap
    rng, found = random.Random(3), [0, 0]
    buf = torch.zeros(4096, dtype=torch.int16)
    for _ in range(3000):
        pair = []
        for _ in range(2):
            n = rng.choice([1, 2, 3])
            shape = [rng.choice([1, 2, 3, 5]) for _ in range(n)]
            stride = [rng.choice([0, 1, 2, 4, 6, 8, 16, 24, 48, 96]) for _ in range(n)]
            x = buf.as_strided(shape, stride, rng.randrange(200))
            pair.append(x if rng.random() < 0.8 or any(s % 2 for s in stride) else
                        buf.view(torch.float32).as_strided(shape, [s // 2 for s in stride], rng.randrange(100)))
        a, b = pair
        shares = bool(addresses(a) & addresses(b))
        assert overlap(a, b) == overlap(b, a)
        assert overlap(a, b) or not shares, (a.shape, a.stride(), a.storage_offset(), b.shape, b.stride(), b.storage_offset())
        found[shares] += 1
    assert min(found) > 300


def test_slices_of_one_buffer_share_nothing():
    """What a user keeps side by side in one buffer: columns of a projection, a head's parts, blocks of rows."""
    from onecomp_runtime.layers._block_ops import overlap
    b = zeros(7, 6 * 64)
    q, o = b[:, :128].unflatten(1, (2, 64)), b[:, 256:].unflatten(1, (2, 64))
    heads, wide = zeros(7, 4, 3, 64), zeros(6, 8, 64)
    batch = zeros(2, 5, 96)
    for x, y in ((q, o), (b[:, :100], b[:, 100:]), (heads[:, :, 0], heads[:, :, 2]), (batch[..., :32], batch[..., 32:]),
                 (b[:3], b[3:]), (b[:, :64], b[2, 64:]), (b[1:, :8], b[:-1, 376:]), (heads[:, 0], heads[:, 1:]),
                 (heads[:, :, 1, :8], heads[:, :, 1, 8:]), (wide[:, ::2], wide[:, 1:2]), (wide[::2], wide[1:2, 3:]),
                 (wide[:, ::4], wide[1:3, 2::4])):
        assert not overlap(x, y) and not overlap(y, x) and not addresses(x) & addresses(y)
    for x, y in ((q, b[:, 64:192].unflatten(1, (2, 64))), (b[:, :101], b[:, 100:]), (b[:4], b[3:]), (b, b), (b[:, 64:], b[2, 64:])):
        assert overlap(x, y) and overlap(y, x)


def test_rotary_in_place_refuses_shared_memory(monkeypatch):
    """q and k that meet anywhere would be rotated twice or half; slices beside one another go on (here to the device's
    refusal, which comes first, so it is taken out of the way and the launch with it)."""
    from onecomp_runtime.layers import RotaryEmbedding, rotary
    rope, pos, launched = RotaryEmbedding(64), torch.arange(6), []
    monkeypatch.setattr(rotary, "one_device", lambda what, q, *more: q.device)
    monkeypatch.setattr(rotary.RotaryEmbedding, "_table", lambda self, dev: (pos, None))
    monkeypatch.setattr(rotary, "on_device", lambda dev: torch.no_grad())
    monkeypatch.setattr(rotary._lib, "stream_of", lambda dev: 0)
    monkeypatch.setattr(rotary._lib, "call", lambda *a: launched.append(a))
    b = zeros(6, 8 * 64)

    def heads(lo, hi):
        return b[:, lo * 64:hi * 64].unflatten(1, (hi - lo, 64))

    inner = zeros(6, 4, 3, 64)
    for q, k in ((heads(0, 4), heads(4, 6)), (heads(4, 8), heads(0, 4)), (b[:3].view(3, 8, 64), b[3:].view(3, 8, 64)),
                 (inner[:, :, 0], inner[:, :, 1]), (zeros(6, 2, 64), zeros(6, 2, 64)), (heads(0, 2)[:1], heads(1, 3)[1:2])):
        rope(q, k, pos[:len(q)], inplace=True)
    assert len(launched) == 6
    rope(heads(0, 4), heads(2, 2), pos, inplace=True)      # no key head: nothing to share
    launched.pop()
    for q, k in ((heads(0, 4), heads(0, 4)), (heads(0, 4), heads(3, 6)), (heads(2, 4), heads(1, 3)), (heads(3, 4), heads(0, 8)),
                 (b[:4].view(4, 8, 64), b[2:].view(4, 8, 64)), (inner[:, :, 0], inner[:, 0]),
                 (b[:, 1:129].unflatten(1, (2, 64)), heads(2, 3))):
        with pytest.raises(ValueError, match="share memory"):
            rope(q, k, pos[:len(q)], inplace=True)
    assert len(launched) == 6


def test_dense_tile_query_refuses():
    import ctypes
    from onecomp_runtime import _lib
    lib, n, f = _lib.lib(), ctypes.c_int(), ctypes.c_int()
    for args in ((0, 8, 8), (8, 0, 8), (8, 8, -8), (1 << 30, 8, 8), (8, 1 << 30, 8), (8, 8, 1 << 30)):
        assert lib.oc_b200_dense_gemm_tile(*args, ctypes.byref(n), ctypes.byref(f)) == 1
    assert lib.oc_b200_dense_gemm_tile(8, 8, 8, None, ctypes.byref(f)) == 1
    assert lib.oc_b200_dense_gemm_tile(8, 8, 8, ctypes.byref(n), None) == 1


def test_rotary_odd_heads_out_of_place_are_refused():
    """The values behind the rotated part are copied in pairs; in place nothing is copied (and the CPU is refused)."""
    import ctypes
    from onecomp_runtime import _lib
    from onecomp_runtime.layers import RotaryEmbedding
    rope, x = RotaryEmbedding(65, rotary_dim=64), zeros(3, 2, 65)
    with pytest.raises(ValueError, match="even out of place"):
        rope(x, None, torch.arange(3))
    with pytest.raises(RuntimeError, match="CUDA"):
        rope(x, None, torch.arange(3), inplace=True)
    p, o = ctypes.c_void_p(0x10000), ctypes.c_void_p(0x20000)
    assert _lib.lib().oc_b200_rope(p, 130, 65, o, 130, 65, 2, None, 0, 0, None, 0, 0, 0, 1, 3, 65, 64, p, 1, 1, p, None, 1.0, 0,
                                   None) == 1
    assert "even out of place" in _lib.last_error()


def test_rotary_counts_of_heads():
    """Heads up to 2^30, as the header says; more are refused before any launch."""
    import ctypes
    from onecomp_runtime import _lib
    from onecomp_runtime.layers import RotaryEmbedding
    p = ctypes.c_void_p(0x10000)
    for Hq, Hk in ((1 << 30, 0), (1, 1 << 30)):
        assert _lib.lib().oc_b200_rope(p, 8, 8, p, 8, 8, Hq, p, 8, 8, p, 8, 8, Hk, 1, 1, 8, 8, p, 1, 1, p, None, 1.0, 0, None) == 1
        assert "below 2^30" in _lib.last_error()
    one = zeros(1, 1, 8)
    with pytest.raises(ValueError, match="2\\*\\*30"):
        RotaryEmbedding(8)(one, one.expand(1, 2**30, 8), torch.arange(1))
