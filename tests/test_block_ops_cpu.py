"""Refusals and host-side formulas of the transformer-block operators (no GPU needed)."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch


def q(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("args,kw,err", [
    ((q(3, 64), q(3, 2, 64), q(3, 2, 64)), {}, "tokens, heads"),
    ((q(3, 4, 64), q(3, 2, 64), q(4, 2, 64)), {}, "do not fit"),
    ((q(3, 4, 64), q(3, 2, 32), q(3, 2, 32)), {}, "do not fit"),
    ((q(3, 5, 64), q(3, 2, 64), q(3, 2, 64)), {}, "query heads"),
    ((q(3, 4, 64), q(3, 0, 64), q(3, 0, 64)), {}, "query heads"),
    ((q(3, 4, 60), q(3, 2, 60), q(3, 2, 60)), {}, "multiple of 8"),
    ((q(3, 4, 264), q(3, 2, 264), q(3, 2, 264)), {}, "multiple of 8"),
    ((q(3, 4, 64), q(3, 2, 64), q(3, 2, 64)), dict(cu_seqlens_q=torch.zeros(2, dtype=torch.int32)), "together"),
    ((q(3, 4, 64), q(3, 2, 64), q(3, 2, 64)), dict(cu_seqlens_q=torch.zeros(2), cu_seqlens_k=torch.zeros(2)), "int32"),
    ((q(3, 4, 64), q(3, 2, 64), q(3, 2, 64)), dict(cu_seqlens_q=torch.zeros(3, dtype=torch.int32),
                                                   cu_seqlens_k=torch.zeros(2, dtype=torch.int32)), "cu_seqlens_k"),
    ((q(3, 4, 64), q(3, 2, 64), q(3, 2, 64)), dict(kv_lens=torch.zeros(2, dtype=torch.int32)), "kv_lens"),
    ((q(3, 4, 64), q(3, 2, 64), q(3, 2, 64)), dict(scale=math.nan), "scale"),
    ((q(3, 4, 64), q(3, 2, 64), q(3, 2, 64)), dict(out=q(3, 4, 32)), "out is"),
])
def test_attention_refuses(args, kw, err):
    from onecomp_runtime.layers import packed_attention
    with pytest.raises(ValueError, match=err):
        packed_attention(*args, **kw)


def test_attention_refuses_types_devices_and_autograd():
    from onecomp_runtime.layers import packed_attention
    a = q(3, 4, 64)
    with pytest.raises(TypeError):
        packed_attention(a.float(), a.float(), a.float())
    with pytest.raises(TypeError):
        packed_attention(a, a.half(), a)
    with pytest.raises(RuntimeError, match="CUDA"):
        packed_attention(a, a, a)
    with pytest.raises(RuntimeError, match="inference only"):
        packed_attention(a.clone().requires_grad_(), a, a)


def test_rope_refuses():
    from onecomp_runtime.layers import RotaryEmbedding
    for kw in (dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=66), dict(layout="pairs"), dict(base=1.0),
               dict(axes=[16, 16]), dict(axes=[63, 1]), dict(axes=[]), dict(scaling={"type": "cubic"}),
               dict(scaling={"type": "linear", "factor": 0.5}), dict(scaling={"type": "linear", "factor": 2, "x": 1}),
               dict(axes=[32, 32], scaling={"type": "linear", "factor": 2}), dict(inv_freq=[1.0]),
               dict(inv_freq=[math.inf] * 32), dict(inv_freq=[1.0] * 32, scaling={"type": "linear", "factor": 2})):
        with pytest.raises(ValueError):
            RotaryEmbedding(64, **kw)
    with pytest.raises(KeyError):
        RotaryEmbedding(64, scaling={"type": "yarn", "factor": 2})
    rope = RotaryEmbedding(64)
    pos = torch.arange(3)
    with pytest.raises(ValueError, match="positions"):
        rope(q(3, 4, 64), None, pos.float())
    with pytest.raises(ValueError, match="positions"):
        rope(q(3, 4, 64), None, torch.arange(4))
    with pytest.raises(ValueError, match="expected"):
        rope(q(3, 4, 32), None, pos)
    with pytest.raises(ValueError, match="k "):
        rope(q(3, 4, 64), q(2, 4, 64), pos)
    with pytest.raises(TypeError):
        rope(q(3, 4, 64), q(3, 4, 64, dtype=torch.float16), pos)
    with pytest.raises(RuntimeError, match="CUDA"):
        rope(q(3, 4, 64), None, pos)
    with pytest.raises(RuntimeError, match="inference only"):
        rope(q(3, 4, 64).requires_grad_(), None, pos)


def test_rope_survives_the_meta_device():
    """Built on the meta device like the loader's models: the table is host data until a call needs it."""
    from onecomp_runtime.layers import RotaryEmbedding
    with torch.device("meta"):
        rope = RotaryEmbedding(128, axes=[16, 56, 56])
    assert len(rope.inv_freq) == 64 and not list(rope.buffers()) and not list(rope.parameters())


def test_rotary_frequencies():
    from onecomp_runtime.layers import RotaryEmbedding, rotary_frequencies
    plain, gain = rotary_frequencies(64)
    assert gain == 1.0 and plain[0] == 1.0 and math.isclose(plain[31], 10000.0 ** (-62 / 64))
    lin, _ = rotary_frequencies(64, scaling={"type": "linear", "factor": 4.0})
    assert all(math.isclose(a, b / 4) for a, b in zip(lin, plain))
    ntk, _ = rotary_frequencies(64, scaling={"type": "ntk", "factor": 8.0})
    assert ntk[0] == 1.0 and math.isclose(ntk[31], plain[31] / 8.0)
    yarn, g = rotary_frequencies(64, scaling={"type": "yarn", "factor": 16.0, "original_max_position": 4096})
    turns = [4096 * f / (2 * math.pi) for f in plain]
    for f, p, t in zip(yarn, plain, turns):
        assert p / 16.0 * (1 - 1e-12) <= f <= p * (1 + 1e-12)
        if t > 2 * 32:
            assert math.isclose(f, p)
        if t < 0.5:
            assert math.isclose(f, p / 16)
    assert math.isclose(g, 0.1 * math.log(16.0) + 1.0)
    # the fixed-point table holds the fraction of a turn to 2^-53 of itself
    rope = RotaryEmbedding(64, inv_freq=[7.5, -0.25] + [1e-3] * 30)
    for f, t in zip(rope.inv_freq, rope._turns):
        assert abs(t / 2.0**64 - f / (2 * math.pi) + round(f / (2 * math.pi) - t / 2.0**64)) < 1e-15


def test_linear_refuses():
    from onecomp_runtime.layers import linear_fused
    x, w = q(3, 64), q(40, 64)
    for args, kw in (((x, q(40, 32)), {}), ((q(3, 12), q(40, 12)), {}), ((x, w, q(41)), {}),
                     ((x, w), dict(activation="tanh")), ((x, w), dict(residual=q(3, 41))),
                     ((x, w), dict(residual=torch.zeros(3, 40))), ((x, w), dict(out=q(4, 40))),
                     ((x, w, torch.zeros(40, dtype=torch.float64)), {})):
        with pytest.raises(ValueError):
            linear_fused(*args, **kw)
    with pytest.raises(TypeError):
        linear_fused(x.float(), w.float())
    with pytest.raises(TypeError):
        linear_fused(x, w.half())
    with pytest.raises(RuntimeError, match="CUDA"):
        linear_fused(x, w)
    with pytest.raises(RuntimeError, match="inference only"):
        linear_fused(x, w.clone().requires_grad_())


def test_c_entry_points_refuse_before_any_launch():
    """Argument checks of the C ABI happen on the host (the pointers are never read); empty work returns."""
    from onecomp_runtime import _lib
    lib = _lib.lib()
    p, odd = ctypes.c_void_p(0x10000), ctypes.c_void_p(0x10002)

    def rope(qp=p, H=4, dt=1, T=5, D=64, R=64, pos=p, gain=1.0, kp=None, Hk=0):
        return lib.oc_b200_rope(qp, 256, 64, qp, 256, 64, H, kp, 0, 0, kp, 0, 0, Hk, dt, T, D, R, pos, 1, 1, p, None,
                                gain, 0, None)

    for kw in (dict(qp=None), dict(dt=3), dict(T=-1), dict(D=0), dict(D=1032), dict(R=66), dict(R=7), dict(R=0),
               dict(pos=None), dict(gain=math.inf), dict(H=-1), dict(Hk=2)):
        assert rope(**kw) == 1, kw
    assert rope(T=0) == 0 and rope(H=0) == 0

    def attn(qp=p, kp=p, dt=1, Tq=8, Tk=8, Hq=4, Hkv=2, D=64, st=256, cq=p, ck=p, B=1, scale=0.1, ws=p, nws=0, out=p):
        return lib.oc_b200_attention(qp, st, 64, kp, 128, 64, kp, 128, 64, out, 256, 64, dt, Tq, Tk, Hq, Hkv, D, cq, ck,
                                     None, B, 1, scale, 0, 0, ws, nws, None)

    for kw in (dict(dt=2), dict(Tq=-1), dict(Hq=3), dict(Hkv=0), dict(B=-1), dict(cq=None), dict(cq=None, ck=None, B=2),
               dict(scale=math.nan), dict(qp=None), dict(kp=None), dict(out=None), dict(qp=odd), dict(kp=odd), dict(st=257)):
        assert attn(**kw) == 1, kw
    assert attn(D=60) == 2 and attn(D=264) == 2
    assert attn(Tq=0) == 0 and attn(B=0) == 0
    assert lib.oc_b200_attention_workspace(4, 4, 1, 4, 2, 0, 0) == 0 and lib.oc_b200_attention_workspace(4, 4, 1, 4, 3, 64, 0) == 0

    def dense(x=p, w=p, dt=1, M=4, N=40, K=64, ldx=64, act=0, bdt=0, ldc=40, c=p, res=None, ldr=0, bias=None):
        return lib.oc_b200_dense_gemm(x, ldx, w, 64, dt, M, N, K, bias, bdt, res, ldr, act, c, ldc, None)

    for kw in (dict(x=None), dict(w=None), dict(c=None), dict(dt=2), dict(M=-1), dict(K=60), dict(K=0), dict(act=5),
               dict(act=-1), dict(bias=p, bdt=9), dict(x=odd), dict(ldx=60), dict(ldx=56), dict(ldc=39),
               dict(res=p, ldr=39)):
        assert dense(**kw) == 1, kw
    assert dense(M=0) == 0 and dense(N=0) == 0


def test_counts_beyond_the_kernels_integers_are_refused():
    """A count that 32 bits would cut (2^32 + 4 would run as 4 rows) is refused by the layers and by the C ABI."""
    from onecomp_runtime import _lib
    from onecomp_runtime.layers import RotaryEmbedding, linear_fused, packed_attention
    a, many = q(3, 2, 8), 2**32 + 4
    with pytest.raises(ValueError, match="2\\*\\*30"):
        packed_attention(q(1, 2, 8).expand(many, 2, 8), a, a)
    with pytest.raises(ValueError, match="2\\*\\*30"):
        packed_attention(a, q(1, 2, 8).expand(many, 2, 8), q(1, 2, 8).expand(many, 2, 8))
    with pytest.raises(ValueError, match="2\\*\\*30"):
        linear_fused(q(1, 8).expand(many, 8), q(40, 8))
    with pytest.raises(ValueError, match="2\\*\\*30"):
        linear_fused(q(3, 8), q(1, 8).expand(many, 8))
    pos = torch.zeros(1, dtype=torch.int64).expand(many)
    with pytest.raises(ValueError, match="2\\*\\*30"):
        RotaryEmbedding(8)(q(1, 1, 8).expand(many, 1, 8), None, pos)
    with pytest.raises(ValueError, match="2\\*\\*30"):
        RotaryEmbedding(8)(q(1, 1, 8).expand(1, many, 8), None, pos[:1])

    lib, p, big = _lib.lib(), ctypes.c_void_p(0x10000), 1 << 30
    assert lib.oc_b200_rope(p, 8, 8, p, 8, 8, 1, None, 0, 0, None, 0, 0, 0, 1, big, 8, 8, p, 1, 1, p, None, 1.0, 0,
                            None) == 1
    for Tq, Tk, B, H in ((big, 4, 1, 1), (4, big, 1, 1), (4, 4, big, 1), (4, 4, 1, big)):
        assert lib.oc_b200_attention(p, 8, 8, p, 8, 8, p, 8, 8, p, 8, 8, 1, Tq, Tk, H, H, 8, p, p, None, B, 1, 0.1, 0, 0, p,
                                     0, None) == 1
    for M, N, K in ((big, 8, 8), (4, big, 8), (4, 8, big)):
        assert lib.oc_b200_dense_gemm(p, big, p, big, 1, M, N, K, None, 0, None, 0, 0, p, big, None) == 1
