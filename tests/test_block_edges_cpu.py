"""Calls of the transformer-block operators at the edges of what their documentation allows: what the host decides."""
from __future__ import annotations

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
