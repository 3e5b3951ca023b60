"""Calls of the transformer-block operators at the edges of what their documentation allows: waits between the
stages of a kernel, infinities, empty batches, tables that decrease, shared buffers, every tile size."""
from __future__ import annotations

import math

import pytest
import torch

import block_ref as ref

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def randn(dev, *shape, dtype=BF, seed=0, std=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=dev) * std).to(dtype)


def table(dev, *values):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def starts(dev, lens):
    return torch.tensor([0, *lens], dtype=torch.int32).cumsum(0).to(torch.int32).to(dev)


def error_word(dev):
    from onecomp_runtime import _lib
    return _lib.read_device_error(dev)


# ------------------------------------------------------------------------------------------ attention
@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("grows", [False, True])
def test_attention_products_done_before_they_are_read(cuda_device, D, grows):
    """The output, and what is accumulated when the maximum grows, are read once the product before is done, however
    early the scores after it were there: one block of keys to many, many tiles, many times."""
    from onecomp_runtime.layers import packed_attention
    dev = cuda_device
    lens = [128, 129, 256, 1, 257, 700, 385, 1100]
    T = sum(lens)
    q, k, v = randn(dev, T, 4, D, seed=1), randn(dev, T, 2, D, seed=2), randn(dev, T, 2, D, seed=3)
    if grows:   # every block of keys raises the maximum of every row by more than the reference's step
        q = q.abs()
        at = torch.cat([torch.arange(n, device=dev) for n in lens]).float()
        k = (k.float().abs() * 0.01 + (at // 128 + 1).view(T, 1, 1) * 20.0 * D ** -0.5).to(BF)
    c = starts(dev, lens)
    seqs = [(sum(lens[:i]), n, sum(lens[:i]), n) for i, n in enumerate(lens)]
    for causal in (False, True):
        want, tol = ref.attention(q, k, v, seqs, causal, D ** -0.5)
        for _ in range(30):
            with torch.no_grad():
                ref.check(packed_attention(q, k, v, c, c, causal=causal, max_seqlen_q=1100), want, tol, f"D={D}")
    assert error_word(dev) == 0
