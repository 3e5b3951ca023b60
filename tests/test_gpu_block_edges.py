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


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("case", [([3], [3]), ([1], [2000]), ([5], [3]), ([200], [200]), ([40], [3000]), ([300, 2], [150, 2])])
def test_attention_rows_of_minus_infinity(cuda_device, D, case):
    """A row that sees keys, all with scores of minus infinity, is NaN, as its softmax is; a row that sees no key is
    zero; one finite score is enough for a finite row. Few rows, prompts, and keys split over CTAs."""
    from onecomp_runtime.layers import packed_attention
    dev = cuda_device
    lq, lk = case
    q, k, v = (randn(dev, sum(n), h, D, seed=i) for i, (n, h) in enumerate(((lq, 4), (lk, 2), (lk, 2))))
    q[..., 0] = q[..., 0].abs() + 1
    k[..., 0] = -math.inf
    finite = k.clone()
    finite[0, :, 0] = 1.0                       # the first key of the first sequence
    for causal in (True, False):
        sees = torch.cat([torch.arange(a, device=dev) + (b - a if causal else b) >= 0 for a, b in zip(lq, lk)])
        with torch.no_grad():
            o = packed_attention(q, k, v, starts(dev, lq), starts(dev, lk), causal=causal, max_seqlen_q=max(lq))
            f = packed_attention(q, finite, v, starts(dev, lq), starts(dev, lk), causal=causal, max_seqlen_q=max(lq))
        assert bool(torch.isnan(o[sees]).all()) and bool((o[~sees] == 0).all())
        first = v[:1].repeat_interleave(2, 1)   # a weight of one on the first key
        here = sees.clone()
        here[lq[0]:] = False
        assert bool((f[here] == first).all()) and bool((f[:lq[0]][~sees[:lq[0]]] == 0).all())
        assert bool(torch.isnan(f[lq[0]:]).all())
    assert error_word(dev) == 0


@pytest.mark.parametrize("nq", [3, 200])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_attention_zero_and_tiny_scales(cuda_device, nq, D):
    """A scale of zero weighs every visible key alike, whatever the scores' size (infinite ones give NaN), and a tiny
    scale still tells scores apart that are large enough."""
    from onecomp_runtime.layers import packed_attention
    dev = cuda_device
    nk = 500
    q, k, v = randn(dev, nq, 4, D, seed=1, std=1e14), randn(dev, nk, 2, D, seed=2, std=1e15), randn(dev, nk, 2, D, seed=3)
    with torch.no_grad():
        for causal in (True, False):
            o = packed_attention(q, k, v, causal=causal, scale=0.0)
            ref.check(o, *ref.attention(q, k, v, [(0, nq, 0, nk)], causal, 0.0), "scale zero")
            for scale in (1e-30, -3e-31):
                o = packed_attention(q, k, v, causal=causal, scale=scale)
                ref.check(o, *ref.attention(q, k, v, [(0, nq, 0, nk)], causal, scale), f"scale {scale}")
            big = k.clone()
            big[7] = math.inf                        # q . k is infinite or NaN: times zero it is NaN
            assert bool(torch.isnan(packed_attention(q, big, v, causal=causal, scale=0.0)).all())
    assert error_word(dev) == 0


def dirty(dev, t):
    """Leave NaN in the block that the allocator hands to the next tensor of this size."""
    junk = torch.full_like(t, math.nan, memory_format=torch.contiguous_format)
    torch.cuda.synchronize(dev)
    del junk


@pytest.mark.parametrize("first", [0, 2, 5, 9])
def test_attention_without_sequences_is_zero_everywhere(cuda_device, first):
    """Tables of one entry hold no sequence, whatever the entry says: a new output is all zeros, a given one stays."""
    from onecomp_runtime.layers import packed_attention
    dev = cuda_device
    q = randn(dev, 5, 4, 64)
    with torch.no_grad():
        dirty(dev, q)
        o = packed_attention(q, q, q, table(dev, first), table(dev, first))
        assert bool((o == 0).all())
        kept = torch.full_like(q, 3.0)
        packed_attention(q, q, q, table(dev, first), table(dev, first), out=kept)
        assert bool((kept == 3).all())
    error_word(dev)


def test_attention_of_an_empty_batch_with_lengths(cuda_device):
    from onecomp_runtime.layers import packed_attention
    dev = cuda_device
    q, none = randn(dev, 5, 4, 64), torch.zeros(0, dtype=torch.int32, device=dev)
    with torch.no_grad():
        assert bool((packed_attention(q, q, q, table(dev, 0), table(dev, 0), kv_lens=none) == 0).all())
        e = packed_attention(q[:0], q, q, table(dev, 0), table(dev, 0), kv_lens=none)
    assert e.shape == (0, 4, 64) and error_word(dev) == 0


@pytest.mark.parametrize("heads", [(4, 2, 64), (2, 1, 128), (2, 2, 256)])
@pytest.mark.parametrize("cq", [(0, 10, 4), (0, 4, 2, 10), (7, 3), (0, 6, 4, 300), (0, 300, 299), (200, 0, 300),
                                tuple(range(0, 280, 7)) + (0, 300), tuple(range(0, 280, 7)) + (278, 279, 5)])
def test_attention_runs_no_sequence_of_a_decreasing_table(cuda_device, cq, heads):
    """Rows would have several owners, or none: the table is reported, a new output is all zeros and a given one stays
    as it was. Few rows, prompts, and keys split over CTAs; then the same call with a table in order."""
    from onecomp_runtime.layers import packed_attention
    dev = cuda_device
    Hq, Hkv, D = heads
    for Tk in (300, 6000):
        q, k = randn(dev, 300, Hq, D, seed=1), randn(dev, Tk, Hkv, D, seed=2)
        bad, ck = table(dev, *cq), table(dev, *(Tk * i // (len(cq) - 1) for i in range(len(cq))))
        for max_q in (1, 300, None):
            with torch.no_grad():
                assert error_word(dev) == 0
                dirty(dev, q)
                o = packed_attention(q, k, k, bad, ck, max_seqlen_q=max_q)
                assert error_word(dev) == 0x302 and bool((o == 0).all())
                kept = torch.full_like(q, 3.0)
                packed_attention(q, k, k, bad, ck, max_seqlen_q=max_q, out=kept)
                assert error_word(dev) == 0x302 and bool((kept == 3).all())
        good = table(dev, *sorted(cq))
        seqs = [(a, b - a, c, d - c) for a, b, c, d in zip(sorted(cq), sorted(cq)[1:], ck.tolist(), ck.tolist()[1:])]
        with torch.no_grad():
            o = packed_attention(q, k, k, good, ck)
        ref.check(o, *ref.attention(q, k, k, seqs, True, D ** -0.5), "table in order")
        assert error_word(dev) == 0


@pytest.mark.parametrize("T", [3, 300])
def test_attention_writes_beside_its_inputs(cuda_device, T):
    """q, k, v and the output as columns of one buffer share no memory: the result is that of separate tensors and
    nothing else in the buffer changes. Columns that do meet are refused."""
    from onecomp_runtime.layers import packed_attention
    dev = cuda_device
    buf = randn(dev, T, 10 * 64, seed=1)
    q, k, v, out, rest = (buf[:, a * 64:b * 64].unflatten(1, (-1, 64)) for a, b in ((0, 2), (2, 4), (4, 6), (6, 8), (8, 10)))
    before = buf.clone()
    with torch.no_grad():
        want = packed_attention(q.contiguous(), k.contiguous(), v.contiguous())
        got = packed_attention(q, k, v, out=out)
        assert torch.equal(got, want) and torch.equal(buf[:, :384], before[:, :384]) and torch.equal(rest, before[:, 512:].view_as(rest))
        for bad in (q, buf[:, 64:192].unflatten(1, (2, 64)), buf[:, 320:448].unflatten(1, (2, 64))):
            with pytest.raises(ValueError, match="shares memory"):
                packed_attention(q, k, v, out=bad)


@pytest.mark.parametrize("D", [8, 64, 128, 256])
def test_attention_tensors_of_one_row(cuda_device, D):
    """One query row with many heads (a tile of its own), one key row, one of each, heads kept in other orders: a
    dimension of one row may have any stride."""
    from onecomp_runtime.layers import packed_attention
    dev = cuda_device
    for Tq, Tk, Hq, Hkv in ((1, 1, 40, 1), (1, 700, 64, 2), (40, 1, 4, 4), (300, 1, 6, 2), (1, 1, 1, 1), (2, 1, 96, 3)):
        q, k, v = randn(dev, Tq, Hq, D, seed=1), randn(dev, Tk, Hkv, D, seed=2), randn(dev, Tk, Hkv, D, seed=3)

        def other(t):   # heads 3 rows apart, tokens at an odd pitch behind them
            T, H, _ = t.shape
            return torch.zeros(H, 3, T, D + 8, dtype=BF, device=dev)[:, 1, :, :D].transpose(0, 1).copy_(t)

        for causal in (True, False):
            want, tol = ref.attention(q, k, v, [(0, Tq, 0, Tk)], causal, D ** -0.5)
            with torch.no_grad():
                ref.check(packed_attention(q, k, v, causal=causal), want, tol, f"{Tq} {Tk}")
                ref.check(packed_attention(other(q), other(k), other(v), causal=causal, out=other(q)), want, tol, f"{Tq} {Tk} strided")
    assert error_word(dev) == 0


# ---------------------------------------------------------------------------------------- rotary
@pytest.mark.parametrize("scaling", [None, {"type": "ntk", "factor": 8.0}])
def test_rope_far_positions_against_long_arithmetic(cuda_device, scaling):
    """Positions up to 2^50, against angles in fractions with a pi of 50 digits. Beside the bound of the near
    positions (its sine and cosine hold 2^-25 of a half turn) the table counts: a fraction of a turn is off by 2^-52 of
    itself and, rounded to a unit of 2^-64 turns, by half of that (pi 2^-64 as an angle), times the position."""
    from fractions import Fraction
    from test_block_edges_cpu import pi_by_machin
    from onecomp_runtime.layers import RotaryEmbedding
    dev = cuda_device
    rope = RotaryEmbedding(64, scaling=scaling)
    where = [2**31, -2**31, 2**33 + 12345, 2**40 + 1, 2**45 - 7, 2**50 + 3, -2**50]
    pi = pi_by_machin(50)
    turn = [[float((Fraction(f) * p / (2 * pi)) % 1) for f in rope.inv_freq] for p in where]
    ang = torch.tensor(turn, dtype=torch.float64, device=dev) * (2 * math.pi)
    q = randn(dev, len(where), 5, 64, dtype=torch.float32, seed=6)
    with torch.no_grad():
        y, _ = rope(q, None, torch.tensor(where, device=dev))
    want, tol = ref.rope(q, ang, rope.gain, 64, False)
    mag = q.double()[..., :32].abs() + q.double()[..., 32:].abs()
    far = torch.tensor([[abs(p) * (abs(f) * 2.0 ** -52 + math.pi * 2.0 ** -64) for f in rope.inv_freq] for p in where],
                       dtype=torch.float64, device=dev)
    mag = mag * far.unsqueeze(1)
    tol = tol + torch.cat([mag, mag], -1)
    ref.check(y, want, tol, "far positions")


def test_rope_odd_head_size_in_place(cuda_device):
    from onecomp_runtime.layers import RotaryEmbedding
    dev = cuda_device
    for layout in ("half", "interleaved"):
        rope, pos = RotaryEmbedding(65, rotary_dim=62, layout=layout), torch.arange(9, device=dev)
        q = randn(dev, 9, 3, 65, seed=2)
        want = ref.rope(q, pos.double()[:, None] * torch.tensor(rope.inv_freq, dtype=torch.float64, device=dev), 1.0, 62,
                        layout == "interleaved")
        with torch.no_grad():
            ref.check(rope(q, None, pos, inplace=True)[0], *want, layout)


@pytest.mark.parametrize("T", [1, 3, 700])
def test_rope_many_heads(cuda_device, T):
    """More heads than a grid dimension holds."""
    from onecomp_runtime.layers import RotaryEmbedding
    dev = cuda_device
    rope, pos = RotaryEmbedding(8), torch.arange(T, device=dev) * 77
    ang = pos.double()[:, None] * torch.tensor(rope.inv_freq, dtype=torch.float64, device=dev)
    q, k = randn(dev, T, 70001, 8, seed=1), randn(dev, T, 65536, 8, seed=2)
    with torch.no_grad():
        for x, y in zip((q, k), rope(q, k, pos)):
            ref.check(y, *ref.rope(x, ang, 1.0, 8, False), f"T={T}")


# ---------------------------------------------------------------------------------------- dense linear
@pytest.mark.parametrize("M", [5, 60, 300])
def test_linear_writes_beside_its_inputs(cuda_device, M):
    """x, the residual and the output as columns of one buffer, on 16-byte boundaries and off them."""
    from onecomp_runtime.layers import linear_fused
    dev = cuda_device
    K, N = 128, 200
    for shift in (0, 3):
        buf = randn(dev, M, K + 3 * N, seed=M)
        w = randn(dev, N, K, seed=2, std=K ** -0.5)
        x, r, out = buf[:, :K], buf[:, K + shift:K + N + shift], buf[:, K + N + shift:K + 2 * N + shift]
        before = buf.clone()
        with torch.no_grad():
            got = linear_fused(x, w, residual=r, out=out)
            ref.check(got, *ref.linear(before[:, :K], w, None, None, before[:, K + shift:K + N + shift]), "beside")
            assert torch.equal(buf[:, :K + N + shift], before[:, :K + N + shift])
            assert torch.equal(buf[:, K + 2 * N + shift:], before[:, K + 2 * N + shift:])
            for bad in (buf[:, K - 1:K - 1 + N], buf[:, K + shift + 1:K + shift + 1 + N]):
                with pytest.raises(ValueError):
                    linear_fused(x, w, residual=r, out=bad)
    assert error_word(dev) == 0


def dense_tile(M, N, K):
    import ctypes
    from onecomp_runtime import _lib
    tokens, splits = ctypes.c_int(), ctypes.c_int()
    _lib.call("oc_b200_dense_gemm_tile", M, N, K, ctypes.byref(tokens), ctypes.byref(splits))
    return tokens.value, bool(splits.value)


def test_linear_tile_rule(cuda_device):
    """Few tokens split K; the pairs' tiles are multiples of 32 tokens, no longer than the call needs."""
    for M in (1, 16, 17, 32, 33, 64, 65, 128, 129, 300, 517, 1024, 4099):
        for N, K in ((8, 8), (2560, 2560), (1024, 8192), (8200, 5120), (95000, 64)):
            tokens, splits = dense_tile(M, N, K)
            assert splits or (64 <= tokens <= 256 and tokens % 32 == 0)
            assert splits or -(-M // tokens) * tokens - M < 32 * -(-M // tokens)
            assert splits == (M <= 32 or (M <= 128 and K > 4096 and -(-N // 256) * -(-M // 32) <= 24))


PAIR_TILES = [   # M, N, K, tokens of a tile: at least 5 tiles for each of 74 pairs, ragged in both dimensions
    (57, 94984, 72, 64), (91, 95001, 136, 96), (113, 94984, 200, 128), (155, 95001, 72, 160), (187, 94984, 72, 192),
    (211, 95001, 72, 224), (251, 94984, 72, 256), (449, 40008, 1032, 160), (513, 31992, 72, 192), (577, 31997, 136, 224),
    (673, 31992, 264, 256), (1300, 20104, 520, 224), (4099, 6344, 1032, 256)]


@pytest.mark.parametrize("case", PAIR_TILES)
@pytest.mark.parametrize("dtype", [BF, HF])
def test_linear_many_tiles_for_each_pair(cuda_device, case, dtype):
    """Every tile size over many tiles: both accumulators and every buffer are used again and again, bands of feature
    tiles end early, and both epilogues write, with a residual, the residual as the output, and without one."""
    from onecomp_runtime.layers import linear_fused
    dev = cuda_device
    M, N, K, tokens = case
    assert dense_tile(M, N, K) == (tokens, False)
    tiles_n = -(-N // 256)
    assert tiles_n * -(-M // tokens) >= 5 * 74 and tiles_n > 8 and tiles_n % 8 and M % tokens and N % 256
    x, w, b = randn(dev, M, K, dtype=dtype, seed=1), randn(dev, N, K, dtype=dtype, seed=2, std=K ** -0.5), \
        randn(dev, N, dtype=torch.float32, seed=3)
    r = randn(dev, M, N, dtype=dtype, seed=4)
    with torch.no_grad():
        want, tol = ref.linear(x, w, b, "gelu_tanh", None)
        first = linear_fused(x, w, b, activation="gelu_tanh")
        ref.check(first, want, tol, f"{case}")
        assert all(torch.equal(first, linear_fused(x, w, b, activation="gelu_tanh")) for _ in range(3))
        del want, tol, first
        want, tol = ref.linear(x, w, b, "relu", r)
        ref.check(linear_fused(x, w, b, activation="relu", residual=r), want, tol, f"{case} residual")
        acc = r.clone()
        ref.check(linear_fused(x, w, b, activation="relu", residual=acc, out=acc), want, tol, f"{case} onto the residual")
        wide = torch.full((M, N + 3), 7.0, dtype=dtype, device=dev)    # rows off 16-byte boundaries
        wide[:, 1:N + 1] = r
        at = wide[:, 1:N + 1]
        ref.check(linear_fused(x, w, b, activation="relu", residual=at, out=at), want, tol, f"{case} direct stores")
        assert bool((wide[:, 0] == 7).all()) and bool((wide[:, N + 1:] == 7).all())
    assert error_word(dev) == 0


@pytest.mark.parametrize("act", [None, "gelu_tanh", "gelu", "silu", "relu"])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("M", [24, 290])
def test_linear_activations_of_extreme_values(cuda_device, act, dtype, M):
    """Sums that are huge, tiny, infinite or NaN come out of every activation as its formula has them."""
    from onecomp_runtime.layers import linear_fused
    dev = cuda_device
    top = torch.finfo(dtype).max
    vals = [0.0, 1e-7, -1e-7, 0.5, -0.5, 5.0, -5.0, 12.0, -12.0, 44.0, -44.0, 100.0, -100.0, 6e4, -6e4, top, -top, math.inf,
            -math.inf, math.nan]
    x = torch.zeros(M, 16, dtype=dtype, device=dev)
    x[:, 0] = torch.tensor(vals, dtype=torch.float64, device=dev).to(dtype).repeat(-(-M // len(vals)))[:M]
    w = torch.zeros(264, 16, dtype=dtype, device=dev)
    w[:, 0] = 1
    with torch.no_grad():
        y = linear_fused(x, w, activation=act)
    v = x[:, :1].double().expand(M, 264)
    # (the normal distribution function through erfc: 1 + erf loses it below -6, where it is 1e-9 and less)
    want = 0.5 * v * torch.special.erfc(-v / math.sqrt(2.0)) if act == "gelu" else ref.act64(v, act)
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    ok = ~torch.isnan(want)
    exact = want.to(dtype).double()      # infinities and what rounds to them
    inf = ok & torch.isinf(exact)
    assert torch.equal(y[inf].double(), exact[inf])
    fin = ok & ~inf
    # the exponent of the fast exponential is off by 2^-16 of the result at most; below the type's normal range one step
    tol = want.abs() * (ref.half_step(dtype) + 2.0 ** -16) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    ref.check(y[fin], want[fin], tol[fin], f"{act}")
    assert error_word(dev) == 0


@pytest.mark.parametrize("M", [1, 20, 40, 300])
@pytest.mark.parametrize("N", [1, 2, 7, 8, 33])
def test_linear_few_features(cuda_device, M, N):
    """Down to one feature and one block of 8 values; a column of a wider output."""
    from onecomp_runtime.layers import linear_fused
    dev = cuda_device
    for K in (8, 72):
        x, w, b, r = randn(dev, M, K, seed=1), randn(dev, N, K, seed=2), randn(dev, N, seed=3), randn(dev, M, N, seed=4)
        wide = torch.full((M, N + 4), 7.0, dtype=BF, device=dev)
        with torch.no_grad():
            want, tol = ref.linear(x, w, b, "silu", r)
            ref.check(linear_fused(x, w, b, activation="silu", residual=r), want, tol, f"{M} {N} {K}")
            ref.check(linear_fused(x, w, b, activation="silu", residual=r, out=wide[:, 2:N + 2]), want, tol, "column")
        assert bool((wide[:, :2] == 7).all()) and bool((wide[:, N + 2:] == 7).all())
    assert error_word(dev) == 0


def test_operators_under_inference_mode_and_other_streams(cuda_device):
    """Inference tensors, and tensors made on one stream and used on another after an event."""
    from onecomp_runtime.layers import RotaryEmbedding, linear_fused, packed_attention
    dev = cuda_device
    rope = RotaryEmbedding(64)
    with torch.inference_mode():
        x, w = randn(dev, 70, 256, seed=1), randn(dev, 3 * 256, 256, seed=2, std=1 / 16)
        pos = torch.arange(70, device=dev)

        def step():
            q, k, v = (t.unflatten(1, (4, 64)) for t in linear_fused(x, w).split(256, 1))
            rope(q, k, pos, inplace=True)
            return packed_attention(q, k, v)

        first = step()
        s = torch.cuda.Stream(dev)
        s.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(s):
            second = step()
        torch.cuda.current_stream(dev).wait_stream(s)
        assert torch.equal(first, second)
    assert error_word(dev) == 0
