"""Rotary positions, packed-sequence attention and the dense linear on a B200 against 64-bit restatements
(tests/block_ref.py), at the sizes, strides and masks where they can go wrong."""
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


def cu(dev, lens):
    return torch.tensor([0, *lens], dtype=torch.int32).cumsum(0).to(torch.int32).to(dev)


def error_word(dev):
    from onecomp_runtime import _lib
    return _lib.read_device_error(dev)


# ------------------------------------------------------------------------------------------ attention
def run_attention(dev, lq, lk, Hq, Hkv, D, dtype=BF, causal=True, seed=0, kv_lens=None, max_q=None, scale=None,
                  qkv=None, q_std=1.5):
    from onecomp_runtime.layers import packed_attention
    q = randn(dev, sum(lq), Hq, D, dtype=dtype, seed=seed, std=q_std)
    k, v = randn(dev, sum(lk), Hkv, D, dtype=dtype, seed=seed + 1), randn(dev, sum(lk), Hkv, D, dtype=dtype, seed=seed + 2)
    lens = None if kv_lens is None else torch.tensor(kv_lens, dtype=torch.int32, device=dev)
    with torch.no_grad():
        o = packed_attention(q, k, v, cu(dev, lq), cu(dev, lk), kv_lens=lens, causal=causal, scale=scale,
                             max_seqlen_q=max_q)
    q0 = [sum(lq[:i]) for i in range(len(lq))]
    k0 = [sum(lk[:i]) for i in range(len(lk))]
    seqs = list(zip(q0, lq, k0, kv_lens or lk))
    want, tol = ref.attention(q, k, v, seqs, causal, D ** -0.5 if scale is None else scale)
    ref.check(o, want, tol, f"attention {lq} {lk} {kv_lens} {Hq}/{Hkv} D={D} causal={causal}")
    assert error_word(dev) == 0
    return q, k, v, o


@pytest.mark.parametrize("D", [8, 64, 80, 128, 192, 256])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_attention_head_sizes(cuda_device, D, dtype):
    for causal in (True, False):
        run_attention(cuda_device, [1, 33, 128, 17], [1, 97, 128, 300], 4, 2, D, dtype, causal, seed=D)


@pytest.mark.parametrize("heads", [(1, 1), (3, 3), (8, 1), (24, 4), (40, 2)])
def test_attention_head_groups(cuda_device, heads):
    run_attention(cuda_device, [5, 1, 0, 40], [70, 513, 9, 40], *heads, 128, seed=7)


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 640, 1031])
def test_attention_prompt_lengths(cuda_device, n):
    """One causal prompt of every length around the tile borders; and as the second of two, so that its
    rows start off a border."""
    run_attention(cuda_device, [n], [n], 4, 2, 128, seed=n)
    run_attention(cuda_device, [3, n, 2], [3, n + 5, 2], 2, 2, 64, HF, seed=n)
    run_attention(cuda_device, [n, 1], [n, 1], 2, 1, 256, causal=False, seed=n)


@pytest.mark.parametrize("nk", [1, 15, 16, 17, 64, 65, 1000, 4099, 20011])
@pytest.mark.parametrize("nq", [1, 4])
def test_attention_single_tokens(cuda_device, nk, nq):
    """Few query rows over caches from one key to long ones (one sequence split over every SM)."""
    if nk >= nq:
        run_attention(cuda_device, [nq], [nk], 8, 2, 128, seed=nk, max_q=nq)
        run_attention(cuda_device, [nq] * 3, [nk, nq, nk], 12, 2, 256, HF, seed=nk, max_q=nq)


def test_attention_many_sequences(cuda_device):
    """More sequences than one scan step of the tables holds, ragged, empty ones among them."""
    lk = [(37 * i) % 211 for i in range(150)]
    lq = [min(1, n) for n in lk]
    run_attention(cuda_device, lq, lk, 4, 1, 64, seed=3, max_q=1)
    lq = [min(n, i % 7) for i, n in enumerate(lk)]
    run_attention(cuda_device, lq, lk, 4, 4, 128, seed=4)


@pytest.mark.parametrize("max_q", [None, 1, 300])
def test_attention_rows_without_keys(cuda_device, max_q):
    """No keys at all, and causal rows before the first key (more queries than keys): zeros. The hint of
    the longest run changes nothing."""
    q, k, v, o = run_attention(cuda_device, [2, 300, 0, 9], [0, 11, 5, 9], 4, 2, 128, seed=5, max_q=max_q)
    assert bool((o[:2] == 0).all()) and bool((o[2:2 + 289] == 0).all()) and bool((o[291:] != 0).any())


@pytest.mark.parametrize("max_q", [1, 200])
def test_attention_padded_cache(cuda_device, max_q):
    """kv_lens below the capacity: what lies behind, NaN and infinities too, stays out. A batch of single
    tokens, and of longer runs."""
    from onecomp_runtime.layers import packed_attention
    dev = cuda_device
    cap, lens = 300, [1, 300, 64, 129, 0, 17]
    lq = [1] * 6 if max_q == 1 else [1, 200, 64, 5, 3, 17]
    k, v = randn(dev, 6 * cap, 2, 128, seed=1), randn(dev, 6 * cap, 2, 128, seed=2)
    q = randn(dev, sum(lq), 8, 128, seed=3)
    for b, n in enumerate(lens):
        k[b * cap + n:(b + 1) * cap] = math.nan
        v[b * cap + n:(b + 1) * cap] = math.inf if b % 2 else math.nan
    kl = torch.tensor(lens, dtype=torch.int32, device=dev)
    for causal in (True, False):
        with torch.no_grad():
            o = packed_attention(q, k, v, cu(dev, lq), cu(dev, [cap] * 6), kv_lens=kl, causal=causal, max_seqlen_q=max_q)
        q0 = [sum(lq[:i]) for i in range(6)]
        want, tol = ref.attention(q, k, v, [(q0[b], lq[b], b * cap, lens[b]) for b in range(6)], causal, 128 ** -0.5)
        ref.check(o, want, tol, f"padded cache causal={causal}")


@pytest.mark.parametrize("shape", [(5, 60, 128), (40, 70, 64), (300, 420, 128), (130, 130, 256)])
def test_attention_nonfinite_values_that_rows_do_not_see(cuda_device, shape):
    """An infinite or NaN value at key j reaches the causal rows that see it and no others."""
    from onecomp_runtime.layers import packed_attention
    dev = cuda_device
    nq, nk, D = shape
    q, k, v = randn(dev, nq, 4, D, seed=1), randn(dev, nk, 2, D, seed=2), randn(dev, nk, 2, D, seed=3)
    want, tol = ref.attention(q, k, v, [(0, nq, 0, nk)], True, D ** -0.5)
    j_nan, j_inf = nk - 2, nk - nq // 2
    v[j_nan, 0, 3] = math.nan
    v[j_inf, 1, D - 1] = -math.inf
    with torch.no_grad():
        o = packed_attention(q, k, v, causal=True)
    assert bool(torch.isnan(o[nq - 2:, 0:2, 3]).all())                       # the rows that see j_nan
    first = j_inf - (nk - nq)                                                 # first row that sees j_inf
    assert bool((o[first:, 2:4, D - 1] == -math.inf).all())
    o[nq - 2:, 0:2, 3] = want[nq - 2:, 0:2, 3].to(o.dtype)
    o[first:, 2:4, D - 1] = want[first:, 2:4, D - 1].to(o.dtype)
    ref.check(o, want, tol, "rows beside non-finite values")


def test_attention_nonfinite_keys_that_rows_do_not_see(cuda_device):
    from onecomp_runtime.layers import packed_attention
    dev = cuda_device
    for nq, nk in ((6, 50), (290, 290)):
        q, k, v = randn(dev, nq, 2, 128, seed=1), randn(dev, nk, 2, 128, seed=2), randn(dev, nk, 2, 128, seed=3)
        want, tol = ref.attention(q, k, v, [(0, nq, 0, nk)], True, 128 ** -0.5)
        k[nk - 1, 0, 5] = math.nan
        with torch.no_grad():
            o = packed_attention(q, k, v, causal=True)
        assert bool(torch.isnan(o[nq - 1, 0]).all())
        o[nq - 1, 0] = want[nq - 1, 0].to(o.dtype)
        ref.check(o, want, tol, "rows before a NaN key")


def test_attention_large_and_equal_scores(cuda_device):
    """Scores far from zero (the running maximum moves by hundreds), growing along the keys, and all equal."""
    from onecomp_runtime.layers import packed_attention
    dev = cuda_device
    run_attention(cuda_device, [260], [700], 2, 1, 64, HF, seed=1, scale=2.0)
    run_attention(cuda_device, [3], [900], 8, 2, 128, seed=2, scale=-3.0, max_q=3)
    for D in (64, 128, 256):   # negative and zero scales of a prompt: Q is negated in the product, every weight equal
        run_attention(cuda_device, [300, 40], [700, 40], 4, 2, D, seed=3, scale=-0.5)
        run_attention(cuda_device, [300, 40], [700, 40], 4, 2, D, HF, seed=4, scale=0.0)
    for nq in (2, 333):
        n = 700
        q = torch.full((nq, 2, 64), 0.5, dtype=BF, device=dev)
        k = (torch.arange(n, device=dev, dtype=torch.float32) / 4).to(BF).view(n, 1, 1).expand(n, 2, 64).contiguous()
        v = randn(dev, n, 2, 64, seed=4)
        with torch.no_grad():
            o = packed_attention(q, k, v, causal=False, scale=1.0 / 32)
            z = packed_attention(q, torch.zeros_like(k), v, causal=False)
        ref.check(o, *ref.attention(q, k, v, [(0, nq, 0, n)], False, 1.0 / 32), "growing scores")
        ref.check(z, *ref.attention(q, torch.zeros_like(k), v, [(0, nq, 0, n)], False, 0.125), "equal scores")


@pytest.mark.parametrize("T", [7, 600])
def test_attention_strided_inputs(cuda_device, T):
    """Column slices of one projection, heads-first storage, a last dimension that is not contiguous, rows
    off 16-byte boundaries, an expanded key head: the same results as from contiguous copies."""
    from onecomp_runtime.layers import packed_attention
    dev = cuda_device
    H, G, D = 4, 2, 64
    base = randn(dev, T, (H + 2 * G) * D, seed=11)
    q, k, v = base[:, :H * D].unflatten(1, (H, D)), base[:, H * D:(H + G) * D].unflatten(1, (G, D)), \
        base[:, (H + G) * D:].unflatten(1, (G, D))
    with torch.no_grad():
        want = packed_attention(q.contiguous(), k.contiguous(), v.contiguous())
        assert torch.equal(packed_attention(q, k, v), want)
        hf = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
        assert torch.equal(packed_attention(*hf), want)
        odd = [torch.cat([t, t[..., :1]], -1)[..., :D] for t in (q, k, v)]       # rows of D + 1 values
        assert torch.equal(packed_attention(*odd), want)
        last = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
        assert torch.equal(packed_attention(*last), want)
        k1, v1 = k[:, :1].expand(T, H, D), v[:, :1].expand(T, H, D)
        assert torch.equal(packed_attention(q, k1, v1), packed_attention(q, k1.contiguous(), v1.contiguous()))


def test_attention_out_and_rows_of_no_sequence(cuda_device):
    """A given output (strided) keeps the rows that no sequence owns; a new one holds zeros there."""
    from onecomp_runtime.layers import packed_attention
    dev = cuda_device
    for lq in ([3, 2], [150, 77]):
        T, n = sum(lq) + 6, sum(lq)
        q, k, v = randn(dev, T, 4, 64, seed=1), randn(dev, T, 4, 64, seed=2), randn(dev, T, 4, 64, seed=3)
        c = cu(dev, lq)
        buf = torch.full((T, 4, 128), 7.0, dtype=BF, device=dev)
        out = buf[..., 64:]
        with torch.no_grad():
            fresh = packed_attention(q, k, v, c, c)
            got = packed_attention(q, k, v, c, c, out=out)
        assert got.data_ptr() == out.data_ptr() and torch.equal(got[:n], fresh[:n])
        assert bool((got[n:] == 7).all()) and bool((buf[..., :64] == 7).all()) and bool((fresh[n:] == 0).all())


def test_attention_rows_in_front_of_the_first_sequence(cuda_device):
    from onecomp_runtime.layers import packed_attention
    dev = cuda_device
    for first, lq in ((2, [3, 2]), (70, [150, 77])):
        T = first + sum(lq) + 5
        q, k, v = randn(dev, T, 4, 64, seed=1), randn(dev, T, 4, 64, seed=2), randn(dev, T, 4, 64, seed=3)
        c = cu(dev, [first, *lq])[1:].contiguous()
        with torch.no_grad():
            junk = torch.full((T, 4, 64), math.nan, dtype=BF, device=dev)   # what a new output may hold
            del junk
            o = packed_attention(q, k, v, c, c)
        s0 = first + lq[0]
        want, tol = ref.attention(q, k, v, [(first, lq[0], first, lq[0]), (s0, lq[1], s0, lq[1])], True, 0.125)
        ref.check(o, want, tol, "rows in front")
        assert bool((o[:first] == 0).all()) and bool((o[-5:] == 0).all())


@pytest.mark.parametrize("case", [([20], [3000], 8, 1, 128), ([33, 5], [4001, 90], 6, 2, 64), ([64], [2500], 3, 1, 256),
                                  ([9, 9, 1, 40], [700, 9, 1, 5000], 10, 2, 128), ([130], [130], 12, 4, 64)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_attention_keys_split_over_ctas(cuda_device, case, dtype):
    """Few tiles and many keys: parts of the keys on several CTAs, parts that some rows do not see at all, a
    group that does not divide a tile."""
    lq, lk, Hq, Hkv, D = case
    for causal in (True, False):
        run_attention(cuda_device, lq, lk, Hq, Hkv, D, dtype, causal, seed=5, max_q=max(lq))


@pytest.mark.parametrize("G", [3, 7, 20, 64, 100, 128, 130, 200])
def test_attention_wide_groups(cuda_device, G):
    run_attention(cuda_device, [3, 40, 1], [50, 300, 1], G, 1, 64, seed=G)
    run_attention(cuda_device, [1, 1], [700, 3], 2 * G, 2, 64, HF, seed=G, max_q=1)


def test_attention_offsets_beyond_32_bits(cuda_device):
    """Key rows whose element offset passes 2^31, for single tokens and for a prompt; the same for queries."""
    from onecomp_runtime.layers import packed_attention
    dev = cuda_device
    st, T, n = 65536, 40000, 300
    buf = torch.empty(st * T, dtype=BF, device=dev)
    k, v = buf.as_strided((T, 1, 64), (st, 64, 1)), buf.as_strided((T, 1, 64), (st, 64, 1), 128)
    k[-n:] = randn(dev, n, 1, 64, seed=1)
    v[-n:] = randn(dev, n, 1, 64, seed=2)
    ck = torch.tensor([T - n, T], dtype=torch.int32, device=dev)
    for nq in (1, 200):
        q = randn(dev, nq, 4, 64, seed=3)
        cq = cu(dev, [nq])
        with torch.no_grad():
            o = packed_attention(q, k, v, cq, ck)
            ref.check(o, *ref.attention(q, k[-n:], v[-n:], [(0, nq, 0, n)], True, 0.125), "far keys")
            wide = k[-nq:]                                   # as queries: rows far apart, far into the buffer
            far = packed_attention(k, k[-n:], v[-n:], torch.tensor([T - nq, T], dtype=torch.int32, device=dev),
                                   cu(dev, [n]))[-nq:]
            ref.check(far, *ref.attention(wide.contiguous(), k[-n:], v[-n:], [(0, nq, 0, n)], True, 0.125), "far queries")
    assert error_word(dev) == 0


def test_attention_refuses_bad_outputs(cuda_device):
    from onecomp_runtime.layers import packed_attention
    dev = cuda_device
    q = randn(dev, 6, 4, 64)
    base = torch.empty((6, 4, 65), dtype=BF, device=dev)
    with torch.no_grad():
        for out in (q, base[..., 1:], base[..., :64], torch.empty((1, 4, 64), dtype=BF, device=dev).expand(6, 4, 64),
                    torch.empty(1000, dtype=BF, device=dev).as_strided((6, 4, 64), (64, 8, 1)), q.new_empty(6, 4, 32)):
            with pytest.raises(ValueError):
                packed_attention(q, q, q, out=out)
        with pytest.raises(ValueError, match="tensors on"):
            packed_attention(q, q.cpu(), q)


def test_attention_empty_calls(cuda_device):
    from onecomp_runtime.layers import packed_attention
    dev = cuda_device
    e = torch.empty((0, 4, 64), dtype=BF, device=dev)
    q = randn(dev, 3, 4, 64)
    with torch.no_grad():
        assert packed_attention(e, q, q).shape == (0, 4, 64)
        assert bool((packed_attention(q, e, e) == 0).all())
        z = torch.zeros(1, dtype=torch.int32, device=dev)
        assert bool((packed_attention(q, q, q, z, z) == 0).all())        # no sequence at all


def test_attention_bad_tables_are_clamped_and_reported(cuda_device):
    """Table values outside the tensors read and write nothing outside and set the device error word."""
    from onecomp_runtime.layers import packed_attention
    dev = cuda_device
    q, k = randn(dev, 10, 2, 64, seed=1), randn(dev, 20, 2, 64, seed=2)
    t = lambda *a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    good = (t(0, 4, 10), t(0, 10, 20), t(10, 10))
    for i, bad in ((0, t(0, 4, 99)), (0, t(-3, 4, 10)), (1, t(0, 10, 1000)), (2, t(10, 11)), (2, t(-1, 10)),
                   (0, t(0, 10, 4)), (1, t(0, 30, 20))):
        args = list(good)
        args[i] = bad
        for max_q in (1, 256):
            assert error_word(dev) == 0
            with torch.no_grad():
                o = packed_attention(q, k, k, args[0], args[1], kv_lens=args[2], max_seqlen_q=max_q)
            assert o.shape == q.shape and error_word(dev) == 0x302


def test_attention_repeats_bit_for_bit(cuda_device):
    from onecomp_runtime.layers import packed_attention
    dev = cuda_device
    for lq, lk in (([1] * 5, [3000, 17, 900, 64, 4097]), ([300, 45, 700], [300, 900, 700])):
        q, k, v = randn(dev, sum(lq), 16, 128, seed=1), randn(dev, sum(lk), 2, 128, seed=2), randn(dev, sum(lk), 2, 128, seed=3)
        with torch.no_grad():
            first = packed_attention(q, k, v, cu(dev, lq), cu(dev, lk))
            assert all(torch.equal(first, packed_attention(q, k, v, cu(dev, lq), cu(dev, lk))) for _ in range(5))


def test_attention_wide_heads_many_times(cuda_device):
    """One row tile per CTA (head size 256): the last product of a tile may run long after its scores were
    ready, so the output is read only once both of the last two products are done. Many tiles, many times."""
    from onecomp_runtime.layers import packed_attention
    dev = cuda_device
    lens = [256, 1, 129, 384, 255, 640]
    q, k, v = randn(dev, sum(lens), 12, 256, seed=1, std=1.5), randn(dev, sum(lens), 4, 256, seed=2), randn(dev, sum(lens), 4, 256, seed=3)
    c = cu(dev, lens)
    starts = [sum(lens[:i]) for i in range(len(lens))]
    for causal in (False, True):
        want, tol = ref.attention(q, k, v, [(s, n, s, n) for s, n in zip(starts, lens)], causal, 256 ** -0.5)
        for _ in range(40):
            with torch.no_grad():
                ref.check(packed_attention(q, k, v, c, c, causal=causal), want, tol, "wide heads")


# ---------------------------------------------------------------------------------------- rotary
def angles(dev, pos, freq):
    return pos.double() * torch.tensor(freq, dtype=torch.float64, device=dev)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [BF, HF, torch.float32])
@pytest.mark.parametrize("dims", [(128, 128), (256, 64), (64, 2), (80, 40), (24, 24), (10, 6)])
def test_rope_layouts(cuda_device, layout, dtype, dims):
    from onecomp_runtime.layers import RotaryEmbedding
    dev = cuda_device
    D, R = dims
    rope = RotaryEmbedding(D, rotary_dim=R, layout=layout)
    for T in (1, 5, 2500):
        q, k = randn(dev, T, 6, D, dtype=dtype, seed=T), randn(dev, T, 2, D, dtype=dtype, seed=T + 1)
        pos = torch.randint(-50, 9000, (T,), device=dev, generator=torch.Generator(device=dev).manual_seed(T))
        with torch.no_grad():
            yq, yk = rope(q, k, pos)
        a = angles(dev, pos[:, None], rope.inv_freq)
        for x, y in ((q, yq), (k, yk)):
            ref.check(y, *ref.rope(x, a, 1.0, R, layout == "interleaved"), f"rope T={T}")
        only, none = rope(q, None, pos.to(torch.int32))
        assert none is None and torch.equal(only, yq)


def test_rope_in_place_on_slices(cuda_device):
    """In place on the q and k columns of one projection: the same bits as out of place, v untouched."""
    from onecomp_runtime.layers import RotaryEmbedding
    dev = cuda_device
    for T, D, R in ((3, 128, 64), (1300, 64, 64), (9, 24, 20)):
        rope = RotaryEmbedding(D, rotary_dim=R)
        base = randn(dev, T, 8 * D, seed=T)
        pos = torch.arange(T, device=dev)
        q, k = base[:, :4 * D].unflatten(1, (4, D)), base[:, 4 * D:6 * D].unflatten(1, (2, D))
        before = base.clone()
        with torch.no_grad():
            yq, yk = rope(q, k, pos)
            rope(q, k, pos, inplace=True)
        assert torch.equal(q, yq) and torch.equal(k, yk) and torch.equal(base[:, 6 * D:], before[:, 6 * D:])


def test_rope_refuses_in_place_overlaps_and_takes_empty_batches(cuda_device):
    from onecomp_runtime.layers import RotaryEmbedding
    dev = cuda_device
    rope = RotaryEmbedding(64, device=dev)
    q, pos = randn(dev, 5, 4, 64), torch.arange(5, device=dev)
    with torch.no_grad():
        for a, b in ((q, q), (q[:, :1].expand(5, 4, 64), None), (q, q[:, :2])):
            with pytest.raises(ValueError):
                rope(a, b, pos, inplace=True)
        with pytest.raises(ValueError, match="tensors on"):
            rope(q, None, pos.cpu())
        e, k = rope(q[:0], q[:0, :2], pos[:0])
        assert e.shape == (0, 4, 64) and k.shape == (0, 2, 64)
        ee = rope(q[:0].view(0, 1, 4, 64), None, pos[:0].view(0, 1))[0]
        assert ee.shape == (0, 1, 4, 64)
        one = rope(q, None, torch.full((1,), 7, device=dev).expand(5))[0]      # one position for all tokens
        assert torch.equal(one, rope(q, None, torch.full((5,), 7, device=dev))[0])


def test_rope_leading_dimensions_and_axes(cuda_device):
    from onecomp_runtime.layers import RotaryEmbedding
    dev = cuda_device
    axes = [16, 56, 56]
    rope = RotaryEmbedding(128, axes=axes, layout="interleaved")
    q, k = randn(dev, 2, 70, 4, 128, seed=1), randn(dev, 2, 70, 4, 128, seed=2)
    pos = torch.randint(-40, 300, (2, 70, 3), device=dev)
    freq = [10000.0 ** (-2.0 * i / a) for a in axes for i in range(a // 2)]
    col = torch.tensor([i for i, a in enumerate(axes) for _ in range(a // 2)], device=dev)
    with torch.no_grad():
        yq, yk = rope(q, k, pos)
    a = angles(dev, pos.view(140, 3)[:, col], freq)
    for x, y in ((q, yq), (k, yk)):
        assert y.shape == x.shape
        ref.check(y.view(140, 4, 128), *ref.rope(x.view(140, 4, 128), a, 1.0, 128, True), "axes")


@pytest.mark.parametrize("scaling", [{"type": "linear", "factor": 4.0}, {"type": "ntk", "factor": 8.0},
                                     {"type": "yarn", "factor": 16.0, "original_max_position": 32768},
                                     {"type": "yarn", "factor": 4.0, "original_max_position": 4096,
                                      "attention_factor": 1.0}])
def test_rope_scaled_far_positions(cuda_device, scaling):
    """Positions far beyond where fp32 angles hold (and beyond 32 bits)."""
    from onecomp_runtime.layers import RotaryEmbedding
    dev = cuda_device
    rope = RotaryEmbedding(64, scaling=scaling)
    pos = torch.tensor([0, 1, -1, 99991, 1000003, 2**31 - 1, 2**33 + 12345], device=dev)
    q = randn(dev, len(pos), 3, 64, dtype=torch.float32)
    with torch.no_grad():
        y, _ = rope(q, None, pos)
    # angles modulo one turn in integers: 2^33 positions of a 53-bit frequency leave 2^-20 of a turn, so the
    # table's own rounding of frequency / 2 pi (2^-53) is part of the reference
    turns = torch.tensor([math.fmod(f / (2 * math.pi), 1.0) for f in rope.inv_freq], dtype=torch.float64, device=dev)
    hi = torch.floor(turns * 2**26)
    lo = turns * 2**26 - hi
    p = pos.double()[:, None]
    part = torch.remainder(p * hi, 2.0**26) / 2**26 + torch.remainder(p * lo, 2.0**26) / 2**26
    ref.check(y, *ref.rope(q, part * 2 * math.pi, rope.gain, 64, False), "far positions")


# ---------------------------------------------------------------------------------------- dense linear
@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 33, 64, 65, 128, 129, 255, 257, 700])
@pytest.mark.parametrize("dims", [(256, 512), (264, 384), (8, 40), (1032, 131), (4096, 1000)])
def test_linear_sizes(cuda_device, M, dims):
    from onecomp_runtime.layers import linear_fused
    dev = cuda_device
    K, N = dims
    x, w, b, r = randn(dev, M, K, seed=1), randn(dev, N, K, seed=2, std=K ** -0.5), randn(dev, N, seed=3), \
        randn(dev, M, N, seed=4)
    with torch.no_grad():
        ref.check(linear_fused(x, w), *ref.linear(x, w, None, None, None), f"linear {M} {dims}")
        ref.check(linear_fused(x, w, b, activation="silu", residual=r), *ref.linear(x, w, b, "silu", r),
                  f"linear epilogue {M} {dims}")
    assert error_word(dev) == 0


@pytest.mark.parametrize("shape", [(33, 1000, 8192), (64, 520, 6000), (100, 264, 5120), (128, 1024, 4104), (65, 6400, 4160),
                                   (200, 4100, 1024), (517, 2056, 640), (1030, 300, 72), (2049, 1288, 128)])
def test_linear_kernel_choice(cuda_device, shape):
    """Both kernels around the border of their rule (few tokens and a long K), and every token tile size."""
    from onecomp_runtime.layers import linear_fused
    dev = cuda_device
    M, N, K = shape
    x, w, b, r = randn(dev, M, K, seed=1), randn(dev, N, K, seed=2, std=K ** -0.5), randn(dev, N, seed=3), \
        randn(dev, M, N, seed=4)
    with torch.no_grad():
        ref.check(linear_fused(x, w, b, activation="gelu", residual=r), *ref.linear(x, w, b, "gelu", r), f"{shape}")
    assert error_word(dev) == 0


@pytest.mark.parametrize("act", [None, "gelu_tanh", "gelu", "silu", "relu"])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("M", [3, 300])
def test_linear_activations(cuda_device, act, dtype, M):
    from onecomp_runtime.layers import linear_fused
    dev = cuda_device
    K, N = 512, 520
    x, w = randn(dev, M, K, dtype=dtype, seed=1, std=3.0), randn(dev, N, K, dtype=dtype, seed=2, std=K ** -0.5)
    for bias_dtype in (dtype, torch.float32):
        b = randn(dev, N, dtype=bias_dtype, seed=3)
        with torch.no_grad():
            ref.check(linear_fused(x, w, b, activation=act), *ref.linear(x, w, b, act, None), f"{act}")


def test_linear_strides_and_aliases(cuda_device):
    """Strided x, w, residual and out; odd row pitches; the residual as the output; leading dimensions."""
    from onecomp_runtime.layers import linear_fused
    dev = cuda_device
    for M, N, K in ((5, 96, 128), (300, 200, 64), (520, 264, 192)):
        xb, wb = randn(dev, M, 2 * K, seed=1), randn(dev, N, K + 8, seed=2, std=K ** -0.5)
        x, w = xb[:, K:], wb[:, :K]
        rb = randn(dev, M, N + 3, seed=3)
        r = rb[:, 1:N + 1]
        want, tol = ref.linear(x, w, None, None, r)
        with torch.no_grad():
            ref.check(linear_fused(x, w, residual=r), want, tol, "strided")
            x1 = torch.cat([x, x[:, :1]], 1)[:, :K]                     # rows of K + 1 values
            ref.check(linear_fused(x1, w, residual=r), want, tol, "odd x rows")
            ob = torch.full((M, N + 5), 3.0, dtype=BF, device=dev)
            got = linear_fused(x, w, residual=r, out=ob[:, 2:N + 2])
            ref.check(got, want, tol, "strided out")
            assert bool((ob[:, :2] == 3).all()) and bool((ob[:, N + 2:] == 3).all())
            acc = r.contiguous()
            ref.check(linear_fused(x, w, residual=acc, out=acc), want, tol, "in place")
            rb2 = rb.clone()
            a2 = rb2[:, 1:N + 1]
            ref.check(linear_fused(x, w, residual=a2, out=a2), want, tol, "in place, strided")
            assert torch.equal(rb2[:, :1], rb[:, :1]) and torch.equal(rb2[:, N + 1:], rb[:, N + 1:])
            x3 = x.reshape(1, M, K)
            assert linear_fused(x3, w).shape == (1, M, N)
    e = torch.empty((0, 64), dtype=BF, device=dev)
    with torch.no_grad():
        assert linear_fused(e, randn(dev, 24, 64)).shape == (0, 24)


def test_linear_repeats_bit_for_bit(cuda_device):
    from onecomp_runtime.layers import linear_fused
    dev = cuda_device
    for M in (1, 40, 700):
        x, w = randn(dev, M, 4096, seed=1), randn(dev, 768, 4096, seed=2)
        with torch.no_grad():
            first = linear_fused(x, w)
            assert all(torch.equal(first, linear_fused(x, w)) for _ in range(5))


def test_eager_layer_forward_fused(cuda_device):
    """The dense layer of the eager backend takes forward_fused like the packed ones, and its plain forward
    is F.linear as before."""
    from onecomp_runtime.backend import build_quant_layer
    from onecomp_runtime.testing import gptq_layer
    dev = cuda_device
    t = gptq_layer(256, 384, 64, seed=5)
    entry = dict(name="a", wbits=4, groupsize=64, actorder=False, in_features=256, out_features=384)
    lin, kind = build_quant_layer(entry, t, "eager", BF, dev)
    assert kind == "eager" and isinstance(lin, torch.nn.Linear)
    x, r = randn(dev, 70, 256, seed=1), randn(dev, 70, 384, seed=2)
    y = lin.forward_fused(x, residual=r, activation="gelu_tanh")
    ref.check(y, *ref.linear(x, lin.weight.detach(), lin.bias.detach(), "gelu_tanh", r), "eager forward_fused")
    assert torch.equal(lin(x), torch.nn.functional.linear(x, lin.weight, lin.bias))


# ---------------------------------------------------------------------------------------- together
def block(x, mods, rope, heads, kv_heads, c, pos):
    from onecomp_runtime.layers import packed_attention
    D = rope.head_dim
    qkv = mods["qkv"].forward_fused(x)
    q = qkv[:, :heads * D].unflatten(1, (heads, D))
    k = qkv[:, heads * D:(heads + kv_heads) * D].unflatten(1, (kv_heads, D))
    v = qkv[:, (heads + kv_heads) * D:].unflatten(1, (kv_heads, D))
    rope(q, k, pos, inplace=True)
    o = packed_attention(q, k, v, c, c)
    h = mods["out"].forward_fused(o.flatten(1), residual=x)
    f = mods["fc1"].forward_fused(h, activation="gelu_tanh")
    return mods["fc2"].forward_fused(f, residual=h)


def block_mods(dev, hidden, qkv_out, mlp, kind, seed=0):
    from onecomp_runtime.backend import build_quant_layer
    from onecomp_runtime.testing import gptq_layer
    mods = {}
    for i, (name, K, N) in enumerate((("qkv", hidden, qkv_out), ("out", hidden, hidden), ("fc1", hidden, mlp),
                                      ("fc2", mlp, hidden))):
        t = gptq_layer(K, N, 32, seed=seed + i, scales_range=(0.001, 0.004))
        entry = dict(name=name, wbits=4, groupsize=32, actorder=False, in_features=K, out_features=N)
        mods[name] = build_quant_layer(entry, t, kind, BF, dev)[0]
    return mods


@pytest.mark.parametrize("kind", ["b200", "eager"])
def test_block_runs_together(cuda_device, kind):
    """A decoder block: packed or dense linears, rotary positions in place on the projection, attention on
    its slices, residuals in the epilogues; each step against the 64-bit restatement of that step."""
    from onecomp_runtime.layers import RotaryEmbedding, packed_attention
    dev = cuda_device
    heads, kv, D = 4, 2, 64
    hidden = heads * D
    mods = block_mods(dev, hidden, (heads + 2 * kv) * D, 512, kind)
    rope = RotaryEmbedding(D, rotary_dim=32)
    lens = [1, 70, 200, 13]
    c, T = cu(dev, lens), sum(lens)
    pos = torch.cat([torch.arange(n, device=dev) for n in lens])
    x = randn(dev, T, hidden, seed=9)
    with torch.no_grad():
        got = block(x, mods, rope, heads, kv, c, pos)
        qkv = mods["qkv"].forward_fused(x)
        q, k, v = qkv[:, :heads * D].unflatten(1, (heads, D)), qkv[:, heads * D:(heads + kv) * D].unflatten(1, (kv, D)), \
            qkv[:, (heads + kv) * D:].unflatten(1, (kv, D))
        a = angles(dev, pos[:, None], rope.inv_freq)
        rq, rk = rope(q, k, pos)
        for s, y in ((q, rq), (k, rk)):
            ref.check(y, *ref.rope(s, a, 1.0, 32, False), "rope in the block")
        o = packed_attention(rq, rk, v, c, c)
        seqs = [(sum(lens[:i]), n, sum(lens[:i]), n) for i, n in enumerate(lens)]
        ref.check(o, *ref.attention(rq, rk, v, seqs, True, D ** -0.5), "attention in the block")
        h = mods["out"].forward_fused(o.flatten(1), residual=x)
        f = mods["fc1"].forward_fused(h, activation="gelu_tanh")
        assert torch.equal(got, mods["fc2"].forward_fused(f, residual=h))
    assert bool(torch.isfinite(got.float()).all()) and error_word(dev) == 0


def test_block_captured_and_replayed(cuda_device):
    """Two captured graphs of the block (sharing the stream and module state) replay with new inputs and new
    lengths, at the same time on two streams."""
    from onecomp_runtime.layers import RotaryEmbedding
    dev = cuda_device
    heads, kv, D = 4, 2, 64
    mods = block_mods(dev, heads * D, (heads + 2 * kv) * D, 512, "eager", seed=3)
    rope = RotaryEmbedding(D, device=dev)
    graphs = []
    for lens in ([40, 60, 28], [1, 1, 126]):
        T = sum(lens)
        x, c, pos = randn(dev, T, heads * D, seed=T), cu(dev, lens), torch.arange(T, device=dev)
        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.no_grad(), torch.cuda.stream(side):
            block(x, mods, rope, heads, kv, c, pos)
            side.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                y = block(x, mods, rope, heads, kv, c, pos)
        graphs.append((g, side, x, c, pos, y))
    torch.cuda.synchronize(dev)
    for i, (g, side, x, c, pos, y) in enumerate(graphs):
        x.copy_(randn(dev, *x.shape, seed=100 + i))
        c.copy_(cu(dev, [10 + i, 50, 128 - 60 - i]))
    torch.cuda.synchronize(dev)
    for _ in range(20):
        for g, side, *_ in graphs:
            with torch.cuda.stream(side):
                g.replay()
    torch.cuda.synchronize(dev)
    for g, side, x, c, pos, y in graphs:
        with torch.no_grad():
            assert torch.equal(y, block(x, mods, rope, heads, kv, c, pos))
    assert error_word(dev) == 0


def test_many_streams_at_once(cuda_device):
    """The operators on several streams at a time: every call has its own workspace."""
    from onecomp_runtime.layers import linear_fused, packed_attention
    dev = cuda_device
    q, k, v = randn(dev, 4, 16, 128, seed=1), randn(dev, 9000, 2, 128, seed=2), randn(dev, 9000, 2, 128, seed=3)
    x, w = randn(dev, 4, 2048, seed=4), randn(dev, 1024, 2048, seed=5)
    cq, ck = cu(dev, [1, 1, 1, 1]), cu(dev, [2000, 3000, 1, 3999])
    with torch.no_grad():
        want, y = packed_attention(q, k, v, cq, ck), linear_fused(x, w)
        streams = [torch.cuda.Stream(dev) for _ in range(4)]
        torch.cuda.synchronize(dev)
        got = []
        for _ in range(5):
            for s in streams:
                with torch.cuda.stream(s):
                    got.append((packed_attention(q, k, v, cq, ck), linear_fused(x, w)))
        torch.cuda.synchronize(dev)
    assert all(torch.equal(a, want) and torch.equal(b, y) for a, b in got)
