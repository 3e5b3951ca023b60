"""Workloads of the transformer-block operators beside the packed linears: rotary positions, attention
over packed sequences, and the dense 16-bit linear with its epilogue.

``run`` computes an operator in plain torch (32-bit, elementary operations) or, with ``own`` set, through
``onecomp_runtime``. Sizes follow the framework's own workloads: 32 heads of 128 (hidden 4096, fc1 16384)
of the video-DiT stack, the 5120-wide decode layers; wide heads rotated in part are the other common form.
"""
import math
import random

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one request, one new token, a short cache: the latency of a serving step
        dict(name="attn_decode_one", op="decode", batch=1, nq=1, cap=2048, lo=1531, hi=1531, hq=32, hkv=8, d=128,
             dtype="bf16"),
        # a full serving batch over padded caches of very different fill
        dict(name="attn_decode_batch", op="decode", batch=48, nq=1, cap=8192, lo=3, hi=8192, hq=32, hkv=8, d=128,
             dtype="bf16"),
        # a few tokens per request at once (the last words of a prompt, a drafted run), wide heads
        dict(name="attn_decode_few", op="decode", batch=7, nq=5, cap=4096, lo=900, hi=4096, hq=24, hkv=4, d=256,
             dtype="bf16"),
        # prompts of a serving batch packed without padding, causal, grouped heads
        dict(name="attn_prompt_packed", op="prompt", batch=9, total=16411, ctx=0, causal=True, hq=32, hkv=8, d=128,
             dtype="bf16"),
        # chunks of longer prompts: each chunk also sees what came before it
        dict(name="attn_prompt_chunk", op="prompt", batch=3, total=2999, ctx=6007, causal=True, hq=16, hkv=16, d=64,
             dtype="fp16"),
        # all tokens of a video clip at once, no mask: the DiT stack's attention
        dict(name="attn_video_full", op="prompt", batch=1, total=16384, ctx=0, causal=False, hq=32, hkv=32, d=128,
             dtype="bf16"),
        # the rotation of a decode step: a few tokens
        dict(name="rope_tokens", op="rope", tokens=17, hq=32, hk=8, d=128, rot=128, layout="half", axes="",
             scaling="", far=8192, dtype="bf16"),
        # a long prompt, a quarter of a wide head rotated, frequencies stretched for a long context
        dict(name="rope_long_partial", op="rope", tokens=16411, hq=24, hk=4, d=256, rot=64, layout="half", axes="",
             scaling="yarn", far=1000000, dtype="fp16"),
        # video tokens: time, height and width share the head, neighbouring pairs rotated
        dict(name="rope_video", op="rope", tokens=32768, hq=32, hk=32, d=128, rot=128, layout="interleaved",
             axes="16,56,56", scaling="", far=256, dtype="bf16"),
        # the output projection of one decode token, added to the residual stream
        dict(name="linear_token", op="linear", m=1, k=4096, n=4096, act="none", bias=True, res=True, dtype="bf16"),
        # a ragged mid-sized batch through a gate projection
        dict(name="linear_batch", op="linear", m=517, k=5120, n=8200, act="silu", bias=False, res=False, dtype="fp16"),
        # fc1 of the video stack with its activation
        dict(name="linear_fc1", op="linear", m=16384, k=4096, n=16384, act="gelu_tanh", bias=True, res=False,
             dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["decode", "decode", "prompt", "prompt", "rope", "linear", "linear"])
    if op == "decode":
        hq, hkv, d = rng.choice([(32, 8, 128), (32, 32, 128), (24, 4, 256), (16, 16, 64), (20, 4, 80), (12, 2, 128)])
        cap = _log(rng, 64, 8192)
        return dict(op=op, batch=_log(rng, 1, 32), nq=rng.choice([1, 1, 1, 2, 5, 8]), cap=cap,
                    lo=max(1, cap // rng.choice([2, 10, 100])), hi=cap, hq=hq, hkv=hkv, d=d,
                    dtype=rng.choice(["bf16", "fp16"]))
    if op == "prompt":
        hq, hkv, d = rng.choice([(32, 8, 128), (8, 8, 128), (24, 4, 256), (16, 16, 64), (10, 2, 96)])
        total = _log(rng, 33, 12000)
        return dict(op=op, batch=rng.randint(1, min(12, total)), total=total, ctx=rng.choice([0, 0, _log(rng, 1, 4000)]),
                    causal=rng.random() < 0.7, hq=hq, hkv=hkv, d=d, dtype=rng.choice(["bf16", "fp16"]))
    if op == "rope":
        d = rng.choice([64, 96, 128, 256])
        layout = rng.choice(["half", "interleaved"])
        axes = rng.choice(["", "", "16,24,24"]) if d >= 64 else ""
        rot = 64 if axes else rng.choice([d, d, d // 2, 32])
        hk = rng.choice([1, 2, 8, 32])
        return dict(op=op, tokens=_log(rng, 1, 32768), hq=hk * rng.choice([1, 4]) if hk < 32 else hk, hk=hk, d=min(d, 128) if hk == 32 else d,
                    rot=min(rot, 128) if hk == 32 else rot, layout=layout, axes=axes,
                    scaling="" if axes else rng.choice(["", "linear", "ntk", "yarn"]),
                    far=_log(rng, 1000, 1000000), dtype=rng.choice(["bf16", "fp16", "fp32"]))
    return dict(op=op, m=_log(rng, 1, 8192), k=8 * _log(rng, 8, 640), n=_log(rng, 40, 16384),
                act=rng.choice(["none", "gelu_tanh", "gelu", "silu", "relu"]), bias=rng.random() < 0.6,
                res=rng.random() < 0.5, dtype=rng.choice(["bf16", "fp16"]))


# ------------------------------------------------------------------------------------------ inputs
def _lengths(case, seed):
    """Host lengths of a case: (query lengths, key lengths)."""
    rng = random.Random(f"{seed}-{sorted(case.items())}")
    if case["op"] == "decode":
        lk = [rng.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]
        nq = min(case["nq"], min(lk))
        return [nq] * case["batch"], lk
    cuts = sorted(rng.sample(range(1, case["total"]), case["batch"] - 1)) if case["batch"] > 1 else []
    lq = [b - a for a, b in zip([0] + cuts, cuts + [case["total"]])]
    return lq, [n + (rng.randint(0, case["ctx"]) if case["ctx"] else 0) for n in lq]


def _work_lengths(case):
    """The lengths ``work`` counts: those of the first seed."""
    return _lengths(case, 0)


def _rope_scaling(case):
    return {"": None, "linear": {"type": "linear", "factor": 4.0}, "ntk": {"type": "ntk", "factor": 8.0},
            "yarn": {"type": "yarn", "factor": 16.0, "original_max_position": 32768}}[case["scaling"]]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(1000003 * (seed % 100000) + 17)
    dt = _DT[case["dtype"]]

    def randn(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * std).to(dt)

    op = case["op"]
    if op in ("decode", "prompt"):
        lq, lk = _lengths(case, seed)
        hq, hkv, d = case["hq"], case["hkv"], case["d"]

        def cum(v):
            return torch.tensor([0] + v, dtype=torch.int32).cumsum(0).to(torch.int32).to(dev)

        st = dict(case=case, lq=lq, lk=lk, cu_q=cum(lq), max_q=max(lq))
        if op == "decode":   # padded caches [batch * cap, heads, d]; what lies behind a length is old data
            st["q"] = randn(sum(lq), hq, d, std=1.5)
            st["k"], st["v"] = randn(case["batch"] * case["cap"], hkv, d), randn(case["batch"] * case["cap"], hkv, d)
            st["cu_k"] = cum([case["cap"]] * case["batch"])
            st["kv_lens"] = torch.tensor(lk, dtype=torch.int32, device=dev)
        elif case["ctx"] == 0:   # one projection's output: q, k and v are its column slices
            qkv = randn(sum(lq), (hq + 2 * hkv) * d)
            st["q"] = qkv[:, :hq * d].unflatten(1, (hq, d))
            st["k"] = qkv[:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d))
            st["v"] = qkv[:, (hq + hkv) * d:].unflatten(1, (hkv, d))
            st["cu_k"] = st["cu_q"]
        else:
            st["q"] = randn(sum(lq), hq, d, std=1.5)
            st["k"], st["v"] = randn(sum(lk), hkv, d), randn(sum(lk), hkv, d)
            st["cu_k"] = cum(lk)
        return st
    if op == "rope":
        t, hq, hk, d = case["tokens"], case["hq"], case["hk"], case["d"]
        qkv = randn(t, (hq + 2 * hk) * d)
        axes = [int(a) for a in case["axes"].split(",")] if case["axes"] else None
        shape = (t, len(axes)) if axes else (t,)
        st = dict(case=case, axes=axes, q=qkv[:, :hq * d].unflatten(1, (hq, d)),
                  k=qkv[:, hq * d:(hq + hk) * d].unflatten(1, (hk, d)),
                  pos=torch.randint(0, case["far"], shape, generator=g, device=dev, dtype=torch.int64))
        if own:
            from onecomp_runtime.layers import RotaryEmbedding
            st["rope"] = RotaryEmbedding(d, rotary_dim=case["rot"], layout=case["layout"], axes=axes,
                                         scaling=_rope_scaling(case), device=dev)
        else:
            freq, gain = _frequencies(case, axes)
            st["freq"], st["gain"] = torch.tensor(freq, dtype=torch.float64, device=dev), gain
            if axes:
                st["axis"] = torch.tensor([a for a, n in enumerate(axes) for _ in range(n // 2)], device=dev)
        return st
    m, k, n = case["m"], case["k"], case["n"]
    st = dict(case=case, x=randn(m, k), w=randn(n, k, std=1.0 / math.sqrt(k)), b=None, r=None)
    if case["bias"]:
        st["b"] = randn(n, std=0.1)
    if case["res"]:
        st["r"] = randn(m, n)
    return st


# --------------------------------------------------------------------------------------- the forms
def run(state):
    op = state["case"]["op"]
    with torch.no_grad():
        if own:
            return _run_own(op, state)
        if op == "decode":
            return _plain_decode(state)
        if op == "prompt":
            return _plain_prompt(state)
        if op == "rope":
            return _plain_rope(state)
        return _plain_linear(state)


def _run_own(op, st):
    from onecomp_runtime import layers
    if op in ("decode", "prompt"):
        return layers.packed_attention(st["q"], st["k"], st["v"], st["cu_q"], st["cu_k"], kv_lens=st.get("kv_lens"),
                                       causal=st["case"].get("causal", True), max_seqlen_q=st["max_q"])
    if op == "rope":
        return st["rope"](st["q"], st["k"], st["pos"])
    act = st["case"]["act"]
    return layers.linear_fused(st["x"], st["w"], st["b"], activation=None if act == "none" else act, residual=st["r"])


def _plain_decode(st):
    """All requests at once over the padded caches; invisible keys get weight zero."""
    c = st["case"]
    b, cap, hq, hkv, d = c["batch"], c["cap"], c["hq"], c["hkv"], c["d"]
    nq, grp = st["lq"][0], hq // hkv
    q = st["q"].float().view(b, nq, hkv, grp, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, grp * nq, d)
    k = st["k"].float().view(b, cap, hkv, d).permute(0, 2, 1, 3)
    v = st["v"].float().view(b, cap, hkv, d).permute(0, 2, 1, 3)
    s = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(d))
    last = st["kv_lens"].view(b, 1) - nq + torch.arange(nq, device=s.device)         # last visible key per query
    hidden = torch.arange(cap, device=s.device) > last.unsqueeze(-1)                  # [b, nq, cap]
    s = s.view(b, hkv, grp, nq, cap).masked_fill(hidden[:, None, None], float("-inf")).view(b, hkv, grp * nq, cap)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    return o.view(b, hkv, grp, nq, d).permute(0, 3, 1, 2, 4).reshape(b * nq, hq, d).to(st["q"].dtype)


def _plain_prompt(st):
    """Sequence by sequence, in blocks of queries."""
    c = st["case"]
    grp, d = c["hq"] // c["hkv"], c["d"]
    out = torch.empty_like(st["q"], memory_format=torch.contiguous_format)
    q0 = k0 = 0
    for nq, nk in zip(st["lq"], st["lk"]):
        k = st["k"][k0:k0 + nk].float().transpose(0, 1)
        v = st["v"][k0:k0 + nk].float().transpose(0, 1)
        step = max(16, min(nq, int(2e8 / (c["hq"] * nk))))
        for i in range(0, nq, step):
            n = min(step, nq - i)
            end = nk if not c["causal"] else nk - nq + i + n                  # keys that any of these rows sees
            q = st["q"][q0 + i:q0 + i + n].float().transpose(0, 1).reshape(c["hkv"], grp * n, d)
            s = torch.matmul(q, k[:, :end].transpose(-1, -2)) * (1.0 / math.sqrt(d))
            if c["causal"]:
                row = torch.arange(n, device=s.device) + (nk - nq + i)
                hidden = torch.arange(end, device=s.device) > row.unsqueeze(-1)
                s = s.view(c["hkv"], grp, n, end).masked_fill(hidden, float("-inf")).view(c["hkv"], grp * n, end)
            p = torch.exp(s - s.amax(-1, keepdim=True))
            o = torch.matmul(p, v[:, :end]) / p.sum(-1, keepdim=True)
            out[q0 + i:q0 + i + n] = o.reshape(c["hq"], n, d).transpose(0, 1).to(out.dtype)
        q0, k0 = q0 + nq, k0 + nk
    return out


def _frequencies(case, axes):
    """(angle per position of every rotated pair, gain of the rotated values)."""
    base, rot = 10000.0, case["rot"]
    if axes:
        return [base ** (-2.0 * i / n) for n in axes for i in range(n // 2)], 1.0
    s = _rope_scaling(case)
    if s and s["type"] == "ntk":
        base *= s["factor"] ** (rot / (rot - 2.0))
    freq = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    gain = 1.0
    if s and s["type"] == "linear":
        freq = [f / s["factor"] for f in freq]
    if s and s["type"] == "yarn":
        def pair_at(turns):   # the pair that makes this many turns over the original context
            return rot * math.log(s["original_max_position"] / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))
        low, high = max(math.floor(pair_at(32.0)), 0), min(math.ceil(pair_at(1.0)), rot - 1)
        keep = [1.0 - min(max((i - low) / max(high - low, 1e-3), 0.0), 1.0) for i in range(rot // 2)]
        freq = [f * w + f / s["factor"] * (1.0 - w) for f, w in zip(freq, keep)]
        gain = 0.1 * math.log(s["factor"]) + 1.0
    return freq, gain


def _plain_rope(st):
    c = st["case"]
    pos = st["pos"].double()
    ang = (pos[:, st["axis"]] if st["axes"] else pos.unsqueeze(-1)) * st["freq"]
    cos, sin = (torch.cos(ang) * st["gain"]).float().unsqueeze(1), (torch.sin(ang) * st["gain"]).float().unsqueeze(1)

    def rotate(x):
        y = x.float()
        r = y[..., :c["rot"]]
        if c["layout"] == "half":
            a, b = r[..., :c["rot"] // 2], r[..., c["rot"] // 2:]
            r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        else:
            a, b = r[..., 0::2], r[..., 1::2]
            r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        return torch.cat([r, y[..., c["rot"]:]], -1).to(x.dtype)

    return rotate(st["q"]), rotate(st["k"])


def _plain_linear(st):
    y = torch.matmul(st["x"].float(), st["w"].float().t())
    if st["b"] is not None:
        y = y + st["b"].float()
    act = st["case"]["act"]
    if act == "gelu_tanh":
        y = 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
    elif act == "gelu":
        y = 0.5 * y * torch.special.erfc(y * (-1.0 / math.sqrt(2.0)))
    elif act == "silu":
        y = y / (1.0 + torch.exp(-y))
    elif act == "relu":
        y = torch.clamp_min(y, 0.0)
    if st["r"] is not None:
        y = y + st["r"].float()
    return y.to(st["x"].dtype)


# ------------------------------------------------------------------------- 64 bits, by another route
def exact(case, seed):
    global own
    mine, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = mine
    if case["op"] in ("decode", "prompt"):
        return _exact_attention(st)
    if case["op"] == "rope":
        return _exact_rope(st)
    return _exact_linear(st)


def _exact_attention(st):
    """Head by head: weights through the log of the sum of exponentials."""
    c = st["case"]
    causal = c.get("causal", True)
    out = torch.empty(st["q"].shape, dtype=torch.float64, device=st["q"].device)
    q0, k0 = 0, 0
    for i, (nq, nk) in enumerate(zip(st["lq"], st["lk"])):
        if c["op"] == "decode":
            k0 = i * c["cap"]
        kpos = torch.arange(nk, device=out.device)
        for h in range(c["hq"]):
            kh = st["k"][k0:k0 + nk, h * c["hkv"] // c["hq"]].double()
            vh = st["v"][k0:k0 + nk, h * c["hkv"] // c["hq"]].double()
            for r in range(0, nq, 4096):
                rows = torch.arange(r, min(nq, r + 4096), device=out.device)
                logits = torch.einsum("id,jd->ij", st["q"][q0 + rows, h].double(), kh) / math.sqrt(c["d"])
                if causal:
                    logits[kpos[None, :] > rows[:, None] + (nk - nq)] = -math.inf
                logits -= torch.logsumexp(logits, 1, keepdim=True)
                out[q0 + rows, h] = torch.einsum("ij,jd->id", logits.exp_(), vh)
        q0, k0 = q0 + nq, k0 + nk
    return out


def _exact_rope(st):
    """Every pair as a complex number times gain * e^(i angle), angles as parts of a turn."""
    c = st["case"]
    axis = st["axis"] if st["axes"] else torch.zeros(c["rot"] // 2, dtype=torch.int64, device=st["pos"].device)
    pos = st["pos"].reshape(c["tokens"], -1)[:, axis].double()
    turn = torch.polar(torch.full_like(pos, st["gain"]), pos * st["freq"])

    def rotate(x):
        y = x.double().clone()
        h = c["rot"] // 2
        first, second = (slice(0, h), slice(h, c["rot"])) if c["layout"] == "half" else (slice(0, c["rot"], 2), slice(1, c["rot"], 2))
        z = torch.complex(y[..., first], y[..., second]) * turn[:, None, :]
        y[..., first], y[..., second] = z.real, z.imag
        return y

    return rotate(st["q"]), rotate(st["k"])


def _exact_linear(st):
    c = st["case"]
    w = st["w"].double()
    out = torch.empty(c["m"], c["n"], dtype=torch.float64, device=w.device)
    for i in range(0, c["m"], 2048):
        y = torch.nn.functional.linear(st["x"][i:i + 2048].double(), w, None if st["b"] is None else st["b"].double())
        if c["act"] == "gelu_tanh":
            y = y * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3))
        elif c["act"] == "gelu":
            y = y * torch.special.ndtr(y)
        elif c["act"] == "silu":
            y = y * torch.sigmoid(y)
        elif c["act"] == "relu":
            y = torch.where(y > 0, y, torch.zeros_like(y))
        out[i:i + 2048] = y if st["r"] is None else y + st["r"][i:i + 2048].double()
    return out


# -------------------------------------------------------------------------------------------- work
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    op = case["op"]
    if op in ("decode", "prompt"):
        lq, lk = _work_lengths(case)
        causal = case.get("causal", True)
        pairs = sum(nq * nk - (nq * (nq - 1) // 2 if causal else 0) for nq, nk in zip(lq, lk))
        rows = 2 * sum(lq) * case["hq"] + 2 * sum(lk) * case["hkv"]
        return {"bytes": rows * case["d"] * e, "flops": 4 * pairs * case["hq"] * case["d"]}
    if op == "rope":
        rows = case["tokens"] * (case["hq"] + case["hk"])
        pos = 8 * case["tokens"] * (case["axes"].count(",") + 1)
        return {"bytes": 2 * rows * case["d"] * e + pos, "flops": 3 * rows * case["rot"]}
    m, k, n = case["m"], case["k"], case["n"]
    moved = m * k + n * k + m * n * (2 if case["res"] else 1) + (n if case["bias"] else 0)
    return {"bytes": moved * e, "flops": 2 * m * n * k}
