"""64-bit restatements of the transformer-block operators, with bounds on what their kernels may be off."""
from __future__ import annotations

import math

import torch


def half_step(dtype: torch.dtype) -> float:
    """Largest relative error of one rounding to ``dtype``."""
    return torch.finfo(dtype).eps / 2


def attention(q, k, v, seqs, causal, scale):
    """``seqs``: (q0, nq, k0, nk) per sequence. Returns (out, tol) in float64; rows of no sequence are zero.

    The bound, per output: the scores are fp32 sums of D products (each addition and the product with the
    scale off by 2^-23 of the magnitudes at most), so a weight is off by a factor 1 + 2 d with
    d = D 2^-23 scale sum|q k|, through numerator and denominator; the exponential adds 2^-21; the weight is
    rounded to 16 bits once (half a step; below fp16's normal range 2^-25 absolute, the largest weight
    being at least 1); sums over keys add nk 2^-24; the result is rounded once."""
    Tq, Hq, D = q.shape
    G = Hq // k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    h = half_step(q.dtype)
    for q0, nq, k0, nk in seqs:
        if nq == 0 or nk == 0:
            continue
        qq = q[q0:q0 + nq].double().transpose(0, 1)
        kk = k[k0:k0 + nk].double().transpose(0, 1).repeat_interleave(G, 0)
        vv = v[k0:k0 + nk].double().transpose(0, 1).repeat_interleave(G, 0)
        s = (qq @ kk.transpose(1, 2)) * scale
        d = (qq.abs() @ kk.abs().transpose(1, 2)) * abs(scale) * D * 2.0 ** -23
        if causal:
            seen = torch.arange(nk, device=q.device)[None] <= torch.arange(nq, device=q.device)[:, None] + nk - nq
        else:
            seen = torch.ones(nq, nk, dtype=torch.bool, device=q.device)
        s = s.masked_fill(~seen, -math.inf)
        d = d.masked_fill(~seen, 0.0).amax(-1, keepdim=True)
        mx = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(torch.isinf(mx), torch.zeros_like(mx), mx)).masked_fill(~seen, 0.0)
        l = p.sum(-1, keepdim=True)
        w = torch.where(l > 0, p / l, torch.zeros_like(p))
        o = w @ vv
        a = w @ vv.abs()
        extra = nk * 2.0 ** -25 * vv.abs().amax() if q.dtype == torch.float16 else 0.0
        t = h * o.abs() + (h + 2 * d + 2.0 ** -20 + nk * 2.0 ** -24) * a * (1 + h) + extra
        out[q0:q0 + nq] = o.transpose(0, 1)
        tol[q0:q0 + nq] = t.transpose(0, 1)
    return out, tol


def rope(x, ang, gain, rot, interleaved):
    """``x`` [T, H, D], ``ang`` [T, rot/2] float64. Bound: one rounding of the result, plus 2^-22 of the
    pair's magnitude for sine, cosine (2^-25 of a half turn and the functions' own error) and three fp32
    operations."""
    y = x.double().clone()
    n = rot // 2
    i1 = torch.arange(0, rot, 2, device=x.device) if interleaved else torch.arange(n, device=x.device)
    i2 = i1 + (1 if interleaved else n)
    a, b = x.double()[..., i1], x.double()[..., i2]
    c, s = (torch.cos(ang) * gain).unsqueeze(1), (torch.sin(ang) * gain).unsqueeze(1)
    y[..., i1], y[..., i2] = a * c - b * s, b * c + a * s
    tol = half_step(x.dtype) * y.abs()
    mag = (a.abs() + b.abs()) * abs(gain) * 2.0 ** -21
    tol[..., i1] += mag
    tol[..., i2] += mag
    if x.dtype == torch.float16:
        tol += 2.0 ** -25
    tol[..., rot:] = 0
    return y, tol


def act64(y, name):
    if name == "gelu_tanh":
        return y * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3))
    if name == "gelu":
        return y * torch.special.ndtr(y)
    if name == "silu":
        return y * torch.sigmoid(y)
    if name == "relu":
        return torch.clamp_min(y, 0.0)
    return y


def linear(x, w, bias, act, residual):
    """Bound: fp32 sums of K products, 2^-23 of the magnitudes per addition at most; the activations change
    by at most 1.13 times their input's change, plus 2^-19 of their value for exponential and division;
    the residual's addition 2^-24; one rounding."""
    K = x.shape[-1]
    y = x.double() @ w.double().t()
    mag = x.double().abs() @ w.double().abs().t()
    if bias is not None:
        y = y + bias.double()
        mag = mag + bias.double().abs()
    d = mag * (K + 2) * 2.0 ** -23
    z = act64(y, act)
    tol = 1.13 * d + z.abs() * 2.0 ** -19
    if residual is not None:
        z = z + residual.double()
        tol = tol + z.abs() * 2.0 ** -23
    tol = tol + half_step(x.dtype) * (z.abs() + tol)
    if x.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    return z, tol


def check(got, want, tol, what=""):
    """Every value within its bound; the message names the worst one."""
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    if bool(bad.any()):
        r = torch.where(torch.isnan(err), torch.full_like(err, math.inf), err - tol)
        i = int(r.flatten().argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values off; worst at {i} (shape "
                             f"{tuple(got.shape)}): got {got.flatten()[i].item()}, want {want.flatten()[i].item()}, "
                             f"bound {tol.flatten()[i].item()}")
