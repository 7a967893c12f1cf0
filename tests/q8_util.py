"""The 8-bit KV format and attention over it in 64 bits (torch, on the
tensors' own device), written from the definitions for the tests of 8-bit
pools."""

from __future__ import annotations

import math

import torch

EPS = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step


def pow2(e):
    """2^e in f64, by its exponent field."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def stored(x):
    """Values of head vectors x [..., head_dim] after a trip through the cache, in f64."""
    x = x.double()
    finite = torch.isfinite(x).all(-1, keepdim=True)
    x = torch.where(finite, x, torch.zeros_like(x))
    mant, e = torch.frexp(x.abs().amax(-1, keepdim=True) / 448.0)
    e = torch.where(mant == 0.5, e - 1, e).clamp(min=-126)
    t = x * pow2(-e)
    _, te = torch.frexp(t)
    quantum = pow2((te - 1).clamp(min=-6) - 3)
    v = torch.round(t / quantum) * quantum * pow2(e)
    return torch.where(finite, v, torch.full_like(v, math.nan))


def row_ranges(positions, window, causal=True):
    """Keys [lo, hi) of rows of one chunk (attn.wgsl:78-88,169)."""
    n = len(positions)
    out = []
    for i, p in enumerate(positions):
        kv_len = positions[min((i // 8) * 8 + 8, n) - 1] + 1 if causal else positions[-1] + 1
        lo = max(0, p + 1 - window) if causal and window else 0
        out.append((lo, min(kv_len, p + 1) if causal else kv_len))
    return out


def attend(q, k, v, ranges, scale, softcap=0.0):
    """(y, bound) in f64: q [m, heads, hd] over stored keys and values [n,
    kv_heads, hd], row i reading keys [lo, hi) of ranges[i].  bound is how far
    an implementation may be off that multiplies codes exactly, sums in f32 and
    splits the probabilities into 16 bits: with A = scale * max sum|q_d k_d|, a
    score is off by head_dim f32 roundings of at most A (and two more for an f32
    query's 22 bits), which a weight takes over relatively, twice (numerator
    and sum); each term by 2^-17, twice; sums over n keys by at most n / 8 + 64
    roundings in a row, in the numerator and in the denominator."""
    q, k, v = q.double(), k.double(), v.double()
    m, nq, hd = q.shape
    g = nq // k.shape[1]
    y = torch.full((m, nq, hd), math.nan, dtype=torch.float64, device=q.device)
    bound = torch.zeros(m, nq, 1, dtype=torch.float64, device=q.device)
    for i, (lo, hi) in enumerate(ranges):
        if hi <= lo:
            continue
        for h in range(k.shape[1]):
            kk, vv, qq = k[lo:hi, h], v[lo:hi, h], q[i, h * g:(h + 1) * g]
            s = qq @ kk.t() * scale
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            w = torch.exp(s - s.amax(-1, keepdim=True))
            y[i, h * g:(h + 1) * g] = w @ vv / w.sum(-1, keepdim=True)
            a = (qq.abs() @ kk.abs().t()).amax() * abs(scale)
            if softcap:  # + the tanh's own: 2^-22 of the cap (a difference of 1 and an f32 quotient)
                a = a + softcap * 4.0 / hd
            bound[i, h * g:(h + 1) * g] = vv.abs().amax() * (2.0 ** -16 + 2 * (hd + 2) * 2.0 ** -24 * a +
                                                             ((hi - lo) / 8 + 64) * 2.0 ** -23)
    return y, bound


def check(name, got, want, bound, dtype):
    """got (the kernel's, of dtype) against want within bound plus the output's rounding."""
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{name}: NaN in other places"
    want = torch.nan_to_num(want)
    err = (torch.nan_to_num(got) - want).abs()
    lim = bound + (want.abs() + bound) * EPS[dtype] + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    worst = (err / lim.clamp(min=1e-300)).max().item() if err.numel() else 0.0
    print(f"[q8-test] {name}: max err {err.max().item() if err.numel() else 0:.3g}, {worst:.3f} of the bound", flush=True)
    assert worst <= 1.0, name
