"""Plain 64-bit forms of the attention layer's operators and the error that the kernels may make.

Each reference returns (value, tolerance), elementwise. U16 = 2^-11 is half a binary16 step relative to
the value, TINY = 2^-25 half the smallest step, U32 = 2^-24 half an fp32 step.
"""
import math

import torch

U16, TINY, U32 = 2.0 ** -11, 2.0 ** -25, 2.0 ** -24


def token_adapters(T, seg_start, seg_adapter, adapters):
    """Adapter of every token, -1 for none."""
    ids = [-1] * T
    for s, a in enumerate(seg_adapter):
        for t in range(max(0, seg_start[s]), min(T, seg_start[s + 1])):
            ids[t] = a if 0 <= a < adapters else -1
    return ids


def lora(X, W, down, up, scale, ids):
    """One rounding of the sum (U16 |y|); the scaled low-rank row is rounded as an operand (U16, TINY);
    K + rank + 8 fp32 additions and the scale's product, each U32 of the sum of magnitudes."""
    x = X.double()
    K, r = X.shape[1], down.shape[2]
    y, mag = x @ W.double(), x.abs() @ W.double().abs()
    tol = (K + 8) * U32 * mag
    for a in sorted(set(ids) - {-1}):
        rows = torch.tensor([i for i, b in enumerate(ids) if b == a], device=X.device)
        s, u, d = scale[a].double(), up[a].double(), down[a].double()
        h = s * (x[rows] @ d)
        hmag = s.abs() * (x[rows].abs() @ d.abs())
        y[rows] += h @ u
        tol[rows] += (U16 * h.abs() + TINY + (K + 8) * U32 * hmag) @ u.abs()
        tol[rows] += (K + r + 8) * U32 * (h.abs() @ u.abs())
    return y, tol + U16 * y.abs() + TINY


def qk_norm_rope(x, w, positions, inv_freq, axis, eps, interleaved):
    """One rounding (U16 |y|); in fp32 a sum of squares (13 additions), rsqrt, four products and the
    rotation's two, sin and cos of an angle rounded to fp32 over pi: under 64 U32 of |n1| + |n2|."""
    rot = 2 * inv_freq.numel()
    x = x.double()
    n = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    y, mag = n.clone(), n.abs()
    if rot:
        pos = positions.reshape(-1, x.shape[0]).double()
        ang = pos[axis.long()].t() * inv_freq.double()
        c, s = ang.cos()[:, None], ang.sin()[:, None]
        i = torch.arange(rot // 2, device=x.device)
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        y[..., a] = n[..., a] * c - n[..., b] * s
        y[..., b] = n[..., b] * c + n[..., a] * s
        mag[..., a] = mag[..., b] = n[..., a].abs() + n[..., b].abs()
    return y, U16 * y.abs() + 64 * U32 * mag + TINY


def attn(q, k, v, q_lens, k_lens, scale, causal, out_rows=None):
    """(out, tolerance, lse, lse tolerance); rows behind the last sequence are NaN.

    Scores: head_dim + 4 fp32 operations, so a weight is off by the factor 1 + e with
    e = scale (d + 4) U32 sum|q||k| + 8 U32 (exp). Weights relative to a running maximum that is at most 2^8
    behind are rounded to binary16: U16 relative, TINY absolute each (their sum is at least 1),
    and n + 16 fp32 additions in the sums; one rounding of the output."""
    Tq, hq, d = q.shape
    hkv = k.shape[1]
    g = hq // hkv
    out = torch.full((Tq, hq, d), math.nan, dtype=torch.float64, device=q.device)
    tol, lse = torch.zeros_like(out), out[..., 0].clone()
    ltol = torch.zeros_like(lse)
    iq = ik = 0
    for nq, nk in zip(q_lens, k_lens):
        for h in range(hq):
            qq = q[iq:iq + nq, h].double()
            kk, vv = (t[ik:ik + nk, h // g].double() for t in (k, v))
            s = scale * (qq @ kk.t())
            e = abs(scale) * (d + 4) * U32 * (qq.abs() @ kk.abs().t()) + 8 * U32
            see = torch.ones((nq, nk), dtype=torch.bool, device=q.device)
            if causal:
                see = see.tril(nk - nq)
            none = ~see.any(-1) if nk else torch.ones(nq, dtype=torch.bool, device=q.device)
            s = s.masked_fill(~see, -math.inf)
            top = s.amax(-1, keepdim=True) if nk else s.new_zeros((nq, 1))
            top = top.masked_fill(none[:, None], 0.0)
            p = (s - top).exp()
            l = p.sum(-1, keepdim=True)
            w = (p / l).masked_fill(none[:, None], 0.0)
            # A masked place holds no value: what stands there must not reach the row.
            clean = torch.nan_to_num(vv, nan=0.0, posinf=0.0, neginf=0.0)
            o = w @ clean
            bad = ~torch.isfinite(vv)
            if bad.any():
                touched = (see.double() @ bad.double()) > 0
                o = o.masked_fill(touched, math.nan)
            err = (w * (U16 + 2 * e.masked_fill(~see, 0.0) + (nk + 16) * U32)) @ clean.abs()
            err += TINY * (see.double() @ clean.abs())
            out[iq:iq + nq, h] = o
            tol[iq:iq + nq, h] = err + U16 * o.abs() + TINY
            z = (top + l.log())[:, 0].masked_fill(none, -math.inf)
            lse[iq:iq + nq, h] = z
            ltol[iq:iq + nq, h] = (4 * U32 * z.abs().masked_fill(none, 0.0) +
                                   (nk + 16) * U32 + 2 * e.masked_fill(~see, 0.0).amax(-1)
                                   if nk else 0.0)
        iq, ik = iq + nq, ik + nk
    return out, tol, lse, ltol


def close(got, want, tol, what=""):
    """Every element within its tolerance; NaN where and only where it is wanted."""
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN in other places"
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]), f"{what}: infinities differ"
    ok = want.isfinite()
    bad = ((got - want).abs() > tol) & ok
    if bad.any():
        at = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {at}: "
                             f"{got[at].item()} for {want[at].item()}, tolerance {tol[at].item()}")
