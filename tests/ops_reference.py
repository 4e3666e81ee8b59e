"""Plain float64 forms of the operators around the attention, and the error bounds their kernels are held to."""
from __future__ import annotations

import math

import torch


def half_step(dtype) -> float:
    """A rounding's largest error relative to the value."""
    return torch.finfo(dtype).eps / 2


def attend64(q, k, v, *, causal=True, scale=None, softcap=0.0, slopes=None, prefix=None, ids=None):
    """One sequence: q (Hq, Sq, D), k and v (Hkv, Skv, D).  Returns o, lse and the error bound of each:

    P is rounded to the inputs' type (half a step of each probability, so of sum p |v| / l), o once more; a score is off by at most D 2^-24
    times its sum of absolute products (fp32 accumulation), the cap's tanh by 2^-22 of the cap, the bias by 2^-23 of itself, and a score's error is
    a probability's relative error, doubled here for the exp2 and the sums.  fp16 probabilities below 2^-14 are off by up to 2^-25 each."""
    Hq, Sq, D = q.shape
    G, Skv = Hq // k.shape[0], k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    kk, vv = (t.double().repeat_interleave(G, 0) for t in (k, v))
    qq = q.double()
    s = (qq @ kk.transpose(1, 2).contiguous()) * scale
    err = D * 2.0 ** -24 * scale * float((qq.abs().amax(1) @ kk.abs().amax(1).T).max()) if Skv and Sq else 0.0
    if softcap:
        s = softcap * torch.tanh(s / softcap)
        err += 2.0 ** -22 * softcap
    p = torch.arange(Sq, device=q.device)[:, None] + (Skv - Sq)
    j = torch.arange(Skv, device=q.device)[None, :]
    if slopes is not None:
        bias = slopes.double().view(Hq, 1, 1) * (p - j).abs()
        s = s - bias
        err += 2.0 ** -23 * min(float(bias.max()) if bias.numel() else 0.0, 200.0)  # (a key 200 below the others weighs nothing)
    seen = torch.ones(Sq, Skv, dtype=torch.bool, device=q.device)
    if causal:
        seen = j <= p
        if prefix:
            seen = seen | (j < prefix)
    if ids is not None:
        mine = ids[Skv - Sq:] if Sq else ids[:0]
        seen = seen & (mine[:, None] == ids[None, :]) & (mine >= 0)[:, None]
    s = s.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1) if Skv else torch.full((Hq, Sq), -math.inf, dtype=torch.float64, device=q.device)
    w = torch.exp(s - torch.where(lse == -math.inf, torch.zeros_like(lse), lse)[..., None])
    o = w @ vv
    u = half_step(q.dtype)
    tol = (u + 2 * err) * (w @ vv.abs()) + u * o.abs() + 2.0 ** -20
    if q.dtype == torch.float16 and Skv:
        tol = tol + min(Skv, 4096) * 2.0 ** -25 * float(v.abs().max()) + 2.0 ** -25
    lse_tol = 2 * err + 2.0 ** -19 + 2.0 ** -22 * lse.abs().nan_to_num(posinf=0.0)
    return o, lse, tol, lse_tol


def check_attention(got, lse, want):
    """`want`: attend64's answer."""
    o, l64, tol, lse_tol = want
    bad = (got.double() - o).abs() > tol
    assert torch.isfinite(got.float()).all()
    assert not bad.any(), f"{int(bad.sum())} outputs off, the worst by {float(((got.double() - o).abs() / tol).max()):.2f} of its bound"
    if lse is not None:
        empty = l64 == -math.inf
        assert torch.equal(lse.double() == -math.inf, empty)
        d = (lse.double() - l64).abs().masked_fill(empty, 0.0)
        assert (d <= lse_tol).all(), f"LSE off by {float(d.max()):.2e}"


def rope64(x, weight, eps, positions, *, rotary_dim, interleaved, inv_freq, axes):
    """x (..., D), positions (A, ...) without x's last dimension; returns the rows and their error bound."""
    D, R = x.shape[-1], rotary_dim
    y = x.double()
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + eps) * weight.double()
    size = y.abs().amax(-1, keepdim=True)
    if positions is not None:
        theta = positions.double()[torch.tensor(axes, device=x.device)].movedim(0, -1) * inv_freq.to(x.device).double()
        c, s = theta.cos(), theta.sin()
        y = y.clone()
        a, b = (slice(0, R // 2), slice(R // 2, R)) if not interleaved else (slice(0, R, 2), slice(1, R, 2))
        ya, yb = y[..., a].clone(), y[..., b].clone()
        y[..., a] = ya * c - yb * s
        y[..., b] = yb * c + ya * s
    # fp32 throughout (the sum of D squares, the root, five products: under 2^-19 of the row's largest), one rounding.
    u = half_step(x.dtype)
    return y, u * y.abs() + 2.0 ** -18 * size + (2.0 ** -25 if x.dtype == torch.float16 else 0.0)
