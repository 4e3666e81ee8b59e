"""Softcaps where they bend: scores of exact products on both sides of every form's border, against float64, with bounds that a cap off by
one in a hundred does not keep."""
import math

import pytest
import torch

from gqa_kernels import gqa_flash_attn
from gqa_kernels.paged import paged_attention
from ops_reference import half_step

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def whole_numbers(B, Hq, Hkv, Sq, Skv, D, dtype, factors, seed=0, turned=1):
    """q, k of whole numbers up to 3 (their products' sums stay below 2^24: exact in any order), q's rows times powers of two in turn (turned by
    `turned` places a head)."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(-3, 4, (B, Hq, Sq, D), generator=g).float()
    q *= torch.tensor([[factors[(i + turned * h) % len(factors)] for i in range(Sq)] for h in range(Hq)]).view(1, Hq, Sq, 1)
    k = torch.randint(-3, 4, (B, Hkv, Skv, D), generator=g).float()
    v = torch.randn(B, Hkv, Skv, D, generator=g)
    return tuple(t.to(dtype).cuda() for t in (q, k, v))


def capped64(q, k, v, cap, causal):
    """One sequence's o and lse in float64, and their bounds.

    The products are exact.  cap tanh(s / cap): 2^-20 of a row's largest value under caps above 128 (the cap and its reciprocal in fp32 2^-22; the
    polynomial 2^-23; past its end 2^-22 of the cap, which is under 2^-20.5 of the value there; the exponent's scale and sum 2^-23), 2^-21 of the cap
    under others (reciprocal and sum 2^-22 of it, the exponential's own and its argument's rounding each 2^-23).  An error of a score is one of its
    probability, doubled for the exponential and the sums.  P is rounded to the inputs' type (half a step of each), o once more."""
    G, (Hq, Sq, D), Skv = q.shape[0] // k.shape[0], q.shape, k.shape[1]
    kk, vv = (t.double().repeat_interleave(G, 0) for t in (k, v))
    s = cap * torch.tanh((q.double() @ kk.transpose(1, 2).contiguous()) * D ** -0.5 / cap)
    seen = torch.arange(Skv, device=q.device)[None] <= torch.arange(Sq, device=q.device)[:, None] + Skv - Sq if causal \
        else torch.ones(Sq, Skv, dtype=torch.bool, device=q.device)
    err = 2.0 ** -20 * (s.abs() * seen).amax(-1, keepdim=True) if cap > 128 else torch.full_like(s[..., :1], 2.0 ** -21 * cap)
    s = s.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1)
    w = torch.exp(s - lse[..., None])
    o, u = w @ vv, half_step(q.dtype)
    tol = (u + 2 * err.clamp(max=50.0).expm1()) * (w @ vv.abs()) + u * o.abs() + 2.0 ** -20
    if q.dtype == FP:
        tol = tol + Skv * 2.0 ** -25 * float(v.abs().max()) + 2.0 ** -25
    return o, lse, tol, 2 * err[..., 0] + 2.0 ** -19 + 2.0 ** -22 * lse.abs()


def kept(o, lse, want):
    d = (o.double() - want[0]).abs() - want[2]
    return bool((d <= 0).all()) and bool(((lse.double() - want[1]).abs() <= want[3]).all())


def check(o, lse, q, k, v, cap, causal=True):
    assert torch.isfinite(o).all() and torch.isfinite(lse).all()
    for b in range(q.shape[0]):
        want = capped64(q[b], k[b], v[b], cap, causal)
        d, dl = ((o[b].double() - want[0]).abs() / want[2]).max(), ((lse[b].double() - want[1]).abs() / want[3]).max()
        assert d <= 1 and dl <= 1, f"o off by {float(d):.2f} of its bound, LSE by {float(dl):.2f}"
        for wrong in (0.99, 1.01):  # (what the bounds are worth)
            other = capped64(q[b], k[b], v[b], cap * wrong, causal)
            assert not kept(other[0], other[1], want)


SHAPES = [(1, 8, 2, 150, 150, 128), (1, 8, 2, 150, 150, 64), (2, 8, 2, 1, 1500, 128), (2, 8, 2, 1, 1500, 64), (1, 8, 2, 20, 700, 128),
          (1, 8, 2, 20, 700, 64), (1, 16, 4, 130, 2000, 128), (1, 8, 2, 5, 2100, 128)]


def factors_of(cap, D, dtype):
    """Powers of two that bring a row's largest score (about 60 / sqrt(D) deviations of 4 a product: 100 for factor 1) to a sixteenth of the cap, near
    the polynomial's end, past the cap and far past it."""
    top = math.floor(math.log2(cap / 20.0))
    most = 14 if dtype == FP else 60
    return [2.0 ** min(max(top + e, -4), most) for e in (-4, -2, -1, 0, 1, 3)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("cap", [130.0, 500.0, 2000.0, 1e4, 1e5, 1e6, 8e6])
def test_wide_caps_on_both_sides_of_their_bend(shape, cap):
    dtype = FP if cap in (500.0, 1e4) else BF
    q, k, v = whole_numbers(*shape, dtype, factors_of(cap, shape[-1], dtype), seed=int(math.log2(cap)))
    for causal in (True, False):
        o, lse = gqa_flash_attn(q, k, v, causal, return_lse=True, softcap=cap)
        check(o, lse, q, k, v, cap, causal)


@pytest.mark.parametrize("cap", [3000.0, 1e6, 8e6])
@pytest.mark.parametrize("D", [64, 128])
def test_ordinary_rows_beside_rows_of_large_scores(cap, D):
    """Rows whose scores are a few units, among rows whose scores are past the cap: each as accurate as alone."""
    q, k, v = whole_numbers(1, 8, 2, 150, 400, D, BF, [2.0 ** -4] * 7 + [2.0 ** math.ceil(math.log2(cap / 10.0))], seed=3, turned=0)
    o, lse = gqa_flash_attn(q, k, v, return_lse=True, softcap=cap)
    check(o, lse, q, k, v, cap)
    rows = torch.tensor([i for i in range(150) if i % 8 != 7], device="cuda")
    o64, l64, tol, ltol = capped64(q[0], k[0], v[0], cap, True)
    assert float(ltol[:, rows].max()) < 1e-4  # (their own scores' bound, not the large rows')
    assert ((o[0].double() - o64).abs() <= tol)[:, rows].all() and ((lse[0].double() - l64).abs() <= ltol)[:, rows].all()


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("cap", [0.5, 5.0, 50.0, 128.0])
def test_usual_caps_far_past_their_bend(shape, cap):
    """Scores up to a thousand caps: tanh is 1 to the last bit."""
    dtype = FP if cap == 50.0 else BF
    q, k, v = whole_numbers(*shape, dtype, [cap / 128.0 * 2.0 ** e for e in (-1, 2, 4, 10)] if cap == 128.0 else [2.0 ** e for e in (-3, 0, 4, 9)],
                            seed=5)
    o, lse = gqa_flash_attn(q, k, v, return_lse=True, softcap=cap)
    check(o, lse, q, k, v, cap)


@pytest.mark.parametrize("route", ["split", "single", "chunks", "short", None])
@pytest.mark.parametrize("cap", [5.0, 2000.0, 1e6])
def test_caps_over_pages(route, cap):
    lens, bs, D = [400, 37], 16, 128
    q, k, v = whole_numbers(2, 8, 2, 20, 400, D, BF, factors_of(max(cap, 200.0), D, BF), seed=7)
    pages = torch.randperm(60, generator=torch.Generator().manual_seed(1))[:50].view(2, 25).int()
    kv = torch.zeros(2, 60, bs, 2, D, dtype=BF, device="cuda")
    for cache, x in zip(kv, (k, v)):
        for b in range(2):
            cache[pages[b].long().cuda()] = x[b].transpose(0, 1).reshape(25, bs, 2, D)
    o, lse = paged_attention(q, kv[0], kv[1], pages.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), True, return_lse=True, softcap=cap,
                             route=route)
    for b, n in enumerate(lens):
        check(o[b:b + 1], lse[b:b + 1], q[b:b + 1], k[b:b + 1, :, :n], v[b:b + 1, :, :n], cap)
