"""Attention with changed scores (softcap, distance bias, prefix and document masks) against float64, over contiguous and paged K/V."""
import math
import threading

import pytest
import torch

from gqa_kernels import document_spans, gqa_flash_attn
from gqa_kernels.paged import GQAPagedAttention, PagedAttentionMetadata, paged_attention, scored_split
from ops_reference import attend64, check_attention

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def make(B, Hq, Hkv, Sq, Skv, D, dtype=BF, seed=0, qscale=3.0):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(B, Hq, Sq, D, generator=g) * qscale
    k, v = torch.randn(B, Hkv, Skv, D, generator=g), torch.randn(B, Hkv, Skv, D, generator=g)
    return tuple(t.to(dtype).cuda() for t in (q, k, v))


def slopes_of(Hq):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / Hq) for h in range(Hq)], dtype=torch.float32).cuda()


def check(q, k, v, causal=True, softcap=None, slopes=None, prefix=None, ids=None):
    docs = None if ids is None else document_spans(ids)
    p = None if prefix is None else torch.tensor(prefix, dtype=torch.int32).cuda()
    o, lse = gqa_flash_attn(q, k, v, causal, return_lse=True, softcap=softcap, alibi_slopes=slopes, prefix_lens=p, documents=docs)
    torch.cuda.synchronize()
    assert o.shape == q.shape and o.dtype == q.dtype
    for b in range(q.shape[0]):
        check_attention(o[b], lse[b], attend64(q[b], k[b], v[b], causal=causal, softcap=softcap or 0.0, slopes=slopes,
                                               prefix=None if prefix is None else prefix[b], ids=None if ids is None else ids[b]))
    return o, lse


SHAPES = [  # B, Hq, Hkv, Sq, Skv, D: the routes' shapes (short, single, chunks, split, flat) and odd sizes
    (1, 4, 1, 1, 1, 128), (1, 8, 2, 65, 65, 64), (2, 8, 2, 300, 300, 128), (1, 32, 8, 1, 700, 128), (1, 32, 8, 1, 4097, 128),
    (1, 32, 8, 5, 2047, 64), (1, 32, 8, 13, 2047, 128), (5, 8, 8, 1, 8192, 128), (1, 8, 2, 130, 5000, 128), (3, 8, 2, 257, 1025, 64),
    (1, 28, 4, 77, 333, 128), (1, 8, 2, 1500, 1500, 128), (1, 32, 8, 2100, 2100, 64), (2, 64, 8, 33, 1200, 128), (4, 6, 6, 40, 39, 64),
    (2, 16, 4, 1600, 1600, 128),
]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
def test_softcap(shape, dtype):
    q, k, v = make(*shape, dtype=dtype)
    check(q, k, v, softcap=20.0)


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_alibi(shape):
    q, k, v = make(*shape, seed=1)
    check(q, k, v, slopes=slopes_of(shape[1]))


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_alibi_softcap_without_causal(shape):
    q, k, v = make(*shape, dtype=FP, seed=2)
    check(q, k, v, causal=False, softcap=30.0, slopes=slopes_of(shape[1]))


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_prefix(shape):
    q, k, v = make(*shape, seed=3)
    B, Skv = shape[0], shape[4]
    check(q, k, v, prefix=[(Skv * (b + 1) // (B + 1) + 3 * b) for b in range(B)], slopes=slopes_of(shape[1]) if B == 1 else None)


def test_prefix_outside_the_keys():
    q, k, v = make(4, 8, 2, 90, 200, 128, seed=4)
    check(q, k, v, prefix=[-5, 0, 200, 100000])
    q, k, v = make(3, 8, 2, 2, 3000, 128, seed=4)
    check(q, k, v, prefix=[-2 ** 31, 2999, 2 ** 31 - 1], softcap=10.0)


def ids_of(lengths, S, B=1, pad=-1):
    rows = []
    for b in range(B):
        row = []
        for i, n in enumerate(lengths[b:] + lengths[:b]):
            row += [i] * n
        rows.append((row + [pad] * S)[:S])
    return torch.tensor(rows, dtype=torch.int32).cuda()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("S,D,lengths,Hq,Hkv", [
    (64, 128, [64], 4, 1), (200, 128, [1, 1, 62, 64, 1, 70], 8, 2), (1000, 64, [500, 3, 200], 8, 2), (1000, 128, [130, 65, 64, 63, 300, 20], 8, 8),
    (2300, 128, [700, 1, 900, 64, 128], 16, 4), (333, 64, [10] * 30, 28, 4), (257, 128, [], 8, 2), (1, 128, [1], 8, 2), (4100, 128, [4100], 8, 2),
])
def test_documents(S, D, lengths, Hq, Hkv, causal):
    q, k, v = make(2, Hq, Hkv, S, S, D, seed=5)
    check(q, k, v, causal=causal, ids=ids_of(lengths, S, 2), softcap=25.0 if S == 1000 else None)


@pytest.mark.parametrize("Sq", [1, 3, 100, 700])
def test_documents_of_a_chunk(Sq):
    q, k, v = make(1, 16, 4, Sq, 1500, 128, seed=6)
    check(q, k, v, ids=ids_of([600, 200, 650], 1500), prefix=[900], slopes=slopes_of(16))


def test_documents_whose_ids_come_back_and_a_padded_start():
    ids = torch.tensor([[-1] * 70 + [3] * 100 + [5] * 30 + [3] * 90 + [-7] * 20 + [0] * 90], dtype=torch.int32).cuda()
    q, k, v = make(1, 8, 2, 400, 400, 128, seed=7)
    spans = document_spans(ids)
    change = [0, 70, 170, 200, 290, 310, 400]
    for a, e in zip(change, change[1:]):
        neg = ids[0, a] < 0
        assert (spans.starts[0, a:e] == (0 if neg else a)).all() and (spans.ends[0, a:e] == (0 if neg else e)).all()
    runs = ids.clone()
    runs[0, 200:290] = 9  # another document in the float64 form, which goes by the id
    o, lse = gqa_flash_attn(q, k, v, return_lse=True, documents=spans)
    check_attention(o[0], lse[0], attend64(q[0], k[0], v[0], ids=runs[0]))
    assert (o[0, :, :70] == 0).all()


@pytest.mark.parametrize("S", [1, 63, 1023, 1024, 1025, 5000, 100003])
def test_document_spans(S):
    g = torch.Generator().manual_seed(S)
    ids = (torch.rand(3, S, generator=g) < 0.01).cumsum(1).to(torch.int32)
    ids[1] = 0
    ids[2, S // 2:] = -1
    change = torch.ones(3, S, dtype=torch.bool)
    change[:, 1:] = ids[:, 1:] != ids[:, :-1]
    at = torch.arange(S).expand(3, S)
    start = torch.where(change, at, torch.zeros_like(at)).cummax(1).values
    nxt = torch.full((3, S), S)
    nxt[:, :-1] = torch.where(change[:, 1:], at[:, 1:], torch.full((3, S - 1), S))
    end = nxt.flip(1).cummin(1).values.flip(1)
    start, end = (torch.where(ids < 0, torch.zeros_like(x), x).int() for x in (start, end))
    spans = document_spans(ids.cuda())
    assert torch.equal(spans.starts.cpu(), start) and torch.equal(spans.ends.cpu(), end)
    wide = torch.zeros(3, S + 5, dtype=torch.int32).cuda()
    wide[:, 2:2 + S] = ids.cuda()
    spans = document_spans(wide[:, 2:2 + S])  # rows apart
    assert torch.equal(spans.starts.cpu(), start) and torch.equal(spans.ends.cpu(), end)


@pytest.mark.parametrize("cap", [0.002, 0.5, 3.0, 100.0, 5e3, 1e6])
@pytest.mark.parametrize("D", [64, 128])
def test_caps_from_tiny_to_none(cap, D):
    q, k, v = make(1, 8, 2, 150, 150, D, seed=8)
    check(q, k, v, softcap=cap)
    q, k, v = make(2, 8, 2, 1, 1500, D, seed=8)
    check(q, k, v, softcap=cap)


def test_large_scores_under_a_cap():
    """Scores far past the cap: tanh is 1 to the last bit."""
    q, k, v = make(1, 8, 2, 200, 200, 128, seed=9, qscale=300.0)
    o, lse = gqa_flash_attn(q, k, v, return_lse=True, softcap=5.0)
    want = attend64(q[0], k[0], v[0], softcap=5.0)
    # (The bound's product term counts scores that the cap has flattened: tanh' <= 1 keeps it an upper bound.)
    check_attention(o[0], lse[0], want)


def test_keys_of_infinity_and_nan_where_they_are_hidden():
    q, k, v = make(1, 8, 2, 300, 300, 128, seed=10)
    ids = ids_of([128, 100], 300)  # padding from 228 on
    k2, v2 = k.clone(), v.clone()
    k2[:, :, 228:260], k2[:, :, 260:] = math.inf, math.nan
    v2[:, :, 228:] = math.nan
    o = gqa_flash_attn(q, k2, v2, documents=document_spans(ids), softcap=20.0)
    assert torch.equal(o, gqa_flash_attn(q, k, v, documents=document_spans(ids), softcap=20.0))


def test_rows_that_see_nothing():
    q, k, v = make(2, 8, 2, 100, 60, 128, seed=12)  # 40 queries before the first key
    check(q, k, v, softcap=20.0)
    check(q, k, v, prefix=[0, 17])
    q, k, v = make(2, 8, 2, 4, 0, 128, seed=12)
    o, lse = gqa_flash_attn(q, k, v, return_lse=True, softcap=20.0)
    assert (o == 0).all() and (lse == -math.inf).all()
    q, k, v = make(1, 8, 2, 3, 2, 128, seed=13)
    check(q, k, v, slopes=slopes_of(8))


def test_strides_and_copies():
    q, k, v = make(2, 8, 2, 150, 400, 128, seed=14)
    want = gqa_flash_attn(q, k, v, softcap=20.0, alibi_slopes=slopes_of(8))
    qt, kt, vt = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v))
    assert torch.equal(gqa_flash_attn(qt, kt, vt, softcap=20.0, alibi_slopes=slopes_of(8)), want)
    odd = torch.empty(2, 8, 150, 129, dtype=BF, device="cuda")[..., 1:]
    odd.copy_(q)
    assert torch.equal(gqa_flash_attn(odd, k, v, softcap=20.0, alibi_slopes=slopes_of(8)), want)


def test_another_stream_and_no_change_of_the_plain_call():
    q, k, v = make(1, 8, 2, 500, 500, 128, seed=15)
    plain = gqa_flash_attn(q, k, v)
    want = gqa_flash_attn(q, k, v, softcap=20.0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = gqa_flash_attn(q, k, v, softcap=20.0)
    s.synchronize()
    assert torch.equal(got, want) and torch.equal(gqa_flash_attn(q, k, v, softcap=0.0), plain)
    assert torch.equal(gqa_flash_attn(q, k, v, softcap=None), plain)


@pytest.mark.parametrize("shape", [(1, 8, 2, 500, 500, 128), (3, 32, 8, 1, 5000, 128), (1, 16, 4, 130, 4000, 128), (2, 16, 4, 1500, 1500, 64)], ids=str)
def test_captured_calls(shape):
    q, k, v = make(*shape, seed=16)
    sl, pre = slopes_of(shape[1]), torch.full((shape[0],), 50, dtype=torch.int32).cuda()
    kw = dict(softcap=20.0, alibi_slopes=sl, prefix_lens=pre, return_lse=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gqa_flash_attn(q, k, v, **kw)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = gqa_flash_attn(q, k, v, **kw)
    for i in range(4):
        q.copy_(make(*shape, seed=20 + i)[0])
        pre.fill_(10 * i)
        want = gqa_flash_attn(q, k, v, **kw)
        o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1])


# ---------------------------------------------------------------------------
# Paged
# ---------------------------------------------------------------------------
def make_paged(lens, Hq, Hkv, Sq, D, block, dtype=BF, seed=0, layout="NHD"):
    g = torch.Generator().manual_seed(seed)
    pages = [-(-n // block) for n in lens]
    width = max(1, max(pages))
    order = torch.randperm(sum(pages) + 3, generator=g)
    table, at = torch.zeros(len(lens), width, dtype=torch.int32), 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    shape = (2, sum(pages) + 3, block, Hkv, D) if layout == "NHD" else (2, sum(pages) + 3, Hkv, block, D)
    kv = torch.randn(*shape, generator=g).to(dtype).cuda()
    if layout != "NHD":
        kv = kv.transpose(2, 3)
    q = (torch.randn(len(lens), Hq, Sq, D, generator=g) * 3).to(dtype).cuda()
    return q, kv[0], kv[1], table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()


def rows_of(cache, table, n):
    bs = cache.shape[1]
    j = torch.arange(n, device=cache.device)
    return cache[table[j // bs].long(), j % bs].transpose(0, 1)


PAGED = [  # lens, Hq, Hkv, Sq, D, block
    ([1], 8, 2, 1, 128, 16), ([700], 32, 8, 1, 128, 64), ([1, 100, 8000, 3001, 0, 64], 32, 8, 1, 128, 16), ([5000, 90, 1200], 32, 8, 1, 64, 16),
    ([3000, 2999], 32, 8, 4, 128, 32), ([1500, 70], 32, 8, 13, 64, 64), ([900, 2000], 8, 2, 300, 128, 16), ([4100], 8, 2, 150, 128, 16),
    ([500, 700, 600], 8, 2, 290, 64, 128), ([260, 300], 8, 8, 2, 128, 2), ([60, 100], 8, 2, 9, 64, 4), ([130, 40, 129], 8, 2, 33, 128, 4),
    ([6000, 6100, 6200, 6300], 16, 4, 600, 128, 64), ([2000] * 20, 16, 2, 1, 128, 16),
]


@pytest.mark.parametrize("case", PAGED, ids=str)
@pytest.mark.parametrize("kind", ["cap", "alibi", "prefix", "all"])
def test_paged(case, kind):
    lens, Hq, Hkv, Sq, D, block = case
    dtype = FP if kind == "alibi" else BF
    q, kc, vc, table, sl = make_paged(*case, dtype=dtype, seed=len(lens), layout="HND" if block == 64 else "NHD")
    cap = 20.0 if kind in ("cap", "all") else None
    slopes = slopes_of(Hq) if kind in ("alibi", "all") else None
    prefix = [n // 2 + 5 for n in lens] if kind in ("prefix", "all") else None
    o, lse = paged_attention(q, kc, vc, table, sl, True, return_lse=True, softcap=cap, alibi_slopes=slopes,
                             prefix_lens=None if prefix is None else torch.tensor(prefix, dtype=torch.int32).cuda())
    torch.cuda.synchronize()
    for b, n in enumerate(lens):
        check_attention(o[b], lse[b], attend64(q[b], rows_of(kc, table[b], n), rows_of(vc, table[b], n), softcap=cap or 0.0, slopes=slopes,
                                               prefix=None if prefix is None else prefix[b]))


@pytest.mark.parametrize("Hkv,D", [(8, 64), (4, 128)])
def test_paged_long_flat_splits(Hkv, D):
    """Unequal lengths, two slots of the flat split a compute unit."""
    lens = [3600 if b == 3 else 1 + 171 * b for b in range(20)]
    slots = scored_split(20, 2 * Hkv, Hkv, 1, 3600 if Hkv == 8 else 7000, 256, 16, D, True)[0]
    assert slots == 512 // Hkv
    q, kc, vc, table, sl = make_paged(lens if Hkv == 8 else [2 * n - 200 * (n == 3600) for n in lens], 2 * Hkv, Hkv, 1, D, 16, seed=5)
    slopes = slopes_of(2 * Hkv)
    o, lse = paged_attention(q, kc, vc, table, sl, True, return_lse=True, softcap=15.0, alibi_slopes=slopes)
    for b, n in enumerate(sl.tolist()):
        check_attention(o[b], lse[b], attend64(q[b], rows_of(kc, table[b], n), rows_of(vc, table[b], n), softcap=15.0,
                                               slopes=slopes))


@pytest.mark.parametrize("Sq", [1, 4])
def test_rows_far_apart(Sq):
    """K and V rows that 32-bit offsets cannot span, before and after calls of the same shape with rows close by."""
    q, k, v = make(1, 8, 2, Sq, 300, 64, seed=6)
    step = (1 << 30) // 492 // 8 * 8 + 8
    base = torch.empty(2, 299 * step + 128, dtype=BF, device="cuda")
    kf, vf = (t.as_strided((1, 2, 300, 64), (300 * step, 64, step, 1)) for t in base)
    kf.copy_(k)
    vf.copy_(v)
    first = check(q, kf, vf, softcap=20.0)
    near = check(q, k, v, softcap=20.0)
    again = check(q, kf, vf, softcap=20.0)
    assert torch.equal(first[0], again[0])
    assert torch.equal(near[0], check(q, k, v, softcap=20.0)[0])
    with pytest.raises(Exception, match="stride|aligned"):
        gqa_flash_attn(q, kf, vf, documents=document_spans(torch.zeros(1, 300, dtype=torch.int32).cuda()))


@pytest.mark.parametrize("route", ["split", "single", "chunks", "short"])
@pytest.mark.parametrize("causal", [True, False])
def test_paged_forced_routes(route, causal):
    lens = [1000, 1100, 37]
    q, kc, vc, table, sl = make_paged(lens, 8, 2, 20, 128, 16, seed=3)
    slopes = slopes_of(8)
    prefix = [900, 30, 37] if causal else None
    for splits in ((None, 3) if route in ("split", "chunks") else (None,)):
        o, lse = paged_attention(q, kc, vc, table, sl, causal, return_lse=True, softcap=15.0, alibi_slopes=slopes, route=route, splits=splits,
                                 prefix_lens=torch.tensor(prefix, dtype=torch.int32).cuda() if causal else None)
        for b, n in enumerate(lens):
            check_attention(o[b], lse[b], attend64(q[b], rows_of(kc, table[b], n), rows_of(vc, table[b], n), causal=causal, softcap=15.0,
                                                   slopes=slopes, prefix=prefix[b] if causal else None))


@pytest.mark.parametrize("max_q", [1, 6, 200])
def test_paged_variable_query_lengths(max_q):
    lens, qlens = [900, 300, 0, 2000], [max_q, 0, 1, max(1, max_q // 2)]
    _, kc, vc, table, sl = make_paged(lens, 8, 2, 1, 128, 16, seed=4)
    total = sum(qlens)
    g = torch.Generator().manual_seed(1)
    q = (torch.randn(total + 3, 8, 128, generator=g) * 3).to(BF).cuda()
    start = [0, qlens[0], qlens[0], qlens[0] + 1]
    out = torch.full_like(q, 7.0)
    slopes = slopes_of(8)
    ints = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    o, lse = paged_attention(q, kc, vc, table, sl, True, query_start=ints(start), query_lens=ints(qlens), max_query_len=max_q, out=out,
                             return_lse=True, softcap=20.0, alibi_slopes=slopes)
    for b, n in enumerate(lens):
        a, e = start[b], start[b] + qlens[b]
        want = attend64(q[a:e].transpose(0, 1), rows_of(kc, table[b], n), rows_of(vc, table[b], n), softcap=20.0, slopes=slopes)
        check_attention(o[a:e].transpose(0, 1), lse[a:e].T, want)
    assert (o[total:] == 7.0).all()  # rows behind the last sequence


def test_paged_scale_and_refusals():
    lens = [300, 40]
    q, kc, vc, table, sl = make_paged(lens, 8, 2, 1, 128, 16, seed=5)
    o = paged_attention(q, kc, vc, table, sl, True, scale=0.31, softcap=9.0)
    for b, n in enumerate(lens):
        check_attention(o[b], None, attend64(q[b], rows_of(kc, table[b], n), rows_of(vc, table[b], n), scale=0.31, softcap=9.0))
    for bad in (-1.0, 1e-9, 1e30, math.nan):
        with pytest.raises(ValueError):
            paged_attention(q, kc, vc, table, sl, True, softcap=bad)
    with pytest.raises(ValueError):
        paged_attention(q, kc, vc, table, sl, True, softcap=9.0, scale=-0.1)
    with pytest.raises(AssertionError):
        paged_attention(q, kc, vc, table, sl, False, prefix_lens=sl)
    with pytest.raises(AssertionError):
        paged_attention(q, kc, vc, table, sl, True, alibi_slopes=slopes_of(4))
    with pytest.raises(AssertionError):
        paged_attention(q, kc, vc, table, sl, True, alibi_slopes=slopes_of(8).double())
    with pytest.raises(NotImplementedError):
        paged_attention(q.clone().requires_grad_(), kc, vc, table, sl, True, softcap=9.0)


def test_layer_with_changed_scores():
    """GQAPagedAttention hands its scores on: uniform and mixed batches."""
    lens, Hq, Hkv, D = [700, 90, 1300, 64], 8, 2, 128
    _, kc, vc, table, sl = make_paged(lens, Hq, Hkv, 1, D, 16, seed=6)
    slopes = slopes_of(Hq)
    layer = GQAPagedAttention(Hq, D, num_kv_heads=Hkv, softcap=20.0, alibi_slopes=slopes)
    kv = torch.stack([kc, vc])
    pre = torch.tensor([100, 0, 1300, 3], dtype=torch.int32).cuda()
    for qlens in ([1, 1, 1, 1], [130, 1, 200, 40]):
        q = (torch.randn(sum(qlens), Hq * D, generator=torch.Generator().manual_seed(2)) * 3).to(BF).cuda()
        md = PagedAttentionMetadata(torch.empty(0, dtype=torch.int64, device="cuda"), table, sl, query_lens=qlens, prefix_lens=pre)
        o = layer(q, None, None, kv, md)
        t = 0
        for b, n in enumerate(lens):
            qb = q[t:t + qlens[b]].view(-1, Hq, D).transpose(0, 1)
            want = attend64(qb, rows_of(kc, table[b], n), rows_of(vc, table[b], n), softcap=20.0, slopes=slopes, prefix=int(pre[b]))
            check_attention(o[t:t + qlens[b]].view(-1, Hq, D).transpose(0, 1), None, want)
            t += qlens[b]


@pytest.mark.parametrize("chunks", [2, 8, 9, 32, 40])
@pytest.mark.parametrize("D", [64, 128])
def test_key_chunks_and_their_combine(chunks, D):
    """Chunk counts on both sides of the combine's forms, chunks that no row sees, a sequence shorter than a chunk and one without keys."""
    lens = [2600, 130, 0, 1999]
    q, kc, vc, table, sl = make_paged(lens, 6, 2, 43, D, 16, seed=chunks)
    slopes = slopes_of(6)
    o, lse = paged_attention(q, kc, vc, table, sl, True, return_lse=True, softcap=15.0, alibi_slopes=slopes, route="chunks",
                             splits=chunks)
    for b, n in enumerate(lens):
        check_attention(o[b], lse[b], attend64(q[b], rows_of(kc, table[b], n), rows_of(vc, table[b], n), softcap=15.0,
                                               slopes=slopes))
    start, qlens = [0, 43, 44, 44], [43, 1, 0, 20]
    ints = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    tokens = torch.cat([q[b, :, :n].transpose(0, 1) for b, n in enumerate(qlens)] + [q[0, :, :2].transpose(0, 1)]).contiguous()
    out = torch.full_like(tokens, 7.0)
    o, lse = paged_attention(tokens, kc, vc, table, sl, True, query_start=ints(start), query_lens=ints(qlens), max_query_len=43,
                             out=out, return_lse=True, softcap=15.0, alibi_slopes=slopes, route="chunks", splits=chunks)
    for b, n in enumerate(lens):
        a, e = start[b], start[b] + qlens[b]
        check_attention(o[a:e].transpose(0, 1), lse[a:e].T, attend64(tokens[a:e].transpose(0, 1), rows_of(kc, table[b], n),
                                                                     rows_of(vc, table[b], n), softcap=15.0, slopes=slopes))
    assert (o[64:] == 7.0).all()


@pytest.mark.parametrize("B,Hkv", [(2, 8), (4, 8), (8, 4), (6, 4), (6, 8), (3, 8), (5, 8)])
def test_batches_over_pages_of_every_dealing(B, Hkv):
    """Pairs of (sequence, kv head) per compute die: 2, 4, 4, 3, 6, 3 and 5, each item once, in one pass and in chunks."""
    lens = [40 + (977 * b) % 1100 for b in range(B)]
    q, kc, vc, table, sl = make_paged(lens, 2 * Hkv, Hkv, 150, 64, 16, seed=B)
    for route, splits in (("single", None), ("chunks", 3), (None, None)):
        o, lse = paged_attention(q, kc, vc, table, sl, True, return_lse=True, softcap=15.0, route=route, splits=splits)
        for b, n in enumerate(lens):
            check_attention(o[b], lse[b], attend64(q[b], rows_of(kc, table[b], n), rows_of(vc, table[b], n), softcap=15.0))


def test_two_threads_at_once():
    """Calls of two threads, on one stream and on streams of their own: each as it is alone."""
    shapes = [(1, 16, 4, 1, 3000, 128), (1, 16, 4, 130, 4000, 128)]
    sl = slopes_of(16)
    data = [make(*s, seed=30 + i) for i, s in enumerate(shapes)]
    paged = make_paged([900, 2500], 16, 4, 1, 64, 16, seed=31)
    calls = [lambda d=d: gqa_flash_attn(*d, softcap=20.0, alibi_slopes=sl, return_lse=True) for d in data]
    calls.append(lambda: paged_attention(*paged, True, softcap=20.0, return_lse=True))
    want = [c() for c in calls]
    torch.cuda.synchronize()
    for own in (False, True):
        bad, streams = [], [torch.cuda.Stream() for _ in range(2)]

        def work(i):
            with torch.cuda.stream(streams[i] if own else torch.cuda.default_stream()):
                for n in range(60):
                    k = (n + i) % len(calls)
                    o, lse = calls[k]()
                    if not (torch.equal(o, want[k][0]) and torch.equal(lse, want[k][1])):
                        bad.append((own, i, n, k))

        threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert not bad
