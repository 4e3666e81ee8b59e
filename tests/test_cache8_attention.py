"""Attention over a paged cache in 8 bits against float64 over the values that its codes stand for (in the queries' type, as the products take them)."""
import threading

import pytest
import torch

from cache8_reference import CODES, gather, new_cache, power
from gqa_kernels import _lib, cache8
from gqa_kernels.paged import paged_attention
from ops_reference import attend64, check_attention

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def rand(*shape, dtype=BF, seed=0, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def ints(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


class Batch:
    """Queries (B, Hq, Sq, D), a cache and tables of sequences of `lens` keys, pages in random order, table entries behind them that must not be read."""

    def __init__(self, lens, Hq, Hkv, Sq, D, bs, dtype=BF, seed=0, layout="NHD", spread=2, width=None, scale=1.0):
        pages = [-(-n // bs) for n in lens]
        blocks = sum(pages) + 2
        order = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).tolist()
        self.width = max(1, max(pages)) if width is None else width
        rows, at = [], 0
        for n in pages:
            rows.append(order[at:at + n] + [-12345] * (self.width - n))
            at += n
        self.table, self.lens, self.n = ints(rows), ints(lens), lens
        self.q = rand(len(lens), Hq, Sq, D, dtype=dtype, seed=seed + 1, scale=scale)
        self.kc, self.vc, self.ke, self.ve = new_cache(blocks, bs, Hkv, D, seed=seed, layout=layout, spread=spread)
        self.e = dict(k_exponents=self.ke, v_exponents=self.ve)

    def run(self, q=None, **kw):
        return paged_attention(self.q if q is None else q, self.kc, self.vc, self.table, self.lens, kw.pop("causal", True), **self.e, **kw)

    def want(self, b, q=None, prefix=None, **kw):
        q = self.q[b] if q is None else q
        k, v = (gather(c, e, self.table[b], self.n[b], q.dtype) for c, e in ((self.kc, self.ke), (self.vc, self.ve)))
        return attend64(q, k, v, prefix=None if prefix is None else max(0, min(int(prefix[b]), self.n[b])), **kw)

    def check(self, routes=(None,), **kw):
        prefix = kw.get("prefix")
        call = {("softcap" if k == "softcap" else "alibi_slopes" if k == "slopes" else "prefix_lens" if k == "prefix" else k): v for k, v in kw.items()}
        for route in routes:
            o, lse = self.run(return_lse=True, route=route[0] if route else None, splits=route[1] if route else None, **call)
            for b in range(len(self.n)):
                check_attention(o[b], lse[b], self.want(b, **{**kw, "prefix": prefix}))
        return o, lse


FEW = [("split", n) for n in (1, 3, 16)] + [("chunks", 1), ("chunks", 3), ("single", None), None]
WIDE = 4096  # keys
MANY = [("chunks", 1), ("chunks", 2), ("chunks", 5), ("single", None), None]


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bs", [16, 32, 64, 256])
@pytest.mark.parametrize("Hq,Hkv,Sq", [(32, 8, 1), (8, 8, 1), (7, 1, 2), (16, 1, 1), (6, 2, 5), (4, 4, 16), (32, 8, 8), (23, 1, 1), (6, 2, 7), (2, 2, 32)])
def test_few_rows(Hq, Hkv, Sq, bs, D, dtype):
    """Up to 16 and up to 32 packed rows; lengths from none over one, a tile's ends and a unit's to many; every route."""
    lens = [0, 1, Sq, 15, 16, 17, 31, 33, 127, 128, 129, 255, 300, 1000]
    Batch(lens, Hq, Hkv, Sq, D, bs, dtype, seed=Sq).check(FEW)


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hkv,Sq,lens", [
    (32, 8, 8, [8, 100, 513, 64]), (28, 4, 3, [3, 0, 700, 65]), (8, 8, 17, [17, 500, 129]), (4, 1, 130, [130, 131, 1000]), (128, 1, 1, [1, 63, 900]),
    (5, 1, 77, [77, 300]), (12, 4, 200, [200, 264, 1111]), (8, 2, 333, [333, 64]),
])
@pytest.mark.parametrize("wide", [False, True], ids=["", "wide"])
def test_many_rows(Hq, Hkv, Sq, lens, D, dtype, wide):
    """Up to several blocks of 128 packed rows, or (under a large bound on the lengths) of 256; a sequence shorter than its queries leaves rows
    empty: zeros and LSE -inf."""
    bs = 16 if Sq % 2 else 64
    Batch(lens, Hq, Hkv, Sq, D, bs, dtype, seed=Sq, layout="HND" if Sq % 3 else "NHD", width=(WIDE // bs if wide else None)).check(MANY)


@pytest.mark.parametrize("Hq,Hkv,Sq", [(8, 2, 1), (8, 2, 4), (8, 2, 6), (8, 2, 40), (8, 2, 100)])
@pytest.mark.parametrize("D", [64, 128])
def test_without_a_mask(Hq, Hkv, Sq, D):
    Batch([1, 50, 3 * 64, 700], Hq, Hkv, Sq, D, 16, width=WIDE // 16 if Sq > 64 else None).check((None, ("single", None), ("chunks", 3)), causal=False)


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
@pytest.mark.parametrize("Hq,Hkv,Sq", [(16, 4, 1), (16, 4, 4), (16, 4, 7), (16, 4, 50), (16, 4, 90)])
@pytest.mark.parametrize("D", [64, 128])
def test_changed_scores(Hq, Hkv, Sq, D, dtype):
    lens = [1, 70, 129, 640, 0, 333]
    b = Batch(lens, Hq, Hkv, Sq, D, 32, dtype, seed=3, scale=2.0, width=WIDE // 32 if Sq > 64 else None)
    slopes = torch.tensor([2.0 ** (-8 * (h + 1) / Hq) for h in range(Hq)]).cuda()
    prefix = ints([0, 50, 200, 640, 5, -3])
    routes = (None, ("single", None), ("chunks", 4)) + ((("split", 5),) if Hq // Hkv * Sq <= 32 else ())
    for kw in (dict(softcap=20.0), dict(softcap=500.0), dict(slopes=slopes), dict(prefix=prefix), dict(softcap=30.0, slopes=slopes, prefix=prefix)):
        b.check(routes, **kw)


def test_exponents_near_the_types_ends():
    """Scales whose products with codes leave fp16's normal numbers, and bf16 far ones: the value in the queries' type is what counts."""
    for dtype, lo, hi in ((FP, -24, 6), (BF, -60, 40)):
        for Sq in (1, 40):
            b = Batch([200, 77], 8, 2, Sq, 128, 16, dtype, seed=5)
            g = torch.Generator().manual_seed(2)
            b.ve.copy_(torch.randint(lo, hi, b.ve.shape, generator=g, dtype=torch.int32))
            b.ke.copy_(torch.randint(-14, -6, b.ke.shape, generator=g, dtype=torch.int32))
            b.check()
    b = Batch([40], 8, 2, 1, 64, 16)
    b.ke.fill_(-2 ** 31)  # clamped: keys next to nothing, an even mean of the values
    o = b.run()
    v = gather(b.vc, b.ve, b.table[0], 40, BF).double().mean(1).repeat_interleave(4, 0)
    assert ((o[0, :, 0].double() - v).abs() <= 2.0 ** -8 * v.abs() + 2.0 ** -8 * gather(b.vc, b.ve, b.table[0], 40, BF).double().abs().mean(1).repeat_interleave(4, 0)).all()


@pytest.mark.parametrize("Hq,Hkv,lens,ql", [(8, 2, [40, 9, 300, 0, 64], [1, 2, 4, 0, 3]), (8, 2, [140, 9, 300, 512], [100, 1, 0, 37]), (8, 2, [5000, 90, 400], [150, 70, 1]), (4, 1, [30] * 70, [1, 0, 2] * 23 + [4])])
def test_variable_query_lengths(Hq, Hkv, lens, ql):
    """Token-major queries; sequences without any, tokens that belong to none (left as they were)."""
    D, start, at = 64, [], 2
    for n in ql:
        start.append(at)
        at += n
    b = Batch(lens, Hq, Hkv, 1, D, 16, seed=1)
    q = rand(at + 3, Hq, D, seed=4)
    for route in (None, ("single", None), ("chunks", 2)):
        out = torch.full_like(q, 7.0)
        o, lse = b.run(q, query_start=ints(start), query_lens=ints(ql), max_query_len=max(ql), return_lse=True, out=out,
                       route=route[0] if route else None, splits=route[1] if route else None)
        assert o.data_ptr() == out.data_ptr() and lse.shape == (at + 3, Hq)
        for i, (s, n) in enumerate(zip(start, ql)):
            if n:
                want = b.want(i, q[s:s + n].transpose(0, 1))
                check_attention(o[s:s + n].transpose(0, 1), lse[s:s + n].t(), want)
        assert (o[:2] == 7.0).all() and (o[at:] == 7.0).all()


def test_layouts_and_strides():
    """Queries and outputs of other orders, a table that is part of a larger one, a bound on the lengths, pages of a larger tensor."""
    lens, Hq, Hkv, Sq, D = [200, 31, 77], 8, 2, 3, 128
    b = Batch(lens, Hq, Hkv, Sq, D, 16)
    o, _ = b.check()
    q = b.q.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)
    out = torch.zeros(3, Sq, Hq, D, dtype=BF, device="cuda").transpose(1, 2)
    assert torch.equal(b.run(q, out=out), o) and torch.equal(out, o)
    wide = torch.full((3, b.width + 9), -5, dtype=torch.int32, device="cuda")
    wide[:, 4:4 + b.width] = b.table
    odd = torch.empty(3, Hq, Sq, D + 1, dtype=BF, device="cuda")[..., 1:].copy_(b.q)  # rows on no 16 bytes
    for kw in (dict(table=wide[:, 4:4 + b.width]), dict(q=odd), dict(scale=0.0883883476), dict(max_seq_len=200)):
        t = b.table
        b.table, q = kw.pop("table", t), kw.pop("q", None)
        got = b.run(q, **kw)
        b.table = t
        assert torch.equal(got, o) or ((got.float() - o.float()).abs() <= 2.0 ** -7 * o.float().abs() + 2.0 ** -9).all()
    short = b.run(max_seq_len=64)  # keys past the bound are not read: as if the sequences ended there
    n, b.n = b.n, [min(x, 64) for x in lens]
    for i in range(3):
        check_attention(short[i], None, b.want(i))
    b.n = n
    both = torch.stack([b.kc.view(torch.uint8), b.vc.view(torch.uint8)], 2)  # (blocks, bs, 2, Hkv, D)
    e = torch.stack([b.ke, b.ve], -1)
    got = paged_attention(b.q, both[:, :, 0].view(CODES), both[:, :, 1].view(CODES), b.table, b.lens, k_exponents=e[..., 0], v_exponents=e[..., 1])
    assert torch.equal(got, o)


def test_what_lies_past_a_sequence_is_not_read():
    """NaN codes in pages' ends and other pages, and exponents of pages that belong to nobody: no output changes."""
    for Sq, Hq in ((1, 8), (40, 8), (100, 8)):
        b = Batch([35, 100, 17], Hq, 2, Sq, 128, 16, seed=2, width=WIDE // 16 if Sq > 64 else None)
        o = b.run()
        used = torch.zeros(b.kc.shape[0], 16, dtype=torch.bool, device="cuda")
        for i, n in enumerate(b.n):
            at = torch.arange(n, device="cuda")
            used[b.table[i][at // 16].long(), at % 16] = True
        for c in (b.kc, b.vc):
            u = c.view(torch.uint8)
            u[~used] = 127
        free = ~used.any(1)
        b.ke[free], b.ve[free] = 2 ** 31 - 1, 2 ** 31 - 1
        assert torch.equal(b.run(), o)


def test_results_repeat_and_two_calls_at_once():
    """The same bits every time, on two streams at once and from two threads."""
    b = Batch([3000, 17, 900, 2222], 32, 8, 1, 128, 16, seed=8)
    c = Batch([600, 900], 16, 4, 30, 64, 32, FP, seed=9)
    want = [b.run(), c.run()]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]

    def work(i, x):
        with torch.cuda.stream(streams[i]):
            for _ in range(20):
                got[i].append(x.run())

    threads = [threading.Thread(target=work, args=(i, x)) for i, x in enumerate((b, c))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        assert len(got[i]) == 20 and all(torch.equal(x, want[i]) for x in got[i])


@pytest.mark.parametrize("Sq", [1, 6, 60, 100])
def test_captured_and_replayed(Sq):
    """Two graphs over one cache, replayed in turn and at once with eager calls in between; lengths and queries that change under them."""
    b = Batch([900, 33, 512, 129], 8, 2, Sq, 128, 16, seed=4, width=WIDE // 16 if Sq > 64 else None)
    b.run()
    graphs, outs, qs = [], [], []
    for i in range(2):
        qs.append(rand(4, 8, Sq, 128, seed=20 + i))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(b.run(qs[i], return_lse=True))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for step, lens in enumerate(([900, 33, 512, 129], [100, 33, 500, 60], [899, 0, 1, 128], [880, 32, 77, 64])):
        b.lens.copy_(ints(lens))
        b.n = lens
        for i in range(2):
            qs[i].copy_(rand(4, 8, Sq, 128, seed=100 * step + i))
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            eager, lse = b.run(qs[i], return_lse=True)
            assert torch.equal(outs[i][0], eager) and torch.equal(outs[i][1], lse)
            for s in range(4):
                check_attention(outs[i][0][s], outs[i][1][s], b.want(s, qs[i][s]))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq", [1, 7, 30, 100])
def test_one_sequence_in_many_parts(Sq, D):
    """Joined by a workgroup a row; pieces beyond the query block's last key."""
    Batch([4999], 8, 2, Sq, D, 16, seed=Sq).check((None, ("split", 39) if Sq <= 8 else ("chunks", 70), ("chunks", 9)))


def test_pieces_of_very_unequal_sequences():
    """One long sequence among those of a tile or none: it takes what they leave, down to a piece each."""
    for lens, splits in (([1] * 40 + [0, 4000] + [64] * 30, 2), ([0] * 65 + [1300, 3], 1), ([700, 100, 0, 1], 256), ([129] * 9, 3)):
        b = Batch(lens, 8, 2, 40, 64, 16, seed=len(lens))
        o, lse = b.run(return_lse=True, route="chunks", splits=splits)
        for i in range(len(lens)):
            if lens[i] != 1 or i < 3:
                check_attention(o[i], lse[i], b.want(i))


def test_many_sequences():
    """More sequences than a wave has lanes, more than the slots, of unequal lengths."""
    g = torch.Generator().manual_seed(0)
    for B, top, Hq, Hkv in ((150, 60, 4, 4), (700, 9, 8, 8), (65, 500, 4, 1)):
        lens = torch.randint(0, top, (B,), generator=g).tolist()
        b = Batch(lens, Hq, Hkv, 1, 64, 16, seed=B)
        o, lse = b.run(return_lse=True)
        for i in range(0, B, 7):
            check_attention(o[i], lse[i], b.want(i))
        assert torch.isfinite(o.float()).all()


def test_pages_past_2_gib():
    """Byte offsets past 32 bits, few rows and many."""
    bs, Hkv, D = 16, 8, 128
    blocks = (1 << 31) // (bs * Hkv * D) + 100
    kc, vc = (torch.zeros(blocks, bs, Hkv, D, dtype=torch.uint8, device="cuda") for _ in range(2))
    ke, ve = (torch.full((blocks, Hkv), -7, dtype=torch.int32, device="cuda") for _ in range(2))
    table = ints([[blocks - 1, 0, blocks - 3, 5, blocks - 2, 1]])
    g = torch.Generator().manual_seed(1)
    for c in (kc, vc):
        c[table[0].long()] = torch.randint(0, 120, (6, bs, Hkv, D), generator=g, dtype=torch.uint8).cuda()
    kc, vc = kc.view(CODES), vc.view(CODES)
    k, v = (gather(c, e, table[0], 90, BF) for c, e in ((kc, ke), (vc, ve)))
    for Sq in (1, 40):
        q = rand(1, 32, Sq, D, seed=Sq)
        o, lse = paged_attention(q, kc, vc, table, ints([90]), return_lse=True, k_exponents=ke, v_exponents=ve)
        check_attention(o[0], lse[0], attend64(q[0], k, v))
    del kc, vc
    torch.cuda.empty_cache()


def test_refusals():
    b = Batch([40, 9], 8, 2, 1, 64, 16)
    a = dict(q=b.q, k_cache=b.kc, v_cache=b.vc, block_table=b.table, seq_lens=b.lens, k_exponents=b.ke, v_exponents=b.ve)
    for kw in (dict(q=b.q.float()), dict(q=b.q[:, :7]), dict(q=b.q[..., :32]), dict(k_exponents=None), dict(v_exponents=b.ve[:1]), dict(k_cache=b.kc[:, :8], v_cache=b.vc[:, :8]),
               dict(k_cache=b.kc.view(torch.uint8)), dict(k_cache=b.kc[..., :32], v_cache=b.vc[..., :32]), dict(seq_lens=b.lens.long()), dict(seq_lens=b.lens[:1]),
               dict(block_table=b.table.long()), dict(block_table=b.table[0]), dict(max_seq_len=b.width * 16 + 1), dict(max_seq_len=-1), dict(route="short"),
               dict(route="single", splits=2), dict(out=torch.empty_like(b.q[:1])), dict(prefix_lens=ints([1, 2]), causal=False),
               dict(alibi_slopes=torch.ones(7, device="cuda")), dict(query_start=ints([0, 1]), query_lens=ints([1, 1]), max_query_len=1), dict(v_cache=b.vc.cpu()),
               dict(k_exponents=b.ke.long())):
        with pytest.raises(AssertionError):
            paged_attention(**{**a, **kw})
    for kw in (dict(scale=0.0), dict(scale=-0.1), dict(softcap=-1.0), dict(softcap=1e30)):
        with pytest.raises(ValueError):
            paged_attention(**{**a, **kw})
    for kw in (dict(route="split", splits=1025), dict(route="chunks", splits=0)):
        with pytest.raises(_lib.GQAError):
            paged_attention(**{**a, **kw})
    with pytest.raises(_lib.GQAError):  # more rows than the flat split takes
        paged_attention(**{**a, "q": rand(2, 8, 9, 64), "route": "split"})
    with pytest.raises(NotImplementedError):
        paged_attention(**{**a, "q": b.q.clone().requires_grad_()})
    wide = Batch([40], 2 * 129, 2, 1, 64, 16)
    with pytest.raises(AssertionError, match="128"):
        wide.run()
    assert power(b.ke).isfinite().all()


def test_nothing_to_do():
    b = Batch([40, 9], 8, 2, 1, 64, 16)
    assert b.run(b.q[:, :, :0]).shape == (2, 8, 0, 64)
    o, lse = paged_attention(b.q[:0], b.kc, b.vc, b.table[:0], b.lens[:0], return_lse=True, **b.e)
    assert o.shape == (0, 8, 1, 64) and lse.shape == (0, 8, 1)
    o, lse = b.run(max_seq_len=0, return_lse=True)
    assert not o.any() and (lse == -float("inf")).all()
    b.lens.copy_(ints([-5, 0]))
    for kw in ({}, dict(route="chunks", splits=2), dict(route="single")):
        o, lse = b.run(return_lse=True, **kw)
        assert not o.any() and (lse == -float("inf")).all()


@pytest.mark.parametrize("Sq", [1, 33])
def test_both_bindings_agree(Sq, monkeypatch):
    b = Batch([700, 33, 64], 8, 2, Sq, 128, 32, seed=6)
    slopes = torch.rand(8, generator=torch.Generator().manual_seed(0)).cuda()
    calls = ({}, dict(softcap=20.0, alibi_slopes=slopes, prefix_lens=ints([9, 40, 0])), dict(scale=0.2, causal=False))
    b.run()  # (loads the binding)
    native = [b.run(return_lse=True, **kw) for kw in calls]
    monkeypatch.setattr(_lib, "_host", None)
    monkeypatch.setattr(cache8, "_decode_host", lambda: None)
    for (o, lse), kw in zip(native, calls):
        o2, lse2 = b.run(return_lse=True, **kw)
        assert torch.equal(o, o2) and torch.equal(lse, lse2)
