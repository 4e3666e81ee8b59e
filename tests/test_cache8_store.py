"""Writes into, and reads out of, a paged cache in 8 bits against the plain forms: codes and exponents to the last bit where no fp32 arithmetic goes before."""
import pytest
import torch

from cache8_reference import CODES, LEAST, decode, encode, exponents_of, limit_of, new_cache, power, stored, values
from gqa_kernels import RotaryTable, _lib, qk_norm_rope, qk_norm_rope_write
from gqa_kernels.paged import read_kv, write_kv
from ops_reference import rope64

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def rand(*shape, dtype=BF, seed=0, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def slots_of(spans, bs, seed=0, pad=()):
    """Slots of sequences (first offset, tokens), each in pages of its own, pages in random order; negative ones at the places of `pad`."""
    need = [-(-(a + n) // bs) for a, n in spans]
    pages = torch.randperm(sum(need) + 3, generator=torch.Generator().manual_seed(seed)).tolist()
    out, at = [], 0
    for (a, n), p in zip(spans, need):
        out += [pages[at + i // bs] * bs + i % bs for i in range(a, a + n)]
        at += p
    for i in pad:
        out.insert(i, -1)
    return torch.tensor(out, dtype=torch.int64).cuda(), sum(need) + 3


def check_store(k, v, slots, blocks, bs, dtype, layout="NHD", seed=0, full=True):
    kc, vc, ke, ve = new_cache(blocks, bs, k.shape[1], k.shape[2], seed=seed, layout=layout, full=full)
    want = [stored(c, e, x.double(), slots, limit_of(dtype)) for c, e, x in ((kc, ke, k), (vc, ve, v))]
    write_kv(k, v, kc, vc, slots, k_exponents=ke, v_exponents=ve)
    for c, e, (codes, exps) in ((kc, ke, want[0]), (vc, ve, want[1])):
        assert torch.equal(e, exps), f"{int((e != exps).sum())} exponents differ"
        c, codes = (torch.where((x & 127) == 127, x & 127, x) for x in (c.view(torch.uint8), codes))  # (NaN of either sign)
        differ = c != codes
        assert not differ.any(), f"{int(differ.sum())} codes differ"
    return kc, vc, ke, ve


SPANS = [(1, [(0, 1)]), (1, [(5, 1)]), (3, [(0, 1), (15, 1), (7, 1)]), (2, [(0, 16), (3, 40)]), (8, [(9, 1)] * 20), (5, [(0, 333)]), (4, [(15, 2), (1, 15), (0, 17)])]


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
@pytest.mark.parametrize("D,layout", [(128, "NHD"), (64, "HND")])
@pytest.mark.parametrize("bs", [16, 32, 128])
@pytest.mark.parametrize("i", range(len(SPANS)))
def test_codes_and_exponents(i, bs, D, layout, dtype):
    """Tokens at every kind of place in a page: its first, its last, over several pages; larger and smaller than what stands there."""
    Hkv, spans = SPANS[i]
    slots, blocks = slots_of(spans, bs, seed=i)
    T = slots.shape[0]
    size = torch.exp2(torch.randint(-9, 9, (T, Hkv, 1), generator=torch.Generator().manual_seed(i + 50)).float()).cuda()
    k, v = ((rand(T, Hkv, D, seed=s).float() * f).to(dtype) for s, f in ((1, size), (2, 1.0)))
    check_store(k, v, slots, blocks, bs, dtype, layout, seed=i)


@pytest.mark.parametrize("Hkv", [1, 2, 3, 7, 8, 16, 20, 33])
def test_head_counts(Hkv):
    for D in (64, 128):
        slots, blocks = slots_of([(3, 30), (0, 1), (15, 1)], 16, seed=Hkv)
        k, v = rand(32, Hkv, D, seed=1), rand(32, Hkv, D, seed=2, scale=7.0)
        check_store(k, v, slots, blocks, 16, BF, seed=Hkv)


def test_padding_and_untouched_pages():
    slots, blocks = slots_of([(4, 20), (0, 5)], 16, seed=3, pad=(0, 0, 22, 28))
    k, v = rand(29, 2, 64, seed=4), rand(29, 2, 64, seed=5)
    check_store(k, v, slots, blocks, 16, BF)
    kc, vc, ke, ve = new_cache(4, 16, 2, 64, seed=9)
    before = [x.view(torch.int32).clone() if x.dtype == torch.int32 else x.view(torch.uint8).clone() for x in (kc, vc, ke, ve)]
    write_kv(k, v, kc, vc, torch.full((29,), -1, dtype=torch.int64, device="cuda"), k_exponents=ke, v_exponents=ve)
    write_kv(k[:0], v[:0], kc, vc, slots[:0], k_exponents=ke, v_exponents=ve)
    for x, y in zip((kc, vc, ke, ve), before):
        assert torch.equal(x if x.dtype == torch.int32 else x.view(torch.uint8), y)


def test_tokens_of_a_page_in_any_order():
    bs, order = 32, torch.randperm(25, generator=torch.Generator().manual_seed(0))
    slots = torch.cat([(3 * bs + 7 + order[:20]), (bs + order[20:]) % (2 * bs)]).cuda()  # offsets 7 .. and a page begun by one of them
    k, v = rand(25, 4, 128, seed=6), rand(25, 4, 128, seed=7)
    check_store(k, v, slots, 6, bs, BF)


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
def test_zeros_smallest_largest_and_nan(dtype):
    top, least = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    inf, nan = float("inf"), float("nan")
    for row in ([0.0, -0.0], [top, -top], [inf, 1.0], [-inf, nan], [nan, 0.0], [least, -least / 4], [448.0, 449.0], [1.75, -1.7578125], [1.0, least]):
        k = torch.zeros(3, 2, 64, dtype=dtype)
        k[0, 0, :2], k[1, 1, 5:7] = torch.tensor(row, dtype=dtype), torch.tensor(row, dtype=dtype)
        k, slots = k.cuda(), torch.tensor([2, 3, 16], dtype=torch.int64).cuda()
        kc, vc, ke, ve = check_store(k, k, slots, 2, 16, dtype, full=False)
        got = values(kc, ke)[0, 2, 0, :2]
        for x, y in zip(row, got.tolist()):
            if x == x:  # half a step, and a saturated value is still within one
                assert abs(y - max(min(x, top), -top)) <= 2.0 ** -4 * min(abs(x), top) * (1 + 2.0 ** -8) + 2.0 ** -10 * 2.0 ** float(ke[0, 0])
            else:
                assert y != y
        rows, _ = read_kv(kc, vc, slots, ke, ve, dtype=dtype)
        assert torch.equal(torch.isnan(rows), torch.isnan(k)) and not torch.isinf(rows).any()


def test_a_page_filled_token_by_token():
    """Growing and shrinking tokens, one a call: every call against the plain form, and all of them within a step of what was stored."""
    bs, Hkv, D = 16, 2, 128
    kc, vc, ke, ve = new_cache(2, bs, Hkv, D, seed=3)
    said = []
    for t, size in enumerate([1.0, 0.1, 30.0, 0.5, 1000.0, 3.0, 3.0, 1e-3, 5e4, 1.0, 1e5, 0.0, 2.0, 1e6, 1.0, 1.0]):
        k = rand(1, Hkv, D, seed=t, scale=size)
        slots = torch.tensor([bs + t], dtype=torch.int64).cuda()
        want = stored(kc, ke, k.double(), slots, limit_of(BF))
        write_kv(k, k, kc, vc, slots, k_exponents=ke, v_exponents=ve)
        assert torch.equal(kc.view(torch.uint8), want[0]) and torch.equal(ke, want[1])
        assert torch.equal(vc.view(torch.uint8)[1, :t + 1], want[0][1, :t + 1]) and torch.equal(ve[1], ke[1])
        said.append(k[0].double())
        unit = power(ke[1])[:, None]
        # Half a step of the value, and of the unit once for every exponent that the page has had (at most one a token).
        off = (values(kc, ke)[1, :t + 1] - torch.stack(said)).abs()
        assert (off <= 2.0 ** -4 * torch.stack(said).abs() * (1 + 2.0 ** -4) + (t + 1) * 2.0 ** -10 * unit).all()


def test_strided_rows_and_exponents():
    bs, Hkv, D, T = 16, 4, 64, 50
    slots, blocks = slots_of([(2, T)], bs)
    qkv = rand(T, 3 * Hkv * D)
    k, v = qkv[:, Hkv * D:2 * Hkv * D].unflatten(1, (Hkv, D)), qkv[:, 2 * Hkv * D:].unflatten(1, (Hkv, D))
    odd = rand(T, Hkv, D + 1)[..., 1:]  # rows that begin on no 16 bytes are copied
    for kk, vv in ((k, v), (odd, v), (k[:1].expand(T, Hkv, D), v)):
        check_store(kk, vv, slots, blocks, bs, BF)
    kc, vc, ke, ve = new_cache(blocks, bs, Hkv, D)
    both = torch.stack([ke.t().contiguous(), ve.t().contiguous()], -1)  # (Hkv, blocks, 2)
    views = both[..., 0].t(), both[..., 1].t()
    want = stored(kc, ke, k.double(), slots, limit_of(BF)), stored(vc, ve, v.double(), slots, limit_of(BF))
    write_kv(k, v, kc, vc, slots, k_exponents=views[0], v_exponents=views[1])
    for c, e, (codes, exps) in ((kc, views[0], want[0]), (vc, views[1], want[1])):
        assert torch.equal(c.view(torch.uint8), codes) and torch.equal(e, exps)


def test_exponents_out_of_range_are_clamped():
    kc, vc, ke, ve = new_cache(3, 16, 2, 64)
    ke[0], ke[1] = 2 ** 31 - 1, -2 ** 31
    slots = torch.tensor([5, 21, 32], dtype=torch.int64).cuda()
    k = rand(3, 2, 64)
    want = stored(kc, ke, k.double(), slots, limit_of(BF))
    write_kv(k, k, kc, vc, slots, k_exponents=ke, v_exponents=ve)
    assert torch.equal(kc.view(torch.uint8), want[0]) and torch.equal(ke, want[1]) and int(ke[0].max()) == 126


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
@pytest.mark.parametrize("T,Hq,Hkv,D,bs,R,inter,norm", [
    (1, 32, 8, 128, 16, 128, False, True), (64, 28, 4, 128, 16, 64, True, True), (333, 6, 2, 64, 32, 64, False, False), (40, 8, 8, 64, 16, 32, True, True),
    (5, 5, 1, 128, 64, 128, False, True), (2500, 8, 2, 128, 16, 128, False, True),
])
def test_norm_rope_write(T, Hq, Hkv, D, bs, R, inter, norm, dtype):
    """Queries as qk_norm_rope gives them; keys within half a step of e4m3 (and of the least one) of the rotated float64 ones, which fp32 reaches to 2^-18
    of the row; exponents the least, or beside it where the largest value is that near to the border; values exactly as write_kv stores them."""
    spans = [(b % bs, 1) for b in range(T)] if T <= 64 else [(3, T - 100), (0, 100)]
    slots, blocks = slots_of(spans, bs, seed=T)
    qkv = rand(T, (Hq + 2 * Hkv) * D, dtype=dtype, scale=2.0)
    q, k, v = (x.unflatten(-1, (-1, D)) for x in qkv.split([Hq * D, Hkv * D, Hkv * D], -1))
    wq, wk = ((rand(D, dtype=dtype, seed=s) * 0.3 + 1).to(dtype) if norm else None for s in (2, 3))
    table = RotaryTable(D, 9000, rotary_dim=R, interleaved=inter)
    pos = torch.randint(0, 9000, (T,), generator=torch.Generator().manual_seed(1)).cuda()
    kc, vc, ke, ve = new_cache(blocks, bs, Hkv, D, seed=2, spread=6)
    was = ke.clone()
    wantv = stored(vc, ve, v.double(), slots, limit_of(dtype))
    qo = qk_norm_rope_write(q, k, v, pos, table, kc, vc, slots, q_weight=wq, k_weight=wk, k_exponents=ke, v_exponents=ve)
    inv = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    y, tol = rope64(q, wq, 1e-6, pos[None, :, None], rotary_dim=R, interleaved=inter, inv_freq=inv, axes=[0] * (R // 2))
    assert ((qo.double() - y).abs() <= tol).all()
    assert torch.equal(vc.view(torch.uint8), wantv[0]) and torch.equal(ve, wantv[1])
    y, _ = rope64(k, wk, 1e-6, pos[None, :, None], rotary_dim=R, interleaved=inter, inv_freq=inv, axes=[0] * (R // 2))
    size = y.abs().amax(-1, keepdim=True)
    page, off = slots // bs, slots % bs
    got, unit = values(kc, ke)[page, off], power(ke)[page][..., None]
    assert ((got - y).abs() <= 2.0 ** -4 * y.abs() + 2.0 ** -10 * unit + 2.0 ** -18 * size).all()
    for pg in page.unique().tolist():
        mine = page == pg
        most, near = y[mine].abs().amax((0, 2)), 2.0 ** -18 * size[mine].amax((0, 2))
        old = was[pg] if int(off[mine].min()) > 0 else torch.full_like(was[pg], LEAST)
        assert (ke[pg] >= torch.maximum(exponents_of(most - near), old)).all() and (ke[pg] <= torch.maximum(exponents_of(most + near), old)).all()


def test_axes_in_place_and_norms_alone():
    T, Hq, Hkv, D = 37, 4, 2, 128
    slots, blocks = slots_of([(1, T)], 16)
    q, k, v = rand(T, Hq, D), rand(T, Hkv, D, seed=1), rand(T, Hkv, D, seed=2)
    table = RotaryTable(D, 500, axes=RotaryTable.sections([16, 24, 24]))
    pos = torch.randint(0, 500, (3, T), generator=torch.Generator().manual_seed(1), dtype=torch.int32).cuda()
    w = rand(D, seed=3).float() + 1
    for t, p, kw in ((table, pos, {}), (None, None, dict(q_weight=w, k_weight=w)), (None, None, dict(k_weight=w))):
        qr, kr = qk_norm_rope(q, k, p, t, **kw)
        kc, vc, ke, ve = new_cache(blocks, 16, Hkv, D, full=False)
        mine = q.clone()
        qo = qk_norm_rope_write(mine, k, v, p, t, kc, vc, slots, q_out=mine, k_exponents=ke, v_exponents=ve, **kw)
        assert qo is mine
        # (both round fp32 values that agree to 2^-18 of the row: a step of bf16 apart at most)
        assert ((qo.float() - qr.float()).abs() <= torch.finfo(BF).eps * qr.float().abs() + 2.0 ** -17 * qr.float().abs().amax(-1, keepdim=True)).all()
        # kr has been rounded to bf16 before: half a step of it more.
        got, unit = values(kc, ke)[slots // 16, slots % 16], power(ke)[slots // 16][..., None]
        assert ((got - kr.double()).abs() <= (2.0 ** -4 + 2.0 ** -7) * kr.double().abs() + 2.0 ** -10 * unit + 2.0 ** -17 * kr.double().abs().amax(-1, keepdim=True)).all()


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
@pytest.mark.parametrize("D,layout,bs", [(128, "NHD", 16), (64, "HND", 64), (128, "HND", 16)])
def test_read(D, layout, bs, dtype):
    kc, vc, ke, ve = new_cache(9, bs, 3, D, layout=layout, spread=12)
    slots = torch.randint(-1, 9 * bs, (217,), generator=torch.Generator().manual_seed(1)).cuda()
    slots[5] = -7
    key, value = read_kv(kc, vc, slots, ke, ve, dtype=dtype)
    for got, c, e in ((key, kc, ke), (value, vc, ve)):
        want = values(c, e).flatten(0, 1)[slots.clamp(min=0)]
        want[slots < 0] = 0
        assert got.dtype == dtype and torch.equal(got, want.to(dtype))
    into = torch.zeros(217, 2, 3, D, dtype=dtype, device="cuda")
    a, b = read_kv(kc, vc, slots, ke, ve, dtype=dtype, key=into[:, 0], value=into[:, 1])
    assert a.data_ptr() == into.data_ptr() and torch.equal(into[:, 0], key) and torch.equal(into[:, 1], value)
    for n in (0, 1):
        a, b = read_kv(kc, vc, slots[:n], ke, ve, dtype=dtype)
        assert a.shape == (n, 3, D) and torch.equal(b, value[:n])


def test_refusals():
    kc, vc, ke, ve = new_cache(4, 16, 2, 64)
    slots = torch.zeros(3, dtype=torch.int64, device="cuda")
    k = rand(3, 2, 64)
    ok = dict(k_exponents=ke, v_exponents=ve)
    for args, kw in (((k.float(), k.float(), kc, vc, slots), ok), ((k, k[:2], kc, vc, slots), ok), ((k, k, kc, vc, slots.int()), ok),
                     ((k, k, kc, vc, slots[:2]), ok), ((k[:, :1], k[:, :1], kc, vc, slots), ok), ((k, k, kc, vc[:3], slots), ok),
                     ((k, k, kc, vc, slots), dict(k_exponents=ke[:3], v_exponents=ve)), ((k, k, kc, vc, slots), dict(k_exponents=ke.long(), v_exponents=ve)),
                     ((k, k, kc, vc, slots), dict(k_exponents=ke.cpu(), v_exponents=ve)), ((k, k, kc[:, :8], vc[:, :8], slots), ok),
                     ((k, k, kc.view(torch.uint8), vc.view(torch.uint8), slots), ok), ((k, k, kc.view(torch.float8_e5m2), vc, slots), ok)):
        with pytest.raises(AssertionError):
            write_kv(*args, **kw)
    with pytest.raises(AssertionError):
        read_kv(kc, vc, slots, ke, ve, dtype=torch.float32)
    with pytest.raises(AssertionError):
        read_kv(kc, vc, slots, ke, ve, key=k)
    with pytest.raises(AssertionError):
        qk_norm_rope_write(rand(3, 4, 64), k, k, None, None, kc, vc, slots, **ok)  # neither rotation nor norm
    with pytest.raises(NotImplementedError):
        write_kv(k.clone().requires_grad_(), k, kc, vc, slots, **ok)


def test_another_stream_and_a_graph():
    """The pool as a captured step leaves it, replayed over new tokens with eager work in between."""
    bs, Hkv, D, T = 16, 2, 128, 8
    kc, vc, ke, ve = new_cache(T, bs, Hkv, D, seed=1)
    k = rand(T, Hkv, D)
    slots = (torch.arange(T) * bs + 3).cuda()
    copy = [x.clone() for x in (kc, vc, ke, ve)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        write_kv(k, k, kc, vc, slots, k_exponents=ke, v_exponents=ve)
    side.synchronize()
    want = stored(copy[0], copy[2], k.double(), slots, limit_of(BF))
    assert torch.equal(kc.view(torch.uint8), want[0]) and torch.equal(ke, want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        write_kv(k, k, kc, vc, slots, k_exponents=ke, v_exponents=ve)
        rows, _ = read_kv(kc, vc, slots, ke, ve)
    for step in range(4):
        k.copy_(rand(T, Hkv, D, seed=10 + step, scale=4.0 ** step))
        slots += 1
        want = stored(kc, ke, k.double(), slots, limit_of(BF))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kc.view(torch.uint8), want[0]) and torch.equal(ke, want[1])
        assert torch.equal(rows, values(kc, ke)[slots // bs, slots % bs].to(BF))


def test_pages_past_2_gib():
    """Byte offsets past 32 bits: the last pages of a cache of 2.1 GiB of keys."""
    bs, Hkv, D = 16, 8, 128
    blocks = (1 << 31) // (bs * Hkv * D) + 500
    kc, vc = (torch.zeros(blocks, bs, Hkv, D, dtype=torch.uint8, device="cuda").view(CODES) for _ in range(2))
    ke, ve = (torch.full((blocks, Hkv), LEAST, dtype=torch.int32, device="cuda") for _ in range(2))
    slots = torch.cat([torch.arange((blocks - 2) * bs, blocks * bs - 3), torch.arange(5)]).cuda()
    k, v = rand(slots.shape[0], Hkv, D), rand(slots.shape[0], Hkv, D, seed=1)
    write_kv(k, v, kc, vc, slots, k_exponents=ke, v_exponents=ve)
    key, value = read_kv(kc, vc, slots, ke, ve)
    for got, x in ((key, k), (value, v)):
        for run in (slice(0, 16), slice(16, 29), slice(29, 34)):
            e = exponents_of(x[run].double().abs().amax((0, 2)))
            want = decode(encode(x[run].double() * power(-e)[:, None]).view(CODES)) * power(e)[:, None]
            assert torch.equal(got[run].double(), want)
    assert int(kc.view(torch.uint8)[1:-2].max()) == 0
    del kc, vc
    torch.cuda.empty_cache()


@pytest.mark.parametrize("native", [True, False], ids=["native", "ctypes"])
def test_both_bindings(native, monkeypatch):
    if not native:
        monkeypatch.setattr(_lib, "_host", None)
        import gqa_kernels.cache8 as m
        import gqa_kernels.rotary as r
        monkeypatch.setattr(m, "_decode_host", lambda: None)
        monkeypatch.setattr(r, "_decode_host", lambda: None)
    slots, blocks = slots_of([(3, 40)], 16)
    k, v = rand(40, 2, 64), rand(40, 2, 64, seed=1)
    kc, vc, ke, ve = check_store(k, v, slots, blocks, 16, BF)
    key, value = read_kv(kc, vc, slots, ke, ve, dtype=FP)
    assert torch.equal(key, values(kc, ke)[slots // 16, slots % 16].to(FP)) and torch.equal(value, values(vc, ve)[slots // 16, slots % 16].to(FP))
