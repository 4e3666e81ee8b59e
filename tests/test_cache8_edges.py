"""The paged cache in 8 bits at the edges of what its calls allow."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from cache8_reference import CODES, LEAST, exponents_of, gather, limit_of, new_cache, power, stored, values
from gqa_kernels import RotaryTable, _lib, cache8, paged, qk_norm_rope, qk_norm_rope_write
from gqa_kernels.paged import PagedKVCache, paged_attention, read_kv, write_kv
from ops_reference import attend64, check_attention, rope64

BF = torch.bfloat16


def rand(*shape, dtype=BF, seed=0, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def ints(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def python_alone(monkeypatch):
    """Calls go through Python's checks and ctypes."""
    monkeypatch.setattr(_lib, "_host", None)
    monkeypatch.setattr(cache8, "_decode_host", lambda: None)


# ---------------------------------------------------------------------------
# A sequence that comes more than once in an append
# ---------------------------------------------------------------------------
COMING_BACK = [(["a", "b", "a"], [3, 2, 4]), (["a", "a", "b"], [3, 2, 4]), (["a", "b", "a", "b", "b", "a"], [1, 20, 15, 1, 2, 16]), (["a", "b", "a"], [3, 0, 4]),
               (["b", "a", "c", "b"], [5, 1, 1, 1])]


@pytest.mark.parametrize("ids,new", COMING_BACK)
def test_a_page_is_one_run_of_each_store(ids, new, monkeypatch):
    """Two runs of a page in one store would be two workgroups over one exponent and the same tokens in front (no GPU here)."""
    cache, calls = PagedKVCache(12, 16, 2, 64, dtype=CODES, device="cpu"), []
    for s in "abc":
        cache.add_sequence(s)
    monkeypatch.setattr(paged, "write_kv", lambda k, v, kc, vc, slots, **kw: calls.append((k, slots)))
    for _ in range(2):
        calls.clear()
        key = torch.arange(sum(new)).view(-1, 1, 1).expand(-1, 2, 64)
        slots = cache.append(ids, key, key, new)
        assert torch.equal(torch.cat([s for _, s in calls]), slots) and torch.equal(torch.cat([k[:, 0, 0] for k, _ in calls]), torch.arange(sum(new)))
        assert len(slots.unique()) == sum(new)
        for _, s in calls:
            pages = torch.unique_consecutive(s // 16)
            assert len(pages) == len(pages.unique()), f"pages {pages.tolist()}"
    together = [i for i, n in zip(ids, new) if n]
    together = [i for j, i in enumerate(together) if not j or together[j - 1] != i]
    if len(set(together)) == len(together):
        assert len(calls) == 1
    cache = PagedKVCache(12, 16, 2, 64, device="cpu")  # 16 bits: one store
    for s in "abc":
        cache.add_sequence(s)
    calls.clear()
    cache.append(ids, key, key, new)
    assert len(calls) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("ids,new", COMING_BACK)
def test_append_of_a_sequence_that_comes_back(ids, new):
    """The pool as one store after the other leaves it, and every token within a rounding of what was appended."""
    cache, said = PagedKVCache(12, 16, 2, 64, dtype=CODES), {s: [] for s in "abc"}
    for s in "abc":
        cache.add_sequence(s)
    for step in range(3):
        key = rand(sum(new), 2, 64, seed=step, scale=4.0 ** step)
        size = torch.exp2(torch.arange(sum(new)) % 7 - 3.0).view(-1, 1, 1).cuda()
        key = (key * size).to(BF)
        cache.append(ids, key, -key, new)
        at = 0
        for s, n in zip(ids, new):
            said[s].append(key[at:at + n])
            at += n
    for s in "abc":
        x = torch.cat(said[s] + [key[:0]]).double()
        k, v = cache.read(s)
        assert torch.equal(k, -v) and k.shape == x.shape
        for a in range(0, x.shape[0], 16):
            page = slice(a, a + 16)
            # Half a step of the value twice (stored, brought to a larger exponent) and half the least step of the page's largest value, once a store.
            unit = x[page].abs().amax((0, 2))[:, None] / 224
            assert ((k[page].double() - x[page]).abs() <= 2 * 2.0 ** -4 * x[page].abs() + 16 * 2.0 ** -10 * unit).all()


# ---------------------------------------------------------------------------
# No keys at all
# ---------------------------------------------------------------------------
@pytest.mark.skipif(torch.cuda.is_available(), reason="what follows the checks would launch")
def test_no_table_is_needed_without_keys():
    """The checks let the call pass: what fails is the missing device."""
    P, st = 0x10000, _lib._i64x4(8 * 64 * 128, 64 * 128, 128, 1)
    none, dead = _lib.Cache8(), 100  # hipErrorNoDevice
    for form, parts, ws in ((_lib.FORM_SINGLE, 0, None), (_lib.FORM_CHUNKS, 2, P)):
        assert _lib.load().gqa_paged8_launch(form, P, st, ctypes.byref(none), ctypes.byref(none), None, 0, P, None, None, 16, 0, P, st, P, ws, parts, 1, 8, 2, 4,
                                             128, 0.1, 1, 0, None, None) == dead


@pytest.mark.gpu
@pytest.mark.parametrize("binding", ["native", "python"])
@pytest.mark.parametrize("Sq", [1, 4, 40])
def test_tables_of_no_pages(Sq, binding, monkeypatch):
    """Requests that have no page yet, over a cache with blocks and over one without: zeros and LSE -inf."""
    q = rand(3, 8, Sq, 64)
    table, lens = torch.empty(3, 0, dtype=torch.int32, device="cuda"), ints([0, 0, 0])
    for blocks in (4, 0):
        kc, vc, ke, ve = new_cache(blocks, 16, 2, 64)
        e = dict(k_exponents=ke, v_exponents=ve)
        paged_attention(q, kc, vc, table, lens, **e)  # (loads the binding)
        if binding == "python":
            python_alone(monkeypatch)
        for kw in ({}, dict(causal=False), dict(softcap=20.0), dict(out=torch.full_like(q, 7.0))):
            o, lse = paged_attention(q, kc, vc, table, lens, return_lse=True, **e, **kw)
            assert o.shape == q.shape and not o.any() and (lse == -float("inf")).all()
            assert torch.equal(paged_attention(q, kc, vc, table, lens, **e, **kw), o)
        t = q.transpose(1, 2).flatten(0, 1).contiguous()
        o = paged_attention(t, kc, vc, table, lens, query_start=ints([0, Sq, 2 * Sq]), query_lens=ints([Sq] * 3), max_query_len=Sq, **e)
        assert not o.any()


# ---------------------------------------------------------------------------
# Norms of keys of any size
# ---------------------------------------------------------------------------
def stored_keys(k, wk, eps, *, R, inter=False, bs=16, start=3, seed=0):
    """(keys that the cache then holds, their unit, those of rope64, the row's largest of these)."""
    T, Hkv, D = k.shape
    table = None if R == 0 else RotaryTable(D, 9000, rotary_dim=R, interleaved=inter)
    pos = torch.randint(0, 9000, (T,), generator=torch.Generator().manual_seed(seed)).cuda()
    kc, vc, ke, ve = new_cache((start + T) // bs + 1, bs, Hkv, D, full=False)
    slots = (torch.arange(T) + start).cuda()
    qk_norm_rope_write(k, k, k, pos, table, kc, vc, slots, k_weight=wk, eps=eps, k_exponents=ke, v_exponents=ve)
    inv = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R) if R else None
    y, _ = rope64(k, wk, eps, pos[None, :, None] if R else None, rotary_dim=R, interleaved=inter, inv_freq=inv, axes=[0] * (R // 2))
    page = slots // bs
    return values(kc, ke)[page, slots % bs], power(ke)[page][..., None], y, y.abs().amax(-1, keepdim=True)


@pytest.mark.gpu
@pytest.mark.parametrize("D,R,inter", [(64, 64, False), (128, 64, True), (128, 0, False), (128, 128, False)])
@pytest.mark.parametrize("w32", [False, True], ids=["w16", "w32"])
def test_norms_of_keys_of_any_size(D, R, inter, w32):
    """Rows of bf16 from its smallest numbers to its largest, whose squares and weighted values pass fp32's range (and, below it, vanish): as close as any."""
    T, Hkv = 40, 2
    size = torch.exp2(torch.linspace(-122, 125, T * Hkv).round()).view(T, Hkv, 1).cuda()
    k = (rand(T, Hkv, D).clamp(-3.9, 3.9).float() * size).to(BF)
    assert torch.isfinite(k).all() and float(k.float().abs().max()) > 1e38
    for least, most in ((-1, 1), (9, 12), (-12, -9)):
        w = torch.exp2(torch.empty(D).uniform_(least, most, generator=torch.Generator().manual_seed(1))).cuda()
        w = w if w32 else w.to(BF)
        for eps in (1e-6, 0.0):
            got, unit, y, top = stored_keys(k, w, eps, R=R, inter=inter)
            assert torch.isfinite(y).all() and (y.abs().amax((0, 2)) > 2.0 ** (least - 1)).all()
            assert ((got - y).abs() <= 2.0 ** -4 * y.abs() + 2.0 ** -10 * unit + 2.0 ** -18 * top).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, torch.float16], ids=["bf16", "fp16"])
def test_norms_of_rows_with_infinities_and_nan(dtype):
    """An infinite key, normed: zeros beside it, as 1 / rms = 0 gives, and NaN where 0 meets it (and in what it turns with); a NaN is the whole row's."""
    k = rand(6, 2, 128, dtype=dtype)
    k[1, 0, 3], k[2, 1, 70], k[2, 1, 71], k[4, 0, 5] = float("inf"), -float("inf"), float("inf"), float("nan")
    w = (rand(128, seed=1) * 0.3 + 1).to(dtype)
    for R in (0, 128, 64):
        got, unit, y, top = stored_keys(k, w, 1e-6, R=R, start=0)
        assert torch.equal(torch.isnan(got), torch.isnan(y)) and torch.isnan(y[4, 0]).all()
        top = torch.nan_to_num(y, nan=0.0).abs().amax(-1, keepdim=True)
        ok = ~torch.isnan(y)
        assert ((got - y).abs() <= 2.0 ** -4 * y.abs() + 2.0 ** -10 * unit + 2.0 ** -18 * top)[ok].all()


# ---------------------------------------------------------------------------
# What would lose a derivative
# ---------------------------------------------------------------------------
def losing_calls():
    """name: (tensors that may not carry one, the call)."""
    kc, vc, ke, ve = new_cache(3, 16, 2, 64)
    x = {"kc": kc, "vc": vc, "q": rand(1, 4, 6, 64), "out": rand(1, 4, 6, 64), "slopes": rand(4).float(), "qt": rand(6, 4, 64), "qo": rand(6, 4, 64),
         "kt": rand(6, 2, 64), "vt": rand(6, 2, 64), "w": rand(64), "key": rand(6, 2, 64), "value": rand(6, 2, 64)}
    rot, table, lens, pos, slots = RotaryTable(64, 50), ints([[2, 0, 1]]), ints([40]), ints(range(6)), torch.arange(6).cuda()
    e = dict(k_exponents=ke, v_exponents=ve)
    return x, {
        "attention": (("q", "kc", "vc", "slopes", "out"), lambda x: paged_attention(x["q"], x["kc"], x["vc"], table, lens, softcap=9.0, alibi_slopes=x["slopes"],
                                                                                   out=x["out"], **e)),
        "write": (("kt", "vt", "kc", "vc"), lambda x: write_kv(x["kt"], x["vt"], x["kc"], x["vc"], slots, **e)),
        "rope write": (("qt", "kt", "vt", "w", "kc", "vc", "qo"), lambda x: qk_norm_rope_write(x["qt"], x["kt"], x["vt"], pos, rot, x["kc"], x["vc"], slots,
                                                                                              q_weight=x["w"], k_weight=x["w"], q_out=x["qo"], **e)),
        "read": (("kc", "vc", "key", "value"), lambda x: read_kv(x["kc"], x["vc"], slots, key=x["key"], value=x["value"], **e)),
    }


@pytest.mark.gpu
@pytest.mark.parametrize("binding", ["native", "python"])
@pytest.mark.parametrize("mode", ["forward", "forward under no_grad", "backward"])
@pytest.mark.parametrize("name", ["attention", "write", "rope write", "read"])
def test_what_would_lose_a_derivative_is_refused(name, mode, binding, monkeypatch):
    x, calls = losing_calls()
    names, call = calls[name]
    call(x)  # (loads the binding)
    if binding == "python":
        python_alone(monkeypatch)
    for n in names:
        if mode == "backward":
            y = {**x, n: x[n].detach().clone().requires_grad_()}
            with pytest.raises(NotImplementedError):
                call(y)
            with torch.no_grad():
                call(y)
        elif x[n].dtype is not CODES:  # (torch makes no tangents of codes)
            with forward_ad.dual_level():
                y = {**x, n: forward_ad.make_dual(x[n].clone(), torch.ones_like(x[n]))}
                with pytest.raises(NotImplementedError):
                    if "no_grad" in mode:
                        with torch.no_grad():
                            call(y)
                    else:
                        call(y)
    call(x)


# ---------------------------------------------------------------------------
# Stores into memory that pages, heads, keys or values share
# ---------------------------------------------------------------------------
def sharing(kv, e):
    """Codes (2, blocks, bs, Hkv, D) and exponents (2, blocks, Hkv) of which some share memory: a store's workgroups would race for it."""
    return [(kv, e[:, :, :1].expand_as(e)), (kv, e[:, :1].expand_as(e)), (kv, e[:1].expand_as(e)), (kv, e[0].new_zeros(1).expand_as(e)),
            (kv[:, :, :, :1].expand_as(kv), e), (kv[:, :1].expand_as(kv), e), (kv[:1].expand_as(kv), e)]


@pytest.mark.parametrize("i", range(7))
def test_stores_into_shared_memory_are_refused(i):
    """(No GPU here: the check comes before any other of the device.)"""
    kv, e = sharing(torch.zeros(2, 4, 16, 2, 64, dtype=torch.uint8).view(CODES), cache8.new_exponents(4, 2, "cpu"))[i]
    rows, slots = torch.zeros(1, 2, 64, dtype=BF), torch.zeros(1, dtype=torch.int64)
    with pytest.raises(AssertionError, match="memory of their own"):
        cache8.write(rows, rows, kv[0], kv[1], slots, e[0], e[1])
    with pytest.raises(AssertionError, match="memory of their own"):
        cache8.check_caches(kv[0], kv[1], e[0], e[1], write=True)


@pytest.mark.skipif(torch.cuda.is_available(), reason="what passes the checks would launch")
def test_stores_into_shared_memory_are_refused_by_the_entry_point():
    P, t3 = 0x10000, _lib._i64x3(1024, 128, 1)

    def write(heads=2, vc=2 * P, ve=2 * P, stride=(4096, 256, 128, 1), exp_stride=(2, 1)):
        k, v = (_lib.Cache8(c, (ctypes.c_int64 * 4)(*stride), x, (ctypes.c_int64 * 2)(*exp_stride)) for c, x in ((P, P), (vc, ve)))
        return _lib.load().gqa_cache8_write_launch(None, t3, P, t3, P, t3, None, t3, ctypes.byref(k), ctypes.byref(v), P, None, 4, 0, heads, 128, 16, 0, None)

    for kw in (dict(vc=P), dict(ve=P), dict(stride=(4096, 256, 0, 1)), dict(stride=(4096, 0, 128, 1)), dict(exp_stride=(2, 0))):
        assert write(**kw) == _lib.GQA_E_CACHE8, kw
    for kw in ({}, dict(heads=1, stride=(4096, 128, 0, 1), exp_stride=(1, 0))):
        assert write(**kw) == 100, kw  # hipErrorNoDevice


@pytest.mark.gpu
def test_broadcast_exponents_are_read_and_not_written():
    kc, vc, ke, ve = new_cache(3, 16, 2, 64)
    e = torch.full((1, 1), -7, dtype=torch.int32, device="cuda")
    one, all_ = e.expand(3, 2), e.expand(3, 2).contiguous()
    slots, k, q = torch.arange(20).cuda(), rand(20, 2, 64), rand(1, 4, 1, 64)
    for a, b in zip(read_kv(kc, vc, slots, one, one), read_kv(kc, vc, slots, all_, all_.clone())):
        assert torch.equal(a, b)
    at = ints([[2, 0, 1]]), ints([40])
    assert torch.equal(paged_attention(q, kc, vc, *at, k_exponents=one, v_exponents=one), paged_attention(q, kc, vc, *at, k_exponents=all_, v_exponents=all_))
    w = rand(64)
    for x, y in ((one, ve), (ke, one), (ke, ke)):
        for _ in range(2):  # (through Python's checks first, and past the native call's)
            with pytest.raises(AssertionError, match="memory of their own"):
                write_kv(k, k, kc, vc, slots, k_exponents=x, v_exponents=y)
            with pytest.raises(AssertionError, match="memory of their own"):
                qk_norm_rope_write(rand(20, 4, 64), k, k, None, None, kc, vc, slots, k_weight=w, k_exponents=x, v_exponents=y)
        read_kv(kc, vc, slots, ke, ve)
    assert int(e) == -7
    kc, vc, ke, ve = new_cache(1, 16, 1, 64)  # one page, one head: any stride is their own
    write_kv(k[:8, :1], k[:8, :1], kc, vc, slots[:8], k_exponents=ke.as_strided((1, 1), (0, 0)), v_exponents=ve.as_strided((1, 1), (0, 0)))
    assert int(ke) == int(ve)


# ---------------------------------------------------------------------------
# Pages and exponents that a wave holds by lane, and their next 64
# ---------------------------------------------------------------------------
def long_batch(lens, Hq, Hkv, Sq, D, dtype, bs=16, seed=0):
    """(queries, cache, exponents, table, lengths): pages in random order, exponents spread over 2^13."""
    pages = [-(-n // bs) for n in lens]
    order, width, rows, at = torch.randperm(sum(pages), generator=torch.Generator().manual_seed(seed)).tolist(), max(pages), [], 0
    for n in pages:
        rows.append(order[at:at + n] + [-12345] * (width - n))
        at += n
    kc, vc, ke, ve = new_cache(sum(pages), bs, Hkv, D, seed=seed, spread=6)
    ke -= 4  # (scores of a few units)
    return rand(len(lens), Hq, Sq, D, dtype=dtype, seed=seed + 1), (kc, vc), dict(k_exponents=ke, v_exponents=ve), ints(rows), ints(lens)


def check_long(batch, lens, slopes=None, **kw):
    q, (kc, vc), e, table, n = batch
    o, lse = paged_attention(q, kc, vc, table, n, return_lse=True, alibi_slopes=slopes, **e, **kw)
    for b, m in enumerate(lens):
        k, v = (gather(c, x, table[b], m, q.dtype) for c, x in ((kc, e["k_exponents"]), (vc, e["v_exponents"])))
        check_attention(o[b], lse[b], attend64(q[b], k, v, slopes=slopes))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq", [1, 3, 8])
@pytest.mark.parametrize("lens", [[4096], [4097], [4100, 8192], [4500, 50, 9000], [12345, 4224]])
def test_few_rows_over_long_pieces(lens, Sq, D, dtype):
    """One and two 16-row blocks; pieces of more than 32 tiles a wave, once and several times over, ends on a tile's, a unit's and a wave's share."""
    batch = long_batch(lens, 8, 2, Sq, D, dtype, seed=Sq)
    slopes = torch.tensor([2.0 ** -(h + 4) for h in range(8)]).cuda()
    for splits in (1, 2):
        check_long(batch, lens, route="split", splits=splits)
    check_long(batch, lens, slopes, route="split", splits=1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq", [30, 100])
@pytest.mark.parametrize("lens", [[4096, 4095], [4097, 100], [4160, 8200], [9000, 4225]])
def test_many_rows_over_long_pieces(lens, Sq, D, dtype):
    """Blocks of 128 packed rows, and at head_dim 128 of 256; more than 64 tiles, in order and, with slopes, in reverse."""
    batch = long_batch(lens, 8, 2, Sq, D, dtype, seed=Sq)
    slopes = torch.tensor([2.0 ** -(h + 4) for h in range(8)]).cuda()
    for kw in (dict(route="single"), dict(route="chunks", splits=1)):
        check_long(batch, lens, **kw)
        check_long(batch, lens, slopes, **kw)


# ---------------------------------------------------------------------------
# Stores of normed and rotated keys whose pages take more than one step
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("T,Hkv,D,bs,R,inter", [(300, 2, 64, 128, 64, False), (300, 8, 128, 256, 64, True), (2500, 2, 128, 256, 128, False), (2500, 4, 64, 128, 32, True),
                                                (300, 1, 128, 512, 128, False), (40, 3, 128, 64, 128, True)])
def test_norms_and_rotation_over_pages_of_several_steps(T, Hkv, D, bs, R, inter, dtype):
    """Two sequences that begin inside a page, most of whose tokens are in later steps and beyond the first 64 of their page."""
    first, cut = 7, T - T // 3
    at = torch.cat([torch.arange(first, first + cut), torch.arange(3, T - cut + 3)])
    pages = -(-(first + cut) // bs)
    order = torch.randperm(pages + -(-(T - cut + 3) // bs), generator=torch.Generator().manual_seed(T))
    page = torch.cat([order[at[:cut] // bs], order[pages + at[cut:] // bs]])
    slots = (page * bs + at % bs).cuda()
    k, v, q = (rand(T, h, D, dtype=dtype, seed=h, scale=2.0) for h in (Hkv, Hkv + 1, 5))
    v = v[:, :Hkv]
    w = (rand(D, seed=2) * 0.3 + 1).to(dtype)
    pos = torch.randint(0, 9000, (T,), generator=torch.Generator().manual_seed(1)).cuda()
    table = RotaryTable(D, 9000, rotary_dim=R, interleaved=inter)
    kc, vc, ke, ve = new_cache(len(order), bs, Hkv, D, seed=2, spread=6)
    was, codes = ke.clone(), kc.clone()
    wantv = stored(vc, ve, v.double(), slots, limit_of(dtype))
    qo = qk_norm_rope_write(q, k, v, pos, table, kc, vc, slots, q_weight=w, k_weight=w, k_exponents=ke, v_exponents=ve)
    assert torch.equal(vc.view(torch.uint8), wantv[0]) and torch.equal(ve, wantv[1])
    inv = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    y, tol = rope64(q, w, 1e-6, pos[None, :, None], rotary_dim=R, interleaved=inter, inv_freq=inv, axes=[0] * (R // 2))
    assert ((qo.double() - y).abs() <= tol).all()
    y, _ = rope64(k, w, 1e-6, pos[None, :, None], rotary_dim=R, interleaved=inter, inv_freq=inv, axes=[0] * (R // 2))
    size, (pg, off) = y.abs().amax(-1, keepdim=True), (slots // bs, slots % bs)
    got, unit = values(kc, ke)[pg, off], power(ke)[pg][..., None]
    assert ((got - y).abs() <= 2.0 ** -4 * y.abs() + 2.0 ** -10 * unit + 2.0 ** -18 * size).all()
    for x in pg.unique().tolist():
        mine = pg == x
        most, near = y[mine].abs().amax((0, 2)), 2.0 ** -18 * size[mine].amax((0, 2))
        old = was[x] if int(off[mine].min()) > 0 else torch.full_like(was[x], LEAST)
        assert (ke[x] >= torch.maximum(exponents_of(most - near), old)).all() and (ke[x] <= torch.maximum(exponents_of(most + near), old)).all()
        # The tokens in front as their old codes under the new exponent; what lies behind is left.
        low, behind = int(off[mine].min()), int(off[mine].max()) + 1
        want = values(codes[x:x + 1], was[x:x + 1])[0, :low]
        assert ((values(kc, ke)[x, :low] - want).abs() <= 2.0 ** -10 * power(ke[x])[:, None]).all()
        assert torch.equal(kc[x, behind:].view(torch.uint8), codes[x, behind:].view(torch.uint8))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("D,R,inter", [(64, 64, False), (64, 32, True), (128, 128, False), (128, 128, True), (128, 16, False)])
def test_queries_are_the_same_whatever_stores_the_keys(D, R, inter, dtype):
    """One form of the norm and rotation: the bits of qk_norm_rope, with keys stored in 8 bits, in 16 or not at all."""
    T, Hq, Hkv = 257, 6, 2
    q, k, v = (rand(T, h, D, dtype=dtype, seed=s, scale=3.0) for s, h in ((1, Hq), (2, Hkv), (3, Hkv)))
    table = RotaryTable(D, 9000, rotary_dim=R, interleaved=inter)
    pos, slots = torch.randint(0, 9000, (T,), generator=torch.Generator().manual_seed(1)).cuda(), torch.arange(T).cuda()
    for w in (None, (rand(D, seed=4) * 0.3 + 1).to(dtype), rand(D, seed=4).float() * 0.3 + 1):
        kw = dict(q_weight=w, k_weight=w)
        want, keys = qk_norm_rope(q, k, pos, table, **kw)
        kc, vc, ke, ve = new_cache(17, 16, Hkv, D, full=False)
        assert torch.equal(qk_norm_rope_write(q, k, v, pos, table, kc, vc, slots, k_exponents=ke, v_exponents=ve, **kw), want)
        k16, v16 = (torch.zeros(17, 16, Hkv, D, dtype=dtype, device="cuda") for _ in range(2))
        assert torch.equal(qk_norm_rope_write(q, k, v, pos, table, k16, v16, slots, **kw), want)
        assert torch.equal(k16.flatten(0, 1)[:T], keys)
