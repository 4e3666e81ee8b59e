"""What the entry points of the paged cache in 8 bits refuse before any HIP call, and the forms that calls are given (no GPU here)."""
import ctypes

import pytest
import torch

from cache8_reference import CODES, decode, encode, exponents_of
from gqa_kernels import _lib, cache8
from gqa_kernels.paged import PagedKVCache, paged_attention, read_kv, write_kv

SHAPE, HEAD, DTYPE, STRIDE, SPLITS, GROUP, NULL, BLOCK = -1, -2, -3, -4, -5, -6, -7, -8
E8 = _lib.GQA_E_CACHE8
P = 0x10000  # an aligned address that is never read
ST = _lib._i64x4(8 * 64 * 128, 64 * 128, 128, 1)
T3 = _lib._i64x3(1024, 128, 1)


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def cache(codes=P, exponents=P, stride=(16 * 2 * 128, 2 * 128, 128, 1), exp_stride=(2, 1)):
    return _lib.Cache8(codes, (ctypes.c_int64 * 4)(*stride), exponents, (ctypes.c_int64 * 2)(*exp_stride))


def attend(lib, form=1, parts=0, q=P, q_st=ST, k=None, v=None, table=P, table_stride=8, lens=P, qs=None, ql=None, block=16, max_len=64, o=P, lse=None, ws=None,
           batch=1, heads=8, kv=2, seq_q=4, head_dim=128, scale=0.1, causal=1, dtype=0, score=None):
    k, v = (cache() if x is None else x for x in (k, v))
    return lib.gqa_paged8_launch(form, q, q_st, ctypes.byref(k), ctypes.byref(v), table, table_stride, lens, qs, ql, block, max_len, o, ST, lse, ws, parts, batch,
                                 heads, kv, seq_q, head_dim, scale, causal, dtype, score, None)


BAD_CACHES = [(dict(codes=None), NULL), (dict(exponents=None), NULL), (dict(codes=P + 8), STRIDE), (dict(exponents=P + 2), STRIDE),
              (dict(stride=(4096, 256, 128, 2)), STRIDE), (dict(stride=(4096, 256, 120, 1)), STRIDE), (dict(stride=(4104, 256, 128, 1)), STRIDE),
              (dict(stride=(1 << 40, 1 << 28, 128, 1)), E8), (dict(stride=(4096, -256, 128, 1)), E8)]


def test_attention_refusals(lib):
    for kw, code in BAD_CACHES:
        assert attend(lib, k=cache(**kw)) == code and attend(lib, v=cache(**kw)) == code, kw
    for kw in (dict(block=8), dict(block=0), dict(block=24), dict(block=1 << 17), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
               dict(scale=float("inf")), dict(form=0), dict(form=4), dict(form=7), dict(form=3, parts=1, seq_q=9), dict(form=3, parts=1, max_len=0)):
        assert attend(lib, **kw) == E8, kw
    for kw in (dict(form=2, parts=0), dict(form=2, parts=1025), dict(form=2, parts=2, batch=3), dict(form=3, parts=0), dict(form=3, parts=1025)):
        assert attend(lib, **kw) == SPLITS, kw
    for kw in (dict(q=None), dict(o=None), dict(table=None), dict(lens=None), dict(qs=P), dict(ql=P), dict(form=2, parts=2), dict(form=3, parts=2)):
        assert attend(lib, **kw) == NULL, kw
    for kw in (dict(q=P + 2), dict(q_st=_lib._i64x4(4, 8, 8, 1)), dict(lens=P + 2), dict(table=P + 1), dict(lse=P + 2), dict(qs=P + 2, ql=P),
               dict(form=2, parts=2, ws=P + 4)):
        assert attend(lib, **kw) == STRIDE, kw
    assert attend(lib, head_dim=96) == HEAD and attend(lib, dtype=2) == DTYPE and attend(lib, heads=7) == SHAPE and attend(lib, batch=-1) == SHAPE
    assert attend(lib, max_len=129) == BLOCK and attend(lib, table_stride=-1) == BLOCK
    for form, parts in ((1, 0), (2, 4), (3, 4)):  # keys whose tiles' ends would pass 32 bits
        assert attend(lib, form=form, parts=parts, ws=P, max_len=0x7FFFC001, table_stride=1 << 28) == E8
    assert attend(lib, heads=2 * 129, kv=2) == GROUP
    assert attend(lib, batch=0) == 0 and attend(lib, seq_q=0) == 0
    # More units and slots than the flat split's walk multiplies in 32 bits.
    assert attend(lib, form=3, parts=1024, ws=P, batch=1 << 20, table_stride=1 << 20, max_len=1 << 20) == E8
    for s, code in ((_lib.Score(softcap=-1.0), _lib.GQA_E_SCORE), (_lib.Score(span_lo=P, span_hi=P), _lib.GQA_E_SCORE), (_lib.Score(alibi_slopes=P + 1), STRIDE)):
        assert attend(lib, score=ctypes.byref(s)) == code
    assert b"8 bits" in lib.gqa_strerror(E8)


def test_write_and_read_refusals(lib):
    def write(q=None, k=P, v=P, qo=None, kc=None, vc=None, slots=P, rope=None, tokens=4, heads=8, kv=2, head_dim=128, block=16, dtype=0, t3=T3):
        kc, vc = (cache() if x is None else x for x in (kc, vc))
        return lib.gqa_cache8_write_launch(q, t3, k, t3, v, t3, qo, t3, ctypes.byref(kc), ctypes.byref(vc), slots, rope, tokens, heads, kv, head_dim, block, dtype,
                                           None)

    def read(kc=None, vc=None, slots=P, k=P, v=P, tokens=4, kv=2, head_dim=128, block=16, dtype=0, t3=T3):
        kc, vc = (cache() if x is None else x for x in (kc, vc))
        return lib.gqa_cache8_read_launch(ctypes.byref(kc), ctypes.byref(vc), slots, k, t3, v, t3, tokens, kv, head_dim, block, dtype, None)

    for call in (write, read):
        for kw, code in BAD_CACHES:
            assert call(kc=cache(**kw)) == code and call(vc=cache(**kw)) == code, kw
        for kw in (dict(block=8), dict(block=48)):
            assert call(**kw) == E8
        for kw in (dict(k=None), dict(v=None), dict(slots=None)):
            assert call(**kw) == NULL, kw
        for kw in (dict(k=P + 2), dict(slots=P + 4), dict(t3=_lib._i64x3(1020, 128, 1)), dict(t3=_lib._i64x3(1024, 128, 2))):
            assert call(**kw) == STRIDE, kw
        assert call(head_dim=96) == HEAD and call(dtype=5) == DTYPE and call(tokens=-1) == SHAPE and call(kv=0) == SHAPE
        assert call(tokens=0, slots=None) == 0
    r = _lib.Rope(table=P, max_positions=10, rotary_dim=128, positions=P, axes=1)
    assert write(q=P, qo=P) == NULL  # queries without a rotation or norm
    assert write(q=P, qo=None, rope=ctypes.byref(r)) == NULL and write(q=None, qo=P, rope=ctypes.byref(r)) == NULL
    assert write(tokens=1 << 26) == SHAPE
    r.rotary_dim = 24
    assert write(q=P, qo=P, rope=ctypes.byref(r)) == _lib.GQA_E_ROPE


def test_plans_keep_their_limits(lib):
    for D in (64, 128):
        for batch, heads, kv, sq, n in ((1, 32, 8, 1, 1), (1, 32, 8, 1, 131072), (256, 32, 8, 1, 4000), (3, 8, 8, 16, 77), (1, 128, 1, 1, 500), (7, 28, 4, 9, 8192), (16, 32, 8, 8, 4000), (2, 31, 1, 1, 3000), (2, 11, 1, 3, 900),
                                        (4, 32, 8, 256, 9000), (1, 32, 8, 4096, 4096), (2, 64, 1, 2, 1 << 20), (1 << 16, 8, 8, 1, 1 << 20)):
            form, parts = cache8.plan(batch, heads, kv, sq, n, D, 256)
            few = heads // kv * sq <= 32
            assert form == (_lib.FORM_FLAT if few else form) and 0 <= parts <= 1024
            assert (form == _lib.FORM_SINGLE) == (parts == 0)
            if form == _lib.FORM_FLAT:
                units = -(-n // 128) * batch
                assert few and parts <= units and (units + 1) * (parts + 1) < 1 << 31
            need = lib.gqa_paged8_workspace_bytes(form, parts, batch, heads, sq, D)
            assert (need == 0) == (parts == 0)
    assert cache8.plan(0, 8, 2, 1, 100, 128, 256) == cache8.plan(1, 8, 2, 0, 100, 128, 256) == cache8.plan(1, 8, 2, 1, 0, 128, 256) == (_lib.FORM_SINGLE, 0)
    assert cache8.plan(1, 8, 2, 1, 0x7FFFC000, 128, 256)[0] == _lib.FORM_FLAT
    for bad in ((1, 8, 2, 1, 0x7FFFC001, 128, 256), (1, 8, 2, 100, 2 ** 31 - 1, 128, 256), (1, 7, 2, 1, 64, 128, 256), (1, 8, 2, 1, 64, 96, 256), (-1, 8, 2, 1, 64, 128, 256), (1, 258, 2, 1, 64, 128, 256), (1, 8, 2, 1, 64, 128, 0)):
        with pytest.raises(_lib.GQAError):
            cache8.plan(*bad)
    assert cache8.route(32, 8, 8) == "split" and cache8.route(32, 8, 9) == "single"


def test_python_refusals():
    """CPU tensors: the first check that a call fails names what is wrong."""
    kv = torch.zeros(2, 4, 16, 2, 64, dtype=torch.uint8).view(CODES)
    e = cache8.new_exponents(4, 2, "cpu")
    assert e.shape == (2, 4, 2) and int(e.max()) == int(e.min()) == -126
    q = torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16)
    table, lens, rows = torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    slots = torch.zeros(1, dtype=torch.int64)
    with pytest.raises(AssertionError):
        paged_attention(q, kv[0], kv[1], table, lens, k_exponents=e[0], v_exponents=e[1])  # (not on a GPU)
    for ke, ve in ((None, None), (e[0], None), (None, e[1])):
        with pytest.raises(AssertionError, match="needs k_exponents and v_exponents"):
            write_kv(rows, rows, kv[0], kv[1], slots, k_exponents=ke, v_exponents=ve)
        with pytest.raises(AssertionError, match="needs k_exponents and v_exponents"):
            read_kv(kv[0], kv[1], slots, ke, ve)
    with pytest.raises(AssertionError, match="codes"):
        write_kv(rows, rows, kv[0].view(torch.uint8), kv[1], slots, k_exponents=e[0], v_exponents=e[1])
    with pytest.raises(NotImplementedError, match="no derivative"):
        write_kv(rows.clone().requires_grad_(), rows, kv[0], kv[1], slots, k_exponents=e[0], v_exponents=e[1])
    with pytest.raises(AssertionError, match="16 tokens"):
        PagedKVCache(4, 8, 2, 64, dtype=CODES, device="cpu")
    assert PagedKVCache(4, 16, 2, 64, device="cpu").exponents is None


def test_reference_codes():
    """The reference's own codes against torch's."""
    every = torch.arange(256, dtype=torch.uint8)
    mine, theirs = decode(every.view(CODES)), every.view(CODES).double()
    nan = torch.isnan(theirs)
    assert int(nan.sum()) == 2 and torch.equal(torch.isnan(mine), nan) and torch.equal(mine[~nan], theirs[~nan])
    g = torch.Generator().manual_seed(0)
    y = torch.randn(20000, generator=g).double() * torch.exp2(torch.randint(-12, 7, (20000,), generator=g).double())
    y = torch.cat([y.clamp(-448, 448), mine[~nan], (mine[:126] + mine[1:127]) / 2])
    assert torch.equal(encode(y), y.float().to(CODES).view(torch.uint8)) or torch.equal(encode(y), y.to(CODES).view(torch.uint8))
    most = torch.tensor([0.0, 448.0, 448.0001, 1.75, 1.7500001, 896.0, 3e38, 1e-45], dtype=torch.float64)
    assert exponents_of(most).tolist() == [-126 if m == 0 or m < 1e-40 else next(e for e in range(-126, 127) if m <= 448 * 2.0 ** e) for m in most.tolist()]
