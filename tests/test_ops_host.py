"""What the entry points of changed scores, rotation, spans and block tables refuse, before any HIP call (no GPU here)."""
import ctypes

import pytest
import torch

from gqa_kernels import RotaryTable, _lib, document_spans, qk_norm_rope
from gqa_kernels.dispatch import _cu_count, _scored_route, scored_fine_split
from gqa_kernels.paged import BlockPool, extend_block_tables, scored_split
from gqa_kernels.scores import DocumentSpans, check_score

SHAPE, HEAD, DTYPE, STRIDE, SPLITS, NULL, BLOCK = -1, -2, -3, -4, -5, -7, -8
P = 0x10000  # an aligned address that is never read
ST = _lib._i64x4(8 * 64 * 128, 64 * 128, 128, 1)


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def scored(lib, form=1, parts=0, paged=False, softcap=10.0, slopes=None, prefix=None, lo=None, hi=None, scale=0.1, causal=1, seq_q=4, seq_kv=64,
           ws=None, lse=None, head_dim=128, dtype=0, batch=1):
    s = _lib.Score(softcap, slopes, prefix, lo, hi)
    if paged:
        return lib.gqa_paged_scored_launch(form, P, ST, P, ST, P, ST, P, 8, P, None, None, 16, seq_kv, P, ST, lse, ws, parts, batch, 8, 2, seq_q,
                                           head_dim, scale, causal, dtype, ctypes.byref(s), None)
    return lib.gqa_scored_launch(form, P, ST, P, ST, P, ST, P, ST, lse, ws, parts, batch, 8, 2, seq_q, seq_kv, head_dim, scale, causal, dtype,
                                 ctypes.byref(s), None)


@pytest.mark.parametrize("paged", [False, True])
def test_scored_refusals(lib, paged):
    E = _lib.GQA_E_SCORE
    for kw in (dict(softcap=-1.0), dict(softcap=float("nan")), dict(softcap=1e-5), dict(softcap=1e9), dict(scale=0.0), dict(scale=-1.0),
               dict(scale=float("inf")), dict(prefix=P, causal=0), dict(form=5), dict(form=-1), dict(lo=P, hi=P, form=0), dict(lo=P, hi=P, form=3),
               dict(lo=P, hi=P, seq_q=65)):
        assert scored(lib, paged=paged, **kw) == E, kw
    if paged:
        assert scored(lib, paged=True, lo=P, hi=P) == E
    for kw in (dict(slopes=P + 1), dict(prefix=P + 2), dict(lo=P + 1, hi=P), dict(lse=P + 1)):
        assert scored(lib, paged=paged, **kw) == STRIDE, kw
    assert scored(lib, paged=paged, lo=P) == NULL
    assert scored(lib, paged=paged, head_dim=96) == HEAD and scored(lib, paged=paged, dtype=2) == DTYPE
    assert scored(lib, paged=paged, form=0, parts=0) == SPLITS and scored(lib, paged=paged, form=2, parts=0) == SPLITS
    assert scored(lib, paged=paged, form=0, parts=2) == NULL  # no workspace
    assert scored(lib, paged=paged, form=3, parts=0) == _lib.GQA_E_FLAT
    assert scored(lib, paged=paged, batch=0) == 0 and scored(lib, paged=paged, seq_q=0) == 0
    assert b"softcap" in lib.gqa_strerror(E) and b"rotary_dim" in lib.gqa_strerror(_lib.GQA_E_ROPE)


def test_rope_refusals(lib):
    def call(q=P, k=P, batch=1, seq=4, head_dim=128, dtype=0, q_st=ST, write=False, block=16, slots=P, **kw):
        r = _lib.Rope(table=P, max_positions=10, rotary_dim=128, positions=P, axes=1)
        for n, v in kw.items():
            setattr(r, n, v)
        if write:
            t3 = _lib._i64x3(1024, 128, 1)
            return lib.gqa_qk_norm_rope_write_launch(q, t3, k, t3, P, t3, P, t3, P, ST, P, ST, slots, ctypes.byref(r), seq, 8, 2, head_dim, block, dtype, None)
        return lib.gqa_qk_norm_rope_launch(q, q_st, k, ST, P, ST, P if k else None, ST, ctypes.byref(r), batch, 8, 2, seq, head_dim, dtype, None)

    E = _lib.GQA_E_ROPE
    words = (ctypes.c_uint32 * 4)(2, 0, 0, 0)
    for write in (False, True):
        for kw in (dict(rotary_dim=8), dict(rotary_dim=144), dict(rotary_dim=24), dict(max_positions=0), dict(axes=0), dict(axes=5),
                   dict(axes=2, pair_axis=words), dict(q_weight=P, eps=-1.0), dict(q_weight=P, eps=float("nan"))):
            assert call(write=write, **kw) == E, kw
        for kw in (dict(table=P + 4), dict(positions=P + 2), dict(positions=P + 4, positions64=1), dict(q_weight=P + 8), dict(q=P + 2)):
            assert call(write=write, **kw) == STRIDE, kw
        for kw in (dict(positions=None), dict(q=None)):
            assert call(write=write, **kw) == NULL, kw
        assert call(write=write, head_dim=96) == HEAD and call(write=write, dtype=3) == DTYPE and call(write=write, seq=-1) == SHAPE
        assert call(write=write, seq=0, positions=None) == 0
    assert call(q_st=_lib._i64x4(4, 8, 8, 1)) == STRIDE and call(q_st=_lib._i64x4(8, 8, 8, 2)) == STRIDE
    assert call(batch=1 << 20, seq=1 << 20) == SHAPE
    assert call(write=True, block=12) == BLOCK and call(write=True, slots=None) == NULL and call(write=True, slots=P + 4) == STRIDE


def test_table_and_span_refusals(lib):
    assert lib.gqa_document_spans_launch(P, 8, P, P, -1, 8, None) == SHAPE and lib.gqa_document_spans_launch(None, 8, P, P, 1, 8, None) == NULL
    assert lib.gqa_document_spans_launch(P + 1, 8, P, P, 1, 8, None) == STRIDE and lib.gqa_document_spans_launch(P, 8, P, P, 0, 8, None) == 0
    assert lib.gqa_extend_tables_scratch_bytes(10, 3) == 4 * 17

    def extend(tables=P, stride=8, width=8, rows=P, block=16, batch=2, tokens=2, pool=4, free=P, blocks=5, slots=P, count=P):
        return lib.gqa_extend_tables_launch(tables, stride, width, P, pool, rows, P, free, count, blocks, block, 1, batch, tokens, P, P, P, slots, P, P,
                                            P, P, P, None)

    assert extend(stride=7) == SHAPE and extend(width=0) == SHAPE and extend(tokens=-1) == SHAPE and extend(rows=None, batch=5) == SHAPE
    assert extend(block=3) == BLOCK and extend(width=1 << 20, stride=1 << 20, block=1 << 16) == BLOCK
    assert extend(tables=None) == NULL and extend(free=None) == NULL and extend(slots=None) == NULL and extend(count=None) == NULL
    assert extend(slots=P + 4) == STRIDE and extend(tables=P + 2) == STRIDE

    def release(tables=P, rows=P, block=16, batch=2, width=8):
        return lib.gqa_release_blocks_launch(tables, 8, width, P, 4, rows, batch, P, P, 5, block, P, None)

    assert release(width=9) == SHAPE and release(block=0) == BLOCK and release(rows=None) == NULL and release(tables=P + 1) == STRIDE
    assert release(batch=0) == 0


def test_python_checks_without_a_device():
    dev = torch.device("cpu")
    kw = dict(batch=2, num_heads=4, num_kv_heads=2, seq_q=8, seq_kv=8, causal=True, scale=0.1, device=dev)
    z = torch.zeros(2, 8, dtype=torch.int32)
    assert check_score(0.0, None, None, None, **kw).softcap == 0.0 and check_score(2.0, None, None, None, **kw).softcap == 2.0
    for cap in (-1.0, float("nan"), 1e-6, 1e12, float("inf")):
        with pytest.raises(ValueError):
            check_score(cap, None, None, None, **kw)
    with pytest.raises(ValueError):
        check_score(1.0, None, None, None, **{**kw, "scale": -1.0})
    bad = [(None, torch.zeros(4, dtype=torch.float64), None, None), (None, torch.zeros(2, 4), None, None), (None, torch.zeros(8)[::2], None, None),
           (None, None, torch.zeros(2), None), (None, None, torch.zeros(3, dtype=torch.int32), None), (None, None, None, z),
           (None, None, None, DocumentSpans(z, z[:, :4])), (None, None, None, DocumentSpans(z, z.long())), (None, None, None, DocumentSpans(z.T.contiguous().T, z))]
    for args in bad:
        with pytest.raises(AssertionError):
            check_score(*args, **kw)
    with pytest.raises(AssertionError, match="causal"):
        check_score(None, None, z[:, 0].contiguous(), None, **{**kw, "causal": False})
    with pytest.raises(AssertionError, match="seq_q"):
        check_score(None, None, None, DocumentSpans(z, z), **{**kw, "seq_q": 9})
    for f in (lambda: document_spans(z), lambda: document_spans(z.long()), lambda: document_spans(z[0])):
        with pytest.raises(AssertionError):
            f()
    with pytest.raises(AssertionError):
        qk_norm_rope(torch.zeros(2, 4, 64, dtype=torch.bfloat16), None, z[0, :2], None)
    p = BlockPool(4, 16, 2, 32, device="cpu")
    with pytest.raises(AssertionError):
        extend_block_tables(p.block_tables, p.seq_lens, z[:, 0].contiguous(), p.free_blocks, p.free_count, 16, 2)


def test_rotary_table_values_and_checks():
    t = RotaryTable(64, 70000, base=1000.0, rotary_dim=32, device="cpu")
    pos = 69999
    ang = pos * 1000.0 ** (-torch.arange(0, 32, 2, dtype=torch.float64) / 32)
    assert torch.equal(t.table[pos, :, 0], ang.cos().float()) and torch.equal(t.table[pos, :, 1], ang.sin().float())
    for kw in (dict(head_dim=96), dict(rotary_dim=24), dict(rotary_dim=80), dict(max_positions=0), dict(axes=[0] * 31), dict(axes=[4] * 32),
               dict(axes=[-1] * 32), dict(inv_freq=[1.0]), dict(base=-1.0)):
        with pytest.raises(AssertionError):
            RotaryTable(**{**dict(head_dim=64, max_positions=4, device="cpu"), **kw})
    assert RotaryTable.sections((2, 1, 3)) == [0, 0, 1, 2, 2, 2]


def test_sizes_past_what_a_launch_spans(lib):
    def rope(write, tokens):
        r = _lib.Rope(table=P, max_positions=10, rotary_dim=128, positions=P, axes=1)
        t3 = _lib._i64x3(1024, 128, 1)
        if write:
            return lib.gqa_qk_norm_rope_write_launch(P, t3, P, t3, P, t3, P, t3, P, ST, P, ST, P, ctypes.byref(r),
                                                     tokens, 8, 2, 128, 16, 0, None)
        return lib.gqa_qk_norm_rope_launch(P, ST, P, ST, P, ST, P, ST, ctypes.byref(r), 1, 8, 2, tokens, 128, 0, None)

    assert rope(False, 1 << 26) == SHAPE and rope(True, 1 << 26) == SHAPE
    assert lib.gqa_document_spans_launch(P, 8, P, P, 1, (1 << 30) + 1, None) == SHAPE
    wide = 1 << 20
    assert lib.gqa_extend_tables_launch(P, wide, wide, P, 4096, P, P, P, P, 5, 16, 1, 2048, 2, P, P, P, P, P, P, P, P, P,
                                        None) == SHAPE


def test_scored_split_counts():
    def split(B, ml, Hq=32, Hkv=8, Sq=1, D=128, block=16):
        return scored_split(B, Hq, Hkv, Sq, ml, 256, block, D, True)

    assert split(1, 1) == (0, 1) and split(1, 64) == (0, 1) and split(1, 700) == (0, 11) and split(1, 3000) == (0, 32)
    assert split(1, 0)[0] == 0 and split(0, 700)[1] >= 1
    assert split(32, 8000)[0] == 64  # two workgroups a compute unit
    assert split(32, 8000, Sq=8)[0] in (0, 32)  # 32 rows: one
    assert scored_fine_split(1, 8, 33, 700, 256, 128) == (0, 0) and scored_fine_split(1, 8, 17, 700, 256, 64) == (0, 0)
    for B in (1, 3, 7, 40, 300):
        for ml in (1, 65, 777, 5000, 100000):
            slots, splits = split(B, ml)
            assert 1 <= splits <= _lib.GQA_MAX_SPLITS and 0 <= slots <= _lib.GQA_MAX_SPLITS


def test_scored_routes_of_few_rows():
    def route(B, Skv, Hkv=8, G=4, Sq=1, D=128):
        q, k = torch.empty(B, Hkv * G, Sq, D, device="meta"), torch.empty(B, Hkv, Skv, D, device="meta")
        return _scored_route(q, k, k, True, 0, False)

    _cu_count.cache_clear()
    try:
        with pytest.MonkeyPatch.context() as mp:
            mp.setattr("gqa_kernels.dispatch._cu_count", lambda dev: 256)
            assert (route(1, 700).kind, route(1, 700).splits) == ("split", 11)
            assert (route(8, 300, Hkv=2).kind, route(8, 300, Hkv=2).splits) == ("split", 5)
            for B, Skv in ((64, 300), (32, 64)):  # one launch: a slot a sequence
                assert (route(B, Skv).kind, route(B, Skv).splits) == ("flat", B)
            assert route(1, 3000, Sq=64).kind in ("single", "chunks", "short")
    finally:
        _cu_count.cache_clear()
