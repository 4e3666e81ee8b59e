"""Norms of queries and keys with the rotation of positions, against float64; with and without the paged cache write."""
import pytest
import torch

from gqa_kernels import RotaryTable, qk_norm_rope, qk_norm_rope_write
from gqa_kernels.paged import GQAPagedAttention, PagedAttentionMetadata, write_kv
from ops_reference import rope64

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def rand(*shape, dtype=BF, seed=0, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def inv_freq(R, base=10000.0):
    return base ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)


def expect(x, w, pos, table, inv, eps=1e-6):
    """x (..., D), pos (A, ...) with a place for the heads."""
    return rope64(x, w, eps, pos, rotary_dim=table.rotary_dim, interleaved=table.interleaved, inv_freq=inv,
                  axes=table.axes or [0] * (table.rotary_dim // 2))


def close(got, want):
    y, tol = want
    assert torch.isfinite(got.float()).all()
    assert ((got.double() - y).abs() <= tol).all(), float(((got.double() - y).abs() / tol).max())


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
@pytest.mark.parametrize("B,S,Hq,Hkv,D,R,inter", [
    (1, 1, 1, 1, 64, 64, False), (1, 1, 32, 8, 128, 128, False), (2, 7, 28, 4, 128, 64, False), (3, 33, 8, 8, 64, 32, True), (1, 1000, 16, 4, 128, 128, True),
    (2, 257, 6, 2, 128, 16, False), (1, 65, 40, 8, 64, 48, False), (2, 130, 64, 8, 128, 112, True),
])
@pytest.mark.parametrize("norm", [True, False])
def test_heads_first(B, S, Hq, Hkv, D, R, inter, norm, dtype):
    qkv = rand(B, S, (Hq + Hkv) * D, dtype=dtype, scale=2.0)
    q, k = (t.unflatten(-1, (-1, D)).transpose(1, 2) for t in qkv.split([Hq * D, Hkv * D], -1))
    table = RotaryTable(D, 5000, rotary_dim=R, interleaved=inter)
    pos = torch.randint(0, 5000, (B, S), generator=torch.Generator().manual_seed(1), dtype=torch.int64).cuda()
    wq, wk = (rand(D, dtype=dtype, seed=s) + 1 if norm else None for s in (2, 3))
    before = qkv.clone()
    qo, ko = qk_norm_rope(q, k, pos, table, q_weight=wq, k_weight=wk)
    assert qo.shape == q.shape and torch.equal(qkv, before)
    close(qo, expect(q, wq, pos[None, :, None], table, inv_freq(R)))
    close(ko, expect(k, wk, pos[None, :, None], table, inv_freq(R)))
    q2, k2 = qk_norm_rope(q, k, pos.int(), table, q_weight=wq, k_weight=wk, q_out=q, k_out=k)  # in place, int32 positions
    assert q2 is q and torch.equal(q, qo) and torch.equal(k, ko)


def test_far_positions_and_given_frequencies():
    inv = inv_freq(128, 500000.0) * 0.37
    table = RotaryTable(128, 131072, inv_freq=inv.tolist())
    pos = torch.tensor([0, 1, 65535, 65536, 131071], dtype=torch.int32).cuda()
    q = rand(5, 4, 128)
    qo, ko = qk_norm_rope(q, None, pos, table)
    assert ko is None
    close(qo, expect(q, None, pos[None, :, None], table, inv))


def test_several_axes():
    axes = RotaryTable.sections((16, 24, 24))
    assert len(axes) == 64 and axes.count(1) == 24
    for ax in (axes, [i % 3 for i in range(64)], [3] * 64):
        for inter in (False, True):
            table = RotaryTable(128, 3000, axes=ax, interleaved=inter)
            A = max(ax) + 1
            pos = torch.randint(0, 3000, (A, 2, 41), generator=torch.Generator().manual_seed(3), dtype=torch.int32).cuda()
            q, k = rand(2, 8, 41, 128), rand(2, 2, 41, 128, seed=1)
            w = rand(128, seed=5).float() + 1
            qo, ko = qk_norm_rope(q, k, pos, table, q_weight=w, k_weight=w, eps=1e-5)
            close(qo, expect(q, w, pos[:, :, None], table, inv_freq(128), 1e-5))
            close(ko, expect(k, w, pos[:, :, None], table, inv_freq(128), 1e-5))


def test_norm_alone_and_one_weight():
    q, k = rand(9, 8, 128, scale=5.0), rand(9, 2, 128, seed=1)
    w = rand(128, seed=2)
    table = RotaryTable(128, 16)
    qo, ko = qk_norm_rope(q, k, None, None, q_weight=w, eps=1e-3)
    y = q.double()
    close(qo, rope64(q, w, 1e-3, None, rotary_dim=128, interleaved=False, inv_freq=None, axes=None))
    assert torch.equal(ko, k)
    zero = torch.zeros_like(q)
    qo, _ = qk_norm_rope(zero, None, torch.zeros(9, dtype=torch.int32).cuda(), table, q_weight=w)
    assert (qo == 0).all() and y is not None


def test_positions_outside_the_table():
    table = RotaryTable(64, 10)
    q = rand(4, 2, 64)
    pos = torch.tensor([-1, 0, 9, 10], dtype=torch.int64).cuda()
    qo, _ = qk_norm_rope(q, None, pos, table)
    assert torch.equal(qo[0], q[0]) and torch.equal(qo[1], q[1])  # negative: position 0
    assert torch.isfinite(qo[2].float()).all() and torch.isnan(qo[3].float()).all()
    pos = torch.tensor([-2 ** 63, 2 ** 63 - 1, 2 ** 32, 0], dtype=torch.int64).cuda()
    qo, _ = qk_norm_rope(q, None, pos, table)
    assert torch.equal(qo[0], q[0]) and torch.isnan(qo[1:3].float()).all()


def test_copies_of_unaligned_rows():
    table = RotaryTable(128, 100)
    pos = torch.arange(30, dtype=torch.int32).cuda()
    q = rand(30, 8, 129)[..., 1:]
    qo, _ = qk_norm_rope(q, None, pos, table)
    close(qo, expect(q, None, pos[None, :, None], table, inv_freq(128)))
    w = rand(129)[1:]
    qo, _ = qk_norm_rope(q, None, pos, table, q_weight=w)
    close(qo, expect(q, w, pos[None, :, None], table, inv_freq(128)))


@pytest.mark.parametrize("T,Hq,Hkv,D,block,layout,dtype", [
    (1, 32, 8, 128, 16, "NHD", BF), (64, 32, 8, 128, 64, "HND", BF), (301, 28, 4, 64, 16, "NHD", FP), (1000, 6, 6, 128, 1, "HND", FP), (5, 64, 2, 64, 256, "NHD", BF),
])
def test_write(T, Hq, Hkv, D, block, layout, dtype):
    blocks = -(-T // block) + 3
    shape = (2, blocks, block, Hkv, D) if layout == "NHD" else (2, blocks, Hkv, block, D)
    kv = rand(*shape, dtype=dtype, seed=9)
    kv = kv if layout == "NHD" else kv.transpose(2, 3)
    qkv = rand(T, (Hq + 2 * Hkv) * D, dtype=dtype)
    q, k, v = (t.unflatten(-1, (-1, D)) for t in qkv.split([Hq * D, Hkv * D, Hkv * D], -1))
    g = torch.Generator().manual_seed(4)
    slots = torch.randperm(blocks * block, generator=g)[:T].cuda()
    slots[::7] = -1 - slots[::7]  # padding
    pos = torch.randint(0, 4000, (T,), generator=g, dtype=torch.int32).cuda()
    table = RotaryTable(D, 4000, base=500000.0)
    wq, wk = rand(D, dtype=dtype, seed=2) + 1, rand(D, dtype=dtype, seed=3) + 1
    old = kv.clone()
    qo = qk_norm_rope_write(q, k, v, pos, table, kv[0], kv[1], slots, q_weight=wq, k_weight=wk)
    # The same rows as the two-step form, bit for bit; nothing else in the caches changes.
    q2, k2 = qk_norm_rope(q, k, pos, table, q_weight=wq, k_weight=wk)
    want = old.clone()
    write_kv(k2, v, want[0], want[1], slots)
    assert torch.equal(qo, q2) and torch.equal(kv, want)
    close(qo, expect(q, wq, pos[None, :, None], table, inv_freq(D, 500000.0)))
    close(k2, expect(k, wk, pos[None, :, None], table, inv_freq(D, 500000.0)))


def test_nothing_to_do():
    table = RotaryTable(128, 10)
    q = rand(0, 8, 128)
    qo, _ = qk_norm_rope(q, None, torch.empty(0, dtype=torch.int32).cuda(), table)
    assert qo.shape == q.shape


def test_captured():
    table = RotaryTable(128, 1000)
    q, k = rand(33, 8, 128), rand(33, 2, 128, seed=1)
    pos = torch.arange(33, dtype=torch.int32).cuda()
    w = rand(128, seed=2)
    qk_norm_rope(q, k, pos, table, q_weight=w, k_weight=w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qo, ko = qk_norm_rope(q, k, pos, table, q_weight=w, k_weight=w)
    for i in range(3):
        q.copy_(rand(33, 8, 128, seed=10 + i))
        pos.add_(7)
        want = qk_norm_rope(q, k, pos, table, q_weight=w, k_weight=w)
        qo.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(qo, want[0]) and torch.equal(ko, want[1])


def test_refusals():
    table = RotaryTable(128, 100)
    q, k, pos = rand(9, 8, 128), rand(9, 2, 128), torch.arange(9, dtype=torch.int32).cuda()
    bad = [lambda: qk_norm_rope(q, k, pos, None), lambda: qk_norm_rope(q, k, pos.float(), table), lambda: qk_norm_rope(q, k, pos[:8], table),
           lambda: qk_norm_rope(q, k, pos, RotaryTable(64, 100)), lambda: qk_norm_rope(q.float(), k.float(), pos, table),
           lambda: qk_norm_rope(q, k[:5], pos, table), lambda: qk_norm_rope(q, k, pos, table, q_weight=rand(64)),
           lambda: qk_norm_rope(q, k, pos, table, q_weight=rand(128), k_weight=rand(128).float()),
           lambda: qk_norm_rope(q, k, pos, table, q_weight=rand(128), eps=-1.0), lambda: qk_norm_rope(q, k, pos, table, q_out=k),
           lambda: qk_norm_rope(q, None, pos, table, k_weight=rand(128)), lambda: qk_norm_rope(q, k.half(), pos, table)]
    for f in bad:
        with pytest.raises(AssertionError):
            f()
    with pytest.raises(NotImplementedError):
        qk_norm_rope(q, k, pos, table, q_weight=rand(128).requires_grad_())
    with torch.no_grad():
        qk_norm_rope(q, k, pos, table, q_weight=rand(128).requires_grad_())


@pytest.mark.parametrize("qlens", [[1, 1, 1], [40, 1, 130]])
def test_layer_norms_rotates_and_stores(qlens):
    """GQAPagedAttention with a rotation: as the steps made one by one."""
    Hq, Hkv, D, bs = 8, 2, 128, 16
    cached = [100, 33, 16]
    lens = [a + b for a, b in zip(cached, qlens)]
    W = max(-(-n // bs) for n in lens)
    table = torch.arange(3 * W, dtype=torch.int32).view(3, W).flip(0).contiguous().cuda()
    kv = rand(2, 3 * W, bs, Hkv, D, seed=7)
    T = sum(qlens)
    q, k, v = rand(T, Hq * D), rand(T, Hkv * D, seed=1), rand(T, Hkv * D, seed=2)
    pos = torch.cat([torch.arange(c, n) for c, n in zip(cached, lens)]).to(torch.int32).cuda()
    seq = torch.cat([torch.full((n,), b) for b, n in enumerate(qlens)]).cuda()
    slots = table[seq, pos.long() // bs].long() * bs + pos.long() % bs
    rot, w = RotaryTable(D, 500), rand(D, seed=3)
    md = PagedAttentionMetadata(slots, table, torch.tensor(lens, dtype=torch.int32).cuda(), query_lens=qlens, positions=pos)
    plain, kv2 = GQAPagedAttention(Hq, D, num_kv_heads=Hkv), kv.clone()
    q2, k2 = qk_norm_rope(q.view(T, Hq, D), k.view(T, Hkv, D), pos, rot, q_weight=w, k_weight=w)
    want = plain(q2.reshape(T, -1), k2.reshape(T, -1), v, kv2, md)
    layer = GQAPagedAttention(Hq, D, num_kv_heads=Hkv, rotary=rot, q_norm_weight=w, k_norm_weight=w)
    before = q.clone()
    got = layer(q, k, v, kv, md)
    assert torch.equal(got, want) and torch.equal(kv, kv2) and torch.equal(q, before)
    assert torch.equal(layer(q, None, None, kv, md), want)  # (nothing to store: queries alone)
