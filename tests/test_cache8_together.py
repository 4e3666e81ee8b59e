"""The paged cache in 8 bits as a program uses it: sequences that share a prefix, the layer with mixed batches, a captured decode loop with the block pool."""
import pytest
import torch

from cache8_reference import CODES, gather, power, values
from gqa_kernels import RotaryTable, qk_norm_rope
from gqa_kernels.cache8 import new_exponents
from gqa_kernels.paged import BlockPool, GQAPagedAttention, PagedAttentionMetadata, PagedKVCache, paged_attention, read_kv, write_kv
from ops_reference import attend64, check_attention, rope64

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def rand(*shape, dtype=BF, seed=0, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def ints(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


@pytest.mark.parametrize("layout", ["HND", "NHD"])
@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
def test_shared_prefix(layout, dtype):
    """Forks of a prefix that ends inside a page, each with its own tokens: read back and attended to; one's large tokens do not touch the other's page."""
    Hq, Hkv, D, bs = 8, 2, 128, 16
    cache = PagedKVCache(24, bs, Hkv, D, dtype=CODES, layout=layout)
    said = {}

    def add(ids, n, seed, scale=1.0):
        k, v = (rand(len(ids) * n, Hkv, D, dtype=dtype, seed=seed + s, scale=scale) for s in (0, 100))
        cache.append(ids, k, v)
        for i, s in enumerate(ids):
            old = said.get(s, (k[:0], v[:0]))
            said[s] = tuple(torch.cat([x, y[i * n:(i + 1) * n]]) for x, y in zip(old, (k, v)))

    cache.add_sequence("system")
    add(["system"], 41, 1)
    for s in ("a", "b"):
        cache.fork("system", s)
        said[s] = said["system"]
    before = cache.read("b", dtype)
    add(["a"], 3, 2, scale=300.0)
    assert all(torch.equal(x, y) for x, y in zip(cache.read("b", dtype), before))
    assert cache.exponents[0][cache.blocks("a")[2]].ge(cache.exponents[0][cache.blocks("b")[2]] + 5).all()
    add(["b", "system"], 20, 3)
    ids = ["a", "b", "system"]
    for s in ids:
        got = cache.read(s, dtype)
        for x, y, e in zip(got, said[s], cache.exponents):
            assert x.shape == y.shape == (cache.seq_len(s), Hkv, D) and x.dtype == dtype
            unit = power(e[torch.tensor(cache.blocks(s), device="cuda")]).repeat_interleave(bs, 0)[:x.shape[0], :, None]
            # Half a step of e4m3, and of the page's least one for each of up to three appends to it.
            assert ((x.double() - y.double()).abs() <= 2.0 ** -4 * y.double().abs() * (1 + 2.0 ** -4) + 3 * 2.0 ** -10 * unit).all()
    q = rand(3, Hq, 2, D, dtype=dtype, seed=9)
    o, lse = cache.attend(q, ids, return_lse=True)
    for i, s in enumerate(ids):
        k, v = (x.transpose(0, 1) for x in cache.read(s, dtype))
        check_attention(o[i], lse[i], attend64(q[i], k, v))
    cache.free("a")
    cache.add_sequence("c")  # takes a's pages, whose exponents are large
    said["c"] = (said["system"][0][:0],) * 2
    add(["c"], 7, 5, scale=1e-3)
    k, _ = cache.read("c", dtype)
    assert ((k.double() - said["c"][0].double()).abs() <= 2.0 ** -4 * said["c"][0].double().abs() + 2.0 ** -16 * 1e-2).all()


def test_read_of_a_16_bit_cache():
    cache = PagedKVCache(8, 16, 2, 64)
    cache.add_sequence(0)
    k, v = rand(37, 2, 64), rand(37, 2, 64, seed=1)
    cache.append([0], k, v)
    got = cache.read(0)
    assert torch.equal(got[0], k) and torch.equal(got[1], v)


@pytest.mark.parametrize("kw", [dict(), dict(softcap=25.0)], ids=["plain", "cap"])
def test_layer_with_a_mixed_batch(kw):
    """Prompts' chunks and decode steps together, twice over one cache, with norms and rotation and without."""
    Hq, Hkv, D, bs, B = 8, 2, 64, 16, 5
    w = (1 + rand(D, seed=7).float() * 0.1).to(BF)
    for normed in (False, True):
        rot = RotaryTable(D, 512)
        extra = dict(rotary=rot, q_norm_weight=w, k_norm_weight=w) if normed else {}
        layer = GQAPagedAttention(Hq, D, num_kv_heads=Hkv, **extra, **kw)
        kv = torch.zeros(2, 60, bs, Hkv, D, dtype=torch.uint8, device="cuda").view(CODES)
        exps = new_exponents(60, Hkv)
        perm = torch.randperm(60, generator=torch.Generator().manual_seed(1))[:50].view(B, 10)
        table, lens = perm.int().cuda(), [0] * B
        for step, ql in enumerate(([1, 90, 3, 33, 0], [4, 1, 1, 40, 70])):
            first, lens = lens, [a + b for a, b in zip(lens, ql)]
            pos = torch.cat([torch.arange(a, b) for a, b in zip(first, lens)])
            seq = torch.repeat_interleave(torch.arange(B), torch.tensor(ql))
            slots = (perm[seq, pos // bs] * bs + pos % bs).cuda()
            T = int(sum(ql))
            q, k, v = (rand(T, h * D, seed=10 * step + i) for i, h in enumerate((Hq, Hkv, Hkv)))
            md = PagedAttentionMetadata(slots, table, ints(lens), query_lens=ql, positions=pos.int().cuda())
            o = layer(q, k, v, kv, md, kv_exponents=exps).view(T, Hq, D)
            qr = q.view(T, Hq, D)
            if normed:
                want, tol = rope64(k.view(T, Hkv, D), w, 1e-6, pos.cuda()[None, :, None], rotary_dim=D, interleaved=False,
                                   inv_freq=10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D), axes=[0] * (D // 2))
                got, unit = values(kv[0], exps[0])[slots // bs, slots % bs], power(exps[0])[slots // bs][..., None]
                assert ((got - want).abs() <= 2.0 ** -4 * want.abs() + 2.0 ** -10 * unit + tol).all()
                qr, _ = qk_norm_rope(qr, None, pos.int().cuda(), rot, q_weight=w)
            at = 0
            for b, n in enumerate(ql):
                if n:
                    ks, vs = (gather(c, e, table[b], lens[b], BF) for c, e in zip(kv, exps))
                    want = attend64(qr[at:at + n].transpose(0, 1), ks, vs, **kw)
                    # (the layer's own queries may be a step of bf16 away from qk_norm_rope's: 2^-8 of each score's sum of products, doubled)
                    if normed:
                        slack = 2.0 ** -7 * float((qr[at:at + n].double().abs().amax((0, 1)) @ ks.double().abs().amax((0, 1)))) * D ** -0.5
                        want = (want[0], want[1], want[2] + slack * vs.double().abs().amax(), want[3] + slack)
                    check_attention(o[at:at + n].transpose(0, 1), None, want)
                at += n


def test_layer_with_equal_query_lengths():
    Hq, Hkv, D, bs, B = 8, 2, 128, 32, 3
    layer = GQAPagedAttention(Hq, D, num_kv_heads=Hkv)
    kv = torch.zeros(2, 9, bs, Hkv, D, dtype=torch.uint8, device="cuda").view(CODES)
    exps = new_exponents(9, Hkv)
    table = ints([[0, 1, 2], [3, 4, 5], [6, 7, 8]])
    for n, first in ((40, 0), (1, 40), (2, 41)):
        pos = torch.arange(first, first + n).repeat(B)
        seq = torch.arange(B).repeat_interleave(n)
        slots = (table.cpu().long()[seq, pos // bs] * bs + pos % bs).cuda()
        q, k, v = (rand(B * n, h * D, seed=first + i) for i, h in enumerate((Hq, Hkv, Hkv)))
        out = torch.empty_like(q)
        o = layer(q, k, v, kv, PagedAttentionMetadata(slots, table, ints([first + n] * B), query_len=n), output=out, kv_exponents=exps)
        assert o is out
        for b in range(B):
            ks, vs = (gather(c, e, table[b], first + n, BF) for c, e in zip(kv, exps))
            check_attention(o.view(B, n, Hq, D)[b].transpose(0, 1), None, attend64(q.view(B, n, Hq, D)[b].transpose(0, 1), ks, vs))


def test_decode_loop_in_a_graph():
    """Tables, cache write and attention of one token a request, captured once and replayed; requests that end hand their pages to new ones."""
    Hq, Hkv, D, bs, B, steps = 8, 2, 128, 16, 4, 40
    p = BlockPool(12, bs, 6, 64)
    kv = torch.zeros(2, 12, bs, Hkv, D, dtype=torch.uint8, device="cuda").view(CODES)
    exps = new_exponents(12, Hkv)
    rows, new = ints([3, 0, -1, 4]), ints([1, 1, 0, 1])
    qkv = torch.zeros(3, Hq + 2 * Hkv, D, dtype=BF, device="cuda")

    def step():
        s = p.step(new, 3, rows=rows)
        q, k, v = qkv.split([Hq, Hkv, Hkv], 1)
        write_kv(k, v, kv[0], kv[1], s.slot_mapping, k_exponents=exps[0], v_exponents=exps[1])
        return paged_attention(q, kv[0], kv[1], s.block_tables, s.seq_lens, True, query_start=s.query_start, query_lens=s.query_lens, max_query_len=1,
                               k_exponents=exps[0], v_exponents=exps[1]), s

    step()
    p.release(rows)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, s = step()
    said = []
    for t in range(steps):
        x = rand(3, Hq + 2 * Hkv, D, seed=t, scale=1.0 + t % 7)
        qkv.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        said.append(x)
        n = len(said)
        assert s.seq_lens.tolist() == [n, n, 0, n] and s.refused.item() == 0
        every = torch.stack(said, 1)  # (3, n, heads, D)
        for i, b in enumerate((0, 1, 3)):
            ks, vs = (gather(c, e, s.block_tables[b], n, BF) for c, e in zip(kv, exps))
            pages = s.block_tables[b][:-(-n // bs)].long()
            for got, mine, e in ((ks, every[i, :, Hq:Hq + Hkv], exps[0]), (vs, every[i, :, Hq + Hkv:], exps[1])):
                unit = power(e[pages]).repeat_interleave(bs, 0)[:n, :, None]
                assert ((got.transpose(0, 1).double() - mine.double()).abs() <= 2.0 ** -4 * mine.double().abs() * (1 + 2.0 ** -4) + bs * 2.0 ** -10 * unit).all()
            check_attention(out[i].unsqueeze(1), None, attend64(x[i, :Hq].unsqueeze(1), ks, vs))
        if t == 24:
            p.release(rows)
            said.clear()
    k, v = read_kv(kv[0], kv[1], s.slot_mapping, exps[0], exps[1])
    assert torch.equal(k, values(kv[0], exps[0])[s.slot_mapping // bs, s.slot_mapping % bs].to(BF)) and v.shape == (3, Hkv, D)
