"""Block tables and slots built on the device, against a plain loop; the pool that a captured decode loop runs on."""
import pytest
import torch

from gqa_kernels import RotaryTable, qk_norm_rope
from gqa_kernels.paged import (BlockPool, GQAPagedAttention, PagedAttentionMetadata, extend_block_tables, paged_attention, release_blocks)
from ops_reference import attend64, check_attention, rope64

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def plain_step(tables, lens, new, free, block, T, rows):
    """The step on lists: (outputs, tables, lens, free)."""
    tables, lens, free = [list(r) for r in tables], list(lens), list(free)
    W, seen, start, blocks = len(tables[0]), set(), 0, 0
    have = len(free)
    out = {"seq_lens": [], "query_start": [], "query_lens": [], "slots": [-1] * T, "pos": [0] * T, "refused": 0}
    taken, after = 0, list(lens)
    batch = []
    for b, n in enumerate(new):
        r, n = rows[b], max(n, 0)
        ok = 0 <= r < len(tables) and r not in seen
        mine = ok
        old = lens[r] if ok else 0
        if ok:
            seen.add(r)
        out["query_start"].append(start)
        ok = ok and old + n <= W * block and start + n <= T
        need = -(-(old + n) // block) - -(-old // block) if ok else 0
        blocks += need
        ok = ok and (need == 0 or blocks <= have)
        if ok:
            for i in range(need):
                tables[r][-(-old // block) + i] = free[have - 1 - (blocks - need) - i]
            taken += need
            for j in range(n):
                out["pos"][start + j] = old + j
                out["slots"][start + j] = tables[r][(old + j) // block] * block + (old + j) % block
            after[r] = old + n
        elif r >= 0:
            out["refused"] += 1
        out["seq_lens"].append(old + n if ok else old)
        out["query_lens"].append(n if ok else 0)
        pages = -(-out["seq_lens"][-1] // block) if mine else 0
        batch.append((tables[r][:pages] if pages else []) + [0] * (W - pages))
        start += n
    out["tables"] = batch
    return out, tables, after, free[:have - taken]


def compare(tables, lens, new, free, block, T, rows=None, spare=3):
    want, wt, wl, wf = plain_step(tables, lens, new, free, block, T, list(range(len(new))) if rows is None else rows)
    free_dev = ints(free + [0] * spare)
    for update in (False, True):
        td, ld, cd = ints(tables), ints(lens), ints([len(free)])
        r = extend_block_tables(td, ld, ints(new), free_dev, cd, block, T, rows=None if rows is None else ints(rows), update=update)
        got = {"seq_lens": r.seq_lens, "query_start": r.query_start, "query_lens": r.query_lens, "slots": r.slot_mapping, "pos": r.positions,
               "tables": r.block_tables}
        for name, x in got.items():
            assert x.tolist() == want[name], name
        assert r.refused.item() == want["refused"] and r.free_count.item() == len(wf)
        assert td.tolist() == wt and ld.tolist() == (wl if update else lens) and cd.item() == (len(wf) if update else len(free))


def pool(rows, width, block, lens, seed=0, spare=50):
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // block) for n in lens]
    order = torch.randperm(sum(need) + spare, generator=g).tolist()
    tables, at = [], 0
    for n in need:
        tables.append(order[at:at + n] + [0] * (width - n))
        at += n
    return tables, order[at:]


@pytest.mark.parametrize("block", [1, 16, 64])
def test_steps(block):
    lens = [0, 5, 16, 17, 31, 32, 63, 64]
    tables, free = pool(8, 100, block, lens, spare=300)
    compare(tables, lens, [1] * 8, free, block, 8)
    compare(tables, lens, [3, 0, 20, 1, 33, 32, 1, 0], free, block, 100)
    compare(tables, lens, [2, 7, 1], free, block, 10, rows=[6, 0, 3])
    compare(tables, lens, [0, 0], free, block, 0, rows=[1, 2])


def test_refused_requests():
    block = 16
    lens = [10, 16, 64, 0, 30]
    tables, free = pool(5, 5, block, lens, spare=3)
    compare(tables, lens, [1, 17, 17, 1, 40], free, block, 200)  # width, then the free list
    compare(tables, lens, [1, 33, 1, 6, 2], free, block, 200)  # the free list ends; requests that need no page go on
    compare(tables, lens, [5, 5, 5, 5, 5], free, block, 12)  # num_tokens
    compare(tables, lens, [1, 2, 3, 4, 5, 6], free, block, 40, rows=[2, -1, 2, 9, 0, -7])  # twice, empty, outside
    compare(tables, lens, [-3, 1, -2 ** 31], free, block, 40, rows=[0, 1, 2])  # negative counts are none
    compare(tables, lens, [1, 1, 1], [], block, 3, rows=[0, 1, 3])


def test_counts_beyond_32_bits():
    tables, free = pool(3, 4, 16, [0, 0, 0], spare=9)
    r = extend_block_tables(ints(tables), ints([0, 0, 0]), ints([2 ** 31 - 1, 2 ** 31 - 1, 3]), ints(free), ints([9]), 16, 50)
    assert r.refused.item() == 3 and r.query_lens.tolist() == [0, 0, 0] and (r.slot_mapping == -1).all()
    # Lengths and counts that no pool has are taken into range.
    r = extend_block_tables(ints(tables), ints([-5, 2 ** 31 - 1, 3]), ints([1, 1, 1]), ints(free), ints([2 ** 31 - 1]), 16, 3)
    assert r.seq_lens.tolist() == [1, 64, 4] and r.refused.item() == 1


@pytest.mark.parametrize("B", [1, 63, 1023, 1024, 1025, 3000])
def test_many_requests(B):
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 200, (B + 7,), generator=g).tolist()
    tables, free = pool(B + 7, 16, 16, lens, spare=B)
    rows = torch.randperm(B + 7, generator=g)[:B].tolist()
    new = torch.randint(0, 9, (B,), generator=g).tolist()
    compare(tables, lens, new, free, 16, sum(new) + 5, rows=rows)


def test_one_long_prompt():
    tables, free = pool(2, 1300, 16, [100, 7], spare=1300)
    compare(tables, [100, 7], [0, 20000], free, 16, 20000)


def test_pool_gives_and_takes():
    p = BlockPool(40, 16, 6, 200)
    used = lambda: {b for r, n in zip(p.block_tables.tolist(), p.seq_lens.tolist()) for b in r[:-(-n // 16)]}  # noqa: E731
    p.step(ints([100, 50, 1]), 160, rows=ints([0, 2, 5]))
    assert p.seq_lens.tolist() == [100, 0, 50, 0, 0, 1] and len(used()) == 12 and p.free_count.item() == 28
    r = p.step(ints([13, 1]), 14, rows=ints([0, 5]))
    assert r.seq_lens.tolist() == [113, 2] and p.free_count.item() == 27
    p.release(ints([0, 9, 0, -1]))
    assert p.seq_lens.tolist() == [0, 0, 50, 0, 0, 2] and p.free_count.item() == 35
    everything = used() | set(p.free_blocks[:35].tolist())
    assert everything == set(range(40))
    r = p.step(ints([200, 200, 200]), 600, rows=ints([0, 1, 3]))
    assert r.refused.item() == 1 and p.free_count.item() == 35 - 26
    p.release(ints([0, 1, 2, 3, 4, 5]))
    assert p.free_count.item() == 40 and set(p.free_blocks.tolist()) == set(range(40))


def test_release_never_overfills():
    tables, lens = ints([[1, 2, 3]]), ints([48])
    free, count = ints([7, 8, 9, 0]), ints([3])
    release_blocks(tables, lens, ints([0]), free, count, 16)
    assert count.item() == 4 and free.tolist() == [7, 8, 9, 1] and lens.item() == 0


def test_nothing_and_refusals():
    p = BlockPool(4, 16, 2, 32)
    r = extend_block_tables(p.block_tables, p.seq_lens, ints([]), p.free_blocks, p.free_count, 16, 3)
    assert r.slot_mapping.tolist() == [-1, -1, -1] and r.free_count.item() == 4
    a = (p.block_tables, p.seq_lens, ints([1, 1]), p.free_blocks, p.free_count)
    for change in ({0: p.block_tables.long()}, {1: p.seq_lens[:1]}, {2: ints([1, 1]).long()}, {2: ints([1, 1, 1])}, {3: p.free_blocks.float()},
                   {4: ints([1, 2])}, {2: torch.ones(2, dtype=torch.int32)}):
        x = list(a)
        for i, t in change.items():
            x[i] = t
        with pytest.raises(AssertionError):
            extend_block_tables(*x, 16, 2)
    for kw in (dict(block_size=12, num_tokens=2), dict(block_size=16, num_tokens=-1)):
        with pytest.raises(AssertionError):
            extend_block_tables(*a, **kw)
    with pytest.raises(AssertionError):
        extend_block_tables(*a, 16, 2, rows=ints([0]))


def test_decode_loop_in_a_graph():
    """Tables, norms, rotation, cache write and capped attention of one token a request, captured once and replayed: every step against
    float64, with an empty place in the batch."""
    Hq, Hkv, D, bs, B, steps = 8, 2, 64, 16, 4, 20
    p = BlockPool(30, bs, 5, 128)
    kv = torch.zeros(2, 30, bs, Hkv, D, dtype=torch.bfloat16, device="cuda")
    rot = RotaryTable(D, 128)
    w = (1 + torch.rand(D, generator=torch.Generator().manual_seed(1))).to(torch.bfloat16).cuda()
    layer = GQAPagedAttention(Hq, D, num_kv_heads=Hkv, softcap=20.0, rotary=rot, q_norm_weight=w, k_norm_weight=w)
    rows, new = ints([3, 0, -1, 4]), ints([1, 1, 0, 1])
    qkv = torch.zeros(B, (Hq + 2 * Hkv) * D, dtype=torch.bfloat16, device="cuda")

    def step():
        s = p.step(new, 3, rows=rows)
        q, k, v = qkv[:3].split([Hq * D, Hkv * D, Hkv * D], -1)
        rotated = layer._norm_rope(q, k, v, kv[0], kv[1], PagedAttentionMetadata(s.slot_mapping, s.block_tables, s.seq_lens, positions=s.positions))
        return paged_attention(rotated.view(3, Hq, D), kv[0], kv[1], s.block_tables, s.seq_lens, True, query_start=s.query_start,
                               query_lens=s.query_lens, max_query_len=1, softcap=20.0), s

    step()
    p.release(rows)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, s = step()
    g = torch.Generator().manual_seed(2)
    said = []
    inv = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    for t in range(steps):
        x = torch.randn(B, (Hq + 2 * Hkv) * D, generator=g).to(torch.bfloat16).cuda()
        qkv.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        said.append(x[:3])
        assert s.seq_lens.tolist() == [t + 1, t + 1, 0, t + 1] and s.refused.item() == 0
        every = torch.stack(said, 1)  # (3, t + 1, ...)
        pos = torch.arange(t + 1, device="cuda", dtype=torch.int32)
        q, k, v = (y.unflatten(-1, (-1, D)) for y in every.split([Hq * D, Hkv * D, Hkv * D], -1))
        for i, b in enumerate((0, 1, 3)):
            at = s.block_tables[b][pos.long() // bs].long(), pos.long() % bs
            want, tol = rope64(k[i], w, 1e-6, pos[None, :, None], rotary_dim=D, interleaved=False, inv_freq=inv, axes=[0] * (D // 2))
            assert ((kv[0][at].double() - want).abs() <= tol).all() and torch.equal(kv[1][at], v[i])
            qr, _ = qk_norm_rope(q[i, -1:], None, pos[-1:], rot, q_weight=w)
            want = attend64(qr.transpose(0, 1), kv[0][at].transpose(0, 1), kv[1][at].transpose(0, 1), softcap=20.0)
            check_attention(out[i].unsqueeze(1), None, want)


@pytest.mark.parametrize("B,width,new", [(1, 600, 1), (31, 500, 3), (32, 512, 128), (32, 513, 1), (33, 100, 1), (32, 40, 129)])
def test_sizes_around_one_workgroup(B, width, new):
    """Steps on both sides of the form that moves the pool on in its only workgroup: three in a row, against the host."""
    p = BlockPool(B * 30 + 7, 16, B + 3, width * 16)
    rows = ints([(5 * b + 2) % (B + 3) for b in range(B)] if (B + 3) % 5 else list(range(B)))
    for step in range(3):
        table, lens = p.block_tables.tolist(), p.seq_lens.tolist()
        free = p.free_blocks[:int(p.free_count)].tolist()
        r = p.step(ints([new] * B), B * new, rows=rows)
        slots, at = [], 0
        for b, row in enumerate(rows.tolist()):
            first, lens[row] = lens[row], lens[row] + new
            for page in range(-(-first // 16), -(-lens[row] // 16)):
                table[row][page] = free.pop()
            slots += [table[row][i // 16] * 16 + i % 16 for i in range(first, lens[row])]
        assert p.block_tables.tolist() == table and p.seq_lens.tolist() == lens
        assert int(p.free_count) == len(free) == int(r.free_count) and int(r.refused) == 0
        assert r.slot_mapping.tolist() == slots and r.seq_lens.tolist() == [lens[i] for i in rows.tolist()]
        assert r.block_tables.tolist() == [table[i][:-(-lens[i] // 16)] + [0] * (width - -(-lens[i] // 16)) for i in rows.tolist()]
