"""The operators between a projection and the attention output: attention whose scores are changed (capped, biased by distance, with document and
prefix masks), over contiguous K/V and over a paged cache; per-head norms of queries and keys with the rotation of positions, with and without the
paged cache write; block tables and slots built on the device from request lengths.

listed() and draw() give the cases, prepare() what a program holds before the call, run() one pass: the plain form (elementary torch operations in
float32, angles in float64, rounded once at the end), or, with `own`, the calls of gqa_kernels.  exact() is the definition in float64."""
import math
import sys
from pathlib import Path

import torch

own = False

PACKAGE = str(Path(__file__).resolve().parent.parent / "gqa-flash-attn-rtx3060_amd")
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
NEG = -math.inf


def _own():
    if PACKAGE not in sys.path:
        sys.path.insert(0, PACKAGE)
    import gqa_kernels

    return gqa_kernels


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _attn(**kw):
    """Attention over contiguous (B, H, S, D) tensors.  cap: 0 none; alibi: distance bias; prefix: the longest of the batch's prefixes (0: no
    prefix mask); docs: documents packed in a row (0: no document mask); pad: tokens behind the last document."""
    d = dict(op="attn", dtype="bf16", B=1, Hq=32, Hkv=8, Sq=1024, Skv=1024, D=128, causal=True, cap=0.0, alibi=False, prefix=0, docs=0, pad=0)
    d.update(kw)
    return d


def _paged(**kw):
    """Attention of Sq new tokens of each of B sequences over a paged cache; lengths spread from low to high."""
    d = dict(op="paged", dtype="bf16", B=16, Hq=32, Hkv=8, Sq=1, low=100, high=8000, D=128, block=16, cap=0.0, alibi=False, prefix=0)
    d.update(kw)
    return d


def _rope(**kw):
    """Norms of q and k with the rotation: B x S tokens as slices of one projection's output.  axes: position axes (1, or 3 for images and
    video); pairs: "half" or "interleaved"; write: K and V go to a paged cache."""
    d = dict(op="rope", dtype="bf16", B=1, S=4096, Hq=32, Hkv=8, D=128, rotary=128, pairs="half", axes=1, norm=True, base=500000.0, far=131072,
             write=False, block=16)
    d.update(kw)
    return d


def _tables(**kw):
    """Block tables and slots of a step: B requests of low to high cached keys get new tokens (1 each, or up to `new`)."""
    d = dict(op="tables", B=256, low=1, high=8000, new=1, block=16, pool=512, pad=0)
    d.update(kw)
    return d


def listed():
    return [
        # The prompt of a model that caps its attention logits, at the 8K length of this repository's prefill benchmark.
        _attn(name="cap_prompt_8k", Sq=8192, Skv=8192, cap=50.0),
        # Pretraining-style packing (scoring, embedding, long-context evaluation): documents of unequal lengths in each row, a padded end.
        _attn(name="documents_2x8k", B=2, Hq=32, Hkv=8, Sq=8192, Skv=8192, docs=13, pad=237),
        # A chunk of a prompt over the keys before it, with the distance bias, at head_dim 64.
        _attn(name="alibi_chunk_d64", dtype="fp16", B=2, Hq=16, Hkv=4, Sq=500, Skv=6001, D=64, alibi=True),
        # Short prompts with an image or instruction prefix that attends to itself in both directions.
        _attn(name="prefix_prompts", B=4, Sq=777, Skv=777, prefix=300, cap=30.0),
        # A serving batch's decode step with capped scores, lengths unequal, 16-key pages.
        _paged(name="cap_decode_b32", B=32, cap=50.0),
        # One user's next token with the distance bias: the smallest call, latency alone.
        _paged(name="alibi_token", B=1, low=700, high=700, alibi=True, block=64),
        # A chunk of new tokens of four requests over their cached prefixes.
        _paged(name="cap_chunk_4x256", B=4, Sq=256, low=2000, high=9000, cap=30.0),
        # A decode step's queries and keys: normed, rotated, the keys and values written to their pages.
        _rope(name="rope_write_decode", S=64, write=True),
        # A long prompt's.
        _rope(name="rope_prompt_16k", S=16384),
        # A prompt with images: three position axes, into the cache.
        _rope(name="rope_axes_write", S=5003, axes=3, write=True, base=1000000.0),
        # A decode step of a large batch.
        _tables(name="tables_decode_256"),
        # Prompts of a batch: many tokens of few requests.
        _tables(name="tables_prompts", B=48, low=1, high=500, new=2048, pool=96),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "paged", "paged", "rope", "tables"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    Hq, Hkv = rng.choice([(32, 8), (32, 8), (16, 4), (64, 8), (8, 8), (12, 4), (28, 4)])
    D = rng.choice([64, 128, 128])
    cap = rng.choice([0.0, 15.0, 30.0, 50.0])
    if op == "attn":
        B = rng.choice([1, 1, 2, 3, 4, 8])
        Skv = _log(rng, 16, 8192)
        Sq = Skv if rng.random() < 0.6 else _log(rng, 1, Skv)
        while B * Hq * Sq * Skv > 32 * 8192 * 8192:
            B, Sq, Skv = max(1, B // 2), max(1, Sq // 2), Skv if B > 1 else max(Sq, Skv // 2)
        kind = rng.choice(["cap", "alibi", "prefix", "docs", "docs"])
        causal = kind == "prefix" or rng.random() < 0.8
        pad = rng.randint(0, min(Skv // 8, Sq // 2)) if kind == "docs" and rng.random() < 0.5 else 0
        return _attn(dtype=dtype, B=B, Hq=Hq, Hkv=Hkv, Sq=Sq, Skv=Skv, D=D, causal=causal, cap=cap if kind != "cap" else cap or 50.0,
                     alibi=kind == "alibi", prefix=rng.randint(1, Skv) if kind == "prefix" else 0,
                     docs=_log(rng, 1, max(2, (Skv - pad) // 16)) if kind == "docs" else 0, pad=pad)
    if op == "paged":
        B = _log(rng, 1, 48)
        high = _log(rng, 64, 131072 // B)
        low = rng.randint(max(1, high // 20), high)
        Sq = rng.choice([1, 1, 1, 4, rng.randint(2, 8), _log(rng, 16, 512)])
        Sq = max(1, min(Sq, low, 32 * 8192 * 8192 // (B * Hq * high)))
        kind = rng.choice(["cap", "alibi", "prefix"])
        return _paged(dtype=dtype, B=B, Hq=Hq, Hkv=Hkv, Sq=Sq, low=low, high=high, D=D, block=rng.choice([16, 16, 32, 64, 128]),
                      cap=cap if kind != "cap" else cap or 30.0, alibi=kind == "alibi", prefix=rng.randint(1, high) if kind == "prefix" else 0)
    if op == "rope":
        write = rng.random() < 0.5
        T = _log(rng, 1, 16384)
        B = 1 if write else rng.choice([1, 1, 2, 3])
        S = max(1, T // B)
        while S * B * (Hq + Hkv) * D > 16384 * 40 * 128:
            S = max(1, S // 2)
        return _rope(dtype=dtype, B=B, S=S, Hq=Hq, Hkv=Hkv, D=D, rotary=rng.choice([D, D, D // 2]), pairs=rng.choice(["half", "half", "interleaved"]),
                     axes=rng.choice([1, 1, 3]), norm=rng.random() < 0.8, base=rng.choice([10000.0, 500000.0, 1000000.0]),
                     far=max(rng.choice([4096, 32768, 131072]), 2 * S), write=write, block=rng.choice([16, 32, 64]))
    new = rng.choice([1, 1, rng.randint(2, 8), _log(rng, 16, 2048)])
    B = _log(rng, 1, 512 if new < 16 else 48)
    high = _log(rng, 2, 16384 if B <= 256 else 8192)
    return _tables(B=B, low=rng.randint(1, high), high=high, new=new, block=rng.choice([16, 16, 32, 64]), pool=B + rng.randint(0, 64),
                   pad=rng.choice([0, rng.randint(1, 64)]))


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _spread(n, low, high):
    """n whole numbers from low to high, evenly spaced in their logarithm."""
    if n == 1:
        return [high]
    return [int(round(low * (high / low) ** (i / (n - 1)))) for i in range(n)]


def _doc_lengths(case):
    """Lengths of one row's documents: from 1 part to 8 parts, together all tokens but the padding."""
    n, total = case["docs"], case["Skv"] - case["pad"]
    parts = [1.0 + 7.0 * i / max(1, n - 1) for i in range(n)]
    cuts, at = [], 0.0
    for p in parts:
        at += p
        cuts.append(int(round(total * at / sum(parts))))
    return [b - a for a, b in zip([0] + cuts, cuts)]


def _prefixes(case):
    return _spread(case["B"], max(1, case["prefix"] // 4), case["prefix"])


def _slopes(H):
    return [2.0 ** (-8.0 * (h + 1) / H) for h in range(H)]


def _shuffled(values, g):
    return [values[i] for i in torch.randperm(len(values), generator=g).tolist()]


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype).cuda()


def _scores_of(case, st, g):
    st["slopes"] = torch.tensor(_slopes(case["Hq"]), dtype=torch.float32).cuda() if case["alibi"] else None
    st["prefix"] = _ints(_shuffled(_prefixes(case), g)) if case["prefix"] else None
    st["cap"] = case["cap"]
    st["ids"] = None


def prepare(case, seed):
    g = torch.Generator().manual_seed(int(seed) * 7919 + 17)
    gd = torch.Generator(device="cuda").manual_seed(int(seed) * 104729 + 5)
    st = {"case": dict(case)}
    dev = "cuda"

    def normal(*shape, scale=1.0, dtype=None):
        return (torch.randn(*shape, generator=gd, device=dev) * scale).to(dtype or DTYPES[case["dtype"]])

    if case["op"] == "attn":
        B, Hq, Hkv, Sq, Skv, D = (case[n] for n in ("B", "Hq", "Hkv", "Sq", "Skv", "D"))
        # (Queries of three times unit variance: logits of a few units, as trained models have them, some beyond half the cap.)
        st["q"], st["k"], st["v"] = normal(B, Hq, Sq, D, scale=3.0), normal(B, Hkv, Skv, D), normal(B, Hkv, Skv, D)
        _scores_of(case, st, g)
        if case["docs"]:
            rows = []
            for _ in range(B):
                row = []
                for i, n in enumerate(_shuffled(_doc_lengths(case), g)):
                    row += [i] * n
                rows.append(row + [-1] * case["pad"])
            st["ids"] = _ints(rows)
    elif case["op"] == "paged":
        B, Hq, Hkv, Sq, D, bs = (case[n] for n in ("B", "Hq", "Hkv", "Sq", "D", "block"))
        lens = _shuffled(_spread(B, case["low"], case["high"]), g)
        width = -(-case["high"] // bs)
        pages = [-(-n // bs) for n in lens]
        order = torch.randperm(sum(pages) + 7, generator=g).tolist()
        table, at = [], 0
        for n in pages:
            table.append(order[at:at + n] + [0] * (width - n))
            at += n
        kv = normal(2, sum(pages) + 7, bs, Hkv, D)
        st.update(q=normal(B, Hq, Sq, D, scale=3.0), k_cache=kv[0], v_cache=kv[1], table=_ints(table), lens=_ints(lens))
        _scores_of(case, st, g)
    elif case["op"] == "rope":
        B, S, Hq, Hkv, D = (case[n] for n in ("B", "S", "Hq", "Hkv", "D"))
        qkv = normal(B, S, (Hq + 2 * Hkv) * D, scale=2.0)
        q, k, v = (x.unflatten(-1, (-1, D)) for x in qkv.split([Hq * D, Hkv * D, Hkv * D], dim=-1))
        w = [(1.0 + 0.2 * torch.randn(D, generator=gd, device=dev)).to(DTYPES[case["dtype"]]) for _ in range(2)]
        st["wq"], st["wk"] = w if case["norm"] else (None, None)
        A = case["axes"]
        start = torch.randint(0, max(1, case["far"] - S), (A, B, 1), generator=gd, device=dev, dtype=torch.int32)
        step = torch.arange(S, device=dev, dtype=torch.int32).expand(A, B, S)
        pos = start + (step if A == 1 else torch.stack([step[0], step[1] // 32, step[2] % 32]))
        half = case["rotary"] // 2
        st["axis_of_pair"] = [0] * half if A == 1 else [0] * (half - 2 * (half * 3 // 8)) + [1] * (half * 3 // 8) + [2] * (half * 3 // 8)
        if case["write"]:
            q, k, v, pos = q[0], k[0], v[0], pos[:, 0]  # token-major (tokens, heads, D)
            bs = case["block"]
            blocks = -(-S // bs) + 5
            kv = torch.zeros(2, blocks, bs, Hkv, D, dtype=qkv.dtype, device=dev)
            st["k_cache"], st["v_cache"] = kv[0], kv[1]
            st["slots"] = torch.randperm(blocks * bs, generator=g)[:S].to(torch.int64).cuda()
        else:
            q, k, v = (x.transpose(1, 2) for x in (q, k, v))  # (B, H, S, D) over the projection's output
        st.update(q=q, k=k, v=v, pos=(pos if A > 1 else pos[0]).contiguous())
        if own:
            st["rotary"] = _own().RotaryTable(D, case["far"], base=case["base"], rotary_dim=case["rotary"], interleaved=case["pairs"] == "interleaved",
                                              axes=st["axis_of_pair"] if A > 1 else None, device=dev)
    else:
        B, bs, rows_n = case["B"], case["block"], case["pool"]
        lens = _shuffled(_spread(B, case["low"], case["high"]), g)
        new = [1] * B if case["new"] == 1 else _shuffled(_spread(B, max(1, case["new"] // 8), case["new"]), g)
        width = -(-(case["high"] + case["new"]) // bs)
        rows = torch.randperm(rows_n, generator=g)[:B].tolist()
        blocks = sum(-(-n // bs) for n in lens) + sum(-(-n // bs) + 1 for n in new) + 11
        order = torch.randperm(blocks, generator=g).tolist()
        table = torch.zeros(rows_n, width, dtype=torch.int32)
        pool_lens = torch.zeros(rows_n, dtype=torch.int32)
        at = 0
        for r, n in zip(rows, lens):
            p = -(-n // bs)
            table[r, :p] = torch.tensor(order[at:at + p], dtype=torch.int32)
            pool_lens[r] = n
            at += p
        free = order[at:]
        st.update(tables=table.cuda(), lens=pool_lens.cuda(), rows=_ints(rows), new=_ints(new), free=_ints(free + [0] * (blocks - len(free))),
                  count=_ints([len(free)]), tokens=sum(new) + case["pad"])
    return st


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def _visible(B, Sq, Skv, causal, prefix, ids, lens, dev):
    """(B, 1, Sq, Skv) truth values, and the distances |p - j| (B, 1, Sq, Skv) or smaller by broadcasting."""
    j = torch.arange(Skv, device=dev)
    i = torch.arange(Sq, device=dev)
    n = torch.full((B, 1), Skv, device=dev) if lens is None else lens.view(B, 1).long()
    p = (i[None, :] + n - Sq)[:, None, :, None]
    ok = j[None, None, None, :] < n[:, :, None, None]
    if causal:
        seen = j <= p
        if prefix is not None:
            seen = seen | (j < prefix.view(B, 1, 1, 1))
        ok = ok & seen
    if ids is not None:
        mine = ids[:, Skv - Sq:]
        ok = ok & (mine[:, None, :, None] == ids[:, None, None, :]) & (mine >= 0)[:, None, :, None]
    return ok, (p - j).abs()


def _attend(q, k, v, causal, cap, slopes, prefix, ids, lens):
    """Plain attention in float32 over (B, H, S, D), rounded once; (o, lse)."""
    B, Hq, Sq, D = q.shape
    Hkv, Skv = k.shape[1], k.shape[2]
    G = Hq // Hkv
    qf, kf, vf = q.float().view(B, Hkv, G, Sq, D), k.float(), v.float()
    o = torch.empty(B, Hkv, G, Sq, D, dtype=q.dtype, device=q.device)
    lse = torch.empty(B, Hkv, G, Sq, dtype=torch.float32, device=q.device)
    ok, dist = _visible(B, Sq, Skv, causal, prefix, ids, lens, q.device)
    step = max(1, (1 << 29) // (B * G * Sq * Skv))  # kv heads at a time
    for h in range(0, Hkv, step):
        e = min(Hkv, h + step)
        s = torch.matmul(qf[:, h:e].reshape(B, e - h, G * Sq, D), kf[:, h:e].transpose(2, 3)).view(B, e - h, G, Sq, Skv) * D ** -0.5
        if cap:
            s = torch.tanh(s / cap) * cap
        if slopes is not None:
            s = s - slopes[h * G:e * G].view(e - h, G, 1, 1) * dist[:, :, None].float()
        s = s.masked_fill(~ok[:, :, None], NEG)
        m = s.amax(-1, keepdim=True)
        m = torch.where(m == NEG, torch.zeros_like(m), m)
        s = torch.exp(s - m)
        total = s.sum(-1, keepdim=True)
        x = torch.matmul(s.view(B, e - h, G * Sq, Skv), vf[:, h:e]).view(B, e - h, G, Sq, D)
        o[:, h:e] = (x / torch.where(total == 0, torch.ones_like(total), total)).to(q.dtype)
        lse[:, h:e] = (m + torch.log(total))[..., 0]
    return o.view(B, Hq, Sq, D), lse.view(B, Hq, Sq)


def _gather(cache, table):
    """Keys of every sequence in order, (B, Hkv, width * block, D)."""
    B, W = table.shape
    return cache[table.long()].reshape(B, W * cache.shape[1], cache.shape[2], cache.shape[3]).transpose(1, 2)


def _rotate(x, w, eps, pos, case, axis_of_pair):
    """Plain norm and rotation of x (..., D) in float32; pos (A, ...) broadcast against x without its last dimension."""
    D, R = case["D"], case["rotary"]
    y = x.float()
    if w is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + eps) * w.float()
    inv = case["base"] ** (-torch.arange(0, R, 2, dtype=torch.float64, device=x.device) / R)
    ang = pos.double()[torch.tensor(axis_of_pair, device=x.device)].movedim(0, -1) * inv
    c, s = ang.cos().float(), ang.sin().float()
    if case["pairs"] == "half":
        a, b = y[..., :R // 2], y[..., R // 2:R]
        r = torch.cat([a * c - b * s, b * c + a * s, y[..., R:]], -1)
    else:
        a, b = y[..., 0:R:2], y[..., 1:R:2]
        r = torch.cat([torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2), y[..., R:]], -1)
    return r.to(x.dtype)


def _plain_tables(st):
    case, dev = st["case"], st["tables"].device
    bs, W, T, B = case["block"], st["tables"].shape[1], st["tokens"], case["B"]
    rows, new = st["rows"].long(), st["new"].long()
    old = st["lens"][rows].long()
    total = old + new
    start = new.cumsum(0) - new
    fits = (total <= W * bs) & (start + new <= T)
    have = (old + bs - 1) // bs
    need = torch.where(fits, (total + bs - 1) // bs - have, torch.zeros_like(old))
    upto = need.cumsum(0)
    ok = fits & ((need == 0) | (upto <= st["count"]))
    t = torch.arange(T, device=dev)
    b = (torch.searchsorted(start + new, t, right=True)).clamp(max=B - 1)
    j = t - start[b]
    good = ok[b] & (j < new[b])
    pos = torch.where(good, old[b] + j, torch.zeros_like(t))
    page = pos // bs
    fresh = good & (page >= have[b])
    at = (st["count"] - 1 - (upto - need)[b] - (page - have[b])).clamp(min=0)
    blk = torch.where(fresh, st["free"][at].long(), st["tables"][rows[b], page].long())
    flat = torch.cat([st["tables"].flatten(), torch.zeros(1, dtype=torch.int32, device=dev)])
    flat[torch.where(fresh, rows[b] * W + page, torch.full_like(t, flat.numel() - 1))] = blk.int()
    st["tables"].copy_(flat[:-1].view_as(st["tables"]))
    lens = torch.where(ok, total, old)
    cols = torch.arange(W, device=dev)
    batch = torch.where(cols[None, :] < ((lens + bs - 1) // bs)[:, None], st["tables"][rows], torch.zeros_like(st["tables"][rows]))
    slots = torch.where(good, blk * bs + pos % bs, torch.full_like(t, -1))
    return {"seq_lens": lens.int(), "query_start": start.int(), "query_lens": torch.where(ok, new, torch.zeros_like(new)).int(),
            "slot_mapping": slots, "positions": pos.int(), "block_tables": batch, "pool": st["tables"],
            "free_count": (st["count"] - torch.where(ok, need, torch.zeros_like(need)).sum()).int(), "refused": (~ok).sum().int().view(1)}


def run(state):
    st, case = state, state["case"]
    if case["op"] == "attn":
        if own:
            g = _own()
            docs = None if st["ids"] is None else g.document_spans(st["ids"])
            return g.gqa_flash_attn(st["q"], st["k"], st["v"], case["causal"], return_lse=True, softcap=st["cap"] or None,
                                    alibi_slopes=st["slopes"], prefix_lens=st["prefix"], documents=docs)
        return _attend(st["q"], st["k"], st["v"], case["causal"], st["cap"], st["slopes"], st["prefix"], st["ids"], None)
    if case["op"] == "paged":
        if own:
            from gqa_kernels.paged import paged_attention

            return paged_attention(st["q"], st["k_cache"], st["v_cache"], st["table"], st["lens"], True, max_seq_len=case["high"],
                                   softcap=st["cap"] or None, alibi_slopes=st["slopes"], prefix_lens=st["prefix"])
        k, v = _gather(st["k_cache"], st["table"]), _gather(st["v_cache"], st["table"])
        return _attend(st["q"], k, v, True, st["cap"], st["slopes"], st["prefix"], None, st["lens"])[0]
    if case["op"] == "rope":
        if own:
            g = _own()
            if not case["write"]:
                return g.qk_norm_rope(st["q"], st["k"], st["pos"], st["rotary"], q_weight=st["wq"], k_weight=st["wk"], eps=1e-6)
            q = g.qk_norm_rope_write(st["q"], st["k"], st["v"], st["pos"], st["rotary"], st["k_cache"], st["v_cache"], st["slots"],
                                     q_weight=st["wq"], k_weight=st["wk"], eps=1e-6)
            return q, st["k_cache"], st["v_cache"]
        pos = st["pos"] if case["axes"] > 1 else st["pos"][None]
        pos = pos[..., None] if case["write"] else pos[:, :, None]  # against (tokens, heads) or (B, heads, S)
        q = _rotate(st["q"], st["wq"], 1e-6, pos, case, st["axis_of_pair"])
        k = _rotate(st["k"], st["wk"], 1e-6, pos, case, st["axis_of_pair"])
        if not case["write"]:
            return q, k
        bs = case["block"]
        st["k_cache"][st["slots"] // bs, st["slots"] % bs] = k
        st["v_cache"][st["slots"] // bs, st["slots"] % bs] = st["v"]
        return q, st["k_cache"], st["v_cache"]
    if own:
        _own()
        from gqa_kernels.paged import extend_block_tables

        r = extend_block_tables(st["tables"], st["lens"], st["new"], st["free"], st["count"], case["block"], st["tokens"], rows=st["rows"],
                                update=False)
        return {"seq_lens": r.seq_lens, "query_start": r.query_start, "query_lens": r.query_lens, "slot_mapping": r.slot_mapping,
                "positions": r.positions, "block_tables": r.block_tables, "pool": st["tables"], "free_count": r.free_count, "refused": r.refused}
    return _plain_tables(st)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def _pairs_of_span(n_q, first, causal):
    """Visible pairs of n_q queries, the first of which sees `first` keys under causal (all of them see the last one's without)."""
    return n_q * first + n_q * (n_q - 1) // 2 if causal else n_q * (first + n_q - 1)


def _pairs(case):
    """Visible (query, key) pairs of one head over the batch (documents: of a row in listed order, within a few percent for a chunk)."""
    if case["op"] == "paged":
        total = 0
        pre = sorted(_prefixes(case)) if case["prefix"] else [0] * case["B"]
        for n, f in zip(_spread(case["B"], case["low"], case["high"]), pre):
            first = n - case["Sq"] + 1
            total += _pairs_of_span(case["Sq"], first, True)
            total += sum(max(0, min(f, n) - (first + i)) for i in range(case["Sq"])) if f > first else 0
        return total
    B, Sq, Skv = case["B"], case["Sq"], case["Skv"]
    if case["docs"]:
        total, at = 0, 0
        for n in _doc_lengths(case):
            lo, hi = max(at, Skv - Sq), at + n  # its tokens that are queries
            if hi > lo:
                total += _pairs_of_span(hi - lo, lo - at + 1, case["causal"])
            at += n
        return B * total
    if not case["causal"]:
        return B * Sq * Skv
    first = Skv - Sq + 1
    total = B * _pairs_of_span(Sq, first, True)
    if case["prefix"]:
        for f in _prefixes(case):
            total += sum(max(0, f - (first + i)) for i in range(Sq))
    return total


def work(case):
    if case["op"] in ("attn", "paged"):
        B, Hq, Hkv, Sq, D = (case[n] for n in ("B", "Hq", "Hkv", "Sq", "D"))
        if case["op"] == "attn":
            keys, extra = B * case["Skv"], 4 * B * Hq * Sq + (4 * B * case["Skv"] if case["docs"] else 0)
        else:
            lens = _spread(B, case["low"], case["high"])
            keys, extra = sum(lens), 4 * sum(-(-n // case["block"]) for n in lens)
        return {"bytes": 2 * (2 * B * Hq * Sq * D + 2 * keys * Hkv * D) + extra, "flops": 4 * D * Hq * _pairs(case)}
    if case["op"] == "rope":
        T, H, D = case["B"] * case["S"], case["Hq"] + case["Hkv"], case["D"]
        v = 4 * T * case["Hkv"] * D if case["write"] else 0
        return {"bytes": 4 * T * H * D + v + 4 * T * case["axes"] + (8 * T if case["write"] else 0),
                "flops": T * H * (3 * case["rotary"] + (4 * D if case["norm"] else 0))}
    new = [1] * case["B"] if case["new"] == 1 else _spread(case["B"], max(1, case["new"] // 8), case["new"])
    T, bs = sum(new) + case["pad"], case["block"]
    width = -(-(case["high"] + case["new"]) // bs)
    cached = sum(-(-n // bs) for n in _spread(case["B"], case["low"], case["high"]))
    return {"bytes": 12 * T + 4 * case["B"] * width + 4 * cached + 8 * sum(-(-n // bs) for n in new) + 24 * case["B"], "flops": 4 * T}


# ---------------------------------------------------------------------------
# The definitions in float64
# ---------------------------------------------------------------------------
def _exact_rows(q, k, v, first, causal, cap, slope, prefix, ids_q, ids_k):
    """One head: q (Sq, D), k and v (n, D) in float64; query i is position first + i."""
    n, dev = k.shape[0], q.device
    out, lses = [], []
    for a in range(0, q.shape[0], 2048):
        qa = q[a:a + 2048]
        s = (qa @ k.t().contiguous()) / math.sqrt(q.shape[1])
        p = (first + a + torch.arange(qa.shape[0], device=dev, dtype=torch.int64))[:, None]
        j = torch.arange(n, device=dev, dtype=torch.int64)[None, :]
        if cap:
            s = cap * torch.tanh(s / cap)
        if slope is not None:
            s = s - slope * (p - j).abs().double()
        hide = torch.zeros_like(s, dtype=torch.bool)
        if causal:
            hide = (j > p) & (j >= prefix)
        if ids_q is not None:
            i_q = ids_q[a:a + 2048, None]
            hide = hide | (i_q != ids_k[None, :]) | (i_q < 0)
        s[hide] = NEG
        lse = torch.logsumexp(s, 1) if n else torch.full((qa.shape[0],), NEG, dtype=torch.float64, device=dev)
        w = torch.exp(s - torch.where(lse == NEG, torch.zeros_like(lse), lse)[:, None])
        out.append(w @ v)
        lses.append(lse)
    return torch.cat(out), torch.cat(lses)


def _exact_rope(x, w, pos, case, axis_of_pair):
    """x (tokens, heads, D); pos (axes, tokens)."""
    y = x.double()
    if w is not None:
        y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / case["D"] + 1e-6) * w.double()
    half = case["rotary"] // 2
    z = y.clone()
    for i in range(half):
        theta = pos[axis_of_pair[i]].double() / case["base"] ** (2.0 * i / case["rotary"])
        a, b = (i, i + half) if case["pairs"] == "half" else (2 * i, 2 * i + 1)
        c, s = torch.cos(theta)[:, None], torch.sin(theta)[:, None]
        z[..., a] = y[..., a] * c - y[..., b] * s
        z[..., b] = y[..., a] * s + y[..., b] * c
    return z


def exact(case, seed):
    if case["op"] == "tables":
        return None  # whole numbers, compared as they are
    st = prepare(case, seed)
    if case["op"] == "rope":
        pos = st["pos"] if case["axes"] > 1 else st["pos"][None]
        if not case["write"]:
            B, S = case["B"], case["S"]
            r = []
            for x, w in ((st["q"], st["wq"]), (st["k"], st["wk"])):
                y = _exact_rope(x.transpose(1, 2).reshape(B * S, x.shape[1], case["D"]), w, pos.reshape(pos.shape[0], B * S), case, st["axis_of_pair"])
                r.append(y.view(B, S, x.shape[1], case["D"]).transpose(1, 2))
            return tuple(r)
        kc, vc = st["k_cache"].double(), st["v_cache"].double()
        flat = (-1, case["Hkv"], case["D"])
        kc.view(flat)[st["slots"]] = _exact_rope(st["k"], st["wk"], pos, case, st["axis_of_pair"])
        vc.view(flat)[st["slots"]] = st["v"].double()
        return _exact_rope(st["q"], st["wq"], pos, case, st["axis_of_pair"]), kc, vc
    q = st["q"].double()
    B, Hq, Sq, D = q.shape
    G = Hq // case["Hkv"]
    o, lse = torch.empty_like(q), torch.empty(B, Hq, Sq, dtype=torch.float64, device=q.device)
    lens = [case["Skv"]] * B if case["op"] == "attn" else st["lens"].tolist()
    pre = [0] * B if st["prefix"] is None else st["prefix"].tolist()
    slopes = [None] * Hq if st["slopes"] is None else st["slopes"].double().tolist()
    for b, n in enumerate(lens):
        if case["op"] == "paged":
            at = torch.arange(n, device=q.device)
            blk = st["table"][b][at // case["block"]].long()
            ks, vs = (c[blk, at % case["block"]].transpose(0, 1).double() for c in (st["k_cache"], st["v_cache"]))
        else:
            ks, vs = st["k"][b].double(), st["v"][b].double()
        ids = None if st["ids"] is None else st["ids"][b]
        for h in range(Hq):
            o[b, h], lse[b, h] = _exact_rows(q[b, h], ks[h // G], vs[h // G], n - Sq, case.get("causal", True), case["cap"], slopes[h], pre[b],
                                             None if ids is None else ids[n - Sq:], ids)
    return (o, lse) if case["op"] == "attn" else o
