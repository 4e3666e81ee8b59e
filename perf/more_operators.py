"""The operators of a paged K/V cache held in 8 bits (e4m3 values, and for each page and kv head a power of two that they are multiplied with):
attention over it, from single tokens to long chunks, with plain and with changed scores; storing new tokens' keys and values, as they come and normed
and rotated on the way; reading tokens back.

listed() and draw() give the cases, prepare() what a program holds before the call, run() one pass: the plain form (elementary torch operations in
float32, angles and exponents in float64), or, with `own`, the calls of gqa_kernels.  exact() is the definition in float64.  Caches are returned as
the values that they stand for."""
import math
import sys
from pathlib import Path

import torch

own = False

PACKAGE = str(Path(__file__).resolve().parent.parent / "gqa-flash-attn-rtx3060_amd")
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
E4M3 = torch.float8_e4m3fn
LEAST, MOST = -126, 127  # exponents of a page and head
NEG = -math.inf


def _own():
    if PACKAGE not in sys.path:
        sys.path.insert(0, PACKAGE)
    import gqa_kernels
    import gqa_kernels.paged

    return gqa_kernels


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _attn(**kw):
    """Attention of Sq new tokens of each of B sequences over the cache; lengths spread from low to high.  cap: 0 none; alibi: distance bias;
    prefix: the longest of the batch's prefixes (0: none)."""
    d = dict(op="attn", dtype="bf16", B=16, Hq=32, Hkv=8, Sq=1, low=100, high=8000, D=128, block=16, cap=0.0, alibi=False, prefix=0)
    d.update(kw)
    return d


def _append(**kw):
    """S new tokens of each of B sequences, which begin somewhere in a page, into the cache; rotary: rotated dimensions (0: keys and values are
    stored as they come), norm: per-head norms of q and k."""
    d = dict(op="append", dtype="bf16", B=64, S=1, Hq=32, Hkv=8, D=128, block=16, rotary=128, pairs="half", norm=True, base=500000.0, far=131072)
    d.update(kw)
    return d


def _read(**kw):
    """T tokens of the cache back as rows of 16 bits."""
    d = dict(op="read", dtype="bf16", T=16384, Hkv=8, D=128, block=16)
    d.update(kw)
    return d


def listed():
    return [
        # One user's next token: the smallest call, latency alone.
        _attn(name="token_700", B=1, low=700, high=700),
        # A serving batch's decode step, lengths unequal, 16-key pages.
        _attn(name="decode_b32", B=32),
        # The next token of one long context, the 128K tokens of this repository's decode benchmark.
        _attn(name="token_131072", B=1, low=131072, high=131072, block=64),
        # A decode step with the distance bias at head_dim 64.
        _attn(name="alibi_decode_d64", dtype="fp16", B=24, Hq=16, Hkv=4, low=200, high=6000, D=64, alibi=True),
        # Verification of 8 drafted tokens of each of 16 requests.
        _attn(name="verify_16x8", dtype="fp16", B=16, Sq=8, low=500, high=8000, block=32),
        # A chunk of new tokens of four requests over their cached prefixes, with capped scores.
        _attn(name="cap_chunk_4x256", B=4, Sq=256, low=2000, high=9000, cap=30.0),
        # A chunk of a long prompt over what is cached of it.
        _attn(name="prompt_chunk_2048", B=1, Sq=2048, low=16384, high=16384, block=64),
        # A decode step's queries, keys and values: normed, rotated, stored in pages that hold tokens already.
        _append(name="append_decode"),
        # A prompt's.
        _append(name="append_prompt", B=1, S=8192),
        # Keys and values alone, as another kernel left them: chunks of three requests.
        _append(name="store_chunks_d64", dtype="fp16", B=3, S=1667, Hkv=4, D=64, block=32, rotary=0, norm=False),
        # A sequence on its way to another machine or to storage.
        _read(name="read_sequence"),
        # A short one, in half precision.
        _read(name="read_short", dtype="fp16", T=333, block=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "attn", "append", "append", "read"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    Hq, Hkv = rng.choice([(32, 8), (32, 8), (16, 4), (64, 8), (8, 8), (12, 4), (28, 4)])
    D = rng.choice([64, 128, 128])
    block = rng.choice([16, 16, 32, 64, 128])
    if op == "attn":
        B = _log(rng, 1, 48)
        high = _log(rng, 32, 131072 // B)
        low = rng.randint(max(1, high // 20), high)
        Sq = rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 9, 128), _log(rng, 128, 2048)])
        Sq = max(1, min(Sq, low, 32 * 2048 * 16384 // (B * Hq * high)))
        kind = rng.choice(["", "", "", "cap", "alibi", "prefix"])
        return _attn(dtype=dtype, B=B, Hq=Hq, Hkv=Hkv, Sq=Sq, low=low, high=high, D=D, block=block, cap=rng.choice([15.0, 30.0, 50.0]) if kind == "cap" else 0.0,
                     alibi=kind == "alibi", prefix=rng.randint(1, high) if kind == "prefix" else 0)
    if op == "append":
        T = _log(rng, 1, 8192)
        B = min(T, rng.choice([1, 1, 3, 16, 64, 256]))
        rotary = rng.choice([0, D, D, D // 2])
        return _append(dtype=dtype, B=B, S=max(1, T // B), Hq=Hq, Hkv=Hkv, D=D, block=block, rotary=rotary, pairs=rng.choice(["half", "half", "interleaved"]),
                       norm=rotary > 0 and rng.random() < 0.7, base=rng.choice([10000.0, 500000.0, 1000000.0]), far=rng.choice([32768, 131072]))
    return _read(dtype=dtype, T=_log(rng, 1, 32768), Hkv=Hkv, D=D, block=block)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _spread(n, low, high):
    """n whole numbers from low to high, evenly spaced in their logarithm."""
    if n == 1:
        return [high]
    return [int(round(low * (high / low) ** (i / (n - 1)))) for i in range(n)]


def _prefixes(case):
    return _spread(case["B"], max(1, case["prefix"] // 4), case["prefix"])


def _shuffled(values, g):
    return [values[i] for i in torch.randperm(len(values), generator=g).tolist()]


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype).cuda()


def _exponent(most):
    """The least exponent that brings values of up to `most` within 448, the largest of e4m3."""
    m, x = torch.frexp(most.double())
    return (x - 9 + (m > 0.875).to(x.dtype)).clamp(LEAST, MOST).to(torch.int32)


def _two(e):
    """2 ** e in float32 of whole e from -126 to 127, by its bits (a power function may be off by the last bit, which moves values between two codes)."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _filled(blocks, case, gd):
    """A cache of `blocks` pages full of tokens: (k, v, exponents of k, of v).  Keys with channels of unequal size, values whose size differs from
    page to page, as trained models' do."""
    bs, Hkv, D = case["block"], case["Hkv"], case["D"]
    out = []
    for scale in (torch.exp(0.7 * torch.randn(1, 1, Hkv, D, generator=gd, device="cuda")),
                  torch.exp2(torch.randint(-2, 3, (blocks, 1, Hkv, 1), generator=gd, device="cuda").float())):
        x = torch.randn(blocks, bs, Hkv, D, generator=gd, device="cuda") * scale
        e = _exponent(x.abs().amax((1, 3)))
        out.append((x * _two(-e)[:, None, :, None]).to(E4M3))
        out.append(e)
    return out[0], out[2], out[1], out[3]


def prepare(case, seed):
    g = torch.Generator().manual_seed(int(seed) * 7919 + 29)
    gd = torch.Generator(device="cuda").manual_seed(int(seed) * 104729 + 11)
    dt, bs, Hkv, D = DTYPES[case["dtype"]], case["block"], case["Hkv"], case["D"]
    st = {"case": dict(case), "table": None}

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gd, device="cuda") * scale).to(dt)

    if case["op"] == "attn":
        B, Hq = case["B"], case["Hq"]
        lens = _shuffled(_spread(B, case["low"], case["high"]), g)
        pages = [-(-n // bs) for n in lens]
        blocks = sum(pages) + 7
        order = torch.randperm(blocks, generator=g).tolist()
        width, table, at = -(-case["high"] // bs), [], 0
        for n in pages:
            table.append(order[at:at + n] + [0] * (width - n))
            at += n
        # (Queries of three times unit variance: logits of a few units, as trained models have them.)
        st.update(q=normal(B, Hq, case["Sq"], D, scale=3.0), table=_ints(table), lens=_ints(lens))
        st["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / Hq) for h in range(Hq)]).cuda() if case["alibi"] else None
        st["prefix"] = _ints(_shuffled(_prefixes(case), g)) if case["prefix"] else None
    elif case["op"] == "append":
        B, S, Hq, R = case["B"], case["S"], case["Hq"], case["rotary"]
        T = B * S
        qkv = normal(T, (Hq + 2 * Hkv) * D, scale=2.0)
        st["q"], st["k"], st["v"] = (x.unflatten(-1, (-1, D)) for x in qkv.split([Hq * D, Hkv * D, Hkv * D], dim=-1))
        if not R:
            st["q"] = None
        st["wq"], st["wk"] = ([(1.0 + 0.2 * torch.randn(D, generator=gd, device="cuda")).to(dt) for _ in range(2)] if case["norm"] else (None, None))
        start = torch.randint(0, max(1, case["far"] - S), (B, 1), generator=g)
        st["pos"] = (start + torch.arange(S)).flatten().int().cuda()
        # The pages that a sequence's new tokens fall in, from the offset of the first one on.
        first = torch.randint(0, bs, (B, 1), generator=g)
        per = (bs - 1 + S - 1) // bs + 1
        blocks = B * per
        at = first + torch.arange(S)
        page = torch.randperm(blocks, generator=g).view(B, per).gather(1, at // bs)
        st["slots"] = (page * bs + at % bs).flatten().cuda()
        st["every"] = torch.arange(blocks * bs, device="cuda")
        # Tokens in front of the new ones; nothing behind them.
        held = torch.zeros(blocks, bs, dtype=torch.uint8)
        held[page[:, 0]] = (torch.arange(bs) < first).to(torch.uint8)
        st["held"] = held.cuda()[:, :, None, None]
        if own and R:
            st["rotary"] = _own().RotaryTable(D, case["far"], base=case["base"], rotary_dim=R, interleaved=case["pairs"] == "interleaved")
    else:
        blocks = -(-case["T"] // bs) + 5
        at = torch.arange(case["T"])
        st["slots"] = (torch.randperm(blocks, generator=g)[at // bs] * bs + at % bs).cuda()
    st["k8"], st["v8"], st["ke"], st["ve"] = _filled(blocks, case, gd)
    if case["op"] == "append":
        held = st.pop("held")
        st["k8"], st["v8"] = ((x.view(torch.uint8) * held).view(E4M3) for x in (st["k8"], st["v8"]))
    return st


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def _values(codes, exponents):
    """Values of codes (..., block, Hkv, D) under exponents (..., Hkv), in float32."""
    return codes.float() * _two(exponents)[..., None, :, None]


def _gather(codes, exponents, table):
    """Keys or values of every sequence in order, float32 (B, Hkv, width * block, D)."""
    B, W = table.shape
    x = _values(codes.view(torch.uint8)[table.long()].view(E4M3), exponents[table.long()])
    return x.flatten(1, 2).transpose(1, 2)


def _attend(st):
    """Plain attention in float32, rounded once."""
    case, q = st["case"], st["q"]
    B, Hq, Sq, D = q.shape
    Hkv = case["Hkv"]
    G = Hq // Hkv
    k, v = _gather(st["k8"], st["ke"], st["table"]), _gather(st["v8"], st["ve"], st["table"])
    Skv = k.shape[2]
    n = st["lens"].view(B, 1).long()
    j = torch.arange(Skv, device=q.device)
    p = (torch.arange(Sq, device=q.device) + n - Sq)[:, None, :, None]
    seen = j <= p
    if st["prefix"] is not None:
        seen = seen | (j < st["prefix"].view(B, 1, 1, 1))
    seen = seen & (j < n[:, :, None, None])
    o = torch.empty(B, Hkv, G, Sq, D, dtype=q.dtype, device=q.device)
    qf = q.float().view(B, Hkv, G * Sq, D)
    step = max(1, (1 << 29) // (B * G * Sq * Skv))  # kv heads at a time
    for h in range(0, Hkv, step):
        e = min(Hkv, h + step)
        s = torch.matmul(qf[:, h:e], k[:, h:e].transpose(2, 3).contiguous()).view(B, e - h, G, Sq, Skv) * D ** -0.5
        if case["cap"]:
            s = torch.tanh(s / case["cap"]) * case["cap"]
        if st["slopes"] is not None:
            s = s - st["slopes"][h * G:e * G].view(e - h, G, 1, 1) * (p - j).abs()[:, :, None].float()
        s = s.masked_fill(~seen[:, :, None], NEG)
        m = s.amax(-1, keepdim=True)
        s = torch.exp(s - torch.where(m == NEG, torch.zeros_like(m), m))
        total = s.sum(-1, keepdim=True)
        x = torch.matmul(s.view(B, e - h, G * Sq, Skv), v[:, h:e].contiguous()).view(B, e - h, G, Sq, D)
        o[:, h:e] = (x / torch.where(total == 0, torch.ones_like(total), total)).to(q.dtype)
    return o.view(B, Hq, Sq, D)


def _rotate(x, w, case, pos):
    """Plain norm and rotation of token-major x (T, heads, D), in float32."""
    D, R = case["D"], case["rotary"]
    y = x.float()
    if w is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * w.float()
    inv = case["base"] ** (-torch.arange(0, R, 2, dtype=torch.float64, device=x.device) / R)
    ang = pos.double()[:, None, None] * inv
    c, s = ang.cos().float(), ang.sin().float()
    if case["pairs"] == "half":
        a, b = y[..., :R // 2], y[..., R // 2:R]
        return torch.cat([a * c - b * s, b * c + a * s, y[..., R:]], -1)
    a, b = y[..., 0:R:2], y[..., 1:R:2]
    return torch.cat([torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2), y[..., R:]], -1)


def _store(codes, exponents, rows, slots, limit):
    """Rows (T, Hkv, D) of float32 into the cache.  A page's exponent is the least for its new tokens, and not below what it was unless the page
    begins anew (its first slot is among theirs); tokens in front of the new ones are brought to it."""
    blocks, bs, Hkv, D = codes.shape
    page, off = slots // bs, slots % bs
    y = rows.clamp(-limit, limit)
    T = y.shape[0]
    most = torch.zeros(blocks, Hkv, device=y.device).scatter_reduce(0, page[:, None].expand(T, Hkv), y.abs().amax(-1), "amax")
    front = torch.full((blocks,), bs, dtype=off.dtype, device=y.device).scatter_reduce(0, page, off, "amin")
    was = torch.where((front == 0)[:, None], torch.full_like(exponents, LEAST), exponents)
    e = torch.where((front < bs)[:, None], torch.maximum(was, _exponent(most)), exponents)
    less = (exponents - e).clamp(LEAST, 0)
    x = codes.float()
    old = (torch.arange(bs, device=y.device) < front[:, None])[:, :, None, None] & (front < bs)[:, None, None, None]
    x = torch.where(old, x * _two(less)[:, None, :, None], x)
    new = y * _two(-e[page])[..., None]
    x.view(blocks * bs, Hkv, D)[slots] = new
    codes.copy_(x.to(E4M3))
    exponents.copy_(e)


def run(state):
    st, case = state, state["case"]
    dt = DTYPES[case["dtype"]]
    if case["op"] == "attn":
        if own:
            return _own().paged.paged_attention(st["q"], st["k8"], st["v8"], st["table"], st["lens"], True, max_seq_len=case["high"], softcap=case["cap"] or None,
                                                alibi_slopes=st["slopes"], prefix_lens=st["prefix"], k_exponents=st["ke"], v_exponents=st["ve"])
        return _attend(st)
    if case["op"] == "append":
        q = None
        if own:
            g = _own()
            if case["rotary"]:
                q = g.qk_norm_rope_write(st["q"], st["k"], st["v"], st["pos"], st["rotary"], st["k8"], st["v8"], st["slots"], q_weight=st["wq"], k_weight=st["wk"],
                                         eps=1e-6, k_exponents=st["ke"], v_exponents=st["ve"])
            else:
                g.paged.write_kv(st["k"], st["v"], st["k8"], st["v8"], st["slots"], k_exponents=st["ke"], v_exponents=st["ve"])
            return (q, *g.paged.read_kv(st["k8"], st["v8"], st["every"], st["ke"], st["ve"], dtype=dt))
        limit = 1.875 * 2.0 ** (15 if dt == torch.float16 else 127)  # the largest e4m3 multiple of a power of two within the type
        k = st["k"].float()
        if case["rotary"]:
            q = _rotate(st["q"], st["wq"], case, st["pos"]).to(dt)
            k = _rotate(st["k"], st["wk"], case, st["pos"])
        _store(st["k8"], st["ke"], k, st["slots"], limit)
        _store(st["v8"], st["ve"], st["v"].float(), st["slots"], limit)
        return q, _values(st["k8"], st["ke"]).to(dt).flatten(0, 1), _values(st["v8"], st["ve"]).to(dt).flatten(0, 1)
    if own:
        return _own().paged.read_kv(st["k8"], st["v8"], st["slots"], st["ke"], st["ve"], dtype=dt)
    page, off = st["slots"] // case["block"], st["slots"] % case["block"]
    return tuple((c.view(torch.uint8)[page, off].view(E4M3).float() * _two(e[page])[..., None]).to(dt)
                 for c, e in ((st["k8"], st["ke"]), (st["v8"], st["ve"])))


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    Hkv, D, bs = case["Hkv"], case["D"], case["block"]
    if case["op"] == "attn":
        B, Hq, Sq = case["B"], case["Hq"], case["Sq"]
        lens = _spread(B, case["low"], case["high"])
        pre = sorted(_prefixes(case)) if case["prefix"] else [0] * B
        pairs = sum(sum(max(n - Sq + 1 + i, min(f, n)) for i in range(Sq)) for n, f in zip(lens, pre))
        pages = sum(-(-n // bs) for n in lens)
        return {"bytes": 4 * B * Hq * Sq * D + 2 * sum(lens) * Hkv * D + 4 * pages + 8 * pages * Hkv, "flops": 4 * D * Hq * pairs}
    if case["op"] == "append":
        B, S, Hq = case["B"], case["S"], case["Hq"]
        T, pages = B * S, B * ((bs - 1 + S - 1) // bs + 1)
        q = 4 * T * Hq * D + 4 * T if case["rotary"] else 0
        # Keys and values read and stored; the pool read once and written once as 16 bits.
        kv = 6 * T * Hkv * D + 8 * T + 2 * pages * bs * Hkv * (1 + 2) * D + 16 * pages * Hkv + 8 * pages * bs
        return {"bytes": q + kv, "flops": T * ((Hq + Hkv) * (3 * case["rotary"] + (4 * D if case["norm"] else 0)) + 4 * Hkv * D)}
    T = case["T"]
    return {"bytes": 6 * T * Hkv * D + 8 * T + 8 * -(-T // bs) * Hkv, "flops": 2 * T * Hkv * D}


# ---------------------------------------------------------------------------
# The definitions in float64
# ---------------------------------------------------------------------------
def _power(e):
    """2 ** e in float64, by its bits."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _decoded(codes):
    """Values of e4m3 from their bits: sign, 4 bits of exponent (bias 7), 3 of mantissa."""
    c = codes.view(torch.uint8).int()
    ex, man = (c >> 3) & 15, (c & 7).double()
    mag = torch.where(ex == 0, man / 512, (1 + man / 8) * _power(ex - 7))
    return torch.where(c >= 128, -mag, mag)


def _nearest(y):
    """float64 values of at most 448 to the nearest of e4m3, ties to an even last bit, without its types."""
    step = _power(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))).clamp(min=-6.0) - 3)
    return torch.round(y / step) * step


def _exact_rope(x, w, pos, case):
    y = x.double()
    if w is not None:
        y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / case["D"] + 1e-6) * w.double()
    half = case["rotary"] // 2
    z = y.clone()
    for i in range(half):
        theta = pos.double() / case["base"] ** (2.0 * i / case["rotary"])
        a, b = (i, i + half) if case["pairs"] == "half" else (2 * i, 2 * i + 1)
        c, s = torch.cos(theta)[:, None], torch.sin(theta)[:, None]
        z[..., a] = y[..., a] * c - y[..., b] * s
        z[..., b] = y[..., a] * s + y[..., b] * c
    return z


def _exact_store(codes, exponents, y, slots, bs):
    """The pool's values (slots, Hkv, D) after the call, page by page over the pages that are written."""
    value = (_decoded(codes) * _power(exponents)[:, None, :, None]).flatten(0, 1)
    order = torch.argsort(slots)
    slots, y = slots[order], y[order]
    pages, counts = torch.unique_consecutive(slots // bs, return_counts=True)
    ends = counts.cumsum(0).tolist()
    heads = y.abs().amax(-1)
    for pg, n, end in zip(pages.tolist(), counts.tolist(), ends):
        mine = slice(end - n, end)
        most = heads[mine].amax(0)
        e = torch.ceil(torch.log2(most.clamp(min=1e-38) / 448))
        e = torch.where(most <= 448 * _power(e - 1), e - 1, e).clamp(min=LEAST)  # (a logarithm is off by its last bit)
        first = int(slots[end - n]) - pg * bs
        if first:
            e = torch.maximum(e, exponents[pg].double())
        unit = _power(e)[:, None]
        front = slice(pg * bs, pg * bs + first)
        tail = slice(pg * bs + first, (pg + 1) * bs)
        value[front] = _nearest(value[front] / unit) * unit
        # (What was behind the new tokens is read under the page's new exponent.)
        value[tail] = value[tail] * _power(e - exponents[pg].double())[:, None]
        value[slots[mine]] = _nearest(y[mine] / unit) * unit
    return value


def exact(case, seed):
    st = prepare(case, seed)
    bs, D = case["block"], case["D"]
    if case["op"] == "read":
        at, e = st["slots"], [_power(x)[st["slots"] // bs][..., None] for x in (st["ke"], st["ve"])]
        return tuple(_decoded(c).flatten(0, 1)[at] * f for c, f in zip((st["k8"], st["v8"]), e))
    if case["op"] == "append":
        q, k = None, st["k"].double()
        if case["rotary"]:
            q, k = _exact_rope(st["q"], st["wq"], st["pos"], case), _exact_rope(st["k"], st["wk"], st["pos"], case)
        return q, _exact_store(st["k8"], st["ke"], k, st["slots"], bs), _exact_store(st["v8"], st["ve"], st["v"].double(), st["slots"], bs)
    q = st["q"].double()
    B, Hq, Sq, _ = q.shape
    G = Hq // case["Hkv"]
    o = torch.empty_like(q)
    for b, n in enumerate(st["lens"].tolist()):
        blk = st["table"][b, :-(-n // bs)].long()
        ks, vs = ((_decoded(c[blk]) * _power(e[blk])[:, None, :, None]).flatten(0, 1)[:n].transpose(0, 1)
                  for c, e in ((st["k8"], st["ke"]), (st["v8"], st["ve"])))
        see = max(0, int(st["prefix"][b])) if st["prefix"] is not None else 0
        i = torch.arange(n - Sq, n, device=q.device)[:, None]
        j = torch.arange(n, device=q.device)[None, :]
        hide = (j > i) & (j >= see)
        for h in range(Hq):
            s = (q[b, h] @ ks[h // G].t().contiguous()) / math.sqrt(D)
            if case["cap"]:
                s = case["cap"] * torch.tanh(s / case["cap"])
            if st["slopes"] is not None:
                s = s - float(st["slopes"][h]) * (i - j).abs().double()
            s[hide] = NEG
            o[b, h] = torch.softmax(s, -1) @ vs[h // G]
    return o
