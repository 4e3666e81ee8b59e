"""Plain forms of the paged cache in 8 bits, in float64: values of its codes, and what a write leaves."""
from __future__ import annotations

import torch

CODES = torch.float8_e4m3fn
LEAST, MOST = -126, 126


def power(e):
    """2 ** e in float64, by its bits (a power function is off by the last one)."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def decode(codes):
    """float64 values of e4m3 codes, from their bits."""
    c = codes.view(torch.uint8).to(torch.int64)
    ex, man = (c >> 3) & 15, (c & 7).double()
    mag = torch.where(ex == 0, man / 512, (1 + man / 8) * power(ex - 7))
    mag = torch.where((c & 127) == 127, torch.full_like(mag, float("nan")), mag)
    return torch.where(c >= 128, -mag, mag)


def encode(y):
    """Codes (uint8) nearest to float64 y within +-448, ties to an even last bit: through the table of all of them."""
    table = decode(torch.arange(127, dtype=torch.uint8, device=y.device).view(CODES))  # ascending, 0 .. 448
    a = y.abs().contiguous()
    hi = torch.searchsorted(table, a).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    up, down = table[hi] - a, a - table[lo]
    c = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo).to(torch.uint8)
    sign = torch.signbit(y).to(torch.uint8) << 7
    return torch.where(torch.isnan(y), torch.full_like(c, 127), c | sign)


def exponents_of(most):
    """The least exponents with most <= 448 * 2 ** e, clamped; float64 `most`."""
    m, x = torch.frexp(most)
    e = (x - 9 + (m > 0.875).to(x.dtype)).clamp(LEAST, MOST).to(torch.int32)
    return torch.where(most == 0, torch.full_like(e, LEAST), e)


def values(codes, exponents):
    """float64 values of a cache (num_blocks, block_size, Hkv, D)."""
    return decode(codes) * power(exponents.clamp(LEAST, MOST))[:, None, :, None]


def stored(codes, exponents, rows, slots, limit):
    """(codes as uint8, exponents) after the rows (T, Hkv, D) of float64 are stored at `slots`, token runs page by page."""
    out, exps = codes.view(torch.uint8).clone(), exponents.clone()
    bs = codes.shape[1]
    y = torch.where(rows.abs() > limit, rows.sign() * limit, rows)
    by_page = {}
    for t, s in enumerate(slots.tolist()):
        if s >= 0:
            by_page.setdefault(s // bs, []).append((t, s % bs))
    for page, tokens in by_page.items():
        at, off = (torch.tensor(x, device=codes.device) for x in zip(*tokens))
        first = int(off.min())
        e = exponents_of(torch.nan_to_num(y[at], nan=0.0).abs().amax((0, 2)))
        if first > 0:
            was = exps[page].clamp(LEAST, MOST)
            e = torch.maximum(e, was)
            grown = e > was
            front = encode(decode(out[page, :first].view(CODES)) * power(was - e)[:, None])
            # (NaN keeps its sign)
            front = torch.where((out[page, :first] & 127) == 127, out[page, :first], front)
            out[page, :first] = torch.where(grown[:, None], front, out[page, :first])
        exps[page] = e
        out[page, off] = encode(y[at] * power(-e)[:, None])
    return out, exps


def limit_of(dtype):
    return 1.875 * 2.0 ** (15 if dtype == torch.float16 else 127)


def new_cache(blocks, bs, Hkv, D, *, seed=0, layout="NHD", full=True, spread=3):
    """(k, v, k_exponents, v_exponents): random codes but NaN, exponents around -6; `full` False: zeros and the least exponents."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(2):
        c = torch.randint(0, 256, (blocks, bs, Hkv, D), generator=g, dtype=torch.uint8)
        c[(c & 127) == 127] = 0
        if not full:
            c.zero_()
        c = c.cuda()
        if layout == "HND":
            c = c.transpose(1, 2).contiguous().transpose(1, 2)
        out.append(c.view(CODES))
    e = torch.randint(-6 - spread, -5 + spread, (2, blocks, Hkv), generator=g, dtype=torch.int32)
    if not full:
        e.fill_(LEAST)
    e = e.cuda()
    return out[0], out[1], e[0], e[1]


def gather(codes, exponents, table, n, dtype):
    """Keys or values of a sequence of n tokens as the products see them: (Hkv, n, D) of dtype."""
    bs = codes.shape[1]
    blk = table[:-(-n // bs)].long()
    c = codes.view(torch.uint8)[blk].view(CODES)
    x = values(c, exponents[blk]).flatten(0, 1)[:n].transpose(0, 1)
    return x.to(dtype)
