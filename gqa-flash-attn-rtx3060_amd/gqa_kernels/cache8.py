"""A paged K/V cache in 8 bits: attention over it, writes and reads.

The reference keeps K and V in the queries' type and has no cache (reference
gqa_kernels/dispatch.py:14-27).  Here a paged cache (``paged.py``) may hold e4m3
codes (``torch.float8_e4m3fn``, half the bytes) with one whole exponent for the
tokens of a page and kv head, keys and values each: a code stands for its value
times 2 ** exponent.

    codes      (num_blocks, block_size, num_kv_heads, head_dim)
    exponents  int32 (num_blocks, num_kv_heads)

``paged_attention``, ``write_kv``, ``qk_norm_rope_write``, ``read_kv``,
``PagedKVCache`` and ``GQAPagedAttention`` take such caches; this module is what
they call.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import Optional

import torch

from . import _lib
from .gqa_split import _decode_host, stream_handle
from .scores import check_score, refuse_grad
from .scores import workspace as own_workspace

__all__ = ["CODES", "MIN_EXPONENT", "MAX_EXPONENT", "read_kv"]

CODES = torch.float8_e4m3fn
MIN_EXPONENT, MAX_EXPONENT = _lib.GQA_MIN_EXPONENT, _lib.GQA_MAX_EXPONENT
MIN_BLOCK = 16
FEW_ROWS = 32  # packed rows per kv head up to which a call takes the flat split
_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16}
_ROUTES = {"split": _lib.FORM_FLAT, "chunks": _lib.FORM_CHUNKS, "single": _lib.FORM_SINGLE}
_LOG2E = math.log2(math.e)


def takes(k_cache, k_exponents, v_exponents) -> bool:
    """Whether a call's cache is one in 8 bits."""
    return k_exponents is not None or v_exponents is not None or k_cache.dtype is CODES


def new_exponents(num_blocks: int, num_kv_heads: int, device="cuda") -> torch.Tensor:
    """Exponents of keys and values for a cache without tokens: int32 (2,
    num_blocks, num_kv_heads)."""
    return torch.full((2, num_blocks, num_kv_heads), MIN_EXPONENT, dtype=torch.int32, device=device)


def _codes_ready(t: torch.Tensor) -> bool:
    st = t.stride()
    return st[-1] == 1 and (t.data_ptr() | st[0] | st[1] | st[2]) % 16 == 0


def check_caches(k_cache, v_cache, k_exponents, v_exponents, write: bool = False) -> int:
    """The block size of a cache in 8 bits, its tensors checked.  write: they are written, so
    that pages, heads, keys and values have memory of their own."""
    assert k_exponents is not None and v_exponents is not None, \
        "a cache in 8 bits needs k_exponents and v_exponents"
    assert k_cache.dtype is CODES and v_cache.dtype is CODES, \
        "with exponents, k_cache and v_cache hold torch.float8_e4m3fn codes"
    assert k_cache.dim() == 4 and tuple(k_cache.shape) == tuple(v_cache.shape), \
        "k_cache / v_cache must be (num_blocks, block_size, num_kv_heads, head_dim)"
    if write:
        for k, v in ((k_cache, v_cache), (k_exponents, v_exponents)):
            assert not any(s == 0 and n > 1 for t in (k, v) for s, n in zip(t.stride(), t.shape)) and \
                (k.numel() == 0 or k.data_ptr() != v.data_ptr()), \
                "a store needs pages, heads, keys and values with memory of their own (no broadcast codes or exponents)"
    assert k_cache.is_cuda and k_cache.device == v_cache.device
    block_size = k_cache.shape[1]
    assert MIN_BLOCK <= block_size <= _lib.GQA_MAX_BLOCK_SIZE and block_size & (block_size - 1) == 0, \
        f"block_size must be a power of two, {MIN_BLOCK} or more"
    assert _codes_ready(k_cache) and _codes_ready(v_cache), "cache rows must be contiguous and 16-byte aligned"
    for e in (k_exponents, v_exponents):
        assert e.dtype == torch.int32 and tuple(e.shape) == (k_cache.shape[0], k_cache.shape[2]), \
            "exponents must be int32 (num_blocks, num_kv_heads)"
        assert e.device == k_cache.device
    return block_size


def struct(cache, exponents) -> _lib.Cache8:
    c = _lib.Cache8()
    c.codes, c.exponents = cache.data_ptr(), exponents.data_ptr()
    c.stride, c.exp_stride = (ctypes.c_int64 * 4)(*cache.stride()), (ctypes.c_int64 * 2)(*exponents.stride())
    return c


@functools.lru_cache(maxsize=4096)
def plan(batch: int, num_heads: int, num_kv_heads: int, seq_q: int, max_seq_len: int, head_dim: int,
         cu_count: int) -> tuple:
    """(form, parts) of a call, gqa_paged8_plan's."""
    form, parts = ctypes.c_int(), ctypes.c_int()
    _lib.check(_lib.load().gqa_paged8_plan(batch, num_heads, num_kv_heads, seq_q, max_seq_len, head_dim, cu_count,
                                           ctypes.byref(form), ctypes.byref(parts)))
    return form.value, parts.value


def route(num_heads: int, num_kv_heads: int, seq_q: int) -> str:
    """"split" (few packed rows a kv head) or "single", as a mixed batch is
    parted."""
    return "split" if num_heads // num_kv_heads * seq_q <= FEW_ROWS else "single"


def attention(q, k_cache, v_cache, block_table, seq_lens, causal, max_seq_len, scale, splits, return_lse, out, route,
              query_start, query_lens, max_query_len, softcap, alibi_slopes, prefix_lens, k_exponents, v_exponents):
    """``paged_attention`` over a cache in 8 bits."""
    if route is None and splits is None and _lib._host is not None and (max_seq_len is None or max_seq_len >= 0):
        # Every check passed, natively; else None.
        res = _lib._host.paged_attn8(q, k_cache, v_cache, k_exponents, v_exponents, block_table, seq_lens,
                                     bool(causal), -1 if max_seq_len is None else max_seq_len,
                                     (q.shape[-1] ** -0.5 if scale is None else scale) * _LOG2E, bool(return_lse), out,
                                     query_start, query_lens, -1 if max_query_len is None else int(max_query_len),
                                     softcap or 0.0, alibi_slopes, prefix_lens)
        if res is not None:
            return res
    from .paged import _cu_count, _row_strides, _rows_ready

    refuse_grad("paged_attention over a cache in 8 bits", q, k_cache, v_cache, alibi_slopes, out)
    dev = q.device
    varlen = query_start is not None
    assert q.is_cuda and q.dtype in _DTYPES, f"unsupported dtype {q.dtype}"
    if varlen:
        assert query_lens is not None and max_query_len is not None, "varlen needs query_lens and max_query_len"
        assert q.dim() == 3, "varlen q is (num_tokens, num_heads, head_dim)"
        _, num_heads, head_dim = q.shape
        batch, seq_q = seq_lens.shape[0], int(max_query_len)
        for t in (query_start, query_lens):
            assert t.dtype == torch.int32 and tuple(t.shape) == (batch,) and t.device == dev
        query_start, query_lens = query_start.contiguous(), query_lens.contiguous()
    else:
        assert q.dim() == 4, "q is (batch, num_heads, seq_q, head_dim)"
        batch, num_heads, seq_q, head_dim = q.shape
        query_lens = None
    block_size = check_caches(k_cache, v_cache, k_exponents, v_exponents)
    num_kv_heads = k_cache.shape[2]
    assert num_heads % num_kv_heads == 0, "num_heads must be divisible by num_kv_heads"
    assert num_heads <= 128 * num_kv_heads, "groups of at most 128 query heads per kv head"
    assert head_dim in (64, 128), f"unsupported head_dim {head_dim}"
    assert k_cache.shape[3] == head_dim, "cache head_dim differs from q"
    assert k_cache.device == dev and block_table.device == dev and seq_lens.device == dev
    assert block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.shape[0] == batch
    assert seq_lens.dtype == torch.int32 and tuple(seq_lens.shape) == (batch,)
    if block_table.stride(1) != 1 or (batch > 1 and block_table.stride(0) < block_table.shape[1]):
        block_table = block_table.contiguous()
    seq_lens = seq_lens.contiguous()
    if not _rows_ready(q):
        q = q.contiguous()
    table_stride = block_table.stride(0) if batch > 1 else block_table.shape[1]
    capacity = block_table.shape[1] * block_size
    max_seq_len = capacity if max_seq_len is None else int(max_seq_len)
    assert 0 <= max_seq_len <= capacity, "max_seq_len exceeds the block table's capacity"
    assert max_seq_len <= _lib.GQA_MAX_CACHE8_KEYS, f"max_seq_len of at most {_lib.GQA_MAX_CACHE8_KEYS}"
    scale = head_dim ** -0.5 if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"a cache in 8 bits needs a positive scale, not {scale}")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    else:
        assert tuple(out.shape) == tuple(q.shape) and out.dtype == q.dtype and out.device == dev
        assert _rows_ready(out), "out rows must be contiguous and 16-byte aligned"
    score = None
    if softcap or alibi_slopes is not None or prefix_lens is not None:
        score = check_score(softcap, alibi_slopes, prefix_lens, None, batch=batch, num_heads=num_heads,
                            num_kv_heads=num_kv_heads, seq_q=seq_q, seq_kv=max_seq_len, causal=bool(causal),
                            scale=scale, device=dev)
    index = dev.index if dev.index is not None else torch.cuda.current_device()
    form, parts = plan(batch, num_heads, num_kv_heads, seq_q, max_seq_len, head_dim, _cu_count(index))
    if route is not None:
        assert route in _ROUTES, f"a cache in 8 bits has the routes {', '.join(_ROUTES)}"
        if _ROUTES[route] != form:
            form, parts = _ROUTES[route], {"split": 1, "chunks": 2 * batch, "single": 0}[route]
    if splits is not None:
        assert form != _lib.FORM_SINGLE, "the single pass has no parts"
        parts = int(splits) * (batch if form == _lib.FORM_CHUNKS else 1)
    lse = None
    if return_lse:
        lse = torch.empty((q.shape[0], num_heads) if varlen else (batch, num_heads, seq_q), dtype=torch.float32,
                          device=dev)
    lib = _lib.load()
    _decode_host()  # (the native call from here on)
    with torch.cuda.device(dev):
        need = lib.gqa_paged8_workspace_bytes(form, parts, batch, num_heads, seq_q, head_dim)
        ws = own_workspace(need, dev) if need else None
        _lib.check(lib.gqa_paged8_launch(
            form, q.data_ptr(), _row_strides(q, varlen), ctypes.byref(struct(k_cache, k_exponents)),
            ctypes.byref(struct(v_cache, v_exponents)), block_table.data_ptr(), table_stride, seq_lens.data_ptr(),
            query_start.data_ptr() if varlen else None, query_lens.data_ptr() if varlen else None, block_size,
            max_seq_len, out.data_ptr(), _row_strides(out, varlen), None if lse is None else lse.data_ptr(),
            None if ws is None else ws.data_ptr(), parts, batch, num_heads, num_kv_heads, seq_q, head_dim,
            scale * _LOG2E, int(bool(causal)), _DTYPES[q.dtype], None if score is None else ctypes.byref(score),
            stream_handle(dev)))
    return out if lse is None else (out, lse)


def _check_tokens(key, value, k_cache, slot_mapping):
    assert key.is_cuda and key.dtype in _DTYPES, f"unsupported dtype {key.dtype}"
    assert key.dim() == 3 and tuple(value.shape) == tuple(key.shape) and value.dtype == key.dtype, \
        "key and value must be (num_tokens, num_kv_heads, head_dim) of one dtype"
    assert key.shape[2] in (64, 128), f"unsupported head_dim {key.shape[2]}"
    assert tuple(key.shape[1:]) == tuple(k_cache.shape[2:]), "key and the cache differ in heads or head_dim"
    assert key.shape[0] < 1 << 26, f"fewer than {1 << 26} tokens a call"
    assert slot_mapping.dtype == torch.int64 and tuple(slot_mapping.shape) == (key.shape[0],)
    assert key.device == value.device == k_cache.device == slot_mapping.device


def _launch_write(q, k, v, q_out, k_cache, v_cache, k_exponents, v_exponents, slot_mapping, rope, block_size):
    _decode_host()  # (the native call from here on)
    with torch.cuda.device(k.device):
        _lib.check(_lib.load().gqa_cache8_write_launch(
            None if q is None else q.data_ptr(), _lib._i64x3() if q is None else _lib.strides3(q), k.data_ptr(),
            _lib.strides3(k), v.data_ptr(), _lib.strides3(v), None if q is None else q_out.data_ptr(),
            _lib._i64x3() if q is None else _lib.strides3(q_out), ctypes.byref(struct(k_cache, k_exponents)),
            ctypes.byref(struct(v_cache, v_exponents)), slot_mapping.data_ptr(),
            None if rope is None else ctypes.byref(rope), k.shape[0], 0 if q is None else q.shape[1], k.shape[1],
            k.shape[2], block_size, _DTYPES[k.dtype], stream_handle(k.device)))


def write(key, value, k_cache, v_cache, slot_mapping, k_exponents, v_exponents) -> None:
    """``write_kv`` into a cache in 8 bits."""
    if _lib._host is not None and _lib._host.write_kv8(key, value, k_cache, v_cache, slot_mapping, k_exponents,
                                                       v_exponents):
        return
    from .rotary import _ready

    refuse_grad("write_kv into a cache in 8 bits", key, value, k_cache, v_cache)
    block_size = check_caches(k_cache, v_cache, k_exponents, v_exponents, write=True)
    _check_tokens(key, value, k_cache, slot_mapping)
    _launch_write(None, _ready(key), _ready(value), None, k_cache, v_cache, k_exponents, v_exponents,
                  slot_mapping.contiguous(), None, block_size)


def norm_rope_write(q, k, v, positions, table, k_cache, v_cache, slot_mapping, q_weight, k_weight, eps, q_out,
                    k_exponents, v_exponents):
    """``qk_norm_rope_write`` into a cache in 8 bits."""
    from .rotary import _check_out, _check_qk, _out_like, _ready, _rope

    refuse_grad("qk_norm_rope_write", q, k, v, q_weight, k_weight, k_cache, v_cache, q_out)
    _check_qk(q, k, 3)
    assert k.shape[0] == q.shape[0], "q and k have different tokens"
    block_size = check_caches(k_cache, v_cache, k_exponents, v_exponents, write=True)
    _check_tokens(k, v, k_cache, slot_mapping)
    slot_mapping = slot_mapping.contiguous()
    qo = _out_like(q) if q_out is None else _check_out(q_out, q, "q_out")
    keep: list = []
    rope = _rope(q, positions, table, q_weight, k_weight, eps, (q.shape[0],), keep)
    _launch_write(_ready(q), _ready(k), _ready(v), qo, k_cache, v_cache, k_exponents, v_exponents, slot_mapping, rope,
                  block_size)
    return qo


def read_kv(k_cache, v_cache, slot_mapping, k_exponents, v_exponents, *, dtype=torch.bfloat16, key=None, value=None):
    """K and V of the tokens at `slot_mapping` out of a cache in 8 bits, as rows of
    16 bits: what moves a sequence to another machine, to storage, or to a cache of
    16 bits (``write_kv``).

    Args:
        k_cache, v_cache, k_exponents, v_exponents: the cache, as
            ``paged_attention`` takes it.
        slot_mapping: int64 (num_tokens,), slot = block * block_size + offset;
            negative ones (padding) give zeros, every other one lies inside the
            cache.
        dtype: bf16 (which holds every value of the cache) or fp16 (which rounds
            those below its least step and has infinities for those past 65504).
        key, value: tensors (num_tokens, num_kv_heads, head_dim) of dtype with
            16-byte aligned rows to write into (both or neither).

    Returns:
        (key, value), (num_tokens, num_kv_heads, head_dim).
    """
    if _lib._host is not None:
        res = _lib._host.read_kv8(k_cache, v_cache, slot_mapping, k_exponents, v_exponents, dtype is torch.bfloat16
                                  if dtype in _DTYPES else None, key, value)  # every check passed, natively; else None
        if res is not None:
            return res
    from .rotary import _rows_ready

    refuse_grad("read_kv", k_cache, v_cache, key, value)
    block_size = check_caches(k_cache, v_cache, k_exponents, v_exponents)
    assert dtype in _DTYPES, f"unsupported dtype {dtype}"
    assert slot_mapping.dtype == torch.int64 and slot_mapping.dim() == 1 and slot_mapping.device == k_cache.device
    assert k_cache.shape[3] in (64, 128), f"unsupported head_dim {k_cache.shape[3]}"
    assert (key is None) == (value is None), "key and value, both or neither"
    shape = (slot_mapping.shape[0], *k_cache.shape[2:])
    assert shape[0] < 1 << 31
    if key is None:
        key, value = (torch.empty(shape, dtype=dtype, device=k_cache.device) for _ in range(2))
    for t in (key, value):
        assert tuple(t.shape) == shape and t.dtype == dtype and t.device == k_cache.device, \
            "key and value must be (num_tokens, num_kv_heads, head_dim) of dtype"
        assert _rows_ready(t), "key and value rows must be contiguous and 16-byte aligned"
    slot_mapping = slot_mapping.contiguous()
    _decode_host()  # (the native call from here on)
    with torch.cuda.device(k_cache.device):
        _lib.check(_lib.load().gqa_cache8_read_launch(
            ctypes.byref(struct(k_cache, k_exponents)), ctypes.byref(struct(v_cache, v_exponents)),
            slot_mapping.data_ptr(), key.data_ptr(), _lib.strides3(key), value.data_ptr(), _lib.strides3(value),
            shape[0], shape[1], shape[2], block_size, _DTYPES[dtype], stream_handle(k_cache.device)))
    return key, value
