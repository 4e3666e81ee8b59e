"""Norms of queries and keys per head, with the rotation of positions, in one
pass; with or without the paged cache write.

What a model does between its projection and the attention (the reference takes
rotated q and k as they come, gqa_kernels/dispatch.py:14-27):

* ``RotaryTable`` — cos and sin of every position and pair, computed once in
  float64; one or several position axes (time, height, width of images and
  video), half or interleaved pairs, partial rotation, given frequencies.
* ``qk_norm_rope`` — q and k, any layout.
* ``qk_norm_rope_write`` — token-major q, k, v: k (normed, rotated) and v go
  straight to their cache slots, as ``write_kv`` stores them.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import torch

from . import _lib
from .gqa_split import _decode_host, stream_handle
from .scores import refuse_grad

__all__ = ["RotaryTable", "qk_norm_rope", "qk_norm_rope_write"]

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16}
_MAX_AXES = 4
_MAX_TOKENS = 1 << 26  # GQA_MAX_ROPE_TOKENS


class RotaryTable:
    """cos and sin of positions 0 .. max_positions - 1.

    Args:
        head_dim: 64 or 128.
        max_positions: positions held; a larger one gives NaN.
        base: pair i turns by position * base ** (-2 i / rotary_dim).
        rotary_dim: dimensions that are rotated (a multiple of 16; default all).
        interleaved: pairs are dimensions (2 i, 2 i + 1); default (i, i +
            rotary_dim / 2).
        axes: the position axis (0 .. 3) of each of the rotary_dim / 2 pairs, for
            positions of several axes; ``RotaryTable.sections`` makes it from
            section sizes.  Default: one axis.
        inv_freq: the rotary_dim / 2 frequencies themselves (scaled ones),
            instead of base.

    ``table`` is float32 (max_positions, rotary_dim / 2, 2), pairs of (cos, sin)
    rounded from float64.  The attributes are fixed; copies and pickles hold a table
    of their own.
    """

    def __init__(self, head_dim: int, max_positions: int, base: float = 10000.0, rotary_dim: Optional[int] = None,
                 interleaved: bool = False, axes: Optional[Sequence[int]] = None, inv_freq=None, device="cuda"):
        assert head_dim in (64, 128), f"unsupported head_dim {head_dim}"
        rotary_dim = head_dim if rotary_dim is None else int(rotary_dim)
        assert 16 <= rotary_dim <= head_dim and rotary_dim % 16 == 0, \
            "rotary_dim must be a multiple of 16 up to head_dim"
        assert 1 <= max_positions < 1 << 31
        half = rotary_dim // 2
        if axes is not None:
            axes = [int(a) for a in axes]
            assert len(axes) == half, f"axes has {len(axes)} entries for {half} pairs"
            assert all(0 <= a < _MAX_AXES for a in axes), f"axes must be in [0, {_MAX_AXES})"
        if inv_freq is None:
            assert base > 0
            inv = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
        else:
            inv = torch.as_tensor(inv_freq, dtype=torch.float64).cpu()
            assert tuple(inv.shape) == (half,), f"inv_freq must hold {half} frequencies"
        inv = inv.to(device)
        max_positions = int(max_positions)
        table = torch.empty(max_positions, half, 2, dtype=torch.float32, device=device)
        for at in range(0, max_positions, 1 << 16):  # (bounds the float64 temporaries)
            end = min(at + (1 << 16), max_positions)
            ang = torch.arange(at, end, dtype=torch.float64, device=device)[:, None] * inv
            table[at:end, :, 0] = ang.cos()
            table[at:end, :, 1] = ang.sin()
        self.__setstate__(dict(table=table, head_dim=head_dim, interleaved=bool(interleaved), axes=axes))

    def __setstate__(self, state):
        table, axes = state["table"], state["axes"]
        words = [0, 0, 0, 0]
        for i, a in enumerate(axes or ()):
            words[i >> 4] |= a << (2 * (i & 15))
        # For the native calls: the table, its gqa_rope, axes (0: positions
        # without an axis dimension), head_dim.
        r = _lib.Rope()
        r.table, r.max_positions, r.rotary_dim = table.data_ptr(), table.shape[0], 2 * table.shape[1]
        r.interleaved, r.axes = int(state["interleaved"]), 1 if axes is None else max(axes) + 1
        r.pair_axis = (ctypes.c_uint32 * 4)(*words)
        self.__dict__.update(state, max_positions=r.max_positions, rotary_dim=r.rotary_dim, num_axes=r.axes, _rope=r,
                             _native=(table, ctypes.addressof(r), 0 if axes is None else r.axes, state["head_dim"]))

    def __getstate__(self):
        # (Copies and pickles: the gqa_rope is made anew, of the copy's own table.)
        return {n: self.__dict__[n] for n in ("table", "head_dim", "interleaved", "axes")}

    def __setattr__(self, name, value):
        raise AttributeError("a RotaryTable's attributes are fixed: make another one, or write into its table")

    @staticmethod
    def sections(sizes: Sequence[int]) -> list:
        """axes for consecutive sections of pairs: sizes[a] pairs of axis a."""
        return [a for a, n in enumerate(sizes) for _ in range(n)]


def _rows_ready(t: torch.Tensor) -> bool:
    st = t.stride()
    bits = 0
    for x in st[:-1]:
        bits |= x
    return st[-1] == 1 and (t.data_ptr() | bits * t.element_size()) % 16 == 0


def _ready(t: torch.Tensor) -> torch.Tensor:
    return t if _rows_ready(t) else t.clone(memory_format=torch.contiguous_format)


def _out_like(t: torch.Tensor) -> torch.Tensor:
    o = torch.empty_like(t)  # t's dimension order where it is dense
    return o if _rows_ready(o) else torch.empty_like(t, memory_format=torch.contiguous_format)


def _check_out(o: torch.Tensor, t: torch.Tensor, name: str) -> torch.Tensor:
    assert tuple(o.shape) == tuple(t.shape) and o.dtype == t.dtype and o.device == t.device, \
        f"{name} must have its input's shape, dtype and device"
    assert _rows_ready(o), f"{name} rows must be contiguous and 16-byte aligned"
    return o


def _rope(q, positions, table: Optional[RotaryTable], q_weight, k_weight, eps: float, tokens, keep: list):
    """gqa_rope of a call; `keep` holds what its addresses belong to."""
    r = _lib.Rope()
    assert table is not None or q_weight is not None or k_weight is not None, "neither a rotation nor a norm is given"
    if table is not None:
        assert table.head_dim == q.shape[-1], "the table's head_dim differs from q"
        assert table.table.device == q.device, "the table is on another device"
        assert positions is not None and positions.dtype in (torch.int32, torch.int64), \
            "positions must be int32 or int64"
        shape = tokens if table.axes is None else (table.num_axes, *tokens)
        assert tuple(positions.shape) == shape, f"positions must be {shape}, not {tuple(positions.shape)}"
        assert positions.device == q.device
        positions = positions.contiguous()
        keep.append(positions)
        r.table, r.max_positions, r.rotary_dim = table.table.data_ptr(), table.max_positions, table.rotary_dim
        r.interleaved, r.axes, r.pair_axis = int(table.interleaved), table.num_axes, table._rope.pair_axis
        r.positions, r.positions64 = positions.data_ptr(), int(positions.dtype == torch.int64)
    assert (q_weight is None and k_weight is None) or eps >= 0
    w32 = None
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is None:
            continue
        assert tuple(w.shape) == (q.shape[-1],) and w.dtype in (q.dtype, torch.float32), \
            f"{name} must be (head_dim,) in q's dtype or float32"
        assert w.device == q.device
        assert w32 is None or w32 == (w.dtype == torch.float32), "q_weight and k_weight must share one dtype"
        w32 = w.dtype == torch.float32
        w = w if w.is_contiguous() and w.data_ptr() % 16 == 0 else w.clone(memory_format=torch.contiguous_format)
        keep.append(w)
        setattr(r, name, w.data_ptr())
    r.weights32, r.eps = int(bool(w32)), eps
    return r


def _check_qk(q, k, dims: int):
    assert q.dim() == dims and q.is_cuda
    assert q.dtype in _DTYPES, f"unsupported dtype {q.dtype}"
    assert q.shape[-1] in (64, 128), f"unsupported head_dim {q.shape[-1]}"
    if k is not None:
        assert k.dim() == dims and k.dtype == q.dtype and k.device == q.device and k.shape[-1] == q.shape[-1]


def qk_norm_rope(q, k, positions, table: Optional[RotaryTable] = None, *, q_weight=None, k_weight=None,
                 eps: float = 1e-6, q_out=None, k_out=None):
    """RMS norm of every head's rows of q and k, then their rotation, in fp32
    and rounded once.

    Args:
        q: (batch, num_heads, seq, head_dim), or token-major (num_tokens,
            num_heads, head_dim); fp16 or bf16, any strides with 16-byte aligned
            rows (others are copied).
        k: the same with its own number of heads, or None: q alone.
        positions: int32 or int64 (batch, seq) or (num_tokens,); with a table of
            several axes, (axes, ...) of that.  Negative ones (padding) are
            taken as 0.
        table: the rotation; None: norms alone.
        q_weight, k_weight: (head_dim,) norm weights in q's dtype or float32;
            None: that tensor is not normed.
        q_out, k_out: tensors to write into; q and k themselves work in place.

    Returns:
        (q, k) normed and rotated (k None without k).
    """
    if _lib._host is not None:
        # Every check passed, natively; else None.
        res = _lib._host.norm_rope(q, k, None, positions, None if table is None else table._native, None, None, None,
                                   q_weight, k_weight, eps, q_out, k_out)
        if res is not None:
            return res
    refuse_grad("qk_norm_rope", q, k, q_weight, k_weight)
    assert q.dim() in (3, 4), "q must be (batch, num_heads, seq, head_dim) or (num_tokens, num_heads, head_dim)"
    _check_qk(q, k, q.dim())
    assert k is not None or (k_weight is None and k_out is None), "k_weight or k_out without k"
    if q.dim() == 4:
        tokens = (q.shape[0], q.shape[2])
        assert k is None or (k.shape[0], k.shape[2]) == tokens, "q and k have different tokens"
    else:
        tokens = (q.shape[0],)
        assert k is None or k.shape[0] == q.shape[0], "q and k have different tokens"
    qo = _out_like(q) if q_out is None else _check_out(q_out, q, "q_out")
    ko = None
    if k is not None:
        ko = _out_like(k) if k_out is None else _check_out(k_out, k, "k_out")
    keep: list = []
    rope = _rope(q, positions, table, q_weight, k_weight, eps, tokens, keep)

    def four(t):  # (batch, heads, seq, head_dim) strides
        if t is None:
            return _lib._i64x4()
        if t.dim() == 4:
            return _lib.strides(t)
        return _lib._i64x4(0, t.stride(1), t.stride(0), 1)

    batch, seq = tokens if len(tokens) == 2 else (1, tokens[0])
    assert batch * seq < _MAX_TOKENS, f"qk_norm_rope takes fewer than {_MAX_TOKENS} tokens"
    qi, ki = _ready(q), None if k is None else _ready(k)
    _decode_host()  # (the native call from here on)
    with torch.cuda.device(q.device):
        _lib.check(_lib.load().gqa_qk_norm_rope_launch(
            qi.data_ptr(), four(qi), None if ki is None else ki.data_ptr(), four(ki),
            qo.data_ptr(), four(qo), None if ko is None else ko.data_ptr(), four(ko),
            ctypes.byref(rope), batch, q.shape[1], 1 if k is None else k.shape[1], seq, q.shape[-1],
            _DTYPES[q.dtype], stream_handle(q.device)))
    return qo, ko


def qk_norm_rope_write(q, k, v, positions, table: Optional[RotaryTable], k_cache, v_cache, slot_mapping, *,
                       q_weight=None, k_weight=None, eps: float = 1e-6, q_out=None):
    """``qk_norm_rope`` of token-major q (num_tokens, num_heads, head_dim) and k
    (num_tokens, num_kv_heads, head_dim), and ``write_kv`` of the rotated k and of
    v, in one pass; returns q.

    Caches and slot_mapping as ``write_kv`` (negative slots are not stored,
    every other one lies inside the caches, no slot twice)."""
    from .paged import _check_cache

    if _lib._host is not None:
        # Every check passed, natively; else None.
        res = _lib._host.norm_rope(q, k, v, positions, None if table is None else table._native, k_cache, v_cache,
                                   slot_mapping, q_weight, k_weight, eps, q_out, None)
        if res is not None:
            return res
    refuse_grad("qk_norm_rope_write", q, k, v, q_weight, k_weight)
    _check_qk(q, k, 3)
    assert v is not None and tuple(v.shape) == tuple(k.shape) and v.dtype == k.dtype and v.device == k.device
    assert k.shape[0] == q.shape[0], "q and k have different tokens"
    assert q.shape[0] < _MAX_TOKENS, f"qk_norm_rope_write takes fewer than {_MAX_TOKENS} tokens"
    block_size = _check_cache(k_cache, v_cache)
    assert k_cache.shape[2] == k.shape[1] and k_cache.shape[3] == k.shape[2] and k_cache.dtype == k.dtype
    assert k_cache.device == q.device
    assert slot_mapping.dtype == torch.int64 and tuple(slot_mapping.shape) == (q.shape[0],)
    assert slot_mapping.device == q.device
    slot_mapping = slot_mapping.contiguous()
    qo = _out_like(q) if q_out is None else _check_out(q_out, q, "q_out")
    keep: list = []
    rope = _rope(q, positions, table, q_weight, k_weight, eps, (q.shape[0],), keep)
    qi, ki, vi = _ready(q), _ready(k), _ready(v)
    _decode_host()  # (the native call from here on)
    with torch.cuda.device(q.device):
        _lib.check(_lib.load().gqa_qk_norm_rope_write_launch(
            qi.data_ptr(), _lib.strides3(qi), ki.data_ptr(), _lib.strides3(ki), vi.data_ptr(), _lib.strides3(vi),
            qo.data_ptr(), _lib.strides3(qo), k_cache.data_ptr(), _lib.strides(k_cache), v_cache.data_ptr(),
            _lib.strides(v_cache), slot_mapping.data_ptr(), ctypes.byref(rope), q.shape[0], q.shape[1], k.shape[1],
            q.shape[2], block_size, _DTYPES[q.dtype], stream_handle(q.device)))
    return qo
