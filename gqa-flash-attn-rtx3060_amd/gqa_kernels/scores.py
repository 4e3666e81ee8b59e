"""Attention with changed scores: capped, biased by distance, with prefix and
document masks (include/gqa_attn.h, gqa_scored_launch).

The reference's attention has one score and one mask (reference
gqa_kernels/dispatch.py:14-27).  Here ``gqa_flash_attn`` and
``paged_attention`` take the changes of other models as keyword arguments.  The
split passes and the short form run in second instances of their kernels; the
single pass, its key chunks and their combine are kernels of their own
(csrc/gqa_scored.hip).
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _lib
from .gqa_split import _decode_host, stream_handle

__all__ = ["DocumentSpans", "document_spans"]


def _has_tangent(t) -> bool:
    return forward_ad.unpack_dual(t).tangent is not None


def refuse_grad(name: str, *tensors) -> None:
    """There is no backward pass, and none of forward mode: better an error than
    outputs that silently carry no gradient or tangent."""
    backward = torch.is_grad_enabled()
    if any(t is not None and ((backward and t.requires_grad) or _has_tangent(t)) for t in tensors):
        raise NotImplementedError(f"{name} has no derivative: call it under torch.no_grad(), on tensors without tangents")


class DocumentSpans(NamedTuple):
    """For each position of a batch of packed sequences, the first key of its
    document and the first key behind it: int32 (batch, seq_kv), contiguous."""

    starts: torch.Tensor
    ends: torch.Tensor


def document_spans(document_ids: torch.Tensor) -> DocumentSpans:
    """Spans of the documents packed into each row of a batch, for
    ``gqa_flash_attn(..., documents=)``; made once for a batch, used by every
    layer.

    document_ids: int32 (batch, seq_kv).  A document is a run of equal ids (an
    id that comes back later is another document); tokens of negative ids are
    padding, which sees nothing and is seen by nothing.
    """
    ids = document_ids
    if _lib._host is not None:
        both = _lib._host.document_spans(ids)  # every check passed, natively; else None
        if both is not None:
            return DocumentSpans(*both)
    assert ids.dim() == 2 and ids.dtype == torch.int32, "document_ids must be int32 (batch, seq_kv)"
    assert ids.is_cuda
    if ids.stride(1) != 1 or ids.stride(0) < ids.shape[1]:
        ids = ids.contiguous()
    _decode_host()  # (the native call from here on)
    both = torch.empty(2, *ids.shape, dtype=torch.int32, device=ids.device)
    with torch.cuda.device(ids.device):
        _lib.check(_lib.load().gqa_document_spans_launch(ids.data_ptr(), ids.stride(0), both[0].data_ptr(),
                                                         both[1].data_ptr(), ids.shape[0], ids.shape[1],
                                                         stream_handle(ids.device)))
    return DocumentSpans(both[0], both[1])


def check_score(softcap, alibi_slopes, prefix_lens, documents, *, batch: int, num_heads: int, num_kv_heads: int,
                seq_q: int, seq_kv: int, causal: bool, scale: float, device) -> _lib.Score:
    """The changes as the C entry points take them, their arguments checked.
    (The struct holds addresses: the caller keeps the tensors.)"""
    s = _lib.Score()
    assert num_heads <= 128 * num_kv_heads, "changed scores take groups of at most 128 query heads per kv head"
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"changed scores need a positive scale, not {scale}")
    if softcap:
        softcap = float(softcap)
        if not (softcap > 0 and _lib.GQA_MIN_RAW_SOFTCAP <= 0.999 * softcap / scale
                and 1.001 * softcap / scale <= _lib.GQA_MAX_RAW_SOFTCAP):
            raise ValueError(f"softcap must be positive and softcap / scale in [{_lib.GQA_MIN_RAW_SOFTCAP}, "
                             f"{_lib.GQA_MAX_RAW_SOFTCAP:.0e}], not {softcap} / {scale}")
        s.softcap = softcap
    if alibi_slopes is not None:
        assert alibi_slopes.dtype == torch.float32 and tuple(alibi_slopes.shape) == (num_heads,), \
            "alibi_slopes must be float32 (num_heads,)"
        assert alibi_slopes.device == device and alibi_slopes.is_contiguous()
        s.alibi_slopes = alibi_slopes.data_ptr()
    if prefix_lens is not None:
        assert causal, "prefix_lens needs causal=True (without it every key is visible)"
        assert prefix_lens.dtype == torch.int32 and tuple(prefix_lens.shape) == (batch,), \
            "prefix_lens must be int32 (batch,)"
        assert prefix_lens.device == device and prefix_lens.is_contiguous()
        s.prefix_lens = prefix_lens.data_ptr()
    if documents is not None:
        assert isinstance(documents, DocumentSpans), "documents is what document_spans() returns"
        assert seq_q <= seq_kv, "documents needs seq_q <= seq_kv (every query is a key position)"
        for t in (documents.starts, documents.ends):
            assert t.dtype == torch.int32 and tuple(t.shape) == (batch, seq_kv), \
                "document spans must be int32 (batch, seq_kv)"
            assert t.device == device and t.is_contiguous()
        s.span_lo, s.span_hi = documents.starts.data_ptr(), documents.ends.data_ptr()
    return s


def scored_launch(form: int, parts: int, q, k, v, o, lse, workspace, causal: bool, scale_log2: float, dtype: int,
                  score: "_lib.Score", stream: int) -> int:
    """gqa_scored_launch on kernel-ready tensors; its return code."""
    batch, num_heads, seq_q, head_dim = q.shape
    return _lib.load().gqa_scored_launch(
        form, q.data_ptr(), _lib.strides(q), k.data_ptr(), _lib.strides(k), v.data_ptr(), _lib.strides(v),
        o.data_ptr(), _lib.strides(o), None if lse is None else lse.data_ptr(),
        None if workspace is None else workspace.data_ptr(), parts, batch, num_heads, k.shape[1], seq_q,
        k.shape[2], head_dim, scale_log2, int(bool(causal)), dtype, ctypes.byref(score), stream)


def workspace(nbytes: int, device) -> Optional[torch.Tensor]:
    """A call's own workspace.  (The call launches twice without the
    interpreter's lock, so the stream's shared one could be taken by a call of
    another thread in between.)"""
    return torch.empty(max(-(-nbytes // 4), 4), dtype=torch.float32, device=device)
