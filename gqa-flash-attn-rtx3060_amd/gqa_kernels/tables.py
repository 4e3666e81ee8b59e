"""Block tables and slots of a step, built on the device from request lengths.

``PagedKVCache`` (paged.py) allocates blocks on the host and copies slots and
tables to the device each step.  Here the pool itself — tables, lengths and the
list of free blocks — lives on the device: a step is one small kernel, or two (more
than 32 requests), no copy and no wait, and can be captured in a HIP graph, whose replays then serve one
token after another.  (No counterpart in the reference, whose README.md:140-146
names a paged cache as its next step.)
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib
from .gqa_split import _decode_host, stream_handle

__all__ = ["StepTables", "extend_block_tables", "release_blocks", "BlockPool"]


class StepTables(NamedTuple):
    """What ``extend_block_tables`` makes of a step, all on the device: int32 but
    for slot_mapping (int64).

    seq_lens (batch,): keys of each request, its new tokens included.
    query_start, query_lens (batch,): its tokens, behind those of the requests
        before it, refused ones included (query_lens 0 if refused).
    slot_mapping, positions (num_tokens,): each token's cache slot (-1: none)
        and position.
    block_tables (batch, width): the requests' pages in key order, 0 behind
        them.
    free_count, refused (1,): blocks left, requests refused.
    """

    seq_lens: torch.Tensor
    query_start: torch.Tensor
    query_lens: torch.Tensor
    slot_mapping: torch.Tensor
    positions: torch.Tensor
    block_tables: torch.Tensor
    free_count: torch.Tensor
    refused: torch.Tensor


def _check_pool(block_tables, seq_lens, free_blocks, free_count, block_size):
    dev = block_tables.device
    assert block_tables.is_cuda and block_tables.dim() == 2 and block_tables.dtype == torch.int32, \
        "block_tables must be int32 (rows, width) on the device"
    assert block_tables.shape[1] >= 1 and block_tables.stride(1) == 1 and \
        (block_tables.shape[0] <= 1 or block_tables.stride(0) >= block_tables.shape[1]), \
        "block_tables rows must be contiguous and apart"
    for name, t, shape in (("seq_lens", seq_lens, (block_tables.shape[0],)), ("free_count", free_count, (1,))):
        assert t.dtype == torch.int32 and tuple(t.shape) == shape and t.device == dev and t.is_contiguous(), \
            f"{name} must be contiguous int32 {shape} on block_tables' device"
    assert free_blocks.dtype == torch.int32 and free_blocks.dim() == 1 and free_blocks.device == dev and \
        free_blocks.is_contiguous(), "free_blocks must be contiguous int32 (num_blocks,)"
    assert 1 <= block_size <= _lib.GQA_MAX_BLOCK_SIZE and block_size & (block_size - 1) == 0, \
        "block_size must be a power of two"
    assert block_tables.shape[1] * block_size < 1 << 31, "block_tables' capacity must be below 2**31 keys"
    return dev


def _check_ints(name, t, dev, n=None):
    assert t.dtype == torch.int32 and t.dim() == 1 and t.device == dev, f"{name} must be int32 on block_tables' device"
    assert n is None or t.shape[0] == n, f"{name} must have {n} entries"
    return t.contiguous()


def extend_block_tables(block_tables, seq_lens, query_lens, free_blocks, free_count, block_size: int,
                        num_tokens: int, *, rows: Optional[torch.Tensor] = None, update: bool = True) -> StepTables:
    """Append query_lens[b] tokens to the sequences of a batch.

    Args:
        block_tables: int32 (pool rows, width), a sequence's pages in key order;
            the new pages are entered here.
        seq_lens: int32 (pool rows,), keys of each sequence so far.
        query_lens: int32 (batch,), new tokens of each request.
        free_blocks, free_count: the free list, blocks free_blocks[:free_count]
            (int32 (num_blocks,) and (1,)); new pages come from its end, request
            by request.
        num_tokens: length of slot_mapping and positions, at least the sum of
            query_lens (tokens behind it are padding: slot -1, position 0).
        rows: int32 (batch,), the pool row of each request; a negative one is an
            empty place of the batch.  Default: row b.
        update: seq_lens and free_count move on in place.  False leaves them
            (the new values are in the result, the new pages in block_tables
            beyond the sequences' lengths): a plan of the step.

    A request is refused (slots -1, its sequence unchanged, counted in
    ``refused``) if its row is outside the pool or named by an earlier request,
    its tokens pass num_tokens, its pages the table's width, or if the free list
    ends before its pages; requests behind one that the free list refused get
    no page either.
    """
    if _lib._host is not None:
        res = _lib._host.extend_tables(block_tables, seq_lens, query_lens, free_blocks, free_count, block_size,
                                       num_tokens, rows, bool(update))  # every check passed, natively; else None
        if res is not None:
            return StepTables(*res)
    dev = _check_pool(block_tables, seq_lens, free_blocks, free_count, block_size)
    assert query_lens.dim() == 1 and num_tokens >= 0
    batch, (n_rows, width) = query_lens.shape[0], block_tables.shape
    query_lens = _check_ints("query_lens", query_lens, dev)
    if rows is None:
        assert batch <= n_rows, "more requests than pool rows"
    else:
        rows = _check_ints("rows", rows, dev, batch)
    lib = _lib.load()
    _decode_host()  # (the native call from here on)
    # One int32 allocation for the small outputs and the scratch.
    counts = [batch, batch, batch, num_tokens, 1, 1, n_rows + 2 * batch + 1]
    seq, start, qlen, pos, left, refused, scratch = torch.empty(sum(counts), dtype=torch.int32,
                                                                device=dev).split(counts)
    slots = torch.empty(num_tokens, dtype=torch.int64, device=dev)
    tables = torch.empty(batch, width, dtype=torch.int32, device=dev)
    with torch.cuda.device(dev):
        _lib.check(lib.gqa_extend_tables_launch(
            block_tables.data_ptr(), max(block_tables.stride(0), width), width, seq_lens.data_ptr(), n_rows,
            None if rows is None else rows.data_ptr(), query_lens.data_ptr(), free_blocks.data_ptr(),
            free_count.data_ptr(), free_blocks.shape[0], block_size, int(bool(update)), batch, num_tokens,
            seq.data_ptr(), start.data_ptr(), qlen.data_ptr(), slots.data_ptr(), pos.data_ptr(), tables.data_ptr(),
            left.data_ptr(), refused.data_ptr(), scratch.data_ptr(), stream_handle(dev)))
    return StepTables(seq, start, qlen, slots, pos, tables, left, refused)


def release_blocks(block_tables, seq_lens, rows, free_blocks, free_count, block_size: int) -> None:
    """Give the blocks of the sequences in ``rows`` (int32 (batch,)) back to the
    free list, in place; their lengths become 0.  Rows outside the pool and
    second mentions are passed over."""
    dev = _check_pool(block_tables, seq_lens, free_blocks, free_count, block_size)
    rows = _check_ints("rows", rows, dev)
    n_rows, width = block_tables.shape
    scratch = torch.empty(n_rows + 1, dtype=torch.int32, device=dev)
    with torch.cuda.device(dev):
        _lib.check(_lib.load().gqa_release_blocks_launch(
            block_tables.data_ptr(), max(block_tables.stride(0), width), width, seq_lens.data_ptr(), n_rows,
            rows.data_ptr(), rows.shape[0], free_blocks.data_ptr(), free_count.data_ptr(), free_blocks.shape[0],
            block_size, scratch.data_ptr(), stream_handle(dev)))


class BlockPool:
    """Tables, lengths and free blocks of up to max_seqs sequences, on the
    device.  Every block belongs to one sequence (``PagedKVCache`` shares
    prefixes)."""

    def __init__(self, num_blocks: int, block_size: int, max_seqs: int, max_seq_len: int, device="cuda"):
        assert num_blocks > 0 and max_seqs > 0 and max_seq_len > 0
        assert block_size > 0 and block_size & (block_size - 1) == 0, "block_size must be a power of two"
        self.block_size, self.num_blocks = block_size, num_blocks
        width = -(-max_seq_len // block_size)
        self.max_seq_len = width * block_size
        self.block_tables = torch.zeros(max_seqs, width, dtype=torch.int32, device=device)
        self.seq_lens = torch.zeros(max_seqs, dtype=torch.int32, device=device)
        self.free_blocks = torch.arange(num_blocks - 1, -1, -1, dtype=torch.int32, device=device)
        self.free_count = torch.full((1,), num_blocks, dtype=torch.int32, device=device)

    def step(self, query_lens, num_tokens: int, rows: Optional[torch.Tensor] = None) -> StepTables:
        """``extend_block_tables`` of this pool, in place."""
        return extend_block_tables(self.block_tables, self.seq_lens, query_lens, self.free_blocks, self.free_count,
                                   self.block_size, num_tokens, rows=rows)

    def release(self, rows) -> None:
        """``release_blocks`` of this pool."""
        release_blocks(self.block_tables, self.seq_lens, rows, self.free_blocks, self.free_count, self.block_size)
