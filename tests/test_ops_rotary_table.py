"""RotaryTable as an object: its attributes are fixed, its copies hold tables of their own."""
import copy
import ctypes
import io
import pickle

import pytest
import torch

from gqa_kernels import RotaryTable, _lib, qk_norm_rope
from gqa_kernels.paged import GQAPagedAttention


def native(t):
    return ctypes.cast(t._native[1], ctypes.POINTER(_lib.Rope)).contents


def saved(t):
    f = io.BytesIO()
    torch.save(t, f)  # (our own file: pickle may run)
    f.seek(0)
    return torch.load(f, weights_only=False)


@pytest.mark.parametrize("make", [copy.deepcopy, lambda t: pickle.loads(pickle.dumps(t)), saved, copy.copy],
                         ids=["deepcopy", "pickle", "save", "copy"])
def test_copies(make):
    t = RotaryTable(64, 30, rotary_dim=32, interleaved=True, axes=[0] * 10 + [2] * 6, device="cpu")
    c = make(t)
    assert torch.equal(c.table, t.table) and (make is copy.copy or c.table.data_ptr() != t.table.data_ptr())
    for name in ("head_dim", "rotary_dim", "max_positions", "interleaved", "axes", "num_axes"):
        assert getattr(c, name) == getattr(t, name), name
    r = native(c)
    assert c._native[0] is c.table and r.table == c.table.data_ptr() and ctypes.addressof(r) != ctypes.addressof(native(t))
    assert (r.max_positions, r.rotary_dim, r.interleaved, r.axes) == (30, 32, 1, 3) and list(r.pair_axis) == list(native(t).pair_axis)


def test_attributes_are_fixed():
    t = RotaryTable(64, 30, device="cpu")
    for name, value in (("table", torch.zeros(30, 32, 2)), ("interleaved", True), ("max_positions", 40), ("axes", [0] * 32), ("another", 1)):
        with pytest.raises(AttributeError, match="fixed"):
            setattr(t, name, value)


def test_a_layer_with_a_table_can_be_copied():
    layer = GQAPagedAttention(8, 64, num_kv_heads=2, rotary=RotaryTable(64, 30, device="cpu"), q_norm_weight=torch.ones(64))
    c = copy.deepcopy(layer)
    assert torch.equal(c.rotary.table, layer.rotary.table) and c.rotary.table is not layer.rotary.table


@pytest.mark.gpu
def test_the_native_call_reads_the_table_that_there_is():
    g = torch.Generator().manual_seed(1)
    q = torch.randn(5, 4, 64, generator=g).to(torch.bfloat16).cuda()
    pos = torch.arange(5, dtype=torch.int32).cuda()
    t = RotaryTable(64, 30)
    qk_norm_rope(q, None, pos, t)
    qk_norm_rope(q, None, pos, t)
    c = copy.deepcopy(t)
    c.table.mul_(0.5)  # (written into: every call sees it)
    want = qk_norm_rope(q, None, pos, RotaryTable(64, 30))[0]
    assert torch.equal(qk_norm_rope(q, None, pos, t)[0], want) and torch.equal(qk_norm_rope(q, None, pos, c)[0], want * 0.5)
    new = torch.zeros_like(t.table)
    new[..., 0] = 1.0  # no rotation
    t.table.data = new
    assert torch.equal(qk_norm_rope(q, None, pos, t)[0], q)
