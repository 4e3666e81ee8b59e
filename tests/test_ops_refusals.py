"""What the C entry points refuse before any HIP call, and which of them keep the interpreter's lock (no GPU here)."""
import ctypes

import pytest

from gqa_kernels import _lib

SHAPE, STRIDE = -1, -4
P = 0x10000  # an aligned address that is never read


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


@pytest.mark.parametrize("scored", [False, True])
@pytest.mark.parametrize("block,D,rows", [(64, 128, 64), (4096, 64, 64), (16, 128, 16), (32, 64, 16), (4, 128, 4), (8, 64, 8)])
def test_slots_of_a_page_past_32_bit_offsets(lib, block, D, rows, scored):
    """A descriptor's rows end past 4 GiB: the offsets would wrap and other keys be read."""
    q_st = _lib._i64x4(8 * 64 * D, 64 * D, D, 1)
    step = ((1 << 32) - 2 * D) // (2 * (rows - 1)) // 8 * 8 + 8
    for k_step, v_step in ((step, D), (D, step), (1 << 40, D)):
        kst, vst = (_lib._i64x4(1 << 20, s, D, 1) for s in (k_step, v_step))
        common = (1, 8, 2, 4, D, 0.1, 1, 0)
        head = (P, q_st, P, kst, P, vst, P, 8, P, None, None, block, 64 if block > 4 else 32, P, q_st, None)
        if scored:
            s = _lib.Score(softcap=10.0)
            for form, parts, ws in ((1, 0, None), (2, 2, P), (4, 0, None)):
                assert lib.gqa_paged_scored_launch(form, *head, ws, parts, *common, ctypes.byref(s), None) == STRIDE
        else:
            assert lib.gqa_paged_fwd_launch(*head, *common, None) == STRIDE
            assert lib.gqa_paged_fwd_short_launch(*head, *common, None) == STRIDE
            assert lib.gqa_paged_fwd_chunks_launch(*head, P, 2, *common, None) == STRIDE


def test_two_launches_over_a_shared_workspace_keep_the_lock(lib):
    """Another thread's call on the stream would write over the partials between the first pass and its combine."""
    for name in ("gqa_fwd_chunks_launch", "gqa_split_launch", "gqa_split_flat_launch", "gqa_paged_fwd_chunks_launch",
                 "gqa_paged_split_flat_launch"):
        fn = getattr(lib, name)
        assert fn._flags_ & ctypes._FUNCFLAG_PYTHONAPI and fn.argtypes == _lib.SIGNATURES[name][1], name
    assert not lib.gqa_fwd_split_launch._flags_ & ctypes._FUNCFLAG_PYTHONAPI  # (one launch: others run)
