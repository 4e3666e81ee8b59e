"""A step's query starts where requests have more tokens than there is room for: the sums of what was asked, in every form of the step."""
import pytest
import torch

from gqa_kernels.paged import extend_block_tables
from test_ops_tables import compare, ints, pool

pytestmark = pytest.mark.gpu
MOST = 2 ** 31 - 1


@pytest.mark.parametrize("T", [0, 7, 12, 300])
def test_starts_behind_a_request_that_passes_the_tokens(T):
    lens = [10, 16, 64, 0, 30]
    tables, free = pool(5, 40, 16, lens, spare=60)
    compare(tables, lens, [5, 100, 3, 0, 9], free, 16, T)
    compare(tables, lens, [200, 1, 1], free, 16, T, rows=[3, -1, 0])


@pytest.mark.parametrize("B", [3, 1025, 2048, 2049])
@pytest.mark.parametrize("n_rows", [3000, 5000])
def test_counts_past_32_bits_in_both_forms(B, n_rows):
    """Up to 2048 requests of 4096 rows in one launch, others in two: the same starts, the largest int32 where a sum is past it."""
    tables, lens, free = torch.zeros(n_rows, 4, dtype=torch.int32).cuda(), torch.zeros(n_rows, dtype=torch.int32).cuda(), ints(list(range(50)))
    new = [2, MOST, 1 << 20, -5] + [(b * 7919) % 600000 for b in range(B)]
    new = new[:B]
    r = extend_block_tables(tables, lens, ints(new), free, ints([50]), 16, 40, update=False)
    at, want = 0, []
    for n in new:
        want.append(min(at, MOST))
        at += max(n, 0)
    assert r.query_start.tolist() == want
    assert r.query_lens.tolist() == [2] + [0] * (B - 1) and r.refused.item() == B - 1 and r.seq_lens.tolist() == [2] + [0] * (B - 1)
    assert r.slot_mapping.tolist() == [49 * 16, 49 * 16 + 1] + [-1] * 38 and r.free_count.item() == 49
