"""The paged cache in 8 bits at the edges of what its calls allow."""
import pytest
import torch

from cache8_reference import CODES
from gqa_kernels import paged
from gqa_kernels.paged import PagedKVCache

BF = torch.bfloat16


def rand(*shape, dtype=BF, seed=0, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


# ---------------------------------------------------------------------------
# A sequence that comes more than once in an append
# ---------------------------------------------------------------------------
COMING_BACK = [(["a", "b", "a"], [3, 2, 4]), (["a", "a", "b"], [3, 2, 4]), (["a", "b", "a", "b", "b", "a"], [1, 20, 15, 1, 2, 16]), (["a", "b", "a"], [3, 0, 4]),
               (["b", "a", "c", "b"], [5, 1, 1, 1])]


@pytest.mark.parametrize("ids,new", COMING_BACK)
def test_a_page_is_one_run_of_each_store(ids, new, monkeypatch):
    """Two runs of a page in one store would be two workgroups over one exponent and the same tokens in front (no GPU here)."""
    cache, calls = PagedKVCache(12, 16, 2, 64, dtype=CODES, device="cpu"), []
    for s in "abc":
        cache.add_sequence(s)
    monkeypatch.setattr(paged, "write_kv", lambda k, v, kc, vc, slots, **kw: calls.append((k, slots)))
    for _ in range(2):
        calls.clear()
        key = torch.arange(sum(new)).view(-1, 1, 1).expand(-1, 2, 64)
        slots = cache.append(ids, key, key, new)
        assert torch.equal(torch.cat([s for _, s in calls]), slots) and torch.equal(torch.cat([k[:, 0, 0] for k, _ in calls]), torch.arange(sum(new)))
        assert len(slots.unique()) == sum(new)
        for _, s in calls:
            pages = torch.unique_consecutive(s // 16)
            assert len(pages) == len(pages.unique()), f"pages {pages.tolist()}"
    together = [i for i, n in zip(ids, new) if n]
    together = [i for j, i in enumerate(together) if not j or together[j - 1] != i]
    if len(set(together)) == len(together):
        assert len(calls) == 1
    cache = PagedKVCache(12, 16, 2, 64, device="cpu")  # 16 bits: one store
    for s in "abc":
        cache.add_sequence(s)
    calls.clear()
    cache.append(ids, key, key, new)
    assert len(calls) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("ids,new", COMING_BACK)
def test_append_of_a_sequence_that_comes_back(ids, new):
    """The pool as one store after the other leaves it, and every token within a rounding of what was appended."""
    cache, said = PagedKVCache(12, 16, 2, 64, dtype=CODES), {s: [] for s in "abc"}
    for s in "abc":
        cache.add_sequence(s)
    for step in range(3):
        key = rand(sum(new), 2, 64, seed=step, scale=4.0 ** step)
        size = torch.exp2(torch.arange(sum(new)) % 7 - 3.0).view(-1, 1, 1).cuda()
        key = (key * size).to(BF)
        cache.append(ids, key, -key, new)
        at = 0
        for s, n in zip(ids, new):
            said[s].append(key[at:at + n])
            at += n
    for s in "abc":
        x = torch.cat(said[s] + [key[:0]]).double()
        k, v = cache.read(s)
        assert torch.equal(k, -v) and k.shape == x.shape
        for a in range(0, x.shape[0], 16):
            page = slice(a, a + 16)
            # Half a step of the value twice (stored, brought to a larger exponent) and half the least step of the page's largest value, once a store.
            unit = x[page].abs().amax((0, 2))[:, None] / 224
            assert ((k[page].double() - x[page]).abs() <= 2 * 2.0 ** -4 * x[page].abs() + 16 * 2.0 ** -10 * unit).all()
