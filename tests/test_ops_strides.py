"""Changed scores over K and V whose rows lie further apart than 32-bit byte offsets reach."""
import pytest
import torch

from gqa_kernels import gqa_flash_attn
from gqa_kernels._lib import GQAError
from gqa_kernels.dispatch import _scored_route
from gqa_kernels.paged import paged_attention
from ops_reference import attend64, check_attention

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def spread(x, step):
    """x (1, H, S, D) with its rows `step` elements apart."""
    _, H, S, D = x.shape
    far = torch.empty((S - 1) * step + H * D, dtype=x.dtype, device="cuda").as_strided(x.shape, (S * step, D, step, 1))
    far.copy_(x)
    return far


@pytest.mark.parametrize("Hq,Hkv,Sq,Skv,D", [(8, 2, 8, 300, 64), (8, 2, 16, 64, 64), (8, 2, 16, 100, 128), (32, 8, 16, 100, 128), (8, 2, 1, 300, 64)])
def test_a_call_does_not_depend_on_the_one_before(Hq, Hkv, Sq, Skv, D):
    """Few rows per kv head: rows close by in the single pass (but for one token), far ones in the split pass, in any order."""
    g = torch.Generator().manual_seed(Sq)
    q, k, v = (torch.randn(1, h, s, D, generator=g).to(BF).cuda() for h, s in ((Hq, Sq), (Hkv, Skv), (Hkv, Skv)))
    want = attend64(q[0], k[0], v[0], softcap=20.0)
    step = (1 << 30) // (Skv + 192) // 8 * 8 + 8
    kf, vf = spread(k, step), spread(v, step)
    near_kind, far_kind = (_scored_route(q, x, y, True, 0, False).kind for x, y in ((k, v), (kf, vf)))
    assert far_kind == "split" and (near_kind == "single" or Sq == 1)
    first = None
    for far in (True, False, True, True, False):
        o, lse = gqa_flash_attn(q, kf if far else k, vf if far else v, return_lse=True, softcap=20.0)
        check_attention(o[0], lse[0], want)
        if far:
            assert first is None or torch.equal(o, first)
            first = o


@pytest.mark.parametrize("softcap", [None, 20.0])
@pytest.mark.parametrize("route", ["single", "chunks"])
def test_slots_far_apart_over_pages(route, softcap):
    """64 slots of a page as far apart as 32-bit offsets reach; one step more is refused there, and taken by the split pass."""
    bs, D, Hkv, Sq, lens = 64, 128, 2, 40, [130, 64]
    most = ((1 << 32) - 2 * D - 2) // (63 * 2) // 8 * 8
    g = torch.Generator().manual_seed(1)
    q = torch.randn(2, 8, Sq, D, generator=g).to(BF).cuda()
    near = torch.randn(2, 5, bs, Hkv, D, generator=g).to(BF).cuda()
    table = torch.tensor([[4, 0, 2], [1, 0, 0]], dtype=torch.int32).cuda()
    sl = torch.tensor(lens, dtype=torch.int32).cuda()
    call = lambda k, v, r: paged_attention(q, k, v, table, sl, True, softcap=softcap, route=r)  # noqa: E731
    want = call(near[0], near[1], route)
    for step in (most, most + 8):
        far = [torch.empty(63 * step + 5 * Hkv * D, dtype=BF, device="cuda").as_strided((5, bs, Hkv, D), (Hkv * D, step, D, 1)) for _ in range(2)]
        for f, x in zip(far, near):
            f.copy_(x)
        if step == most:
            assert torch.equal(call(*far, route), want)
        else:
            with pytest.raises(GQAError, match="4 GiB"):
                call(*far, route)
        o = call(*far, "split")
        for b, n in enumerate(lens):
            k, v = (x[table[b].long()].reshape(-1, Hkv, D)[:n].transpose(0, 1) for x in near)
            check_attention(o[b], None, attend64(q[b], k, v, softcap=softcap or 0.0))
        del far, f

