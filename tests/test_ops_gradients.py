"""The operators around the attention have no derivative: inputs that would need one are refused, others take the native calls."""
import pytest
import torch
from torch.autograd import forward_ad

from gqa_kernels import RotaryTable, document_spans, gqa_flash_attn, qk_norm_rope, qk_norm_rope_write
from gqa_kernels.paged import paged_attention

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def inputs():
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g).to(BF).cuda()  # noqa: E731
    return {"q": r(1, 4, 6, 64), "k": r(1, 2, 40, 64), "v": r(1, 2, 40, 64), "slopes": torch.rand(4, generator=g).cuda(), "kc": r(3, 16, 2, 64),
            "vc": r(3, 16, 2, 64), "qt": r(6, 4, 64), "kt": r(6, 2, 64), "vt": r(6, 2, 64), "wq": r(64), "wk": r(64)}


def calls():
    rot = RotaryTable(64, 50)
    ints = lambda x, t=torch.int32: torch.tensor(x, dtype=t).cuda()  # noqa: E731
    table, lens, pos, slots = ints([[2, 0, 1]]), ints([40]), ints(range(6)), ints(range(6), torch.int64)
    docs = document_spans(ints([[0] * 40]))
    return {
        "flash": (("q", "k", "v", "slopes"), lambda x: gqa_flash_attn(x["q"], x["k"], x["v"], softcap=9.0, alibi_slopes=x["slopes"])),
        "documents": (("q", "k", "v"), lambda x: gqa_flash_attn(x["q"], x["k"], x["v"], documents=docs)),
        "paged": (("q", "kc", "vc", "slopes"), lambda x: paged_attention(x["q"], x["kc"], x["vc"], table, lens, softcap=9.0, alibi_slopes=x["slopes"])),
        "rope": (("qt", "kt", "wq", "wk"), lambda x: qk_norm_rope(x["qt"], x["kt"], pos, rot, q_weight=x["wq"], k_weight=x["wk"])),
        "write": (("qt", "kt", "vt", "wq", "wk"), lambda x: qk_norm_rope_write(x["qt"], x["kt"], x["vt"], pos, rot, x["kc"], x["vc"], slots,
                                                                               q_weight=x["wq"], k_weight=x["wk"])),
    }


@pytest.mark.parametrize("name", ["flash", "documents", "paged", "rope", "write"])
@pytest.mark.parametrize("mode", ["forward", "forward under no_grad", "backward"])
def test_what_would_lose_a_derivative_is_refused(name, mode):
    names, call = calls()[name]
    x = inputs()
    call(x)  # (the shape is planned: its next calls go natively)
    for n in names:
        if mode == "backward":
            y = {**x, n: x[n].clone().requires_grad_()}
            with pytest.raises(NotImplementedError):
                call(y)
            with torch.no_grad():
                call(y)
            continue
        with forward_ad.dual_level():
            y = {**x, n: forward_ad.make_dual(x[n].clone(), torch.ones_like(x[n]))}
            with pytest.raises(NotImplementedError):
                if "no_grad" in mode:
                    with torch.no_grad():
                        call(y)
                else:
                    call(y)
            call(x)
    call(x)


@pytest.mark.parametrize("name", ["flash", "paged"])
def test_learned_slopes_take_the_native_calls_under_no_grad(name, monkeypatch):
    _, call = calls()[name]
    x = inputs()
    x["slopes"].requires_grad_()
    with torch.no_grad():
        want = call(x)  # (plans the shape)

        def never(*a, **k):
            raise RuntimeError("the call went through Python's checks")

        monkeypatch.setattr("gqa_kernels.dispatch.check_score", never)
        monkeypatch.setattr("gqa_kernels.paged.check_score", never)
        assert torch.equal(call(x), want)
