"""A test's new stream is like one that no test has used, whichever tests ran before."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_every_stream_gets_a_workspace():
    from gqa_kernels import gqa_flash_attn, gqa_split
    q = torch.randn(1, 32, 1, 128, device="cuda").bfloat16()
    k = torch.randn(1, 8, 4096, 128, device="cuda").bfloat16()
    want = gqa_flash_attn(q, k, k)
    torch.cuda.synchronize()
    for _ in range(40):  # (more than there are)
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            assert torch.equal(gqa_flash_attn(q, k, k), want)
        s.synchronize()
        assert (torch.cuda.current_device(), s.cuda_stream) in gqa_split._workspaces


def test_the_next_test_finds_none():
    from gqa_kernels import gqa_split
    assert not gqa_split._workspaces
