"""Operators of token-by-token answers at operands and sizes where they went wrong, or could."""
import pytest
import torch

from mccl_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("offset", [1, 3, 16, 17])
@pytest.mark.parametrize("n,k,group", [(5, 64, 32), (17, 96, 32), (64, 256, 128)])
def test_codes_that_begin_on_any_byte(offset, n, k, group):
    g = torch.Generator().manual_seed(offset)
    codes = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8).cuda()
    zeros = torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8).cuda()
    scales = torch.rand(n, k // group, generator=g).cuda()
    want = ops.W4Weight.from_codes(codes, scales, zeros)

    def moved(t):
        room = torch.full((t.numel() + offset,), 255, dtype=torch.uint8, device="cuda")
        room[offset:] = t.flatten()
        return room[offset:].view(t.shape)

    got = ops.W4Weight.from_codes(moved(codes), scales, moved(zeros))
    assert torch.equal(got.codes, want.codes) and torch.equal(got.params, want.params)
