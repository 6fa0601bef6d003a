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


# Bound of an element of few rows, whose weights are whole numbers times a scale in fp32: rounding of the result (2^-8 of itself), and sums of k exact
# products in fp32, k 2^-24 of their absolute sum at the very worst and less than 2^-19 of it in practice, whose errors are not all of one sign.
@pytest.mark.parametrize("rows,n,k,group", [
    (8, 7104, 8192, 32), (8, 8192, 7328, 32), (8, 7200, 7296, 32), (7, 7104, 9344, 32), (7, 7111, 8352, 32), (4, 7104, 16384, 32), (4, 7120, 14624, 32), (2, 7104, 32768, 32),
    (1, 7104, 65536, 32), (1, 7110, 58784, 32), (8, 7104, 8192, 64), (8, 7104, 8192, 128), (8, 7088, 8192, 32), (16, 7104, 4096, 32), (9, 7104, 7168, 32)])
def test_few_rows_of_many_columns(rows, n, k, group):
    g = torch.Generator(device="cuda").manual_seed(k)
    codes = torch.randint(0, 16, (n, k), generator=g, device="cuda", dtype=torch.uint8)
    zeros = torch.randint(0, 16, (n, k // group), generator=g, device="cuda", dtype=torch.uint8)
    scales = (torch.rand(n, k // group, generator=g, device="cuda") * 0.01 + 0.001).to(torch.bfloat16)
    x = torch.randn(rows, k, generator=g, device="cuda").to(torch.bfloat16)
    y = ops.linear_w4(x, ops.W4Weight.from_codes(codes, scales, zeros)).double()
    want, size = torch.empty_like(y), torch.empty_like(y)
    for at in range(0, n, 1024):
        part = slice(at, at + 1024)
        w = (codes[part].view(-1, k // group, group).double() - zeros[part].double()[..., None]) * scales[part].double()[..., None]
        w = w.view(-1, k)
        want[:, part], size[:, part] = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    assert ((y - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -19 * size).all()


def test_more_rows_than_a_grid_has_in_a_column():
    # 256 rows of x per block and 65535 blocks along them are 16776960; x and y are 1.1 and 0.3 GB
    rows, n, k = 65535 * 256 + 1345, 9, 32
    g = torch.Generator(device="cuda").manual_seed(3)
    weight = ops.W4Weight.from_codes(torch.randint(0, 16, (n, k), generator=g, device="cuda", dtype=torch.uint8), torch.rand(n, 1, generator=g, device="cuda"))
    w = weight.dequantize().float()   # what many rows are multiplied with
    x = torch.randn(rows, k, generator=g, device="cuda", dtype=torch.bfloat16)
    y = ops.linear_w4(x, weight)
    for at in range(0, rows, 1 << 21):
        part = x[at:at + (1 << 21)].float()
        want, size = part @ w.t(), part.abs() @ w.abs().t()
        assert ((y[at:at + (1 << 21)].float() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18 * size).all()   # 32 products each, in fp32 on both sides
