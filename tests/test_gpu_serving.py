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


def _calls():
    """Every operator as a call of its floating operands, and those."""
    def r(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, device="cuda", dtype=dtype)
    table, one = torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2), torch.ones(2, dtype=torch.int32, device="cuda")
    weight = ops.quantize_w4(r(16, 64), 64)
    return {
        "attention": (lambda q, k, v: ops.paged_attention(q, k, v, table, one), [r(2, 4, 16), r(4, 2, 8, 16), r(4, 2, 8, 16)]),
        "append": (lambda k, v, kp, vp, q, cos, sin: ops.paged_append(k, v, kp, vp, table, one, q=q, rope=(cos, sin)),
                   [r(2, 2, 16), r(2, 2, 16), r(4, 2, 8, 16), r(4, 2, 8, 16), r(2, 4, 16), r(9, 8, dtype=torch.float32), r(9, 8, dtype=torch.float32)]),
        "copy": (lambda p: ops.copy_pages(p, one[:1], one[:1] * 2), [r(4, 2, 8, 16)]),
        "w4": (lambda x, b, y: ops.linear_w4(x, weight, b, residual=y), [r(3, 64), r(16, dtype=torch.float32), r(3, 16)]),
    }


@pytest.mark.parametrize("op", ["attention", "append", "copy", "w4"])
def test_operands_whose_derivative_would_be_lost(op):
    import torch.autograd.forward_ad as forward
    call, operands = _calls()[op]
    call(*operands)
    for i, t in enumerate(operands):
        rest = operands[:i], operands[i + 1:]
        leaf = t.clone().requires_grad_()
        with pytest.raises(RuntimeError, match="no_grad"):
            call(*rest[0], leaf, *rest[1])
        with torch.no_grad():
            call(*rest[0], leaf, *rest[1])
        with forward.dual_level():
            dual = forward.make_dual(t.clone(), torch.ones_like(t))
            with pytest.raises(RuntimeError, match="tangent"):
                call(*rest[0], dual, *rest[1])
            call(*rest[0], forward.unpack_dual(dual).primal, *rest[1])
            with torch.inference_mode():
                call(*operands)


@pytest.mark.parametrize("dim", [0, 1, 2])
def test_copies_are_made_in_place(dim):
    pages = torch.randn(4, 6, 8, device="cuda")
    want = pages.clone()
    if dim < 2:
        want.select(dim, 2).copy_(pages.select(dim, 1))
    else:
        want[..., 2] = pages[..., 1]
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    assert ops.copy_pages(pages, one, one * 2, dim=dim) is pages
    assert torch.equal(pages, want)


# A result of many rows: rounding of the result, sums of k products in fp32, weights rounded to bf16 once (six standard deviations of 2^-8 of each, evenly
# spread), all at the GELU's largest slope; and the GELU itself in fp32, whose erf is off by up to two units in the last place: 2^-23 |z|, twice that here.
@pytest.mark.parametrize("rows,n,k,group", [(1, 512, 512, 128), (7, 7200, 256, 64), (16, 300, 96, 32), (20, 512, 512, 128), (48, 3072, 768, 128), (130, 1000, 1088, 64), (300, 2048, 64, 32),
                                            (600, 8192, 256, 128), (1025, 4099, 320, 64)])
@pytest.mark.parametrize("residual", [False, True])
def test_gelu_has_no_error_of_its_own(rows, n, k, group, residual):
    g = torch.Generator(device="cuda").manual_seed(n + rows)
    weight = ops.W4Weight.from_codes(torch.randint(0, 16, (n, k), generator=g, device="cuda", dtype=torch.uint8), torch.rand(n, k // group, generator=g, device="cuda") * 0.04)
    w = weight._plain().double()
    x = torch.randn(rows, k, generator=g, device="cuda").to(torch.bfloat16)
    bias = torch.randn(n, generator=g, device="cuda")
    add = torch.randn(rows, n, generator=g, device="cuda").to(torch.bfloat16) if residual else None
    y = ops.linear_w4(x, weight, bias, act="gelu", residual=add).double()
    z = x.double() @ w.t() + bias.double()
    want = 0.5 * z * torch.special.erfc(-z * 0.5 ** 0.5) + (add.double() if residual else 0.0)
    before = 2.0 ** -19 * (x.double().abs() @ w.abs().t() + bias.double().abs())
    if rows > 16:
        before = before + 6 * 2.0 ** -8 * ((x.double() ** 2) @ (w.t() ** 2) / 3).sqrt()
    assert ((y - want).abs() <= 2.0 ** -8 * want.abs() + 1.13 * before + 2.0 ** -22 * z.abs()).all()


def test_copies_into_pages_that_overlap_are_refused():
    memory = torch.arange(64, dtype=torch.float32, device="cuda")
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    for size, stride in (((2, 4, 8), (8, 8, 1)), ((3, 3, 8), (16, 8, 1)), ((2, 3, 8), (12, 8, 1)), ((2, 4, 8), (4, 16, 1)), ((1, 4, 8), (0, 4, 1))):
        with pytest.raises(RuntimeError, match="overlap"):
            ops.copy_pages(memory.as_strided(size, stride), one, one * 2, dim=1)
    for size, stride in (((2, 4, 8), (32, 8, 1)), ((2, 4, 8), (8, 16, 1)), ((1, 4, 8), (1, 8, 1)), ((2, 1, 8), (8, 1, 1))):     # pages of two layers in turn, too
        pages = memory.clone().as_strided(size, stride)
        want = pages.clone()
        if size[1] > 2:
            want[:, 2] = want[:, 1]
        assert torch.equal(ops.copy_pages(pages, one, one * 2, dim=1), want)


def test_tokens_into_pages_that_overlap_are_refused():
    k, v = torch.randn(2, 2, 2, 16, device="cuda").to(torch.bfloat16)
    table, at = torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2), torch.ones(2, dtype=torch.int32, device="cuda")
    pages = torch.zeros(2, 4, 2, 8, 16, dtype=torch.bfloat16, device="cuda")
    for k_pages, v_pages in ((pages[0, :1].expand(4, -1, -1, -1), pages[1]), (pages[0], pages[1, :, :1].expand(-1, 2, -1, -1)), (pages[0], pages[0]),
                             (pages.view(8, 2, 8, 16)[:4], pages.view(8, 2, 8, 16)[3:7])):
        with pytest.raises(RuntimeError, match="paged_append"):
            ops.paged_append(k, v, k_pages, v_pages, table, at)
    assert not pages.any()
    ops.paged_append(k, v, pages[0], pages[1], table, at)
    both = torch.zeros(4, 2, 2, 8, 16, dtype=torch.bfloat16, device="cuda")     # keys and values of a page side by side
    ops.paged_append(k, v, both[:, 0], both[:, 1], table, at)
    assert torch.equal(both.transpose(0, 1), pages)
