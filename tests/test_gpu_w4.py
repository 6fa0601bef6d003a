"""Products with 4-bit weights against the formula in 64 bits.

Bounds: the result is rounded to bf16 (2^-8 of itself).  Few rows: codes times x are exact in fp32 and sums of k of them lose at most
k 2^-24 sum |x w|, in practice their root; 2^-19 sum |x w| covers both here (k <= 8192).  Many rows: the weights are rounded to bf16 once, 2^-8 of each
with either sign: six standard deviations of that sum, 6 * 2^-8 sqrt(sum (x w)^2 / 3).  The GELU's slope is at most 1.13."""
import pytest
import torch

from mccl_b200 import ops

pytestmark = pytest.mark.gpu


def make(n, k, group, seed=0, zeros=True):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
    scales = (torch.rand(n, k // group, generator=g) * 0.01 + 0.001).to(torch.bfloat16)
    z = torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8) if zeros else None
    w = (codes.view(n, -1, group).double() - (z.double() if zeros else torch.full(scales.shape, 8.0, dtype=torch.float64))[..., None]) * scales.double()[..., None]
    return ops.W4Weight.from_codes(codes.cuda(), scales.cuda(), None if z is None else z.cuda()), w.view(n, k).cuda()


def check(x, weight, w, bias=None, act="none", residual=None):
    y = ops.linear_w4(x, weight, bias, act=act, residual=residual)
    x2 = x.reshape(-1, x.shape[-1]).double()
    z = x2 @ w.t()
    if bias is not None:
        z = z + bias.double()
    want = 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5)) if act == "gelu" else z
    if residual is not None:
        want = want + residual.reshape(want.shape).double()
    bound = 2.0 ** -19 * (x2.abs() @ w.abs().t())
    if x2.shape[0] > 16:   # rows enough for the weights to be rounded
        bound = bound + 6 * 2.0 ** -8 * ((x2 ** 2) @ (w.t() ** 2) / 3).sqrt()
    bound = 2.0 ** -8 * want.abs() + 1.13 * bound + 1e-6
    if act == "gelu" and x2.shape[0] > 16:   # the many-row epilogue's own erf
        bound = bound + 2.0 ** -8 * z.abs()
    assert y.shape == (*x.shape[:-1], w.shape[0]) and y.dtype == torch.bfloat16
    worst = ((y.reshape(want.shape).double() - want).abs() / bound).max().item()
    assert worst <= 1.0, worst


def x_of(*shape, seed=1):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda()


@pytest.mark.parametrize("rows", [1, 2, 3, 7, 8, 9, 15, 16, 17, 31, 33, 48, 64, 65, 100, 128, 129, 250, 600])
@pytest.mark.parametrize("n,k,group", [(512, 512, 128), (200, 1088, 64)])
def test_rows(rows, n, k, group):
    weight, w = make(n, k, group)
    check(x_of(rows, k), weight, w)


@pytest.mark.parametrize("rows", [1, 5, 40])
@pytest.mark.parametrize("n,k,group", [(1, 32, 32), (3, 64, 32), (8, 96, 32), (15, 64, 64), (16, 128, 128), (17, 256, 256), (33, 544, 32), (1000, 2048, 128), (2048, 8192, 128),
                                       (4099, 64, 64), (129, 768, 256), (40, 8160, 32), (32000, 128, 64)])
def test_sizes(n, k, group, rows):
    weight, w = make(n, k, group, seed=n)
    assert torch.equal(weight.dequantize().double(), w.to(torch.bfloat16).double())
    check(x_of(rows, k), weight, w)


@pytest.mark.parametrize("rows", [1, 4, 30, 300])
@pytest.mark.parametrize("act,bias,residual", [("none", True, False), ("none", False, True), ("none", True, True), ("gelu", True, False), ("gelu", False, False), ("gelu", True, True)])
def test_epilogues(rows, act, bias, residual):
    weight, w = make(384, 256, 128, zeros=False)
    check(x_of(rows, 256), weight, w, torch.randn(384, device="cuda") if bias else None, act, x_of(rows, 384, seed=5) if residual else None)


@pytest.mark.parametrize("rows,n,k,group", [(600, 4096, 64, 32), (333, 20000, 128, 64), (1025, 4099, 320, 64), (700, 9000, 96, 32), (2049, 2100, 544, 32), (1000, 32000, 192, 64)])
@pytest.mark.parametrize("act", ["none", "gelu"])
def test_more_tiles_than_sms(rows, n, k, group, act):
    weight, w = make(n, k, group, seed=n)
    check(x_of(rows, k), weight, w, torch.randn(n, device="cuda"), act, x_of(rows, n, seed=3))


@pytest.mark.parametrize("rows", [3, 150])
def test_shapes_and_strides(rows):
    weight, w = make(96, 128, 64)
    wide = x_of(rows, 3, 200)
    check(wide[:, 1, 64:192], weight, w)                       # rows of a wider tensor
    check(wide[:, 1, 63:191], weight, w)                       # not on a 16-byte boundary
    check(wide[..., :128], weight, w, residual=x_of(rows, 3, 104)[..., :96])
    check(x_of(128, rows).t(), weight, w)
    check(x_of(128), weight, w)
    assert ops.linear_w4(x_of(0, 128), weight).shape == (0, 96)
    assert ops.linear_w4(x_of(2, 0, 128), weight).shape == (2, 0, 96)


@pytest.mark.parametrize("rows", [1, 20, 200])
def test_a_row_of_x_stays_its_own(rows):
    """An infinity or a NaN in one row of x reaches that row of the result alone."""
    weight, w = make(64, 256, 64)
    x = x_of(rows + 1, 256)
    want = ops.linear_w4(x, weight)
    x[rows // 2, 7] = float("inf")
    x[rows // 2, 9] = float("nan")
    y = ops.linear_w4(x, weight)
    other = torch.arange(rows + 1, device="cuda") != rows // 2
    assert torch.equal(y[other], want[other]) and y[rows // 2].isnan().any()


def test_the_same_bits_again_and_on_another_stream():
    weight, w = make(2048, 8192, 128)
    for rows in (1, 12, 100):
        x = x_of(rows, 8192)
        want = ops.linear_w4(x, weight)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = [ops.linear_w4(x, weight) for _ in range(3)]
        ops.linear_w4(x_of(3, 8192), weight)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(g, want) for g in got)


@pytest.mark.parametrize("n,k,group", [(1, 32, 32), (17, 96, 32), (16, 64, 64), (100, 256, 256), (130, 1088, 64)])
@pytest.mark.parametrize("zeros", [True, False])
def test_layout_is_the_same_on_both_devices(n, k, group, zeros):
    g = torch.Generator().manual_seed(n)
    codes, scales = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8), torch.randn(n, k // group, generator=g)
    z = torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8) if zeros else None
    cpu = ops.W4Weight.from_codes(codes, scales, z)
    gpu = ops.W4Weight.from_codes(codes.cuda(), scales.cuda(), None if z is None else z.cuda())
    assert torch.equal(cpu.codes, gpu.codes.cpu()) and torch.equal(cpu.params, gpu.params.cpu())
    apart = ops.W4Weight.from_codes(codes.t().contiguous().cuda().t(), scales.cuda(), None if z is None else z.cuda())
    assert torch.equal(apart.codes, gpu.codes)
    for bad_codes, bad_zeros in ((codes.clone().index_fill_(1, torch.tensor([k - 1]), 16), z), (codes, torch.full((n, k // group), 200, dtype=torch.uint8))):
        with pytest.raises(RuntimeError, match="0 to 15"):
            ops.W4Weight.from_codes(bad_codes.cuda(), scales.cuda(), None if bad_zeros is None else bad_zeros.cuda())


def test_quantize():
    w = torch.randn(130, 256, device="cuda") * 0.02
    w[3] = 0.0
    w[4] = 0.5
    weight = ops.quantize_w4(w, 64)
    step = (w.view(130, 4, 64).amax(-1).clamp(min=0) - w.view(130, 4, 64).amin(-1).clamp(max=0)) / 15
    # a code is at most half a step off, the zero point another half, the rounded scale 2^-8 of up to fifteen steps
    bound = (step * 1.06 + 1e-6).repeat_interleave(64, dim=1)
    assert ((weight._plain() - w).abs() <= bound).all()
    assert not weight._plain()[3].any()
    assert weight.shape == (130, 256) and weight.nbytes < 0.7 * 130 * 256
    check(x_of(2, 256), weight, weight._plain().double())


def test_refusals():
    weight, w = make(64, 128, 64)
    x = x_of(2, 128)

    def refused(*args, **kw):
        with pytest.raises(RuntimeError):
            ops.linear_w4(*args, **kw)

    refused(x.float(), weight)
    refused(x[:, :64], weight)
    refused(x, weight, torch.zeros(63, device="cuda"))
    refused(x, weight, torch.zeros(64, device="cuda", dtype=torch.bfloat16))
    refused(x, weight, torch.zeros(64))
    refused(x, weight, act="silu")
    refused(x, weight, residual=x)
    refused(x, weight, residual=x_of(2, 64).float())
    refused(x, weight.to("cpu"))
    refused(x.clone().requires_grad_(), weight)
    codes, scales = torch.zeros(4, 64, dtype=torch.uint8), torch.ones(4, 1)
    for args in ((codes.int(), scales), (codes, scales[:3]), (codes, scales.int()), (codes + 16, scales), (codes, scales, codes[:, :1] + 16), (codes, scales, scales),
                 (codes[:, :48], scales), (codes, torch.ones(4, 4)), (codes, torch.ones(4, 0)), (codes[0], scales)):
        with pytest.raises(RuntimeError, match="W4Weight"):
            ops.W4Weight.from_codes(*args)
    for args in ((torch.zeros(4, 100), 64), (torch.zeros(4, 96), 48), (torch.zeros(64), 64)):
        with pytest.raises(RuntimeError, match="quantize_w4"):
            ops.quantize_w4(*args)


def test_refuses_weights_off_their_boundaries():
    weight, w = make(64, 128, 64)
    x = x_of(2, 128)
    shifted = torch.zeros(weight.codes.numel() + 8, dtype=torch.uint8, device="cuda")[8:].view(weight.codes.shape)
    odd = torch.zeros(weight.params.numel() + 1, dtype=torch.int32, device="cuda")[1:].view(weight.params.shape)
    for codes, params in ((shifted, weight.params), (weight.codes, odd)):
        moved = ops.W4Weight(codes, params, 64, 128, 64)
        with pytest.raises(RuntimeError, match="boundary"):
            ops.linear_w4(x, moved)
        with pytest.raises(RuntimeError, match="boundary"):
            moved.dequantize()
    for group in (48, 16, 512):
        with pytest.raises(RuntimeError, match="laid out"):
            ops.linear_w4(x, ops.W4Weight(weight.codes, weight.params, 64, 128, group))
