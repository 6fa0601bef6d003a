"""Rotary positions against complex multiplication in 64 bits.

Bound of an element: two products and a sum in fp32 (3 * 2^-24 of |a c| + |b s|, at most 1.5 * |(a, b)|) and one rounding to 16 bits (u of the value).
"""
import math

import pytest
import torch

from mccl_b200 import ops

pytestmark = pytest.mark.gpu
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def exact(x, cos, sin, positions, layout):
    pairs = cos.shape[1]
    inside = (positions >= 0) & (positions < cos.shape[0])
    at = positions.long().clamp(0, cos.shape[0] - 1)
    z = torch.complex(cos.double(), sin.double())[at][:, None]
    y = x.detach().double().clone()
    part = y[..., :2 * pairs]
    a, b = (part[..., 0::2], part[..., 1::2]) if layout == "interleaved" else part.chunk(2, -1)
    w = torch.complex(a.contiguous(), b.contiguous()) * z
    y[..., :2 * pairs] = torch.view_as_real(w).flatten(-2) if layout == "interleaved" else torch.cat((w.real, w.imag), -1)
    size = torch.complex(a.contiguous(), b.contiguous()).abs()
    size = torch.stack((size, size), -1).flatten(-2) if layout == "interleaved" else torch.cat((size, size), -1)
    off = torch.zeros_like(y)
    off[..., :2 * pairs] = size
    return torch.where(inside[:, None, None], y, 0.0), off


def close(got, x, cos, sin, positions, layout):
    want, size = exact(x, cos, sin, positions, layout)
    bound = UNIT[x.dtype] * want.abs() + 4.5 * 2.0 ** -24 * size + (2.0 ** -25 if x.dtype == torch.float16 else 1e-38)   # (below fp16's normal numbers: half a step)
    assert got.dtype == x.dtype and got.shape == x.shape and got.is_contiguous()
    assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dim,turned", [(8, 8), (32, 32), (64, 16), (72, 72), (72, 24), (96, 96), (128, 128), (128, 64), (256, 256), (256, 8)])
@pytest.mark.parametrize("tokens,heads,kv_heads", [(1, 1, 1), (37, 8, 2), (700, 12, 12)])
def test_turns(tokens, heads, kv_heads, dim, turned, layout, dtype):
    g = torch.Generator().manual_seed(dim + turned)
    qkv = torch.randn(tokens, heads + 2 * kv_heads, dim, generator=g).to(dtype).cuda()
    q, k, _ = qkv.split([heads, kv_heads, kv_heads], dim=1)
    rope = ops.rotary_tables(500, turned)
    positions = torch.randint(0, 500, (tokens,), generator=g).to(torch.int32).cuda()
    a, b = ops.rotary(q, k, rope=rope, positions=positions, layout=layout)
    close(a, q, *rope, positions, layout)
    close(b, k, *rope, positions, layout)
    assert torch.equal(ops.rotary(q, rope=rope, positions=positions, layout=layout), a)
    if tokens <= 500:
        assert torch.equal(ops.rotary(k, rope=rope, layout=layout), ops.rotary(k, rope=rope, positions=torch.arange(tokens, dtype=torch.int32).cuda(), layout=layout))


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_large(layout):
    q = torch.randn(5000, 40, 128, device="cuda").to(torch.bfloat16)
    rope = ops.rotary_tables(5000, 96)
    close(ops.rotary(q, rope=rope, layout=layout), q, *rope, torch.arange(5000, device="cuda"), layout)


def test_positions_outside_the_tables_give_zeros():
    q = torch.randn(6, 4, 64, device="cuda").to(torch.bfloat16)
    rope = ops.rotary_tables(10, 32)
    positions = torch.tensor([-1, 0, 9, 10, -(1 << 31), (1 << 31) - 1], dtype=torch.int32, device="cuda")
    out = ops.rotary(q, rope=rope, positions=positions)
    close(out, q, *rope, positions, "interleaved")
    assert not out[[0, 3, 4, 5]].any() and out[1:3].any()
    assert not ops.rotary(q, rope=ops.rotary_tables(0, 32)).any()
    assert ops.rotary(q[:0], rope=rope).shape == (0, 4, 64) and ops.rotary(q[:, :0], rope=rope).shape == (6, 0, 64)


def test_agrees_with_what_the_cache_is_given():
    """The same tables and layout as paged_append: the same bits."""
    q, k = (torch.randn(20, h, 64, device="cuda").to(torch.bfloat16) for h in (4, 2))
    rope = ops.rotary_tables(40, 64)
    positions = torch.arange(3, 23, dtype=torch.int32, device="cuda")
    pages = torch.zeros(2, 1, 2, 64, 64, dtype=torch.bfloat16, device="cuda")
    table, rows = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.zeros(20, dtype=torch.int32, device="cuda")
    want = ops.paged_append(k, k, pages[0], pages[1], table, positions, rows=rows, q=q, rope=rope)
    a, b = ops.rotary(q, k, rope=rope, positions=positions)
    assert torch.equal(a, want) and torch.equal(b, pages[0, 0, :, 3:23].transpose(0, 1))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dim,turned", [(64, 64), (72, 24), (128, 64)])
def test_gradients(dim, turned, layout, dtype):
    """The transpose of a rotation is the rotation the other way; sums with any vector agree: <turn(x), g> = <x, turn'(g)> to their roundings."""
    q, k = (torch.randn(300, h, dim, device="cuda").to(dtype).requires_grad_() for h in (6, 2))
    rope = ops.rotary_tables(200, turned)
    positions = torch.randint(-2, 205, (300,), device="cuda").to(torch.int32)
    a, b = ops.rotary(q, k, rope=rope, positions=positions, layout=layout)
    ga, gb = (torch.randn(t.shape[::-1], device="cuda").to(dtype).permute(2, 1, 0) for t in (a, b))   # in any strides
    dq, dk = torch.autograd.grad((a, b), (q, k), (ga, gb))
    for got, g in ((dq, ga), (dk, gb)):
        close(got, g.contiguous(), rope[0], -rope[1], positions, layout)
    for x, y, g, d in ((q, a, ga, dq), (k, b, gb, dk)):
        left, right = (y.double() * g.double()), (x.double() * d.double())
        assert abs(left.sum() - right.sum()).item() <= UNIT[dtype] * (left.abs().sum() + right.abs().sum()).item() + 1e-3
    only, = torch.autograd.grad(ops.rotary(q, k, rope=rope, positions=positions, layout=layout)[0], q, ga)
    assert torch.equal(only, dq)
    alone, = torch.autograd.grad(ops.rotary(q, rope=rope, positions=positions, layout=layout), q, ga[:, :1].expand_as(ga) * 0 + ga)
    assert torch.equal(alone, dq)


def test_strides_and_graphs():
    rope = ops.rotary_tables(64, 64)
    wide = torch.randn(4, 64, 80, device="cuda").to(torch.bfloat16)
    q = wide.transpose(0, 1)[..., :64]   # heads outside, gaps between rows
    want = ops.rotary(q.contiguous(), rope=rope)
    assert torch.equal(ops.rotary(q, rope=rope), want)
    one = q[:, :1].expand(64, 3, 64)
    assert torch.equal(ops.rotary(one, rope=rope), want[:, :1].expand(64, 3, 64))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.rotary(q, rope=rope)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    positions = torch.arange(64, dtype=torch.int32, device="cuda")
    with torch.cuda.graph(graph):
        out = ops.rotary(q, rope=rope, positions=positions)
    positions.copy_(positions.flip(0))
    graph.replay()
    assert torch.equal(out, ops.rotary(q, rope=rope, positions=positions)) and not torch.equal(out, want)


def test_refusals():
    q, k = (torch.randn(8, h, 64, device="cuda").to(torch.bfloat16) for h in (4, 2))
    rope = ops.rotary_tables(8, 64)
    at = torch.arange(8, dtype=torch.int32, device="cuda")
    f = ops.rotary
    calls = [
        lambda: f(q, k, rope=rope, layout="other"), lambda: f(q.float(), rope=rope), lambda: f(q, k.half(), rope=rope), lambda: f(q, k[:5], rope=rope), lambda: f(q, k[..., :32], rope=rope),
        lambda: f(q[0], rope=rope), lambda: f(q, rope=ops.rotary_tables(8, 72)), lambda: f(q, rope=ops.rotary_tables(8, 12)), lambda: f(q, rope=(rope[0], rope[1][:5])),
        lambda: f(q, rope=(rope[0].double(), rope[1].double())), lambda: f(q, rope=(rope[0].cpu(), rope[1].cpu())), lambda: f(q, rope=(rope[0][:, :0], rope[1][:, :0])),
        lambda: f(q, rope=(rope[0].t(), rope[1].t())), lambda: f(q, rope=(rope[0].clone().requires_grad_(), rope[1])), lambda: f(q, rope=rope, positions=at.long()),
        lambda: f(q, rope=rope, positions=at[:5]), lambda: f(q, rope=rope, positions=at.cpu()), lambda: f(q[..., 1:57], rope=ops.rotary_tables(8, 32)), lambda: f(q[..., :60], rope=ops.rotary_tables(8, 32)),
        lambda: f(q.transpose(1, 2), rope=ops.rotary_tables(8, 8)), lambda: f(torch.autograd.forward_ad.make_dual(q, q), rope=ops.rotary_tables(8, 64)),
    ]
    with torch.autograd.forward_ad.dual_level():
        for i, call in enumerate(calls):
            with pytest.raises(RuntimeError):
                call()
                pytest.fail(f"call {i} was not refused")
    leaf = q.requires_grad_()
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(f(leaf, rope=ops.rotary_tables(8, 64)).float().sum(), leaf, create_graph=True)


def test_tables():
    cos, sin = ops.rotary_tables(200000, 64)
    at = torch.tensor([0, 1, 77, 131071, 199999], dtype=torch.float64)
    for i in (0, 5, 31):
        angle = at * 10000.0 ** (-2 * i / 64)
        assert torch.allclose(cos[at.long().cuda(), i].cpu().double(), angle.cos(), atol=2.0 ** -24) and torch.allclose(sin[at.long().cuda(), i].cpu().double(), angle.sin(), atol=2.0 ** -24)
    assert math.isclose(cos[1, 0].item(), math.cos(1.0), rel_tol=1e-6)
