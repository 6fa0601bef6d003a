"""Gradients of packed attention against the formula in 64 bits, and against differences.

Bound of an element, from the roundings there are (u = 2^-8, half a step of bf16).  Weights are off by w = 3e-4 of themselves (scores, sums and the saved
logarithm in fp32) and rounded before the product with dO: dV by u |dV| + (u + w) sum p |dO|.  delta is a sum over the rounded result: off by
sum |dO| (u |o| + (u + w) sum p |v|).  A score's gradient p (dP - delta) is rounded, and its parts are off by w p (|dP| + |delta|), p times delta's error, and
2e-5 p sum |dO v| (128 products in fp32): dQ and dK by u of themselves and the sum of that with |K| and |Q|.
"""
import math

import pytest
import torch

from mccl_b200 import ops
from tests.test_gpu_packed_attention import exact as exact_results
from tests.test_gpu_packed_attention import make, offsets_of

pytestmark = pytest.mark.gpu
U, W = 2.0 ** -8, 3e-4


def exact(q, k, v, g, offsets, k_offsets, scale, window=None, sinks=0):
    """((dq, dk, dv), their bounds) in 64 bits."""
    group = q.shape[1] // k.shape[1]
    grads = [torch.zeros(t.shape, dtype=torch.float64, device=q.device) for t in (q, k, v)]
    bounds = [torch.zeros_like(t) for t in grads]
    starts, keys = offsets.tolist(), (offsets if k_offsets is None else k_offsets).tolist()
    for s in range(len(starts) - 1):
        rows, cols = slice(starts[s], starts[s + 1]), slice(keys[s], keys[s + 1])
        n, m = rows.stop - rows.start, cols.stop - cols.start
        if n == 0 or m == 0:
            continue
        p, j = torch.arange(n, device=q.device)[:, None] + m - n, torch.arange(m, device=q.device)[None]
        seen = j <= p
        if window is not None:
            seen &= (j > p - window) | (j < sinks)
        for h in range(q.shape[1]):
            hk = h // group
            qq, gg, kk, vv = q[rows, h].double(), g[rows, h].double(), k[cols, hk].double(), v[cols, hk].double()
            weight = torch.softmax(((qq @ kk.T) * scale).masked_fill(~seen, -math.inf), 1).masked_fill(~seen, 0.0)
            o, dp = weight @ vv, gg @ vv.T
            delta = (gg * o).sum(1, keepdim=True)
            ds = weight * (dp - delta)
            delta_off = (gg.abs() * (U * o.abs() + (U + W) * (weight @ vv.abs()))).sum(1, keepdim=True)
            off = U * ds.abs() + weight * (delta_off + W * (dp.abs() + delta.abs()) + 2e-5 * (gg.abs() @ vv.abs().T))
            grads[0][rows, h] = scale * ds @ kk
            grads[1][cols, hk] += scale * ds.T @ qq
            grads[2][cols, hk] += weight.T @ gg
            bounds[0][rows, h] = scale * off @ kk.abs()
            bounds[1][cols, hk] += scale * off.T @ qq.abs()
            bounds[2][cols, hk] += (U + W) * weight.T @ gg.abs()
    return grads, [b + U * t.abs() + 1e-7 for t, b in zip(grads, bounds)]


def run(q, k, v, g, offsets, k_offsets=None, **options):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = ops.packed_attention(*leaves, offsets, k_offsets, **options)
    return o, torch.autograd.grad(o, leaves, g)


def check(q, k, v, offsets, k_offsets=None, scale=None, window=None, sinks=0, seed=9):
    g = torch.randn(q.shape, generator=torch.Generator().manual_seed(seed)).to(q.dtype).cuda()
    g[offsets[-1]:], g[:offsets[0]] = math.nan, math.nan
    o, grads = run(q, k, v, g, offsets, k_offsets, scale=scale, window=window, sinks=sinks)
    assert torch.equal(o, ops.packed_attention(q, k, v, offsets, k_offsets, scale=scale, window=window, sinks=sinks))
    want, bounds = exact(q, k, v, g, offsets, k_offsets, q.shape[-1] ** -0.5 if scale is None else scale, window, sinks)
    for name, got, x, bound in zip("qkv", grads, want, bounds):
        assert got.dtype == torch.bfloat16 and got.shape == x.shape
        assert torch.isfinite(got).all(), name
        worst = ((got.double() - x).abs() / bound).max().item() if got.numel() else 0.0
        assert worst <= 1.0, (name, worst)
    again = run(q, k, v, g, offsets, k_offsets, scale=scale, window=window, sinks=sinks)[1]
    assert all(torch.equal(a, b) for a, b in zip(grads, again))   # the same bits again
    return grads


@pytest.mark.parametrize("lengths", [[1], [37], [128], [129], [256], [257], [700], [5, 0, 300, 1, 128, 64]])
def test_lengths(lengths):
    check(*make(lengths, 4, 4, 64))


@pytest.mark.parametrize("dim", [8, 16, 24, 32, 64, 72, 96, 128])
@pytest.mark.parametrize("heads,kv_heads", [(3, 3), (6, 2), (8, 1)])
def test_head_layouts(dim, heads, kv_heads):
    check(*make([130, 61, 300], heads, kv_heads, dim, seed=dim))


@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 128), (4, 1, 64)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 0), (128, 0), (129, 4), (200, 130), (1000, 3), (100, 700), (1 << 40, 5)])
def test_windows(window, sinks, heads, kv_heads, dim):
    check(*make([700, 90, 1, 513], heads, kv_heads, dim, seed=window % 1000), window=window, sinks=sinks)


@pytest.mark.parametrize("window,sinks", [(None, 0), (150, 0), (150, 9)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(3, 3, 128), (4, 2, 64)])
def test_keys_from_before(heads, kv_heads, dim, window, sinks):
    check(*make([1, 130, 64, 0, 257], heads, kv_heads, dim, before=[900, 77, 128, 40, 0], seed=3), window=window, sinks=sinks)


def test_few_rows_over_many_keys():
    """The forward pass shares the keys out there."""
    check(*make([37, 130], 4, 2, 64, before=[3000, 2500], begin=3, spare=5, seed=8))
    check(*make([2100], 2, 2, 128, seed=9), window=1500, sinks=9)


def test_more_queries_than_keys():
    dq, _, _ = check(*make([100, 500, 70], 4, 2, 64, before=[-60, -300, -70]))
    assert not dq[:60].any() and not dq[100:400].any() and not dq[600:].any()


@pytest.mark.parametrize("heads,kv_heads", [(3, 3), (4, 2)])
def test_rows_of_no_text(heads, kv_heads):
    for t in check(*make([40, 200], heads, kv_heads, 64, begin=7, spare=300)):
        assert not t[:7].any() and not t[247:].any()


def test_keys_of_a_text_without_queries():
    _, dk, dv = check(*make([0, 5], 2, 2, 64, before=[200, 0]))
    assert not dk[:200].any() and not dv[:200].any()


def test_no_texts_and_no_tokens():
    q, k, v, _, _ = make([5], 2, 2, 64)
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert not any(t.any() for t in run(q, k, v, torch.ones_like(q), none)[1])
    assert [t.shape[0] for t in run(q[:0], k[:0], v[:0], q[:0], none)[1]] == [0, 0, 0]
    both = torch.tensor([0, 5], dtype=torch.int32).cuda(), torch.zeros(2, dtype=torch.int32).cuda()
    assert not run(q, k[:0], v[:0], torch.ones_like(q), *both)[1][0].any()
    assert not any(t.any() for t in run(q[:0], k, v, q[:0], both[1], both[0])[1])


def test_no_query_heads():
    """Their keys' gradients are zeros, not what was in the memory before."""
    q, k, v, offsets, _ = make([50], 4, 2, 64, poison=False)
    run(q, k, v, torch.ones_like(q), offsets)
    o, grads = run(q[:, :0], k, v, q[:, :0], offsets)
    assert o.shape == (50, 0, 64) and grads[0].shape == (50, 0, 64) and not grads[1].any() and not grads[2].any()


def test_many_texts():
    g = torch.Generator().manual_seed(1)
    check(*make(torch.randint(0, 30, (1500,), generator=g).tolist(), 2, 2, 64))


def test_gradients_in_any_strides_and_expanded_inputs():
    q, k, v, offsets, _ = make([300], 4, 2, 64, poison=False)
    want = run(q, k, v, torch.ones_like(q), offsets)[1]
    one = torch.ones((), dtype=q.dtype, device="cuda")
    for g in (one.expand(q.shape), torch.ones(64, 4, 300, dtype=q.dtype, device="cuda").permute(2, 1, 0), torch.ones(300, 4, 65, dtype=q.dtype, device="cuda")[..., 1:]):
        assert all(torch.equal(a, b) for a, b in zip(run(q, k, v, g, offsets)[1], want))
    # one head of keys that is handed over as two: its gradient is the sum of both
    single = k[:, :1].detach().clone().requires_grad_()
    o = ops.packed_attention(q, single.expand(300, 2, 64), v, offsets)
    got, = torch.autograd.grad(o, single, torch.ones_like(q))
    two = run(q, k[:, :1].expand(300, 2, 64).contiguous(), v, torch.ones_like(q), offsets)[1][1]
    assert torch.allclose(got[:, 0].float(), two.float().sum(1), rtol=2 * U, atol=1e-6)


def test_only_some_inputs_and_the_logarithm():
    q, k, v, offsets, _ = make([300], 4, 2, 64, poison=False)
    g = torch.ones_like(q)
    _, want = run(q, k, v, g, offsets)
    leaf = v.detach().requires_grad_()
    o, lse = ops.packed_attention(q, k, leaf, offsets, return_lse=True)
    assert not lse.requires_grad
    got, = torch.autograd.grad(o, leaf, g)
    assert torch.equal(got, want[2])
    with torch.no_grad():
        assert not ops.packed_attention(q, k, leaf, offsets).requires_grad


def test_against_differences():
    """Central differences of sum o g along the signs of the gradient.  They leave the slope by the truncation, which the formula in 64 bits gives for the same
    two points, by the results' roundings at both, sum |g| (u |o| + (u + w) sum p |v|) over 2 h each, and by the gradient's own bound along the step."""
    q, k, v, offsets, _ = make([200], 2, 1, 64, poison=False)
    g = torch.randn(q.shape, generator=torch.Generator().manual_seed(3)).to(q.dtype).cuda()
    _, grads = run(q, k, v, g, offsets)
    exact_grads, bounds = exact(q, k, v, g, offsets, None, 0.125)
    h = 0.25
    for i in range(3):
        up, down = ([x if j != i else (x + s * h * grads[i].sign()).to(x.dtype) for j, x in enumerate((q, k, v))] for s in (1, -1))
        step = (up[i].double() - down[i].double()) / (2 * h)   # as it is after rounding
        got, want, off = [], [], 0.0
        for x in (up, down):
            got.append((ops.packed_attention(*x, offsets).double() * g.double()).sum().item())
            o, spread, _ = exact_results(*x, offsets, None, 0.125)
            want.append((o * g.double()).sum().item())
            off += (g.double().abs() * (U * o.abs() + (U + W) * spread + 1e-7)).sum().item() / (2 * h)
        slope = (grads[i].double() * step).sum().item()
        truncation = abs((want[0] - want[1]) / (2 * h) - (exact_grads[i] * step).sum().item())
        bound = truncation + off + (bounds[i] * step.abs()).sum().item()
        assert abs((got[0] - got[1]) / (2 * h) - slope) <= bound, (i, got, slope, bound)
        assert bound < 0.6 * abs(slope), (i, slope, bound)   # a missing or doubled part would show


@pytest.mark.parametrize("heads,kv_heads,dim", [(3, 3, 128), (4, 2, 64)])
@pytest.mark.parametrize("lengths,before,window", [([1], None, None), ([1] * 40, None, None), ([1, 0, 5, 1, 100], None, None), ([300, 77, 1], None, 1), ([20, 1, 60], [700, 5, 0], 1),
                                                   ([3, 9], [-2, -9], None)])
def test_rows_of_one_key(lengths, before, window, heads, kv_heads, dim):
    """Their weight is one whatever the score is: no gradient of it, not even a rounded one."""
    dq, dk, _ = check(*make(lengths, heads, kv_heads, dim, before=before, seed=4), window=window)
    keys = lengths if before is None else [max(0, n + m) for n, m in zip(lengths, before)]
    row = key = 0
    for n, m in zip(lengths, keys):
        blind = max(0, n - m)
        assert not dq[row:row + blind].any()
        if window == 1:
            assert not dq[row:row + n].any() and not dk[key:key + m].any()
        elif m <= n and m > 0:
            assert not dq[row + blind].any()
            if m == 1:
                assert not dk[key].any()
        row, key = row + n, key + m


@pytest.mark.parametrize("lengths,before,window,sinks", [([3] * 100, None, None, 0), ([8] * 60, None, None, 0), ([20] * 30, None, None, 0), ([300, 77], None, 2, 0), ([300, 77], None, 5, 3),
                                                         ([4] * 90, [2] * 90, 3, 1), ([500], None, None, 0)])
def test_two_roundings_and_no_more(lengths, before, window, sinks):
    """dQ and dK are rounded themselves and are sums of gradients of scores that were rounded, each time by as much (root mean square): 2^0.5 times what rounding the exact ones
    leaves.  Everything else is a sixth of that at most, 1.5 times in all."""
    q, k, v, offsets, k_offsets = make(lengths, 4, 2, 64, before=before, poison=False, seed=len(lengths))
    g = torch.randn(q.shape, generator=torch.Generator().manual_seed(7)).to(q.dtype).cuda()
    want, _ = exact(q, k, v, g, offsets, k_offsets, 0.125, window, sinks)
    _, got = run(q, k, v, g, offsets, k_offsets, window=window, sinks=sinks)
    for name, a, b in list(zip("qkv", got, want))[:2]:
        assert (a.double() - b).norm() <= 1.5 * (b.to(torch.bfloat16).double() - b).norm(), name


def test_threads_that_have_done_nothing_yet():
    """Tensor maps need a context; a thread whose memory all comes from the cache may have none."""
    import threading
    q, k, v, offsets, _ = make([300, 40], 4, 2, 64, poison=False)
    g = torch.ones_like(q)
    want = run(q, k, v, g, offsets)
    got = []
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    thread = threading.Thread(target=lambda: got.append(ops.packed_attention(*leaves, offsets)))
    thread.start()
    thread.join()
    assert torch.equal(got[0], want[0])
    thread = threading.Thread(target=lambda: got.extend(torch.autograd.grad(got[0], leaves, g)))
    thread.start()
    thread.join()
    assert all(torch.equal(a, b) for a, b in zip(got[1:], want[1])) and len(got) == 4


def test_other_texts_are_other_texts():
    q, k, v, offsets, _ = make([70, 200, 65], 4, 2, 128)
    g = torch.ones_like(q)
    _, want = run(q, k, v, g, offsets)
    for a, b in ((0, 70), (70, 270), (270, 335)):
        x = [t.clone() for t in (q, k, v, g)]
        for t in x:
            t[a:b] = math.nan
        for got, t in zip(run(*x, offsets)[1], want):
            assert torch.equal(got[:a], t[:a]) and torch.equal(got[b:], t[b:])


def test_training_step_in_a_graph():
    q, k, v, offsets, _ = make([300, 77], 4, 2, 64, poison=False)
    g = torch.randn(q.shape, device="cuda").to(q.dtype)
    _, want = run(q, k, v, g, offsets)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(ops.packed_attention(*leaves, offsets), leaves, g)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = torch.autograd.grad(ops.packed_attention(*leaves, offsets), leaves, g)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(grads, want))
    offsets.copy_(offsets_of([10, 367]))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(grads, run(q, k, v, g, offsets)[1]))


def test_offsets_that_do_not_fit_stay_within_the_tensors():
    q, k, v, _, _ = make([300], 2, 2, 64, poison=False)
    for bad in ([-5, 100, 300], [0, 100, 1000], [0, 250, 100], [400, 500, 600], [-(1 << 31), (1 << 31) - 1, 0]):
        run(q, k, v, torch.ones_like(q), torch.tensor(bad, dtype=torch.int32).cuda())
    torch.cuda.synchronize()


def test_refusals():
    q, k, v, offsets, _ = make([30], 4, 2, 64, poison=False)
    leaf = q.detach().requires_grad_()
    o = ops.packed_attention(leaf, k, v, offsets)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(o.float().sum(), leaf, create_graph=True)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.packed_attention(torch.autograd.forward_ad.make_dual(q, q), k, v, offsets)
    o = ops.packed_attention(leaf, k, v, offsets)
    with torch.no_grad():
        leaf.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.float().sum().backward()
