"""The plain forms of the operators around whole prompts (CPU tensors) against loops over single queries and tokens in 64 bits."""
import math

import pytest
import torch

from mccl_b200 import ops


def one_by_one(q, k, v, starts, key_starts, scale, window=None, sinks=0):
    o, lse = torch.zeros(q.shape, dtype=torch.float64), torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    group = q.shape[1] // k.shape[1]
    for s in range(len(starts) - 1):
        n, m = starts[s + 1] - starts[s], key_starts[s + 1] - key_starts[s]
        for i in range(n):
            p = m - n + i
            seen = [j for j in range(max(0, p + 1)) if window is None or j > p - window or j < sinks]
            if not seen:
                continue
            at = torch.tensor(seen) + key_starts[s]
            for h in range(q.shape[1]):
                score = k[at, h // group].double() @ q[starts[s] + i, h].double() * scale
                lse[starts[s] + i, h] = torch.logsumexp(score, 0)
                o[starts[s] + i, h] = torch.softmax(score, 0) @ v[at, h // group].double()
    return o, lse


@pytest.mark.parametrize("window,sinks", [(None, 0), (4, 0), (4, 2), (1, 0), (100, 3)])
@pytest.mark.parametrize("behind", [False, True])
def test_attention(window, sinks, behind):
    g = torch.Generator().manual_seed(1)
    starts = [2, 9, 9, 10, 30]
    key_starts = [0, 20, 25, 25, 40] if behind else starts   # keys from before; a text that has none; more queries than keys
    q = torch.randn(33, 4, 8, generator=g)
    k, v = (torch.randn(40 if behind else 33, 2, 8, generator=g) for _ in range(2))
    offsets = torch.tensor(starts, dtype=torch.int32)
    o, lse = ops.packed_attention(q, k, v, offsets, torch.tensor(key_starts, dtype=torch.int32) if behind else None, window=window, sinks=sinks, return_lse=True)
    want, want_lse = one_by_one(q, k, v, starts, key_starts, 8 ** -0.5, window, sinks)
    assert torch.allclose(o.double(), want, atol=1e-5) and torch.allclose(lse.double(), want_lse, atol=1e-5)
    assert not o[:2].any() and not o[30:].any()


def test_attention_gradients_against_differences():
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(12, h, 8, generator=g).requires_grad_() for h in (2, 1, 1))
    offsets = torch.tensor([0, 5, 12], dtype=torch.int32)
    direction = [torch.randn(t.shape, generator=g) for t in (q, k, v)]
    weight = torch.randn(12, 2, 8, generator=g)
    value = lambda *x: (ops.packed_attention(*x, offsets, window=4, sinks=1).double() * weight).sum()
    grads = torch.autograd.grad(value(q, k, v), (q, k, v))
    h = 1e-2
    up, down = (value(*(t.detach() + s * h * d for t, d in zip((q, k, v), direction))).item() for s in (1, -1))
    slope = sum((a.double() * d).sum().item() for a, d in zip(grads, direction))
    # 192 products of a result in fp32 (some 16 roundings of 2^-24 on values of about 1) and a weight of about 1: off by 2e-4 at most, over h;
    # h^2 / 6 times a third derivative of some 192 x 3 is below that
    assert abs((up - down) / (2 * h) - slope) < 2e-2 * max(1.0, abs(slope))


def test_attention_refusals():
    q = torch.randn(4, 2, 8)
    offsets = torch.tensor([0, 4], dtype=torch.int32)
    for options in ({"window": 0}, {"sinks": 2}):
        with pytest.raises(RuntimeError):
            ops.packed_attention(q, q, q, offsets, **options)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_rotary(layout):
    g = torch.Generator().manual_seed(3)
    q, k = torch.randn(7, 3, 16, generator=g), torch.randn(7, 1, 16, generator=g)
    rope = ops.rotary_tables(20, 8, device="cpu")
    at = torch.tensor([0, 3, 19, 20, -1, 5, 7], dtype=torch.int32)
    a, b = ops.rotary(q, k, rope=rope, positions=at, layout=layout)
    for x, y in ((q, a), (k, b)):
        for t in range(7):
            if not 0 <= at[t] < 20:
                assert not y[t].any()
                continue
            assert torch.equal(y[t, :, 8:], x[t, :, 8:])
            for i in range(4):
                lo, hi = (2 * i, 2 * i + 1) if layout == "interleaved" else (i, i + 4)
                angle = float(at[t]) * 10000.0 ** (-2 * i / 8)
                c, s = math.cos(angle), math.sin(angle)
                assert torch.allclose(y[t, :, lo], x[t, :, lo] * c - x[t, :, hi] * s, atol=1e-5)
                assert torch.allclose(y[t, :, hi], x[t, :, lo] * s + x[t, :, hi] * c, atol=1e-5)
    assert torch.equal(ops.rotary(q[:5], rope=rope, layout=layout), ops.rotary(q[:5], rope=rope, positions=torch.arange(5, dtype=torch.int32), layout=layout))
    with pytest.raises(RuntimeError):
        ops.rotary(q, rope=rope, layout="other")


def test_rotary_tables():
    plain = ops.rotary_tables(300, 64, device="cpu")
    assert plain[0].shape == (300, 32) and plain[0].dtype == torch.float32
    angle = lambda t: torch.atan2(t[1][1].double(), t[0][1].double())   # of position 1
    want = 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    assert torch.allclose(angle(plain), want, rtol=1e-5)
    assert torch.allclose(angle(ops.rotary_tables(2, 64, scaling="linear", factor=4.0, device="cpu")), want / 4, rtol=1e-5)
    base = angle(ops.rotary_tables(2, 64, scaling="base", factor=4.0, device="cpu"))
    assert torch.allclose(base[0], want[0]) and torch.allclose(base[-1], want[-1] / 4, rtol=1e-4)
    bands = angle(ops.rotary_tables(2, 64, scaling="bands", factor=4.0, original=2048, device="cpu"))
    turns = 2048 * want / (2 * math.pi)
    assert torch.allclose(bands[turns >= 32], want[turns >= 32], rtol=1e-5) and torch.allclose(bands[turns <= 1], want[turns <= 1] / 4, rtol=1e-4)
    assert bool((bands <= want * 1.00001).all()) and bool((bands >= want / 4 * 0.9999).all())
    far = ops.rotary_tables(1 << 20, 2, device="cpu")
    assert abs(far[0][-1, 0].item() - math.cos((1 << 20) - 1)) < 1e-7
    assert torch.equal(ops.rotary_tables(5, 8, magnitude=2.0, device="cpu")[0][0], torch.full((4,), 2.0))
    for options in ({"scaling": "other"}, {"scaling": "bands"}, {"factor": 0.0}, {"theta": -1.0}):
        with pytest.raises(RuntimeError):
            ops.rotary_tables(4, 8, device="cpu", **options)
    for bad in ((-1, 8), (4, 7), (4, 0)):
        with pytest.raises(RuntimeError):
            ops.rotary_tables(*bad, device="cpu")


def draw(x, u, t, k, p, low):
    if t == 0:
        return max(range(len(x)), key=lambda i: (x[i], -i))
    top = max(x)
    w = [math.exp((v - top) / t) for v in x]
    order = sorted(range(len(x)), key=lambda i: (-x[i], i))
    if k:
        order = order[:k]
    if p < 1:
        total, sum_, kept = sum(w[i] for i in order), 0.0, []
        for i in order:
            if kept and sum_ >= p * total:
                break
            kept.append(i)
            sum_ += w[i]
        order = kept
    order = sorted(i for i in order if w[i] >= low)
    aim, sum_ = u * sum(w[i] for i in order), 0.0
    for i in order:
        sum_ += w[i]
        if sum_ > aim:
            return i
    return order[-1]


def test_sample():
    g = torch.Generator().manual_seed(4)
    for t, k, p, low in ((1.0, 0, 1.0, 0.0), (0.5, 5, 1.0, 0.0), (2.0, 0, 0.7, 0.0), (1.0, 0, 1.0, 0.2), (0.75, 20, 0.9, 0.01), (0.0, 3, 0.5, 0.0), (1.0, 0, 0.0, 0.0)):
        x = (torch.randn(30, 50, generator=g) * 2).to(torch.bfloat16)
        u = torch.rand(30, generator=g)
        f = lambda v: torch.tensor(v, dtype=torch.float32).item()
        want = [draw(x[i].double().tolist(), u[i].item(), f(t), k, f(p), f(low)) for i in range(30)]
        assert ops.sample(x, u, temperature=t, top_k=k, top_p=p, min_p=low).tolist() == want
        rows = [torch.full((30,), v, dtype=torch.int32 if v is k and isinstance(k, int) else torch.float32) for v in (t, k, p, low)]
        assert ops.sample(x, u, temperature=rows[0], top_k=torch.full((30,), k, dtype=torch.int32), top_p=rows[2], min_p=rows[3]).tolist() == want
    x = torch.zeros(5, 8)
    x[0, 2], x[1, 3], x[2] = math.nan, math.inf, -math.inf
    assert ops.sample(x, torch.full((5,), 0.5), temperature=torch.tensor([1.0, 1.0, 1.0, -1.0, 1.0])).tolist() == [-1, -1, -1, -1, 4]
    for options in ({"temperature": -1.0}, {"top_p": 2.0}, {"min_p": -0.5}, {"top_k": -3}, {"temperature": math.nan}):
        with pytest.raises(RuntimeError):
            ops.sample(x, torch.rand(5), **options)
