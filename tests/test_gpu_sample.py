"""The choice of tokens against sorting in 64 bits, on a CPU.  Tokens are whole numbers and have to be equal.  Random numbers are drawn so that none falls on a
border: one that lies closer than 1e-7 of the whole to where the token changes is drawn again (sums of the kernel are off by less than 1e-10)."""
import math

import numpy as np
import pytest
import torch

from mccl_b200 import ops

pytestmark = pytest.mark.gpu


def kept_of(x, t, k, p, low):
    """(kept token numbers in ascending order, their weights, how near a border of top_p or min_p was) of one row."""
    weight = np.exp((x - x.max()) / t)
    order = np.lexsort((np.arange(len(x)), -x))
    if k > 0:
        order = order[:k]
    near = 1.0
    if p < 1:
        sums = np.cumsum(weight[order])
        near = min(near, np.abs(sums / sums[-1] - p).min())
        order = order[:1 + int(np.searchsorted(sums, p * sums[-1]))]
    if low > 0:
        near = min(near, np.abs(weight[order] - low).min() if low < 1 else 1.0)
        order = order[weight[order] >= low]
    order = np.sort(order)
    return order, weight[order], near


def check(logits, t=1.0, k=0, p=1.0, low=0.0, seed=0, wide=False):
    """Settings: numbers, or lists of one per row."""
    rows = logits.shape[0]
    rng = np.random.default_rng(seed)
    x = logits.double().cpu().numpy()
    each = [v if isinstance(v, list) else [v] * rows for v in (t, k, p, low)]
    f32 = lambda v: float(np.float32(v))
    want, uniform = [], []
    for r in range(rows):
        tt, kk, pp, ll = f32(each[0][r]), each[1][r], f32(each[2][r]), f32(each[3][r])
        if tt == 0:
            want.append(int(np.argmax(x[r])))
            uniform.append(rng.random())
            continue
        kept, weight, near = kept_of(x[r], tt, kk, pp, ll)
        assert near > 1e-9, "inputs that lie on a border"
        sums = np.cumsum(weight)
        while True:
            u = f32(rng.random()) if not wide else rng.random()
            if u < 1 and np.abs(sums / sums[-1] - u).min() > min(1e-7, 0.1 / len(kept)):
                break
        uniform.append(u)
        want.append(int(kept[min(len(kept) - 1, np.searchsorted(sums, u * sums[-1], side="right"))]))
    def arg(v, dtype):
        return torch.tensor(v, dtype=dtype, device="cuda") if isinstance(v, list) else v
    u = torch.tensor(uniform, dtype=torch.float64 if wide else torch.float32, device="cuda")
    call = lambda: ops.sample(logits, u, temperature=arg(t, torch.float32), top_k=arg(k, torch.int32), top_p=arg(p, torch.float32), min_p=arg(low, torch.float32))
    got = call()
    assert got.dtype == torch.int64 and got.tolist() == want
    assert torch.equal(call(), got)


def logits_of(rows, vocab, dtype, seed=0, spread=3.0):
    return (torch.randn(rows, vocab, generator=torch.Generator().manual_seed(seed)) * spread).to(dtype).cuda()


DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 2), (3, 31), (5, 100), (2, 4097), (1, 32000), (7, 32001), (70, 5000), (200, 1000), (2, 200003), (1, 1 << 20)])
def test_sizes(rows, vocab, dtype):
    x = logits_of(rows, vocab, dtype, seed=vocab)
    check(x)
    check(x, t=0.7, k=50, p=0.9, low=0.01, seed=1)
    check(x, t=0.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [0, 1, 2, 50, 1023, 1025, 20000, 49999, 50000, 70000, (1 << 31) - 1])
@pytest.mark.parametrize("p", [1.0, 0.999, 0.5, 0.01, 0.0])
def test_top_k_and_top_p(k, p, dtype):
    check(logits_of(3, 50000, dtype, seed=k % 1000), k=k, p=p, seed=2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t", [1e-20, 0.01, 0.3, 1.0, 5.0, 1000.0, 1e30])
@pytest.mark.parametrize("k,p,low", [(0, 1.0, 0.0), (300, 0.8, 0.0), (0, 0.7, 0.05), (0, 1.0, 1.0)])
def test_temperatures(t, k, p, low, dtype):
    check(logits_of(3, 20000, dtype, seed=4), t=t, k=k, p=p, low=low, seed=3)


@pytest.mark.parametrize("dtype", DTYPES)
def test_equal_logits(dtype):
    """Ties go to the lowest numbers; one step of the logit holds them all."""
    x = torch.zeros(4, 100000, dtype=dtype, device="cuda")
    for k, p in ((0, 1.0), (1, 1.0), (77777, 1.0), (0, 0.30001), (3000, 0.50001)):
        check(x, k=k, p=p, seed=5)
    x[:, ::2] = -1.0
    x[:, 5::1000] = 2.0
    for k, p in ((0, 1.0), (99, 1.0), (101, 1.0), (60000, 0.90001), (0, 0.20001)):
        check(x, k=k, p=p, seed=6)
    x[:, 3] = -0.0   # the same number as 0
    check(x, k=50101, seed=7)


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_tokens_are_not_drawn(dtype):
    x = logits_of(6, 30000, dtype, seed=8)
    x[:, 100:29000] = -math.inf
    check(x, k=500, p=0.95, seed=8)
    check(x, k=2000, seed=9)
    x[:, 100:29000] = torch.finfo(dtype).min
    check(x, t=0.5, k=500, p=0.95, seed=10)
    check(x, t=2.0, p=0.5, seed=11)
    x[:] = -math.inf
    x[:, 17] = -1e4
    assert ops.sample(x, torch.rand(6, device="cuda"), top_p=0.5, top_k=3).tolist() == [17] * 6
    assert ops.sample(x, torch.rand(6, device="cuda")).tolist() == [17] * 6


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_nothing_can_be_drawn_from(dtype):
    x = logits_of(8, 9000, dtype, seed=12)
    good = ops.sample(x, torch.full((8,), 0.25, device="cuda"), top_p=0.9)
    x[1, 4000], x[2, 8999], x[3, 0], x[4] = math.nan, math.inf, -math.nan, -math.inf
    t = torch.ones(8, device="cuda")
    t[5], t[6] = -1.0, math.nan
    for options in ({}, {"top_p": 0.9}, {"top_k": 5}, {"min_p": 0.1}):
        got = ops.sample(x, torch.full((8,), 0.25, device="cuda"), temperature=t, **options).tolist()
        assert got[1:7] == [-1] * 6 and got[0] >= 0 and got[7] >= 0
    assert ops.sample(x, torch.full((8,), 0.25, device="cuda"), temperature=t, top_p=0.9)[0] == good[0]
    assert ops.sample(x, torch.full((8,), 0.25, device="cuda"), temperature=0.0).tolist()[1:5] == [-1] * 4


@pytest.mark.parametrize("k", [0, 2500])
@pytest.mark.parametrize("low", [0.3, 0.9, 1.0, 0.01, 1e-6])
@pytest.mark.parametrize("off", [-1e-2, -1e-5, 1e-5, 1e-2])
def test_min_p_next_to_top_p(k, low, off):
    """What min_p keeps is a share of the weights that is a little above or below top_p."""
    x = torch.cat([torch.zeros(7), torch.full((40,), -1.0), torch.full((3000,), -4.0), torch.full((30000,), -9.0)])[torch.randperm(33047, generator=torch.Generator().manual_seed(3))]
    w = np.sort(np.exp(x.double().numpy()))[::-1][:k or None]
    p = min(0.9999, w[w >= low].sum() / w.sum() * (1 + off))
    check(x[None].expand(9, -1).cuda(), k=k, p=p, low=low)


def test_settings_of_each_row():
    rng = np.random.default_rng(13)
    rows = 90
    t = [0.0 if i % 9 == 0 else float(rng.uniform(0.2, 2.0)) for i in range(rows)]
    k = [int(rng.integers(0, 2000)) if i % 2 else 0 for i in range(rows)]
    p = [float(rng.uniform(0.1, 1.0)) if i % 3 else 1.0 for i in range(rows)]
    low = [float(rng.uniform(0.0, 0.1)) if i % 4 == 0 else 0.0 for i in range(rows)]
    for dtype in DTYPES:
        check(logits_of(rows, 12345, dtype, seed=14), t, k, p, low, seed=15, wide=True)


def test_every_token_has_its_share():
    """Numbers spread evenly over 0 to 1 give each of some tokens as often as its weight says, to one."""
    x = logits_of(1, 40, torch.float32, seed=16, spread=1.0)
    n = 20000
    u = (torch.arange(n, device="cuda", dtype=torch.float64) + 0.5) / n
    got = torch.bincount(ops.sample(x.expand(n, 40), u), minlength=40).double()
    assert bool(((got - n * torch.softmax(x[0].double(), -1)).abs() <= 1.0 + 1e-6).all())
    u = torch.tensor([-1.0, 0.0, 1.0, 2.0, math.nan], device="cuda")
    assert ops.sample(x.expand(5, 40), u).tolist() == [0, 0, 39, 39, 0]


def test_strides_streams_and_graphs():
    wide = logits_of(4, 1001, torch.bfloat16, seed=17)
    for x in (wide[:, :1000], wide[:, 1:], wide[::2], wide[:, 8:]):
        u = torch.rand(x.shape[0], device="cuda")
        assert torch.equal(ops.sample(x, u, top_k=20), ops.sample(x.contiguous(), u, top_k=20))
    x, u = logits_of(3, 40000, torch.float32, seed=18), torch.rand(3, device="cuda")
    t = torch.ones(3, device="cuda")
    want = ops.sample(x, u, temperature=t, top_p=0.9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(ops.sample(x, u, temperature=t, top_p=0.9), want)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.sample(x, u, temperature=t, top_p=0.9)
    graph.replay()
    assert torch.equal(out, want)
    x.copy_(logits_of(3, 40000, torch.float32, seed=19))
    t.fill_(0.5)
    graph.replay()
    assert torch.equal(out, ops.sample(x, u, temperature=0.5, top_p=0.9))
    assert ops.sample(x[:0], u[:0]).shape == (0,)


def test_agrees_with_the_plain_form():
    x, u = logits_of(40, 3000, torch.bfloat16, seed=20), torch.rand(40, generator=torch.Generator().manual_seed(21))
    for options in ({}, {"top_k": 30}, {"top_p": 0.8}, {"min_p": 0.02}, {"temperature": 0.0}, {"temperature": 0.6, "top_k": 100, "top_p": 0.9, "min_p": 0.001}):
        assert torch.equal(ops.sample(x, u.cuda(), **options).cpu(), ops.sample(x.cpu(), u, **options))


@pytest.mark.parametrize("temperature", [0.0, 1e-45, 1e-38, 1.3e-38, 2e-37, 1e-36, 1e-30])
def test_temperatures_next_to_zero(temperature):
    x = torch.randn(5, 1000, generator=torch.Generator().manual_seed(1)).cuda()
    u = torch.full((5,), 0.999, device="cuda")
    for settings in ({}, {"top_k": 7}, {"top_p": 0.5, "min_p": 0.1}):
        assert torch.equal(ops.sample(x, u, temperature=temperature, **settings), x.argmax(1))


def test_refusals():
    x, u = logits_of(2, 100, torch.float32), torch.rand(2, device="cuda")
    f = ops.sample
    calls = [
        lambda: f(x.double(), u), lambda: f(x[0], u), lambda: f(x[:, :0], u), lambda: f(x.t().contiguous().t(), u), lambda: f(x, u.half()), lambda: f(x, u[:1]), lambda: f(x, u.cpu()),
        lambda: f(x, u, temperature=-1.0), lambda: f(x, u, temperature=math.nan), lambda: f(x, u, top_k=-1), lambda: f(x, u, top_k=2.5), lambda: f(x, u, top_k=1 << 31), lambda: f(x, u, top_p=1.5), lambda: f(x, u, top_p=-0.1), lambda: f(x, u, min_p=2.0),
        lambda: f(x, u, temperature=u.double()), lambda: f(x, u, top_k=u), lambda: f(x, u, top_p=u[:1]), lambda: f(x, u, min_p=u.cpu()), lambda: f(x, u, temperature=math.inf),
        lambda: f(torch.zeros(1, (1 << 20) + 1, device="cuda"), u[:1]),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was not refused")
