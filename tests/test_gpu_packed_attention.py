"""Causal attention of packed texts against the formula in 64 bits.

Bound of an element, from the roundings there are: the result is rounded to 16 bits (u |o|), and so are the weights before the product with V
(u sum p |v|); scores and sums are in fp32, which moves a weight by less than 2e-4 of itself (128 products of up to some 30 each, 2^-24 apiece).
"""
import math

import pytest
import torch

from mccl_b200 import ops

pytestmark = pytest.mark.gpu
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def offsets_of(lengths, begin=0):
    return torch.cumsum(torch.tensor([begin, *lengths]), 0).to(torch.int32).cuda()


def make(lengths, heads, kv_heads, dim, dtype=torch.bfloat16, seed=0, before=None, begin=0, spare=0, poison=True):
    """q, k, v as parts of one tensor (or, with keys from before, of two), NaN in all rows of no text, and the offsets."""
    g = torch.Generator().manual_seed(seed)

    def rows(n, h, used):
        x = torch.randn((n, h, dim), generator=g).to(dtype).cuda()
        if poison:
            x[:begin], x[begin + used:] = math.nan, math.nan
        return x

    total = sum(lengths)
    if before is None:
        q, k, v = rows(begin + total + spare, heads + 2 * kv_heads, total).split([heads, kv_heads, kv_heads], dim=1)
        return q, k, v, offsets_of(lengths, begin), None
    keys = [n + m for n, m in zip(lengths, before)]
    q = rows(begin + total + spare, heads, total)
    k, v = rows(begin + sum(keys) + spare, 2 * kv_heads, sum(keys)).split(kv_heads, dim=1)
    return q, k, v, offsets_of(lengths, begin), offsets_of(keys, begin)


def exact(q, k, v, offsets, k_offsets, scale, window=None, sinks=0):
    """(o, sum p |v|, lse) in 64 bits."""
    group = q.shape[1] // k.shape[1]
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    spread, lse = torch.zeros_like(o), torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
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
        any_seen = seen.any(1)
        for h in range(q.shape[1]):
            score = (q[rows, h].double() @ k[cols, h // group].double().T) * scale
            score = score.masked_fill(~seen, -math.inf)
            w = torch.softmax(score, 1).masked_fill(~seen, 0.0)
            o[rows, h] = w @ v[cols, h // group].double()
            spread[rows, h] = w @ v[cols, h // group].double().abs()
            lse[rows, h] = torch.where(any_seen, torch.logsumexp(score, 1), -math.inf)
    return o, spread, lse


def close(o, lse, want, dtype):
    (want, spread, want_lse), u = want, UNIT[dtype]
    assert ((o.double() - want).abs() <= u * want.abs() + (u + 2e-4) * spread + 1e-7).all()
    assert (lse.double() - want_lse).abs().max().item() < 2e-4


def check(q, k, v, offsets, k_offsets=None, scale=None, window=None, sinks=0):
    scale_ = q.shape[-1] ** -0.5 if scale is None else scale
    o, lse = ops.packed_attention(q, k, v, offsets, k_offsets, scale=scale, window=window, sinks=sinks, return_lse=True)
    want, spread, want_lse = exact(q, k, v, offsets, k_offsets, scale_, window, sinks)
    u = UNIT[q.dtype]
    bound = u * want.abs() + (u + 2e-4) * spread + 1e-7
    assert o.shape == q.shape and o.dtype == q.dtype and o.is_contiguous()
    assert torch.isfinite(o).all()
    worst = ((o.double() - want).abs() / bound).max().item() if o.numel() else 0.0
    assert worst <= 1.0, worst
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse), empty)
    assert (lse.double() - want_lse)[~empty].abs().max().item() < 2e-4 if (~empty).any() else True
    assert torch.equal(ops.packed_attention(q, k, v, offsets, k_offsets, scale=scale, window=window, sinks=sinks), o)   # the same bits again
    return o


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths", [[1], [37], [128], [129], [256], [257], [700], [5, 0, 300, 1, 128, 64]])
def test_lengths(lengths, dtype):
    check(*make(lengths, 4, 4, 64, dtype))


@pytest.mark.parametrize("dim", [8, 16, 24, 32, 64, 72, 80, 96, 104, 128])
@pytest.mark.parametrize("heads,kv_heads", [(3, 3), (4, 2), (6, 2), (8, 1)])
def test_head_layouts(dim, heads, kv_heads):
    check(*make([130, 61, 300], heads, kv_heads, dim, seed=dim))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 128), (4, 1, 64)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 0), (128, 0), (129, 4), (200, 130), (1000, 3), (100, 700), (1 << 40, 5)])
def test_windows(window, sinks, heads, kv_heads, dim, dtype):
    check(*make([700, 90, 1, 513], heads, kv_heads, dim, dtype, seed=window % 1000), window=window, sinks=sinks)


@pytest.mark.parametrize("window,sinks", [(None, 0), (150, 0), (150, 9)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(3, 3, 128), (4, 2, 64)])
def test_keys_from_before(heads, kv_heads, dim, window, sinks):
    check(*make([1, 130, 64, 0, 257], heads, kv_heads, dim, before=[900, 77, 128, 40, 0], seed=3), window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1500, 0), (1500, 9), (3, 300)])
@pytest.mark.parametrize("lengths,before,heads,kv_heads,dim", [([1], [5000], 3, 1, 128), ([37, 0, 130], [3000, 10, 2500], 4, 2, 64), ([2100], None, 2, 2, 72), ([200], [1100], 8, 8, 32)])
def test_few_rows_over_many_keys(lengths, before, heads, kv_heads, dim, window, sinks, dtype):
    """Keys are shared out over several blocks and their results joined."""
    check(*make(lengths, heads, kv_heads, dim, dtype, before=before, begin=3, spare=5, seed=8), window=window, sinks=sinks)


def test_infinite_numbers_where_keys_are_shared_out():
    q, k, v, offsets, k_offsets = make([30, 20], 2, 2, 64, before=[2500, 1800], seed=6)
    good = ops.packed_attention(q, k, v, offsets, k_offsets)
    bad_v, bad_k = v.clone(), k.clone()
    bad_v[2520, 0, 5] = math.inf       # the 21st new position of the first text, ...
    bad_k[2520, 1, 7] = math.nan
    bad_v[2530 + 7, 1, 3] = math.nan   # ... and an early one of the second
    o = ops.packed_attention(q, bad_k, bad_v, offsets, k_offsets)
    assert torch.equal(o[:20], good[:20]) and torch.equal(o[30:, 0], good[30:, 0])
    assert not torch.isfinite(o[20:30, 0, 5]).any() and torch.isnan(o[20:30, 1]).all() and torch.isnan(o[30:, 1, 3]).all()
    keep = torch.arange(64, device="cuda")
    assert torch.equal(o[20:30, 0][:, keep != 5], good[20:30, 0][:, keep != 5]) and torch.equal(o[30:, 1][:, keep != 3], good[30:, 1][:, keep != 3])
    # scores that are all minus infinity have no softmax; where some are finite, those count
    low_k = k.clone()
    low_k[:2530] = -math.inf
    assert torch.isnan(ops.packed_attention(q.abs() + 0.1, low_k, v, offsets, k_offsets)[:30]).all()
    low_k[2529] = k[2529]
    o = ops.packed_attention(q.abs() + 0.1, low_k, v, offsets, k_offsets)
    assert torch.isnan(o[:29]).all() and torch.allclose(o[29].float(), v[2529].float(), rtol=2 ** -7)


def test_more_queries_than_keys():
    # the first 60, 300 and all of the queries stand in front of their first key
    o = check(*make([100, 500, 70], 4, 2, 64, before=[-60, -300, -70]))
    assert not o[:60].any() and not o[100:400].any() and not o[600:].any()


@pytest.mark.parametrize("heads,kv_heads", [(3, 3), (4, 2)])
def test_rows_of_no_text(heads, kv_heads):
    o = check(*make([40, 200], heads, kv_heads, 64, begin=7, spare=300))
    assert not o[:7].any() and not o[247:].any()


def test_no_texts_and_no_tokens():
    q, k, v, _, _ = make([5], 2, 2, 64)
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert not ops.packed_attention(q, k, v, none).any()
    assert ops.packed_attention(q[:0], k[:0], v[:0], none).shape == (0, 2, 64)
    o, lse = ops.packed_attention(q, k[:0], v[:0], torch.tensor([0, 5], dtype=torch.int32).cuda(), torch.zeros(2, dtype=torch.int32).cuda(), return_lse=True)
    assert not o.any() and torch.isinf(lse).all()


def test_many_texts():
    g = torch.Generator().manual_seed(1)
    check(*make(torch.randint(0, 30, (1500,), generator=g).tolist(), 2, 2, 64))


@pytest.mark.parametrize("scale", [1e-3, 1.0, 4.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scales(scale, dtype):
    """Scores of up to a hundred and more, whose maximum grows from block to block.  A score is a sum of 64 products, off by up to 2^-24 of the sum of
    their sizes (times 4, some 60 * 4): weights move by e^(1e-4) at most, within the 2e-4 above."""
    q, k, v, offsets, _ = make([900], 2, 2, 64, dtype, seed=5)
    ramp = torch.linspace(0.1, 1.0, 900, device="cuda")[:, None, None]
    check(q * 0.5, (k * ramp).to(dtype), v, offsets, scale=scale)


def test_strides():
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(h, 300, 80, generator=g).to(torch.bfloat16).cuda().transpose(0, 1)[..., :64] for h in (4, 2, 2))   # heads outside, gaps between rows
    assert not q.is_contiguous()
    check(q, k, v, offsets_of([100, 200]))
    one = torch.randn(300, 1, 64, generator=g).to(torch.bfloat16).cuda()
    check(q, one.expand(300, 2, 64), v, offsets_of([100, 200]))


@pytest.mark.parametrize("what", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("window,sinks", [(None, 0), (100, 0), (100, 3)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 128), (4, 2, 64)])
def test_what_is_not_seen_has_no_influence(what, window, sinks, heads, kv_heads, dim):
    """Numbers that are not finite in one value of a head, and in one key of another: rows that do not see them keep their bits, all columns that the
    value does not belong to keep theirs."""
    q, k, v, offsets, _ = make([400, 300], heads, kv_heads, dim, seed=4)
    good = ops.packed_attention(q, k, v, offsets, window=window, sinks=sinks)
    for at in (0, 2, 127, 128, 130, 255, 300, 399):
        bad_v, bad_k = v.clone(), k.clone()
        bad_v[at, 0, 5] = what
        bad_k[at, 1, 7] = what
        o = ops.packed_attention(q, bad_k, bad_v, offsets, window=window, sinks=sinks)
        sees = torch.zeros(700, dtype=torch.bool, device="cuda")
        sees[at:400 if window is None or at < sinks else min(400, at + window)] = True
        assert torch.equal(o[~sees], good[~sees])
        group = heads // kv_heads
        columns = torch.ones(dim, dtype=torch.bool, device="cuda")
        columns[5] = False
        assert torch.equal(o[:, :group][..., columns], good[:, :group][..., columns])
        assert not torch.isfinite(o[sees][:, :group, 5]).any()
        if what != -math.inf and what != math.inf:
            assert torch.isnan(o[sees][:, group:2 * group]).all()


def test_other_texts_are_other_texts():
    q, k, v, offsets, _ = make([70, 200, 65], 2, 2, 128)
    o = ops.packed_attention(q, k, v, offsets)
    for s, (a, b) in enumerate(((0, 70), (70, 270), (270, 335))):
        x, y, z = (t.clone() for t in (q, k, v))
        for t in (x, y, z):
            t[a:b] = math.nan
        again = ops.packed_attention(x, y, z, offsets)
        assert torch.equal(again[:a], o[:a]) and torch.equal(again[b:], o[b:]) and torch.isnan(again[a:b]).all()


def test_graph_and_streams():
    q, k, v, offsets, _ = make([300, 77], 4, 2, 64, poison=False)
    want = ops.packed_attention(q, k, v, offsets)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a, b = ops.packed_attention(q, k, v, offsets), ops.packed_attention(q, k, v, offsets)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, want) and torch.equal(b, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.packed_attention(q, k, v, offsets)
    # other texts in the same tokens: nothing of the lengths is in the graph
    offsets.copy_(offsets_of([10, 367]))
    graph.replay()
    assert torch.equal(out, ops.packed_attention(q, k, v, offsets)) and not torch.equal(out, want)


def test_offsets_that_do_not_fit_stay_within_the_tensors():
    q, k, v, _, _ = make([300], 2, 2, 64, poison=False)
    for bad in ([-5, 100, 300], [0, 100, 1000], [0, 250, 100], [400, 500, 600], [-(1 << 31), (1 << 31) - 1, 0]):
        o = ops.packed_attention(q, k, v, torch.tensor(bad, dtype=torch.int32).cuda())
        assert o.shape == q.shape
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_weights_of_all_sizes(dtype):
    """One key that outweighs the others by up to 2^30, first, in the middle or last, and thousands whose weights count together."""
    n = 4000
    for place in (0, 1900, n - 1):
        q, k, v, offsets, _ = make([n], 2, 1, 64, dtype, poison=False, seed=place)
        q, k, v = (t.contiguous() for t in (q, k, v))
        q[..., 0], k[..., 0] = 8.0, 0.0
        k[place, :, 0] = 20.0   # a score of 20 more
        v.abs_()
        check(q, k, v, offsets)


def test_offsets_beyond_32_bits():
    """Keys and values, and then queries and results, whose elements are numbered past 2^31."""
    many = 1_070_000   # x 16 heads of 128: 2.19e9 elements
    k, v = (torch.empty(many, 16, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    for t in (k, v):
        t[-5000:].normal_()
    q = torch.randn(70, 32, 128, device="cuda").to(torch.bfloat16)
    o, lse = ops.packed_attention(q, k, v, offsets_of([70]), offsets_of([5000], many - 5000), return_lse=True)
    close(o, lse, exact(q, k[-5000:], v[-5000:], offsets_of([70]), offsets_of([5000]), 128 ** -0.5), torch.bfloat16)
    del k, v
    rows = 135_000     # x 128 heads of 128: 2.21e9 elements
    q = torch.empty(rows, 128, 128, dtype=torch.bfloat16, device="cuda")
    q[-300:].normal_()
    k, v = (torch.randn(300, 2, 128, device="cuda").to(torch.bfloat16) for _ in range(2))
    o, lse = ops.packed_attention(q, k, v, offsets_of([300], rows - 300), offsets_of([300]), return_lse=True)
    close(o[-300:], lse[-300:], exact(q[-300:], k, v, offsets_of([300]), None, 128 ** -0.5), torch.bfloat16)
    assert not o[:-300].any() and torch.isneginf(lse[:-300]).all()


def test_two_graphs_and_two_streams_at_once():
    """Each call has its own workspace (keys are shared out here)."""
    sets = [make([40, 60], 4, 2, 64, before=[3000, 2000], seed=s, poison=False) for s in (1, 2)]
    want = [ops.packed_attention(*x) for x in sets]
    graphs, outs = [], []
    for x in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.packed_attention(*x))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_refusals():
    q, k, v, offsets, _ = make([30], 4, 2, 64)
    f = ops.packed_attention
    bad = [
        lambda: f(q.float(), k.float(), v.float(), offsets), lambda: f(q, k.half(), v, offsets), lambda: f(q, k[..., :32], v[..., :32], offsets), lambda: f(q, k, v[:20], offsets),
        lambda: f(q[:, :3], k, v, offsets), lambda: f(q, k[:, :0], v[:, :0], offsets), lambda: f(q[0], k, v, offsets), lambda: f(q, k, v, offsets.long()),
        lambda: f(q, k, v, offsets.cpu()), lambda: f(q, k, v, offsets[:0]), lambda: f(q, k, v, offsets, offsets[:1]), lambda: f(q[:20], k, v, offsets),
        lambda: f(q, k, v, offsets, window=0), lambda: f(q, k, v, offsets, sinks=2), lambda: f(q, k, v, offsets, window=3, sinks=-1), lambda: f(q, k, v, offsets, scale=0.0),
        lambda: f(q, k, v, offsets, scale=-1.0), lambda: f(q, k, v, offsets, scale=math.nan), lambda: f(q[..., 1:57], k[..., 1:57], v[..., 1:57], offsets),
        lambda: f(q[..., ::2], k[..., ::2], v[..., ::2], offsets), lambda: f(q, k, v, torch.stack((offsets, offsets), 1)[:, 0]),
        lambda: f(*(torch.zeros(30, 2, 136, dtype=torch.bfloat16, device="cuda") for _ in range(3)), offsets),
        lambda: f(q.half().requires_grad_(), k.half(), v.half(), offsets),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was not refused")
