"""Attention of single tokens over a paged cache, against the formula in 64 bits.

Bound of an element, from the roundings there are: the result is rounded to 16 bits (u |o|), and so may be the weights before the product with V
(u sum p |v|); scores and sums are in fp32, which moves a weight by less than 2e-4 of itself (256 products of up to some 30 each, 2^-24 apiece).
"""
import math

import pytest
import torch

from mccl_b200 import ops

pytestmark = pytest.mark.gpu
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def make(lengths, heads, kv_heads, dim, page, dtype=torch.bfloat16, seed=0, spare=3, width=None, layout="heads", poison=True):
    """Queries, pages in a random order with NaN wherever no token was written, a table that is -1 behind the last page."""
    g = torch.Generator().manual_seed(seed)
    needed = [-(-n // page) for n in lengths]
    total = sum(needed) + spare
    order = torch.randperm(total, generator=g)
    width = width or max(max(needed), 1)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    shape = (total, kv_heads, page, dim)
    k, v = torch.randn(shape, generator=g).to(dtype).cuda(), torch.randn(shape, generator=g).to(dtype).cuda()
    keep = torch.zeros(total, page, dtype=torch.bool)
    at = 0
    for b, n in enumerate(needed):
        table[b, :n] = order[at:at + n]
        for i in range(n):
            keep[order[at + i], :max(0, lengths[b] - i * page)] = True
        at += n
    if poison:
        hole = ~keep.cuda()[:, None, :, None].expand(shape)
        k[hole], v[hole] = math.nan, math.nan
    if layout == "tokens":   # [pages, page_size, kv_heads, dim] in memory
        k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    q = torch.randn((len(lengths), heads, dim), generator=g).to(dtype).cuda()
    return q, k, v, table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda")


def exact(q, k, v, table, lengths, scale, window=None, sinks=0):
    """(o, sum p |v|, lse) in 64 bits."""
    B, H, D = q.shape
    rep, page = H // k.shape[1], k.shape[2]
    o = torch.zeros(B, H, D, dtype=torch.float64, device=q.device)
    spread, lse = torch.zeros_like(o), torch.full((B, H), -math.inf, dtype=torch.float64, device=q.device)
    for b, n in enumerate(lengths.tolist()):
        j = torch.arange(min(n, table.shape[1] * page), device=q.device)
        n = len(j)
        if window is not None:
            j = j[(j >= n - window) | (j < sinks)]
        if not len(j):
            continue
        i = table[b].long()[j // page]
        kk, vv = (t[i, :, j % page].double().repeat_interleave(rep, dim=1) for t in (k, v))
        s = torch.einsum("hd,jhd->hj", q[b].double(), kk) * scale
        p = torch.softmax(s, -1)
        o[b] = torch.einsum("hj,jhd->hd", p, vv)
        spread[b] = torch.einsum("hj,jhd->hd", p, vv.abs())
        lse[b] = torch.logsumexp(s, -1)
    return o, spread, lse


def check(q, k, v, table, lengths, scale=None, window=None, sinks=0):
    scale_ = q.shape[-1] ** -0.5 if scale is None else scale
    o, lse = ops.paged_attention(q, k, v, table, lengths, scale=scale, window=window, sinks=sinks, return_lse=True)
    want, spread, want_lse = exact(q, k, v, table, lengths, scale_, window, sinks)
    u = UNIT[q.dtype]
    bound = u * want.abs() + (u + 2e-4) * spread + 1e-7
    assert o.shape == q.shape and o.dtype == q.dtype and o.is_contiguous()
    assert torch.isfinite(o).all()
    worst = ((o.double() - want).abs() / bound).max().item()
    assert worst <= 1.0, worst
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse), empty)
    assert (lse.double() - want_lse)[~empty].abs().max().item() < 2e-4 if (~empty).any() else True
    assert torch.equal(ops.paged_attention(q, k, v, table, lengths, scale=scale, window=window, sinks=sinks), o)   # the same bits again
    return o


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [8, 32, 40, 64, 72, 96, 128, 192, 256])
def test_head_dims(dim, dtype):
    check(*make([1, 37, 64, 65, 200], 4, 2, dim, 16, dtype))


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (12, 12), (6, 2), (8, 1), (16, 2), (24, 2), (40, 1), (33, 3), (5, 5)])
def test_head_layouts(heads, kv_heads):
    check(*make([3, 130, 517], heads, kv_heads, 64, 32))


@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 64, 100, 256, 1000])
def test_page_sizes(page):
    check(*make([1, page, page + 1, 2 * page - 1, 333], 4, 2, 64, page))


@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1023, 1025, 4099, 70001])
def test_lengths(length):
    check(*make([length], 8, 4, 128, 64))


@pytest.mark.parametrize("batch", [1, 2, 7, 64, 300])
def test_empty_and_ragged(batch):
    g = torch.Generator().manual_seed(batch)
    lengths = [int(x) for x in torch.randint(0, 400, (batch,), generator=g)]
    lengths[0] = 0
    q, k, v, table, n = make(lengths, 4, 2, 64, 16)
    o = check(q, k, v, table, n)
    assert not o[0].any()


def test_all_empty_and_no_sequences():
    q, k, v, table, n = make([0, 0, 0], 4, 2, 64, 16)
    o, lse = ops.paged_attention(q, k, v, table, n, return_lse=True)
    assert not o.any() and torch.isinf(lse).all() and (lse < 0).all()
    assert ops.paged_attention(q[:0], k, v, table[:0], n[:0]).shape == (0, 4, 64)
    # a table without columns: nothing can be seen
    assert not ops.paged_attention(q, k, v, table[:, :0], n).any()


@pytest.mark.parametrize("few,many", [(1, 30000), (40, 8000)])
def test_one_long_among_short(few, many):
    check(*make([few] * 20 + [many] + [few] * 11, 8, 8, 64, 16))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 3), (16, 16), (64, 4), (100, 37), (1000, 4), (10 ** 12, 7)])
@pytest.mark.parametrize("page", [16, 24])
def test_window_and_sinks(window, sinks, page):
    q, k, v, table, n = make([0, 1, 2, 3, 4, 5, 17, 63, 64, 104, 137, 500, 1003, 2000], 4, 2, 64, page)
    check(q, k, v, table, n, window=window, sinks=sinks)


def test_pages_out_of_the_window_are_not_looked_at():
    q, k, v, table, n = make([700, 333, 64], 4, 2, 64, 16)
    want = ops.paged_attention(q, k, v, table, n, window=50, sinks=5)
    gone = table.clone()
    for b, length in enumerate(n.tolist()):
        first, last = 1, (length - 50) // 16
        for i in range(first, last):
            k[table[b, i]], v[table[b, i]] = math.nan, math.inf   # the page has another owner now
            gone[b, i] = -1
    assert torch.equal(ops.paged_attention(q, k, v, gone, n, window=50, sinks=5), want)


def test_lengths_beyond_the_table_and_pages_outside_the_cache():
    q, k, v, table, n = make([160, 100], 4, 2, 64, 16)
    want, _, _ = exact(q, k, v, table, n, 0.125)
    more = n.clone()
    more[0] = 2 ** 31 - 1
    assert (ops.paged_attention(q, k, v, table, more).double() - want)[0].abs().max() < 0.02
    negative = n.clone()
    negative[1] = -5
    assert not ops.paged_attention(q, k, v, table, negative)[1].any()
    # a visible position without a page is left out
    holes = table.clone()
    holes[0, 0], holes[0, 3], holes[1, 2] = -1, k.shape[0], 2 ** 31 - 1
    o = ops.paged_attention(q, k, v, holes, n)
    for b, left in ((0, [j for j in range(160) if j // 16 not in (0, 3)]), (1, [j for j in range(100) if j // 16 != 2])):
        j = torch.tensor(left, device="cuda")
        kk, vv = (t[table[b].long()[j // 16], :, j % 16].double().repeat_interleave(2, dim=1) for t in (k, v))
        w = torch.einsum("hj,jhd->hd", torch.softmax(torch.einsum("hd,jhd->hj", q[b].double(), kk) * 0.125, -1), vv)
        assert (o[b].double() - w).abs().max() < 0.02
    assert ops.paged_attention(q, k, v, torch.full_like(table, -1), n).isnan().all()


def test_infinities_that_are_seen():
    # one key at -inf beside others takes no part; a NaN goes into its own head alone
    q, k, v, table, n = make([90], 4, 4, 64, 16)
    q.fill_(1.0)
    at = table[0, 2].item()
    k[at, 0, 5] = -math.inf
    k[at, 1, 5, 3] = math.nan
    o = ops.paged_attention(q, k, v, table, n)
    assert torch.isfinite(o[0, [0, 2, 3]]).all() and o[0, 1].isnan().all()
    j = torch.tensor([x for x in range(90) if x != 37], device="cuda")
    kk, vv = (t[table[0].long()[j // 16], 0, j % 16].double() for t in (k, v))
    want = torch.softmax(kk.sum(-1) * 0.125, -1) @ vv
    assert (o[0, 0].double() - want).abs().max() < 0.02


@pytest.mark.parametrize("size", [0.0, 30.0])
def test_scores_far_apart(size):
    # equal scores, and scores of which one decides
    q, k, v, table, n = make([1, 100, 1000], 8, 2, 64, 16)
    check(q * size, k, v, table, n)
    check(q, k, v, table, n, scale=0.9)


@pytest.mark.parametrize("layout", ["heads", "tokens"])
def test_strides(layout):
    q, k, v, table, n = make([5, 77, 300], 8, 2, 64, 16, layout=layout)
    want = check(q, k, v, table, n)
    wide = torch.zeros(3, 20, 96, dtype=q.dtype, device="cuda")[:, 4:12, 16:80]
    wide.copy_(q)
    both = torch.empty(2, *k.shape, dtype=k.dtype, device="cuda")
    both[0], both[1] = k, v
    columns = torch.zeros(3, table.shape[1] + 5, dtype=torch.int32, device="cuda")[:, 2:2 + table.shape[1]]
    columns.copy_(table)
    assert torch.equal(ops.paged_attention(wide, both[0], both[1], columns, n), want)


def test_offsets_beyond_32_bits():
    # a cache of 5 * 2^30 elements for each of K and V (10 GB in one allocation is enough: they overlap but for one page)
    page, dim, heads = 64, 128, 8
    pages = 5 * 2 ** 30 // (page * dim * heads)
    cache = torch.zeros(pages + 1, heads, page, dim, dtype=torch.bfloat16, device="cuda")
    q, k, v, table, n = make([64 * 6 - 3], heads, heads, dim, page, spare=0, poison=False)
    high = torch.tensor([pages - 2, 3, pages // 2 + 7, pages - 9, pages - 20, 11], dtype=torch.int32, device="cuda")
    for i in range(6):
        cache[high[i]] = k[table[0, i]]
    far = torch.stack([high])
    for i in range(6):
        cache[high[i] + 1] = v[table[0, i]]   # V is the same memory one page on
    o = ops.paged_attention(q, cache[:-1], cache[1:], far, n)
    assert torch.equal(o, ops.paged_attention(q, k, v, table, n))


def test_another_stream_and_a_graph():
    q, k, v, table, n = make([50, 3000, 7], 8, 2, 64, 16)
    want = ops.paged_attention(q, k, v, table, n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [ops.paged_attention(q, k, v, table, n) for _ in range(4)]
    # beside it, on this stream, calls of another shape
    for _ in range(4):
        ops.paged_attention(q[:2], k, v, table[:2], n[:2])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(o, want) for o in outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = ops.paged_attention(q, k, v, table, n)
    for lengths in ([50, 3000, 7], [1, 2, 3], [0, 2999, 0]):
        n.copy_(torch.tensor(lengths))
        graph.replay()
        assert torch.equal(captured, ops.paged_attention(q, k, v, table, n))


def test_refusals():
    q, k, v, table, n = make([50, 30], 4, 2, 64, 16)

    def refused(*args, **kw):
        with pytest.raises(RuntimeError, match="paged_attention"):
            ops.paged_attention(*args, **kw)

    refused(q.float(), k.float(), v.float(), table, n)
    refused(q.half(), k, v, table, n)
    refused(q, k, v.half(), table, n)
    refused(q[..., :60], k[..., :60], v[..., :60], table, n)          # head_dim not a multiple of 8
    refused(q[..., :56], k, v, table, n)
    refused(q[:, :3], k, v, table, n)                                  # heads that do not share evenly
    refused(q, k, v[:-1], table, n)
    refused(q, k, v, table.long(), n)
    refused(q, k, v, table, n.long())
    refused(q, k, v, table[:1], n)
    refused(q, k, v, table, n[:1])
    refused(q[0], k, v, table, n)
    refused(q, k[0], v[0], table, n)
    refused(q, k, v, table.cpu(), n)
    refused(q, k.cpu(), v.cpu(), table, n)
    refused(q, k, v, table, n, window=0)
    refused(q, k, v, table, n, sinks=2)
    refused(q, k, v, table, n, window=4, sinks=-1)
    refused(q, k.transpose(2, 3), v.transpose(2, 3), table, n)
    refused(torch.zeros(2 * 4 * 64 + 1, dtype=q.dtype, device="cuda")[1:].view(2, 4, 64), k, v, table, n)   # not on 16 bytes
    refused(q, torch.zeros(10, 2, 16, 324, dtype=q.dtype, device="cuda")[..., :320], torch.zeros(10, 2, 16, 324, dtype=q.dtype, device="cuda")[..., :320], table, n)
    refused(q.clone().requires_grad_(), k, v, table, n)
    with torch.no_grad():
        ops.paged_attention(q.clone().requires_grad_(), k, v, table, n)
