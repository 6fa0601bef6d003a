"""Packed attention and rotary positions at the edges of their operands: last texts that end inside a tile, gradients that begin off a 16-byte boundary, units of work that
take seconds, texts that must not depend on what else is in the batch."""
import math

import pytest
import torch

from mccl_b200 import ops
from tests.test_gpu_packed_attention import close, make, offsets_of
from tests.test_gpu_packed_attention import exact as exact_results
from tests.test_gpu_packed_gradients import exact, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 128), (4, 2, 64), (3, 1, 64)])
@pytest.mark.parametrize("lengths,before", [([100, 412], None), ([412, 28], None), ([300, 1], None), ([3, 5], [700, 2300])])
def test_values_of_the_last_text_that_are_not_finite(lengths, before, heads, kv_heads, dim):
    """The last text ends inside a block of 128 keys and its values are the last ones there are (here the first part of a larger tensor): its rows are put right, and the tile's rows behind
    it look at nothing."""
    q, k, v, offsets, k_offsets = make(lengths, heads, kv_heads, dim, before=before, poison=False, seed=sum(lengths))
    room = torch.full((v.shape[0] + 1024, kv_heads, dim), math.nan, dtype=v.dtype, device="cuda")
    good = ops.packed_attention(q, k, v, offsets, k_offsets)
    last_rows, last_keys = lengths[-1], lengths[-1] + (0 if before is None else before[-1])
    group = heads // kv_heads
    for at in (0, last_keys // 2, last_keys - 1):   # a key of the last text
        room[:v.shape[0]] = v
        room[v.shape[0] - last_keys + at, 0, 5] = math.inf
        o = ops.packed_attention(q, k, room[:v.shape[0]], offsets, k_offsets)
        sees = torch.zeros(q.shape[0], dtype=torch.bool, device="cuda")
        sees[q.shape[0] - last_rows + max(0, at - (last_keys - last_rows)):] = True
        columns = torch.arange(dim, device="cuda") != 5
        assert not torch.isfinite(o[sees][:, :group, 5]).any()
        assert torch.equal(o[~sees], good[~sees]) and torch.equal(o[:, group:], good[:, group:]) and torch.equal(o[:, :group][..., columns], good[:, :group][..., columns])


@pytest.mark.parametrize("elements", [1, 3, 4])
def test_gradients_that_begin_off_a_boundary(elements):
    """What the gradient of a concatenation hands on is contiguous and begins anywhere."""
    q, k, v, offsets, _ = make([300], 4, 2, 64, poison=False)
    front = torch.zeros(elements, dtype=q.dtype, device="cuda")
    g = torch.randn(q.shape, generator=torch.Generator().manual_seed(1)).to(q.dtype).cuda()
    shifted = torch.cat([front, g.flatten()])[elements:].view(q.shape)
    assert shifted.is_contiguous() and shifted.data_ptr() % 16

    def gradients(f, leaves, grad):
        leaves = [t.detach().requires_grad_() for t in leaves]
        return torch.autograd.grad(f(*leaves), leaves, grad)

    rope = ops.rotary_tables(300, 64)
    for f, inputs in ((lambda *x: ops.packed_attention(*x, offsets), (q, k, v)), (lambda x: ops.rotary(x, rope=rope), (q,)),
                      (lambda x, y: ops.rotary(x, y, rope=rope, layout="half")[0], (q, k))):
        want = gradients(f, inputs, g)
        for got in (gradients(f, inputs, shifted), gradients(lambda *x: torch.cat([front, f(*x).flatten()]), inputs, torch.cat([front, g.flatten()]))):
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_units_of_work_that_take_seconds():
    """A block of keys that all rows of 128 heads see: a million steps of one block of the grid, more than a second, in which others of its warps wait for the next unit.

    Every row but the first sees the first position and itself, with scores of zero and so weights of one half; the numbers are small and whole, so every sum is exact."""
    tokens, heads, dim, scale = 1_000_000, 128, 8, 0.25
    gen = torch.Generator(device="cuda").manual_seed(3)
    whole = lambda *sizes: torch.randint(-1, 2, sizes, generator=gen, device="cuda", dtype=torch.int8).to(torch.bfloat16)
    q = torch.zeros(tokens, heads, dim, dtype=torch.bfloat16, device="cuda").requires_grad_()
    k, v = (whole(tokens, 1, dim).requires_grad_() for _ in range(2))
    g = whole(tokens, heads, dim)
    o = ops.packed_attention(q, k, v, offsets_of([tokens]), window=1, sinks=1, scale=scale)
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), g)
    k, v = k.detach().float()[:, 0], v.detach().float()[:, 0]
    assert not dk.any()   # (of queries that are zeros)
    first = torch.zeros(dim, dtype=torch.float64, device="cuda")
    for a in range(0, tokens, 100_000):
        part, kk, vv = slice(a, a + 100_000), k[a:a + 100_000], v[a:a + 100_000]
        gg = g[part].float()
        assert torch.equal(o[part].float(), ((v[0] + vv) / 2)[:, None].expand(-1, heads, -1))
        own = gg.sum(1, dtype=torch.float64) / 2
        first += own.sum(0)
        if a == 0:
            first += own[0]   # the first row sees one key, with a weight of one
        seen = slice(1 if a == 0 else 0, None)
        assert torch.equal(dv[part][seen, 0], own[seen].to(torch.bfloat16))
        ds = ((gg @ v[0])[..., None] - (gg * vv[:, None]).sum(-1, keepdim=True)) / 4   # of the first position's score; the own one's is the opposite
        assert torch.equal(dq[part], (scale * (ds * k[0] - ds * kk[:, None])).to(torch.bfloat16))
    assert torch.equal(dv[0, 0], first.to(torch.bfloat16))


@pytest.mark.parametrize("short,long,window,sinks", [([3] * 160, [5000], None, 0), ([8] * 160, [5000, 0, 3000], None, 0), ([2, 0, 0, 5] * 80, [6000], None, 0), ([1, 4, 7] * 60, [5000], 400, 2)])
def test_gradients_of_short_texts_do_not_depend_on_the_batch(short, long, window, sinks):
    """dQ and dK of short texts beside long ones: rounded themselves, and sums of gradients of scores that were rounded (2^0.5 times what rounding the exact ones leaves, everything else
    a sixth of that at most: 1.5 times), as where they are alone, and the same bits."""
    lengths, rows = short + long, sum(short)
    q, k, v, offsets, _ = make(lengths, 4, 4, 64, poison=False, seed=len(lengths))
    g = torch.randn(q.shape, generator=torch.Generator().manual_seed(7)).to(q.dtype).cuda()
    _, got = run(q, k, v, g, offsets, window=window, sinks=sinks)
    alone = offsets_of(short)
    want, _ = exact(q[:rows], k[:rows], v[:rows], g[:rows], alone, None, 0.125, window, sinks)
    for name, a, b in list(zip("qkv", got, want))[:2]:
        assert (a[:rows].double() - b).norm() <= 1.5 * (b.to(torch.bfloat16).double() - b).norm(), name
    _, again = run(*(t[:rows] for t in (q, k, v, g)), alone, window=window, sinks=sinks)
    assert all(torch.equal(a[:rows], b) for a, b in zip(got, again))
    # and behind the long ones, where they begin at other places of a tile
    behind = offsets_of(long + short)
    moved = [torch.cat((t[rows:], t[:rows])) for t in (q, k, v, g)]
    _, last = run(*moved, behind, window=window, sinks=sinks)
    assert all(torch.equal(a[-rows:], b) for a, b in zip(last, again))


@pytest.mark.parametrize("heads,kv_heads,dim", [(3, 3, 128), (4, 2, 64)])
@pytest.mark.parametrize("lengths,before", [([128, 256], None), ([129, 700], None), ([1, 127, 1000], None), ([300, 260], [-44, -132])])
def test_first_positions_have_no_gradient_of_their_score(lengths, before, heads, kv_heads, dim):
    """A first position sees one key: its weight is one whatever the score is.  With gradients in the rows of first positions alone dQ and dK are zeros, whatever else is in their tiles."""
    q, k, v, offsets, k_offsets = make(lengths, heads, kv_heads, dim, before=before, poison=False, seed=5)
    firsts = torch.tensor([a + max(0, -m) for a, m in zip(offsets.tolist(), before or [0] * len(lengths))], device="cuda")
    g = torch.zeros_like(q)
    g[firsts] = torch.randn((len(lengths), heads, dim), generator=torch.Generator().manual_seed(2)).to(q.dtype).cuda()
    _, (dq, dk, dv) = run(q, k, v, g, offsets, k_offsets)
    assert not dq.any() and not dk.any()
    want = g[firsts].float().view(len(lengths), kv_heads, -1, dim).sum(2)
    got = dv[(offsets if k_offsets is None else k_offsets)[:-1].long()].float()
    # sums of up to three numbers of 8 bits in fp32, rounded once; products with a weight that rounds to one are exact
    assert torch.allclose(got, want, rtol=2.0 ** -8, atol=1e-6)


def test_windows_behind_a_long_cache_take_as_long_as_behind_a_short_one():
    """Where keys are shared out, one tile's share may be the first positions alone while the other has blocks of the window: what lies between (800 blocks here, of which nothing is
    seen) is not walked through."""
    rows, heads, dim, window, sinks = 512, 16, 128, 2048, 4

    def call(keys):
        g = torch.Generator().manual_seed(keys)
        q = torch.randn((rows, heads, dim), generator=g).to(torch.bfloat16).cuda()
        k, v = (torch.randn((keys, heads, dim), generator=g).to(torch.bfloat16).cuda() for _ in range(2))
        at = offsets_of([rows]), offsets_of([keys])
        best = math.inf
        for _ in range(10):
            begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            begin.record()
            for _ in range(5):
                ops.packed_attention(q, k, v, *at, window=window, sinks=sinks)
            end.record()
            end.synchronize()
            best = min(best, begin.elapsed_time(end))
        # what the window and the first positions are: a text of those keys alone, whose first positions stand right in front
        near = torch.cat((torch.arange(sinks), torch.arange(keys - rows - window + 1, keys))).cuda()
        o, lse = ops.packed_attention(q, k, v, *at, window=window, sinks=sinks, return_lse=True)
        close(o, lse, exact_results(q, k[near], v[near], at[0], offsets_of([len(near)]), dim ** -0.5, window, sinks), torch.bfloat16)
        return best

    short, long = call(8000), call(100_000)
    assert long < 5 * short, (short, long)   # twice as long: an average over more shares; 30 times with the blocks between
