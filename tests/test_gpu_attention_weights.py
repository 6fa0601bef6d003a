"""How many bits the weights of paged attention have, with scores that both sides know exactly: queries are the first unit vector, so a score is a
key's first element.

Bound of an element, relative to the largest weight of its row.  The result is rounded to 16 bits, u |o| (fp16 has steps of 2^-24 at its low end).  A weight is
the sum of two 16-bit values, u^2 of itself; the exponent (up to 24, in fp32) is off by a few 2^-21, exp2 by 2^-22 and sums of some hundred fp32
terms by less than that: 2^-18 of a weight covers them, and 2^-15 the sums over 100000 positions.  fp16 weights are kept times 2^15, so the second value
has steps of 2^-39: half of one, 2^-40, per position."""
import pytest
import torch

from mccl_b200 import ops

pytestmark = pytest.mark.gpu
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def paged(scores, values, page, heads, dtype):
    """scores [n], values [n, dim] of one sequence and one head of keys, in pages in a random order."""
    n, dim = values.shape
    pages = -(-n // page)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(n))
    k, v = (torch.zeros(pages, 1, page, dim, dtype=dtype, device="cuda") for _ in range(2))
    room = torch.zeros(pages * page, dim, dtype=dtype, device="cuda")
    room[:n] = values
    v[order.cuda(), 0] = room.view(pages, page, dim)
    keys = torch.zeros_like(room)
    keys[:n, 1:].normal_()      # times zero
    keys[:n, 0] = scores
    k[order.cuda(), 0] = keys.view(pages, page, dim)
    q = torch.zeros(1, heads, dim, dtype=dtype, device="cuda")
    q[:, :, 0] = 1.0
    return q, k, v, order.to(torch.int32)[None].cuda(), torch.tensor([n], dtype=torch.int32, device="cuda")


def exact(scores, values):
    """(o, sum p |v|, sum |v| / sum of weights, lse), the weights relative to the largest."""
    s = scores.double()
    w = torch.exp(s - s.max())
    p = w / w.sum()
    return p @ values.double(), p @ values.double().abs(), values.double().abs().sum(0) / w.sum(), torch.logsumexp(s, 0)


def check(scores, values, page, heads, sums=2.0 ** -18):
    dtype = values.dtype
    o, lse = ops.paged_attention(*paged(scores, values, page, heads, dtype), scale=1.0, return_lse=True)
    want, spread, each, want_lse = exact(scores, values)
    u = UNIT[dtype]
    bound = u * want.abs() + (u * u + sums) * spread + (2.0 ** -40 * each + 2.0 ** -25 if dtype == torch.float16 else 0.0)
    assert ((o[0].double() - want).abs() / bound).max().item() <= 1.0
    assert torch.equal(o[0], o[0, :1].expand_as(o[0]))      # the heads are all the same
    assert (lse.double() - want_lse).abs().max().item() <= 2.0 ** -20 * want_lse.abs().item() + 2 * sums


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [2, 8, 16])
@pytest.mark.parametrize("dim,page", [(32, 16), (64, 64), (128, 16), (256, 8), (64, 100)])
def test_weights_have_more_than_16_bits(dim, page, heads, dtype):
    g = torch.Generator(device="cuda").manual_seed(dim + heads)
    for n in (2, 3, 8, 40, 100):
        scores = (torch.rand(n, generator=g, device="cuda") * 4).to(dtype)
        check(scores, torch.randn(n, dim, generator=g, device="cuda").to(dtype), page, heads)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,dim,page", [(1, 64, 64), (4, 128, 16), (16, 128, 64), (2, 64, 100), (3, 256, 24)])
@pytest.mark.parametrize("above", [10.0, 16.5, 17.4, 20.0, 30.0])
def test_a_first_position_far_above_the_others(above, heads, dim, page, dtype):
    """It has nothing to say itself (its values are zero): what the others say, small as their weights are, is the result."""
    n = 120011
    g = torch.Generator(device="cuda").manual_seed(int(above))
    scores = torch.zeros(n, dtype=dtype, device="cuda")
    scores[0] = above
    values = (1.0 + torch.rand(n, dim, generator=g, device="cuda")).to(dtype)
    values[0] = 0.0
    check(scores, values, page, heads, sums=2.0 ** -15)
