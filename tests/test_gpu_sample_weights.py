"""How exact the weights are that tokens are drawn by.  Of two tokens the first is drawn while the uniform number is below its weight's share, so halving intervals of that number finds the
weight itself, to 2^-52.

A weight is a whole number of 2^-43: half of one is its last rounding, and before that it is off by less than 2^-36 of itself."""
import math

import pytest
import torch

from mccl_b200 import ops

pytestmark = pytest.mark.gpu
ROWS = 20000


def weights(logits, **settings):
    """The first token's weight over the second's (the likelier one's), as the draws have it."""
    low, high = (torch.full((logits.shape[0],), v, dtype=torch.float64, device="cuda") for v in (0.0, 0.500001))
    for _ in range(70):
        middle = (low + high) / 2
        below = ops.sample(logits, middle, **settings) == 0
        low, high = torch.where(below, middle, low), torch.where(below, high, middle)
    return high / (1.0 - high)


@pytest.mark.parametrize("temperature", [1.0, 0.7, 3.3, 1e-4, 1e4, None])
@pytest.mark.parametrize("middle", [0.0, 17.3, -250.0])
def test_weights_are_exact_to_2_36(temperature, middle):
    g = torch.Generator().manual_seed(5)
    t = torch.full((ROWS,), temperature) if temperature is not None else torch.rand(ROWS, generator=g) * 3 + 0.01
    t = t.float()
    top = (torch.randn(ROWS, generator=g) + middle) * t
    x = torch.minimum(top, top - t * 30.4 * torch.rand(ROWS, generator=g) ** 2)
    logits = torch.stack((x, top), 1).float()
    got = weights(logits.cuda(), temperature=t.cuda()).cpu()
    want = torch.exp((logits[:, 0].double() - logits[:, 1].double()) / t.double())
    off = (got - want).abs()
    bound = 0.51 * 2.0 ** -43 + 2.0 ** -36 * want   # (0.01: the interval that is left, and the product with the sum of both)
    assert (off <= bound).all(), (off / bound).max().item()


def test_a_border_of_min_p():
    """A token whose weight is above min_p by 1e-10 of it stays, one as far below does not, wherever it stands."""
    g = torch.Generator().manual_seed(6)
    low = torch.rand(ROWS, generator=g).float() * 0.9 + 0.01
    # the largest logit (fp32, near zero: steps of 2^-24 and less of the weight) whose weight is below min_p, and the next one
    x = (torch.log(low.double())).float()
    below = torch.where(torch.exp(x.double()) < low.double(), x, torch.nextafter(x, torch.tensor(-math.inf)))
    above = torch.nextafter(below, torch.tensor(0.0))
    for logit in (below, above):
        weight = torch.exp(logit.double())
        clear = (weight / low.double() - 1.0).abs() > 1e-10
        logits = torch.stack((logit, torch.zeros(ROWS)), 1).cuda()
        drawn = ops.sample(logits, torch.zeros(ROWS, device="cuda"), min_p=low.cuda()).cpu()
        assert torch.equal((drawn == 0)[clear], (weight >= low.double())[clear])
        assert clear.float().mean() > 0.99
