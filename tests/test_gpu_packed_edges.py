"""Packed attention and rotary positions at the edges of their operands: last texts that end inside a tile, gradients that begin off a 16-byte boundary, units of work that
take seconds, texts that must not depend on what else is in the batch."""
import math

import pytest
import torch

from mccl_b200 import ops
from tests.test_gpu_packed_attention import make, offsets_of

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
