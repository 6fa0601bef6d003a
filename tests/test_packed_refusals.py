"""Arguments of the operators around whole prompts that are refused on any device."""
import math

import pytest
import torch

from mccl_b200 import ops


@pytest.mark.parametrize("scale", [0.0, -1.0, math.nan, math.inf, 1e300, 3e38])
def test_scales_that_no_score_can_have(scale):
    """Times log2 e the last two are infinite in 32 bits, and every result would be NaN."""
    q = torch.randn(4, 2, 8)
    with pytest.raises(RuntimeError, match="scale"):
        ops.packed_attention(q, q, q, torch.tensor([0, 4], dtype=torch.int32), scale=scale)
