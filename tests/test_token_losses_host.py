"""The losses over rows of logits on the host side (no GPU needed): their oracle where differences are infinite."""
import math

import pytest
import torch
import torch.nn.functional as F

from oracle import token_ops as O


@pytest.mark.parametrize("smoothing", [0.0, 0.2])
@pytest.mark.parametrize("side", [0, 1])
def test_the_oracle_of_a_pair_with_a_masked_label(side, smoothing):
    x = torch.randn(2, 7, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    x[side, 3] = -math.inf
    loss, rewards, grad = O.preference(x, torch.tensor([3, 3]), [(0, 1), (1, 2)], smoothing=smoothing)
    z = torch.tensor(math.inf if side else -math.inf, dtype=torch.float64)
    want = -(1 - smoothing) * F.logsigmoid(z) - (smoothing * F.logsigmoid(-z) if smoothing else 0.0)
    assert loss == float(want) and not torch.isnan(grad).any()
