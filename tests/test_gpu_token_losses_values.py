"""Losses over rows of logits at the values where digits or signs are lost first (csrc/token_losses.hip, csrc/token_distill.hip):
infinite differences, rows with one dominant logit, teachers and students that leave next to nothing for the rest, references
between two ranges.  Against the formulas in 64 bits; no counterpart in the reference: parity unpinned.

U = 2^-24 is half a step of fp32, relative to the value."""
import math

import pytest
import torch
import torch.nn.functional as F

from oracle import token_ops as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
INF = math.inf


# ---- preference loss: differences of +-inf ------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["sigmoid", "hinge"])
def test_a_masked_label_in_one_sequence_of_a_pair(dtype, kind):
    """A label that the mask leaves no probability: -inf for its sequence.  In the rejected one the pair's loss is 0 and nothing
    moves; in the chosen one it is +inf.  Beside an ordinary pair."""
    from style_transfer_amd.losses import preference_loss
    vocab, beta = 300, 0.5
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(4, 2, vocab, generator=g) * 2).to(dtype)   # chosen 0, 1, rejected 2, 3
    t = torch.randint(0, vocab, (4, 2), generator=g)
    for side, pair_loss in ((2, 0.0), (0, INF)):
        masked = x.clone()
        masked[side, 1, t[side, 1]] = -INF
        logp = torch.log_softmax(masked.double(), -1).gather(-1, t[..., None])[..., 0].sum(1)
        h = logp[:2] - logp[2:]
        each = -F.logsigmoid(beta * h) if kind == "sigmoid" else (1 - beta * h).clamp(min=0)
        assert float(each[0]) == pair_loss
        leaf = masked.cuda().requires_grad_(True)
        loss, chosen, rejected = preference_loss(leaf, t.cuda(), beta=beta, kind=kind)
        loss.backward()
        want = each.mean()
        # the ordinary pair: 4 rows, each within (V / 64 + 64) U of its log-probability of at most 20; Lipschitz with beta in h
        bound = beta * 4 * (vocab / 64 + 64 + 40) * U
        assert float(loss.detach()) == INF if pair_loss else abs(float(loss.detach()) - float(want)) <= bound
        assert float((chosen if side == 0 else rejected)[0]) == -INF
        assert torch.isfinite(leaf.grad).all() and leaf.grad[1].any() and leaf.grad[3].any()
        assert bool(leaf.grad[side].any()) == (pair_loss > 0)   # its slope is 0 where the pair is settled, -beta where it is lost


@pytest.mark.parametrize("smoothing", [0.0, 0.1])
def test_the_smoothed_part_of_an_infinite_difference(smoothing):
    """-eps log sigmoid(-z) is what makes z = +inf cost anything: nothing without it, +inf with it."""
    from style_transfer_amd.losses import preference_loss
    x = torch.zeros(2, 1, 8)
    x[1, 0, 3] = -INF
    t = torch.full((2, 1), 3)
    loss = preference_loss(x.cuda(), t.cuda(), label_smoothing=smoothing).loss
    assert float(loss) == (INF if smoothing else 0.0)
    loss = preference_loss(x.flip(0).cuda(), t.cuda(), label_smoothing=smoothing).loss
    assert float(loss) == INF
