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


# ---- distillation: what a confident teacher leaves for the rest -----------------------------------------------------------------
@pytest.mark.parametrize("vocab", [1000, 20000])
@pytest.mark.parametrize("k,left", [(1, 1e-5), (1, 1e-6), (64, 1e-4), (64, 1e-5), (64, 1e-6)])
def test_distill_teacher_that_leaves_next_to_nothing(vocab, k, left):
    """1 - sum p where p was stored as fp32 log-probabilities: they hold the digits, and an entry's own rounding may not take them.
    The student leaves a tenth of that off the list, so that the rest decides the gradient there."""
    from style_transfer_amd.losses import topk_distill_loss
    g = torch.Generator().manual_seed(k)
    x = torch.randn(3, vocab, generator=g)
    idx = torch.stack([torch.randperm(vocab, generator=g)[:k] for _ in range(3)])
    x.scatter_(1, idx, x.gather(1, idx) + math.log(vocab / k) + math.log(10 / left))
    val = (torch.log_softmax(torch.randn(3, k, generator=g, dtype=torch.float64), 1) + math.log1p(-left)).float()
    loss, want = O.distill(x, idx, val, None, 1.0, True)
    leaf = x.cuda().requires_grad_(True)
    got = topk_distill_loss(leaf, idx.cuda(), val.cuda(), tail=True)
    got.backward()
    # off the list an entry is q_j - rest e_j / S_off, over the rows: q_j and e_j / S_off have a row's error R each (sums of V terms,
    # the exponential's argument of up to 40 bits), rest the fp64 sum's, K 2^-46 / left, which is nothing.  With r = rest / q_rest
    # that is R (1 + r) of the |1 - r| q_j that are left, and a few roundings.
    off = torch.ones(3, vocab, dtype=torch.bool).scatter_(1, idx, False)
    grad = leaf.grad.cpu().double()
    q_rest = torch.stack([O.row(r, 1.0)[1] for r in x]).mul(off).sum(1)
    r = ((1 - val.double().exp().sum(1)) / q_rest)[:, None]
    bound = want.abs() * ((vocab / 64 + 64 + 80) * (1 + r) / (1 - r).abs() + 20) * U
    assert float(r.max()) > 1 and bool(((grad - want).abs() <= bound)[off].all())
    # a listed entry p_k (log p_k - log q_k) has a row's error, the rest's term next to none
    assert abs(float(got.detach()) - loss) <= (vocab / 64 + 64 + 80) * U


# ---- distillation: entries without any mass ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("vocab,k", [(9000, 128), (20000, 300), (131072, 2000)])
@pytest.mark.parametrize("value", [-1e9, -300.0, torch.finfo(torch.float32).min])
def test_distill_entries_that_both_models_mask(vocab, k, tail, value):
    """A list filled up with masked tokens: the teacher's values are a mask's, the student's logits -inf.  Where they have no mass in 64
    bits, what the student says of them does not count, whichever wave they are in; exp(-300) is a mass that the student denies."""
    from style_transfer_amd.losses import topk_distill_loss
    g = torch.Generator().manual_seed(k)
    x = torch.randn(2, vocab, generator=g)
    idx = torch.stack([torch.randperm(vocab, generator=g)[:k] for _ in range(2)])
    val = torch.log_softmax(torch.randn(2, k, generator=g), 1) - 0.2
    x[0].index_fill_(0, idx[0, 40:], -INF)                      # all behind the first 40; a few in the middle
    val[0, 40:] = value
    x[1].index_fill_(0, idx[1, 5:9], -INF)
    val[1, 5:9] = value
    loss, want = O.distill(x, idx, val, None, 1.0, tail)
    assert math.isfinite(loss) == (value != -300)
    leaf = x.cuda().requires_grad_(True)
    got = topk_distill_loss(leaf, idx.cuda(), val.cuda(), tail=tail)
    got.backward()
    row = (vocab / 64 + 64) * U
    bound = 2 * row + 60 * U + k / 16 * U + abs(loss) * 4 * U
    assert float(got.detach()) == loss if math.isinf(loss) else abs(float(got.detach()) - loss) <= bound
    # rows are halved by the mean: an entry q_j Q - p_j, each with a row's error and 40 bits of its exponent
    grad = leaf.grad.cpu().double()
    assert bool(((grad - want).abs() <= (2 * row + k / 16 * U + 200 * U) * (want.abs() + 2e-4) + 2.0 ** -126).all())


# ---- references on both sides of 2^24 ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("vocab", [1000, 20000, 131072])
def test_parts_whose_references_lie_on_both_sides_of_a_border(vocab, sign):
    """Up to |m c| < 2^24 a reference is the whole number next to m c, beyond it m itself: a part of each kind, one unit of the
    last place apart in x, joins without the up to half a bit between the two readings."""
    from style_transfer_amd.losses import token_logprobs, topk_distill_loss
    x = torch.full((2, vocab), sign * 11629077.0)               # x c = 16777211.49
    x[:, vocab // 2:] = sign * 11629080.0                       # 16777215.82, which is 2^24 in fp32
    x[1] = x[1].flip(0)
    t = torch.tensor([0, 0])
    logp, h, log_q, q = O.token_logprobs(x, t)
    got, entropy = token_logprobs(x.cuda(), t.cuda(), return_entropy=True)
    row = (vocab / 64 + 64) * U
    assert float((got.cpu().double() - logp).abs().max()) <= row + 2 * U * float(logp.abs().max())
    assert float((entropy.cpu().double() - h).abs().max()) <= (float(h.max()) + 2) * row + 2 * U * float(h.max())
    idx = torch.tensor([[0, 1], [vocab - 1, vocab - 2]])        # the list on one side of the border, most of the row on the other
    val = torch.tensor([[-0.5, -1.5]]).repeat(2, 1)
    for tail in (False, True):
        loss, want = O.distill(x, idx, val, None, 1.0, tail)
        leaf = x.cuda().requires_grad_(True)
        got = topk_distill_loss(leaf, idx.cuda(), val.cuda(), tail=tail)
        got.backward()
        assert abs(float(got.detach()) - loss) <= 2 * row + 60 * U + abs(loss) * 8 * U
        assert bool(((leaf.grad.cpu().double() - want).abs() <= (2 * row + 60 * U) * (want.abs() + 2 / vocab)).all())


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("vocab", [300, 9000])
def test_distill_a_position_without_entries_contributes_nothing(vocab, tail):
    """Whatever its logits hold: a row of -inf, one with an infinity or a NaN, an ordinary one.  It counts in the mean."""
    from style_transfer_amd.losses import topk_distill_loss
    x = torch.randn(5, vocab, generator=torch.Generator().manual_seed(2))
    x[1] = -INF
    x[2, 7] = INF
    x[3, 8] = math.nan
    idx, val = torch.full((5, 3), -1), torch.zeros(5, 3)
    idx[4], val[4] = torch.tensor([1, 2, 5]), torch.tensor([-1.0, -1.5, -2.0])
    loss, want = O.distill(x[4:], idx[4:], val[4:], None, 1.0, tail)
    leaf = x.cuda().requires_grad_(True)
    got = topk_distill_loss(leaf, idx.cuda(), val.cuda(), tail=tail)
    got.backward()
    assert abs(float(got.detach()) - loss / 5) <= (2 * (vocab / 64 + 64) + 60) * U
    assert not leaf.grad[:4].any() and leaf.grad[4].any()
    (2 * topk_distill_loss(leaf, idx.cuda(), val.cuda(), tail=tail)).backward()      # computed again
    assert not leaf.grad[:4].any()


# ---- rows with one dominant logit ---------------------------------------------------------------------------------------------------
#: a row for each kernel: a wave's and a block's, held and in part read again
ROWS = [(torch.float32, 1000), (torch.bfloat16, 2040), (torch.float16, 7001), (torch.bfloat16, 16000), (torch.float32, 16001),
        (torch.bfloat16, 50001), (torch.bfloat16, 80000), (torch.bfloat16, 131072), (torch.float32, 131072)]


@pytest.mark.parametrize("dtype,vocab", ROWS)
@pytest.mark.parametrize("gap", [30.0, 38.0, 45.0, 52.0])
def test_policy_of_a_token_that_the_model_is_sure_of(dtype, vocab, gap):
    """The dominant logit is far above the first vectors of its row, and of its wave; the model's log-probability is its own old
    one.  All others together are below V exp(0.5 - gap) <= 2e-8 of the sum, so that adding them in any order changes it by no more
    than that: what is left is the dominant element's own error, 2 U of the exponential and U of its argument, which therefore
    has to be near 0."""
    from style_transfer_amd.losses import clipped_policy_loss, token_logprobs
    n = 3
    x = torch.randn(n, vocab, generator=torch.Generator().manual_seed(vocab))
    at = torch.tensor([vocab * 3 // 5, vocab - 1, vocab // 2 + 1])
    x[torch.arange(n), at] = gap
    x = x.to(dtype)
    label = at.clone()
    label[2] = 0                                                # an improbable token, and a ratio of 1 as well
    logp, h, log_q, q = O.token_logprobs(x, label)
    old = logp.float()
    others = vocab * math.exp(1.0 - gap)
    err = others + 4 * U
    for r in range(n):
        leaf = x[r:r + 1].cuda().requires_grad_(True)
        got = clipped_policy_loss(leaf[None], label[r:r + 1][None].cuda(), old[r:r + 1][None].cuda(), torch.ones(1, 1).cuda(), entropy_coef=0.01)
        got.loss.backward()
        ratio = math.exp(float(logp[r]) - float(old[r]))
        stats = got.stats.cpu().double()
        assert abs(float(stats[0]) + ratio) <= ratio * (err + U)
        # H = ln S - ln2 W / S: the argument's share of the dominant element, at most 2 bits, cancels but for three roundings
        assert abs(float(stats[2]) - float(h[r])) <= err + gap * others + 2 * math.log(2) * 3 * U
        a = torch.tensor([-ratio], dtype=torch.float64)
        _, _, want = O.policy(x[r:r + 1], label[r:r + 1], [(0, 1)], old[r:r + 1], torch.ones(1), ent=0.01)
        grad = leaf.grad.cpu().double()
        half = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
        tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126
        bound = a.abs() * q[r] * (err + 6 * U + (log_q[r] - log_q[r].max()).abs().clamp(max=200) * 2 * U) + want.abs() * half * 1.01 + tiny
        bound[0, label[r]] += 4 * U                             # 1 - q there
        bound += 0.01 * q[r] * (log_q[r].abs().clamp(max=200) + h[r]) * (err + 40 * U)
        assert bool(((grad - want).abs() <= bound).all())
    both = clipped_policy_loss(x[None].cuda(), label[None].cuda(), token_logprobs(x.cuda(), label.cuda())[None], torch.ones(1, n).cuda())
    assert abs(float(both.stats[0]) + 1) <= 2 * err + float(logp.abs().max()) * U        # an old log-probability is rounded to fp32


# ---- policy: a token that another model rules out -------------------------------------------------------------------------------------
@pytest.mark.parametrize("vocab", [50, 9000])
def test_policy_reference_that_masks_the_token(vocab):
    """ref = -inf: the estimate is +inf, its derivative -kl_coef (exp(ref - logp) - 1) = kl_coef."""
    from style_transfer_amd.losses import clipped_policy_loss
    x = torch.randn(2, vocab, generator=torch.Generator().manual_seed(9))
    t = torch.tensor([3, 4])
    logp, h, log_q, q = O.token_logprobs(x, t)
    ref = torch.stack([torch.tensor(-INF), logp[1].float() - 0.5])
    leaf = x.cuda().requires_grad_(True)
    got = clipped_policy_loss(leaf[None], t[None].cuda(), logp.float()[None].cuda(), torch.zeros(1, 2).cuda(), ref[None].cuda(), kl_coef=0.25)
    got.loss.backward()
    assert float(got.loss.detach()) == INF and float(got.stats[1]) == INF
    a = torch.stack([torch.tensor(0.125, dtype=torch.float64), -0.125 * torch.expm1(ref[1].double() - logp[1])])
    want = O.row_gradient(t, 1.0, h, log_q, q, a, a * 0)
    err = (vocab / 64 + 64) * U                                # a row's; an entry of it has 40 bits of its exponent besides
    bound = a.abs()[:, None] * q * (2 * err + 80 * U) + want.abs() * 4 * U + 0.125 * 2 * err * (q > 0.01)
    bound[torch.arange(2), t] += 0.125 * (2 * err + 8 * U)
    assert bool(((leaf.grad.cpu().double() - want).abs() <= bound + 2.0 ** -126).all())


# ---- policy: a token's terms --------------------------------------------------------------------------------------------------------
def one_token(old, adv=1.0, ref=None, vocab=8, **settings):
    """stats and loss of one token over equal logits: S = V exactly, log-probability -ln V to the last digit of 64 bits."""
    from style_transfer_amd.losses import clipped_policy_loss
    x = torch.zeros(1, 1, vocab, device="cuda", requires_grad=True)
    t = torch.zeros(1, 1, dtype=torch.long, device="cuda")
    f = lambda v: None if v is None else torch.full((1, 1), v, device="cuda")  # noqa: E731
    got = clipped_policy_loss(x, t, f(old), f(adv), f(ref), **settings)
    got.loss.backward()
    return got.stats.cpu().double(), float(got.loss.detach()), x.grad.cpu().double().view(-1)


def test_policy_ratio_and_estimate_have_one_rounding():
    """exp(logp - old) and exp(d) - 1 - d in 64 bits, rounded once."""
    g = torch.Generator().manual_seed(1)
    for vocab in (8, 4096):
        logp = -math.log(vocab)
        for old, ref in zip((logp + torch.randn(24, generator=g)).tolist(), (logp + torch.randn(24, generator=g) * 2).tolist()):
            old, ref = float(torch.tensor(old)), float(torch.tensor(ref))
            stats, loss, _ = one_token(old, -1.0, ref, vocab, clip_high=1e30, clip_low=0.0)      # A < 0: the ratio above 1 is not held
            ratio, d = max(1.0, math.exp(logp - old)), ref - logp
            assert abs(float(stats[0]) - ratio) <= 1.001 * U * ratio
            kl = math.expm1(d) - d
            assert abs(float(stats[1]) - kl) <= 1.001 * U * kl


def test_policy_advantage_of_zero_costs_nothing():
    """0 times a ratio that fp32 cannot hold, but 64 bits can."""
    stats, loss, grad = one_token(-120.0, adv=0.0)
    assert loss == 0 and not stats[0] and not grad.any()


def test_policy_terms_that_cancel():
    """Rows' terms of both signs, whose sum is far smaller than they are: rounded once, at the end."""
    from style_transfer_amd.losses import clipped_policy_loss
    n, vocab = 200, 8
    g = torch.Generator().manual_seed(5)
    old = (-math.log(vocab) + torch.randn(n, generator=g) * 0.05)
    adv = torch.randn(n, generator=g) * 1000
    terms = -adv.double() * torch.exp(-math.log(vocab) - old.double())
    adv[-1] += float(terms.sum() / torch.exp(-math.log(vocab) - old.double())[-1])
    terms = -adv.double() * torch.exp(-math.log(vocab) - old.double())
    want = float(terms.mean())
    assert abs(want) < 1e-4 * float(terms.abs().mean())
    x, t = torch.zeros(n, 1, vocab, device="cuda"), torch.zeros(n, 1, dtype=torch.long, device="cuda")
    got = clipped_policy_loss(x, t, old[:, None].cuda(), adv[:, None].cuda(), clip_low=0.9, clip_high=9.0)
    assert abs(float(got.loss) - want) <= 1.001 * U * abs(want) + float(terms.abs().mean()) * 2.0 ** -48


# ---- distillation: the rounding of log2(e) / tau --------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,vocab", [(torch.float32, 1000), (torch.float32, 16384), (torch.bfloat16, 32768)])
@pytest.mark.parametrize("tail", [False, True])
def test_distill_at_a_temperature_that_rounds_badly(dtype, vocab, tail):
    """tau for which log2(e) / tau lies between two fp32 numbers, 5.8e-8 of it away from either, and rows half of whose mass is far
    below the other half: every ln S would be off in the same direction by that times the mean distance, about 5 U.  Over 64 rows
    what is random goes down: a row's sum has up to 10 joins of U each, 10 U / sqrt(3 * 64) = 0.7 U of the mean, two of those are
    1.4 U; the exponential's own mean error is 0.06 U."""
    from style_transfer_amd.losses import topk_distill_loss
    rows, tau = 64, 1 / (math.log(2) * (1 + 0.98 * 2.0 ** -24))
    g = torch.Generator().manual_seed(vocab)
    x = (torch.rand(rows, vocab, generator=g) - 0.5 - math.log(vocab)) * tau
    x[torch.arange(rows), torch.arange(rows) * 3] = torch.rand(rows, generator=g) * 0.1
    x = x.to(dtype)
    idx = (torch.arange(rows) * 3)[:, None]
    val = torch.full((rows, 1), math.log(0.5) if tail else 0.0)
    loss, _ = O.distill(x, idx, val, None, tau, tail)
    got = float(topk_distill_loss(x.cuda(), idx.cuda(), val.cuda(), temperature=tau, tail=tail))
    assert abs(got - loss) <= tau * tau * 1.5 * U + U * abs(loss)


# ---- the gradient that the forward pass leaves --------------------------------------------------------------------------------------
def early(t, idx, val, old):
    from style_transfer_amd import losses
    return [lambda v: losses.clipped_policy_loss(v, t, old, old + 9).loss, lambda v: losses.topk_distill_loss(v, idx, val, tail=True)]


def steps_of(vocab, seed=4):
    from style_transfer_amd import losses
    g = torch.Generator().manual_seed(seed)
    x, t = torch.randn(4, 6, vocab, generator=g).cuda(), torch.randint(0, vocab, (4, 6), generator=g).cuda()
    idx = torch.arange(24 * 5).view(4, 6, 5).cuda() % vocab
    val = torch.log_softmax(torch.randn(4, 6, 5, generator=g), -1).cuda() - 0.1
    return x, early(t, idx, val, losses.token_logprobs(x, t) + 0.1)


def test_the_early_gradient_goes_where_saved_tensors_go():
    """Saved tensors that are kept on the host, or dropped by a checkpoint: nothing of the logits' size stays on the device but the
    logits themselves."""
    from torch.utils.checkpoint import checkpoint
    vocab = 60000
    x, fns = steps_of(vocab)
    size = x.numel() * 4
    for fn in fns:
        want = []
        for mode in ("plain", "host", "checkpoint"):
            leaf = x.clone().requires_grad_(True)
            torch.cuda.synchronize()
            before = torch.cuda.memory_allocated()
            if mode == "host":
                with torch.autograd.graph.save_on_cpu():
                    loss = fn(leaf)
            else:
                loss = checkpoint(fn, leaf, use_reentrant=False) if mode == "checkpoint" else fn(leaf)
            torch.cuda.synchronize()
            held = torch.cuda.memory_allocated() - before
            assert mode == "plain" or held < size // 4, (mode, held)
            loss.backward()
            want.append(leaf.grad)
            del loss, leaf                                     # or the next measurement begins with them
        assert torch.equal(want[0], want[1]) and torch.equal(want[0], want[2])


def test_a_gradient_that_was_given_away_may_be_changed():
    """Twice through one graph, with the first gradient changed in place between: the second is as the first was."""
    x, fns = steps_of(700)
    for fn in fns:
        leaf = x.clone().requires_grad_(True)
        loss = fn(leaf)
        one, = torch.autograd.grad(loss, [leaf], retain_graph=True)
        kept = one.clone()
        one.mul_(7).add_(1)
        two, = torch.autograd.grad(loss, [leaf], retain_graph=True)
        assert torch.equal(two, kept)
        two.zero_()
        loss.backward()
        assert torch.equal(leaf.grad, kept)


@pytest.mark.parametrize("vocab", [700, 20000])
def test_a_backward_pass_in_a_graph_of_its_own(vocab):
    """Forward and backward captured into two graphs, as make_graphed_callables does, and the second replayed more than once: each
    replay gives the gradient for the upstream gradient that it finds, whatever the buffer held."""
    x, fns = steps_of(vocab)
    for fn in fns:
        eager = x.clone().requires_grad_(True)
        one, = torch.autograd.grad(fn(eager), [eager])
        leaf, up = x.clone().requires_grad_(True), torch.ones((), device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(fn(leaf), [leaf], [up])
        torch.cuda.current_stream().wait_stream(side)
        forward, backward = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(forward, stream=side):
            loss = fn(leaf)
        with torch.cuda.graph(backward, pool=forward.pool(), stream=side):
            grad, = torch.autograd.grad(loss, [leaf], [up])
        for first in range(3):
            forward.replay()
            for factor in (1.0, 3.0, 1.0, 0.0, 1.0):
                up.fill_(factor)
                backward.replay()
                torch.cuda.synchronize()
                assert torch.allclose(grad, one * factor, rtol=8 * U, atol=16 * U * 3 * float(one.abs().max())), factor
                assert factor != 1 or torch.equal(grad, one)
                grad.add_(0.25)                                 # the program's own use of it


def test_the_early_gradient_is_used_where_its_forward_pass_is_repeated(monkeypatch):
    """Eagerly and within one graph it is handed over; across graphs, or captured after an eager forward pass, it is not."""
    from style_transfer_amd import token_losses
    taken = []
    real = token_losses._take_grad
    monkeypatch.setattr(token_losses, "_take_grad", lambda *a: taken.append(real(*a)) or taken[-1])
    x, fns = steps_of(700)
    side = torch.cuda.Stream()
    for fn in fns:
        leaf = x.clone().requires_grad_(True)
        torch.autograd.grad(fn(leaf), [leaf])
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(fn(leaf), [leaf])
            loss = fn(leaf)
        torch.cuda.current_stream().wait_stream(side)
        one, first, second, late = (torch.cuda.CUDAGraph() for _ in range(4))
        with torch.cuda.graph(late, stream=side):
            torch.autograd.grad(loss, [leaf])
        with torch.cuda.graph(one, stream=side):
            torch.autograd.grad(fn(leaf), [leaf])
        with torch.cuda.graph(first, stream=side):
            loss = fn(leaf)
        with torch.cuda.graph(second, pool=first.pool(), stream=side):
            torch.autograd.grad(loss, [leaf])
        assert [for_one for _, for_one in taken] == [1, 1, 0, 1, 0]
        taken.clear()


# ---- ordinary rows: how many digits are right -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,vocab", [(torch.float32, 1000), (torch.bfloat16, 5001), (torch.float32, 32768), (torch.bfloat16, 65536),
                                         (torch.bfloat16, 131072), (torch.float32, 131072), (torch.bfloat16, 2 ** 20)])
@pytest.mark.parametrize("lift", [0.0, 8.0, 20.0])
def test_large_vocabularies_keep_their_digits(dtype, vocab, lift):
    """A bound that does not grow with the vocabulary.  The roundings of a sum of positive terms are independent, to either side and
    at most U of what has been added up so far: a thread's n <= 2048 terms are worth at most sqrt(n / 3) U of its share, and T >= 64
    threads' errors average to 1 / sqrt(T) of that, 3.3 U with n = 2048 and T = 64, less for longer rows, which have more threads;
    then about 12 joins of U / sqrt(3) each, sqrt(12 / 3) = 2 U, and the exponentials, whose errors average out but for 0.06 U.
    Five standard deviations of both are 20 U of S, and so 20 U of a log-probability; of the entropy by a factor of its distances
    from it, which average to H - ln2 sum q d <= 12 nats, weighted like the terms: 3 times as much at most."""
    from style_transfer_amd.losses import clipped_policy_loss, token_logprobs, topk_distill_loss
    n = 4
    g = torch.Generator().manual_seed(vocab)
    x = torch.randn(n, vocab, generator=g) * 2
    t = torch.randint(0, vocab, (n,), generator=g)
    x[torch.arange(n), t] += lift
    x = x.to(dtype)
    logp, h, log_q, q = O.token_logprobs(x, t)
    got, entropy = token_logprobs(x.cuda(), t.cuda(), return_entropy=True)
    assert bool(((got.cpu().double() - logp).abs() <= 20 * U + U * logp.abs()).all())
    assert bool(((entropy.cpu().double() - h).abs() <= 60 * U + U * h).all())
    # each row alone, so that nothing averages: the ratio is 1, its error the log-probability's
    for r in range(n):
        leaf = x[r:r + 1].cuda().requires_grad_(True)
        old = logp[r:r + 1].float()
        loss, stats = clipped_policy_loss(leaf[None], t[r:r + 1][None].cuda(), old[None].cuda(), -torch.ones(1, 1).cuda())
        loss.backward()
        ratio = math.exp(float(logp[r]) - float(old))
        assert abs(float(stats[0]) - ratio) <= 22 * U and abs(float(stats[2]) - float(h[r])) <= 60 * U + U * float(h[r])
        # an entry: 20 U of S, its own exponent of up to 32 bits, a few roundings; at the label 1 - q is left of both
        want = O.row_gradient(t[r:r + 1], 1.0, h, log_q[r:r + 1], q[r:r + 1], torch.tensor([ratio], dtype=torch.float64), torch.zeros(1))[0]
        half = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}[dtype]
        bound = want.abs() * half + 50 * U * ratio * q[r]
        bound[t[r]] += 4 * U
        assert bool(((leaf.grad[0].cpu().double() - want).abs() <= bound + 2.0 ** -126).all())
        if vocab <= 131072:
            idx = torch.stack([t[r], (t[r] + 1) % vocab])[None]
            val = torch.tensor([[-0.25, -2.0]])
            for tail in (False, True):
                want, _ = O.distill(x[r:r + 1], idx, val, None, 1.0, tail)
                got = topk_distill_loss(x[r:r + 1].cuda(), idx.cuda(), val.cuda(), tail=tail)
                assert abs(float(got) - want) <= 40 * U + U * abs(want)


@pytest.mark.parametrize("vocab,k,tail,tau", [(1000, 40, True, 1.0), (20000, 300, True, 1.7), (9000, 40, False, 1.7), (60000, 1500, False, 1.0)])
def test_distill_listed_entries_have_the_digits_of_their_probabilities(vocab, k, tail, tau):
    """Listed entries are tau (Q q_j - p_j) over the rows, however far apart the values are: p_j within 6 U, since its exponent is a
    whole number and a fraction of at most 1/2 (0.4 U), the exponential is within 2 U, the row's coefficient, the product and the
    entry are rounded; q_j, with an exponent of up to 32 bits that is rounded once, within 20 U of S as any row's, 22 U and 6 U."""
    from style_transfer_amd.losses import topk_distill_loss
    g = torch.Generator().manual_seed(k)
    x = torch.randn(2, vocab, generator=g) * 4
    idx = torch.stack([torch.randperm(vocab, generator=g)[:k] for _ in range(2)])
    val = torch.randn(2, k, generator=g) * 4
    if tail:
        val = torch.log_softmax(val, 1) - 0.05
    _, want = O.distill(x, idx, val, None, tau, tail)
    leaf = x.cuda().requires_grad_(True)
    loss = topk_distill_loss(leaf, idx.cuda(), val.cuda(), temperature=tau, tail=tail)
    got, = torch.autograd.grad(loss, [leaf], retain_graph=True)
    again, = torch.autograd.grad(loss, [leaf])                  # computed from the saved coefficients
    q = torch.stack([O.row(r, tau)[1] for r in x])
    p = (val.double() if tail else torch.log_softmax(val.double() / tau, 1)).exp()
    bound = tau / 2 * (q.gather(1, idx) * 48 * U + p * 6 * U) + 2.0 ** -126
    assert torch.equal(got, again)
    assert bool(((got.cpu().double() - want).gather(1, idx).abs() <= bound).all())


# ---- rows in which the reference moves -------------------------------------------------------------------------------------------------
def moving_rows(dtype, vocab):
    """Rising, falling, stepping up and down, up from a mask, into the low range at the end or in one element, past it and back."""
    up = torch.linspace(-60, 60, vocab)
    x = torch.stack([up, up.flip(0), torch.where(torch.arange(vocab) % 512 < 256, up, -up), up, up, up / 60])
    x[2] += 0.25 * torch.randn(vocab, generator=torch.Generator().manual_seed(vocab))
    x[3, : vocab * 3 // 4] = -INF
    if dtype != torch.float16:
        x[4, vocab - 3:] = 3e7
        x[5, vocab // 2] = 2.5e7
    return x.to(dtype)


@pytest.mark.parametrize("dtype,vocab", ROWS + [(torch.bfloat16, 170001), (torch.float32, 90000)])
def test_rows_in_which_the_reference_moves(dtype, vocab):
    from style_transfer_amd.losses import clipped_policy_loss, topk_distill_loss
    x = moving_rows(dtype, vocab)
    n = x.shape[0]
    t = torch.tensor([vocab - 1, 0, vocab - 1, vocab - 2, vocab - 1, vocab // 2])
    logp, h, log_q, q = O.token_logprobs(x, t)
    row = (vocab / 64 + 64) * U
    half, tiny = {torch.float32: (U, 2.0 ** -126), torch.bfloat16: (2.0 ** -8, 2.0 ** -126), torch.float16: (2.0 ** -11, 2.0 ** -25)}[dtype]
    for r in range(n):
        leaf = x[r:r + 1].cuda().requires_grad_(True)
        old = logp[r:r + 1].float()
        loss, stats = clipped_policy_loss(leaf[None], t[r:r + 1][None].cuda(), old[None].cuda(), -torch.ones(1, 1).cuda(), entropy_coef=0.1)
        loss.backward()
        ratio = math.exp(float(logp[r]) - float(old))
        assert abs(float(stats[0]) - ratio) <= row + 2 * U
        assert abs(float(stats[2]) - float(h[r])) <= (float(h[r]) + 2) * row + 2 * U * float(h[r])
        a, b = torch.tensor([ratio], dtype=torch.float64), torch.tensor([-0.1], dtype=torch.float64)
        want = O.row_gradient(t[r:r + 1], 1.0, h[r:r + 1], log_q[r:r + 1], q[r:r + 1], a, b)
        low = log_q[r].clamp(min=-200.0).abs()
        # as any row's: S, the exponent of an entry, roundings; and the exponential is 0 below 2^-126, an entry this many times that
        size = ratio + 0.1 * (low + h[r])
        fp32 = q[r] * size * (row + 10 * U + 3 * low * U) + size * 2.0 ** -126
        fp32[t[r]] += 8 * U
        assert bool(((leaf.grad.cpu().double() - want)[0].abs() <= (want[0].abs() + fp32) * half * 1.01 + fp32 + tiny).all()), r
        idx, val = torch.tensor([[int(t[r]), vocab // 2 + 1, vocab - 5]]), torch.tensor([[-0.5, -2.0, -2.5]])
        val = val.masked_fill(x[r].gather(0, idx[0])[None] == -INF, -INF)
        for tail in (False, True):
            want_loss, want = O.distill(x[r:r + 1], idx, val, None, 1.0, tail)
            leaf.grad = None
            got = topk_distill_loss(leaf, idx.cuda(), val.cuda(), tail=tail)
            got.backward()
            # p (log p - log q): q is up to e^-120, or e^-3e7, of which fp32 keeps 2 U
            assert abs(float(got.detach()) - want_loss) <= 2 * row + 60 * U + abs(want_loss) * 4 * U
            fp32 = (2 * q[r] + (want[0] - q[r]).abs()) * (2 * row + 40 * U + 6 * low * U)
            assert bool(((leaf.grad.cpu().double() - want)[0].abs() <= (want[0].abs() + fp32) * half * 1.01 + fp32 + tiny).all()), r


@pytest.mark.parametrize("dtype,vocab", ROWS)
@pytest.mark.parametrize("value", [INF, math.nan])
def test_a_value_without_a_softmax_anywhere_in_a_row(dtype, vocab, value):
    """+inf or NaN in the first vector, in the middle or outside the vectors: the row is NaN, and no other."""
    from style_transfer_amd.losses import clipped_policy_loss
    x = torch.randn(4, vocab, generator=torch.Generator().manual_seed(1)).to(dtype)
    for r, at in enumerate((1, vocab // 2, vocab - 1)):
        x[r, at] = value
    leaf = x.cuda().requires_grad_(True)
    t = torch.tensor([[5, 6, 7, 8]]).cuda()
    for r in range(4):
        loss, stats = clipped_policy_loss(leaf[None, r:r + 1], t[:, r:r + 1], torch.full((1, 1), -9.0).cuda(), -torch.ones(1, 1).cuda(), clip_low=0.0)
        assert math.isnan(float(stats[2])) == (r < 3)
    old = torch.full((1, 4), -9.0).cuda()
    clipped_policy_loss(leaf[None], t, old, -torch.ones(1, 4).cuda(), clip_low=0.0, entropy_coef=0.1).loss.backward()
    assert torch.isnan(leaf.grad[:3]).all() and torch.isfinite(leaf.grad[3]).all()
