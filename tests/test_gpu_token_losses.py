"""Losses over rows of logits (csrc/token_losses.hip, style_transfer_amd/token_losses.py) against oracle/token_ops.py, which
computes the formulas in 64 bits.  No counterpart in the reference: parity unpinned.

Tolerances.  U = 2^-24 is half a step of fp32.  A row's sum S has V positive terms; a thread adds at most V / 64 of them
(and at most 16 more joins and batch ends follow), each term carries the rounding of its exponent, d = (x - m) c with two
roundings, |d| ln2 2 U, and of the exponential, 2 U.  Weighted by the probabilities |d| averages to the entropy in bits plus
a constant, under 20 for the vocabularies here.  So ln S, and a log-probability, is off by at most
R = (V / 64 + 16 + 2 * 20 + 8) U, plus the rounding of the result.  A gradient entry has the relative error
R + 2 |log2 q_j| U + 8 U in fp32 and half a step of its own type; at a label two such terms are subtracted.
"""
import math

import pytest
import torch

from oracle import token_ops as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
#: Half a step relative to the value, and what is lost near 0: half the smallest step of fp16's subnormals; for the types with
#: fp32's range, the exponential itself, whose result is 0 below the smallest normal number 2^-126 (times coefficients of at
#: most 1, so an entry below it is off by at most that).
HALF = {torch.float32: (2.0 ** -24, 2.0 ** -126), torch.bfloat16: (2.0 ** -8, 2.0 ** -126), torch.float16: (2.0 ** -11, 2.0 ** -25)}


def row_error(vocab):
    return (vocab / 64 + 64) * U


def close(got, want, bound, what):
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape, what
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), what
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), what
    fine = ~(nan | inf)
    bound = torch.as_tensor(bound, dtype=torch.float64).expand(want.shape)
    over = ((got - want).abs() - bound)[fine]
    assert over.numel() == 0 or float(over.max()) <= 0, f"{what}: {float(over.max()):.3g} over the bound"


def grad_bound(want, dtype, log_q, a, b=None, h=None, tau=1.0, extra=0.0):
    """Elementwise bound of a gradient [N, V] whose rows have the coefficients a (of the log-probability) and b (of the
    entropy); extra: the relative error of the coefficients themselves."""
    half, tiny = HALF[dtype]
    vocab = want.shape[1]
    q = log_q.clamp(min=-1e300).exp()
    low = log_q.clamp(min=-200.0).abs() / math.log(2)
    size = a.abs()[:, None] * q
    if b is not None:
        size = size + b.abs()[:, None] * q * (log_q.clamp(min=-200.0).abs() + h[:, None])
    rel = row_error(vocab) + 8 * U + extra + 2 * low * U
    label = a.abs()[:, None] * (8 * U + extra)
    fp32 = (size * rel + label) / tau
    return (want.abs() + fp32) * half * 1.01 + fp32 + tiny


def logits(n, vocab, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, vocab, generator=g) * spread).to(dtype)


def labels_for(n, vocab, seed, share=5):
    g = torch.Generator().manual_seed(seed + 77)
    t = torch.randint(0, vocab, (n,), generator=g)
    if share:
        t[::share] = -100
    return t


def rand(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


# ---- log-probabilities ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,vocab", [(1, 1), (3, 2), (5, 7), (9, 64), (7, 1000), (6, 1025), (33, 2047), (2, 2049), (3, 8193), (1, 50001),
                                     (5, 131072)])
def test_token_logprobs(dtype, n, vocab):
    from style_transfer_amd.losses import token_logprobs
    tau = 0.7
    x, t = logits(n, vocab, dtype, vocab), labels_for(n, vocab, n, 5 if n > 1 else 0)
    logp, h, log_q, q = O.token_logprobs(x, t, tau)
    leaf = x.cuda().requires_grad_(True)
    got, got_h = token_logprobs(leaf, t.cuda(), temperature=tau, return_entropy=True)
    err = row_error(vocab)
    close(got, logp, err + logp.abs() * 2 * U, "logp")
    close(got_h, h, (h + 2) * err + 2 * h * U, "entropy")
    a, b = rand(1, n).double(), rand(2, n).double()
    torch.autograd.backward([got, got_h], [a.float().cuda(), b.float().cuda()])
    a, b = a.float().double() * (t != -100), b.float().double() * (t != -100)
    want = O.row_gradient(t, tau, h, log_q, q, a, b)
    assert leaf.grad.dtype == dtype
    close(leaf.grad, want, grad_bound(want, dtype, log_q, a, b, h, tau), "gradient")
    with torch.no_grad():                                     # the form without a gradient, one output, int32 labels
        again = token_logprobs(leaf, t.int().cuda(), temperature=tau)
    assert torch.equal(again, got.detach())


def test_one_gradient_of_the_two_outputs():
    from style_transfer_amd.losses import token_logprobs
    x, t = logits(4, 300, torch.float32, 3), labels_for(4, 300, 3)
    logp, h, log_q, q = O.token_logprobs(x, t)
    keep = (t != -100).double()
    for which in (0, 1):
        leaf = x.cuda().requires_grad_(True)
        token_logprobs(leaf, t.cuda(), return_entropy=True)[which].sum().backward()
        a, b = (keep, keep * 0) if which == 0 else (keep * 0, keep)
        want = O.row_gradient(t, 1.0, h, log_q, q, a, b)
        close(leaf.grad, want, grad_bound(want, torch.float32, log_q, a, b, h), f"output {which}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [5, 1000, 20000])
def test_masked_logits_and_empty_rows(dtype, vocab):
    from style_transfer_amd.losses import token_logprobs
    x = logits(8, vocab, dtype, 11)
    low = torch.finfo(dtype).min
    x[0, 1:] = -math.inf                                       # one token is left
    x[1, ::2] = low
    x[2, :] = low                                              # nothing but the mask's value: the formula's uniform row
    x[3, :] = -math.inf                                        # no distribution
    x[4, :] = math.nan                                         # does not count, so nobody looks
    x[5, 2:] = -math.inf                                       # the label itself is masked
    x[6, 0] = math.inf                                         # no finite softmax
    x[7, vocab // 2] = math.nan
    t = torch.tensor([0, 1, vocab - 1, 2, -100, 4, 1, 0])
    logp, h, log_q, q = O.token_logprobs(x[:6], t[:6])
    leaf = x.cuda().requires_grad_(True)
    got, got_h = token_logprobs(leaf, t.cuda(), return_entropy=True)
    err = row_error(vocab)
    close(got[:6], logp, err + logp.abs().nan_to_num(posinf=0) * 2 * U, "logp")
    close(got_h[:6], h, (h + 2) * err + 2 * h * U, "entropy")
    assert got[3] == -math.inf and got_h[3] == 0 and got[4] == 0 and got_h[4] == 0 and got[5] == -math.inf
    assert torch.isnan(got[6:]).all()
    got[[0, 1, 2, 3, 4, 6, 7]].sum().backward()
    a = torch.tensor([1.0, 1, 1, 1, 0, 0], dtype=torch.float64)
    want = O.row_gradient(t[:6], 1.0, h, log_q, q, a, a * 0)
    close(leaf.grad[:6], want, grad_bound(want, dtype, log_q, a), "gradient")
    assert not leaf.grad[3:6].any() and torch.isnan(leaf.grad[6:]).all()


@pytest.mark.parametrize("dtype,vocab", [(torch.float32, 1030), (torch.bfloat16, 4097), (torch.float16, 8000), (torch.bfloat16, 16383), (torch.float32, 8193)])
def test_many_rows_of_middle_size(dtype, vocab):
    """From 2048 rows on a row of up to 32 KB is a wave's: the same as of fewer rows at a time, and as the formula."""
    from style_transfer_amd.losses import token_logprobs
    rows = 2050
    x, t = logits(40, vocab, dtype, vocab).repeat(rows // 40 + 1, 1)[:rows], labels_for(rows, vocab, 3)
    x[1::40, : vocab // 2] = -math.inf
    t[t >= 0] = t[t >= 0] // 2 + vocab // 2                     # not a masked one
    leaf = x.cuda().requires_grad_(True)
    got, h = token_logprobs(leaf, t.cuda(), temperature=0.9, return_entropy=True)
    w = rand(4, rows).cuda()
    (got * w + h).sum().backward()
    few = x.cuda().requires_grad_(True)
    for part in range(0, rows, 1025):
        a, b = token_logprobs(few[part:part + 1025], t[part:part + 1025].cuda(), temperature=0.9, return_entropy=True)
        err = row_error(vocab)
        assert torch.allclose(got[part:part + 1025], a, atol=2 * err, rtol=4 * U) and torch.allclose(h[part:part + 1025], b, atol=24 * err, rtol=4 * U)
        (a * w[part:part + 1025] + b).sum().backward()
    # per unit of a probability: the row's error times what multiplies it, |w| + |log q| + h
    half, tiny = HALF[dtype]
    size = 2 * row_error(vocab) * (float(w.abs().max()) + 40)
    assert torch.allclose(leaf.grad.float(), few.grad.float(), rtol=2 * half, atol=size + tiny)
    some = slice(0, 44)
    logp, entropy, log_q, q = O.token_logprobs(x[some], t[some], 0.9)
    close(got[some], logp, row_error(vocab) + logp.abs() * 2 * U, "logp")
    close(h[some], entropy, (entropy + 2) * row_error(vocab) + 2 * entropy * U, "entropy")
    a, b = w[some].cpu().double(), torch.ones(44, dtype=torch.float64)
    want = O.row_gradient(t[some], 0.9, entropy, log_q, q, a, b)
    close(leaf.grad[some], want, grad_bound(want, dtype, log_q, a, b, entropy, 0.9), "gradient")


def test_labels_outside_the_vocabulary_are_nan_and_touch_nothing():
    from style_transfer_amd.losses import token_logprobs
    x = logits(4, 130, torch.float32, 5)
    t = torch.tensor([130, -1, 2 ** 40, 3])
    leaf = x.cuda().requires_grad_(True)
    got = token_logprobs(leaf, t.cuda())
    got.sum().backward()
    assert torch.isnan(got[:3]).all() and torch.isnan(leaf.grad[:3]).all()
    assert torch.isfinite(got[3]) and torch.isfinite(leaf.grad[3]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [333, 5001])
def test_strides_and_alignments(dtype, vocab):
    """Slices of a larger tensor in every alignment, read in place: the same numbers as of a copy."""
    from style_transfer_amd.losses import token_logprobs
    base = logits(3 * 6, vocab + 11, dtype, 21).view(3, 6, vocab + 11).cuda()
    t = labels_for(3 * 4, vocab, 9).view(3, 4).cuda()
    for off in range(9):
        leaf = base.clone().requires_grad_(True)
        view = leaf[:, 1:5, off:off + vocab]
        assert not view.is_contiguous()
        copy = view.detach().contiguous().requires_grad_(True)
        w = rand(off, 3, 4).cuda()
        for v in (view, copy):
            (token_logprobs(v, t) * w).sum().backward()
        want, err = token_logprobs(copy, t).detach(), row_error(vocab)
        assert torch.allclose(token_logprobs(view, t), want, atol=4 * err, rtol=4 * U)
        inner = leaf.grad[:, 1:5, off:off + vocab]
        half, tiny = HALF[dtype]
        assert torch.allclose(inner.float(), copy.grad.float(), atol=4 * err, rtol=2 * half)     # two roundings of nearly one value
        outer = leaf.grad.clone()
        outer[:, 1:5, off:off + vocab] = 0
        assert not outer.any()


def test_expanded_rows_and_long_offsets():
    from style_transfer_amd.losses import token_logprobs
    x, t = logits(1, 900, torch.float32, 4), torch.tensor([5, 5, 5])
    leaf = x.cuda().requires_grad_(True)
    token_logprobs(leaf.expand(3, 900), t.cuda()).sum().backward()      # a broadcast row: the gradients add up
    logp, h, log_q, q = O.token_logprobs(x, t[:1])
    want = 3 * O.row_gradient(t[:1], 1.0, h, log_q, q, torch.ones(1, dtype=torch.float64), torch.zeros(1, dtype=torch.float64))
    close(leaf.grad, want, grad_bound(want, torch.float32, log_q, 3 * torch.ones(1, dtype=torch.float64)) + 4 * U * want.abs(), "gradient")
    rows = torch.empty_strided((3, 1000), (1_500_000_000, 1), dtype=torch.bfloat16, device="cuda")   # row 2 starts beyond 2^31 elements
    x = logits(3, 1000, torch.bfloat16, 6)
    rows.copy_(x)
    assert torch.equal(token_logprobs(rows, t.cuda()), token_logprobs(x.cuda(), t.cuda()))


# ---- preference loss -------------------------------------------------------------------------------------------------------
def sequence_labels(n, vocab, seed, longest):
    t = labels_for(n * longest, vocab, seed, 4).view(n, longest)
    for s in range(n):
        t[s, longest - (s * 3) % longest:] = -100              # ragged ends
    return t


def packed(x, t):
    """The counted stretch of each padded sequence without the padding behind it: rows, labels, cu_seqlens."""
    n, longest = t.shape
    keep = [max([i + 1 for i in range(longest) if int(t[s, i]) != -100], default=0) for s in range(n)]
    rows = torch.cat([x[s, :k] for s, k in enumerate(keep)])
    return rows, torch.cat([t[s, :k] for s, k in enumerate(keep)]), torch.tensor([0, *torch.tensor(keep).cumsum(0).tolist()])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["padded", "packed"])
@pytest.mark.parametrize("kind,smoothing,average,beta", [("sigmoid", 0.0, False, 0.1), ("sigmoid", 0.2, True, 2.0), ("ipo", 0.0, True, 0.3),
                                                         ("hinge", 0.0, False, 0.05)])
def test_preference_loss(dtype, layout, kind, smoothing, average, beta):
    from style_transfer_amd.losses import PreferenceLoss
    pairs, longest, vocab = 3, 9, 517
    x = logits(2 * pairs * longest, vocab, dtype, 31).view(2 * pairs, longest, vocab)
    t = sequence_labels(2 * pairs, vocab, 8, longest)
    cu = None
    if layout == "packed":
        x, t, cu = packed(x, t)
    seqs = O.sequences_of(t, cu)
    flat, rows = t.reshape(-1), x.reshape(-1, vocab)
    ref = -rand(5, 2 * pairs).abs() * (1 if average else 30)
    loss, rewards, want = O.preference(rows, flat, seqs, ref, beta, kind, smoothing, average)
    leaf = x.cuda().requires_grad_(True)
    got = PreferenceLoss(beta=beta, kind=kind, label_smoothing=smoothing, average=average)(
        leaf, t.cuda(), ref.cuda(), None if cu is None else cu.int().cuda())
    # a sequence's sum is off by its rows' errors; h by two of them; every loss is Lipschitz in h near its value here
    each = longest * (row_error(vocab) + 20 * U)
    close(torch.cat([got.chosen_rewards, got.rejected_rewards]), rewards, beta * each + rewards.abs() * 2 * U, "rewards")
    gap = (rewards[:pairs] - rewards[pairs:]).abs().max() / beta
    steep = beta if kind != "ipo" else 2 * (float(gap) + 0.5 / beta)
    close(got.loss, torch.tensor(loss), 2 * steep * each + abs(loss) * 2 * U, "loss")
    got.loss.backward()
    logp, h, log_q, q = O.token_logprobs(rows, flat)
    a = want.gather(1, flat.clamp(min=0)[:, None])[:, 0] / (1 - q.gather(1, flat.clamp(min=0)[:, None])[:, 0])
    bend = 2 if kind == "ipo" else beta * beta / 4              # how far a slope moves with h
    extra = 2 * bend * each / pairs / max(1e-30, float(a.abs()[a != 0].min()) if bool(a.any()) else 1)
    close(leaf.grad.reshape(-1, vocab), want, grad_bound(want, dtype, log_q, a, extra=extra), "gradient")


def test_preference_empty_sequences_and_rows_behind_the_last():
    from style_transfer_amd.losses import preference_loss
    x, t = logits(9, 70, torch.float32, 2), labels_for(9, 70, 2, 0)
    cu = torch.tensor([1, 4, 4, 6, 7], dtype=torch.int32)       # row 0 and rows 7, 8 lie outside; the second chosen one is empty
    loss, rewards, want = O.preference(x, t, O.sequences_of(t, cu))
    leaf = x.cuda().requires_grad_(True)
    got = preference_loss(leaf, t.cuda(), cu_seqlens=cu.cuda())
    got.loss.backward()
    assert abs(float(got.loss.detach()) - loss) <= 1e-5 * abs(loss)
    close(leaf.grad, want, 1e-5 * want.abs() + 1e-7, "gradient")
    assert not leaf.grad[[0, 7, 8]].any() and float(got.chosen_rewards[1]) == 0
    # no rows at all: the references alone
    none = torch.empty(4, 0, 70, device="cuda", requires_grad=True)
    ref = torch.tensor([1.0, 2.0, 3.0, 5.0])
    got = preference_loss(none, torch.empty(4, 0, dtype=torch.long, device="cuda"), ref.cuda(), beta=1.0)
    got.loss.backward()
    want = sum(math.log1p(math.exp(-(-ref[i] + ref[i + 2]))) for i in range(2)) / 2
    assert abs(float(got.loss.detach()) - want) < 1e-6 and none.grad.shape == none.shape
    assert float(preference_loss(torch.empty(0, 3, 7, device="cuda"), torch.empty(0, 3, dtype=torch.long, device="cuda")).loss) == 0


# ---- clipped policy loss --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["padded", "packed"])
@pytest.mark.parametrize("reduction,per_sequence,kl,ent,tau", [("token", False, 0.0, 0.0, 1.0), ("sequence", True, 0.05, 0.0, 1.3),
                                                               ("token", True, 0.1, 0.02, 0.8), ("sequence", False, 0.0, 0.5, 1.0)])
@pytest.mark.parametrize("vocab", [411, 4099])
def test_clipped_policy_loss(dtype, layout, reduction, per_sequence, kl, ent, tau, vocab):
    from style_transfer_amd.losses import ClippedPolicyLoss
    count, longest = 4, 7
    x = logits(count * longest, vocab, dtype, 41).view(count, longest, vocab)
    t = sequence_labels(count, vocab, 3, longest)
    cu = None
    if layout == "packed":
        x, t, cu = packed(x, t)
    flat, rows = t.reshape(-1), x.reshape(-1, vocab)
    n = flat.numel()
    seqs = O.sequences_of(t, cu)
    logp, h, log_q, q = O.token_logprobs(rows, flat, tau)
    step = torch.linspace(-0.6, 0.6, n)[torch.randperm(n, generator=torch.Generator().manual_seed(1))]     # none near a border: a ratio is off by 2e-5 at most
    assert min(abs(math.exp(-float(v)) - e) for v in step for e in (0.75, 1.3)) > 1e-4
    old, ref = (logp.float() + step), logp.float() + rand(6, n) * 0.5
    adv = rand(7, count) if per_sequence else rand(7, n)
    each = torch.zeros(n)
    for s, (b, e) in enumerate(seqs):
        each[b:e] = adv[s] if per_sequence else adv[b:e]
    loss, stats, want = O.policy(rows, flat, seqs, old, each, ref if kl else None, 0.25, 0.3, kl, ent, tau, reduction == "sequence")
    leaf = x.cuda().requires_grad_(True)
    got = ClippedPolicyLoss(0.25, 0.3, kl, ent, tau, reduction)(
        leaf, t.cuda(), old.view(t.shape).cuda(), (adv if per_sequence else adv.view(t.shape)).cuda(),
        ref.view(t.shape).cuda() if kl else None, None if cu is None else cu.int().cuda())
    # a log-probability's error moves a ratio by as much relatively, a KL estimate by |exp(d) - 1|, the entropy by itself
    err = row_error(vocab) + 30 * U
    top = float(each.abs().max()) * 2
    close(got.stats, stats, torch.tensor([top * err, 4 * err, 14 * err, 2 * U]) + stats.abs() * 2 * U, "stats")
    close(got.loss, torch.tensor(loss), top * err + 4 * kl * err + 14 * ent * err + 4 * U * float(stats.abs().sum()), "loss")
    got.loss.backward()
    w = torch.zeros(n, dtype=torch.float64)
    for b, e in seqs:
        held = [r for r in range(b, e) if int(flat[r]) != -100]
        w[held] = 1.0 if reduction == "token" else 1.0 / max(1, len(held))
    w = w / (w.sum() if reduction == "token" else sum(any(int(flat[r]) != -100 for r in range(b, e)) for b, e in seqs))
    # coefficients: |A r| and kl |exp(d) - 1| move with the log-probability's error
    a = w * (each.double().abs() * 2 + kl * 4)
    close(leaf.grad.reshape(-1, vocab), want, grad_bound(want, dtype, log_q, a, w * ent, h, tau, extra=err), "gradient")


def test_policy_counts_only_what_is_there():
    from style_transfer_amd.losses import clipped_policy_loss
    x = logits(6, 50, torch.float32, 1)
    x[1] = math.nan
    t = torch.tensor([[3, -100], [-100, -100], [7, 9]])
    old, adv = torch.zeros(3, 2), torch.tensor([1.0, math.nan, -1.0])
    adv[1] = 2.0
    leaf = x.view(3, 2, 50).cuda().requires_grad_(True)
    for reduction, weights in (("token", [1 / 3] * 3), ("sequence", [1 / 2, 1 / 4, 1 / 4])):
        leaf.grad = None
        loss, stats = clipped_policy_loss(leaf, t.cuda(), old.cuda() - 3, adv.cuda(), reduction=reduction)
        loss.backward()
        logp = O.token_logprobs(x, t.view(-1))[0]
        want = sum(w * -min(r * a, min(max(r, 0.8), 1.2) * a)
                   for w, r, a in zip(weights, (logp[[0, 4, 5]] + 3).exp().tolist(), (1.0, -1.0, -1.0)))
        assert abs(float(loss.detach()) - want) < 1e-5
        assert torch.isfinite(leaf.grad).all() and not leaf.grad[0, 1].any() and not leaf.grad[1].any()
    # nothing counts: 0, and a zero gradient
    none = torch.full_like(t, -100).cuda()
    leaf.grad = None
    loss, stats = clipped_policy_loss(leaf, none, old.cuda(), adv.cuda(), old.cuda(), kl_coef=0.1, entropy_coef=0.1)
    loss.backward()
    assert float(loss.detach()) == 0 and not stats.any() and not leaf.grad.any()
    empty = torch.empty(0, 50, device="cuda", requires_grad=True)
    z = torch.empty(0, device="cuda")
    loss, stats = clipped_policy_loss(empty, z.long(), z, torch.ones(2, device="cuda"), cu_seqlens=torch.zeros(3, dtype=torch.int32, device="cuda"))
    loss.backward()
    assert float(loss.detach()) == 0 and empty.grad.shape == (0, 50)


def test_rows_outside_the_sequences_do_not_count():
    from style_transfer_amd.losses import clipped_policy_loss
    x, t = logits(8, 90, torch.float32, 3), labels_for(8, 90, 1, 0)
    old, adv = torch.full((8,), -4.0), rand(3, 8)
    for reduction in ("token", "sequence"):
        leaf = x.cuda().requires_grad_(True)
        cu = torch.tensor([2, 4, 4, 7], dtype=torch.int32)
        loss, stats = clipped_policy_loss(leaf, t.cuda(), old.cuda(), adv.cuda(), cu_seqlens=cu.cuda(), reduction=reduction)
        loss.backward()
        want, _, grad = O.policy(x, t, O.sequences_of(t, cu), old, adv, per_sequence=reduction == "sequence")
        assert abs(float(loss.detach()) - want) < 1e-5
        close(leaf.grad, grad, 2e-5 * grad.abs() + 1e-6, "gradient")
        assert not leaf.grad[[0, 1, 7]].any()


@pytest.mark.parametrize("rows,sequences", [(700, 1), (900, 64), (900, 65), (3000, 700), (20000, 5000), (300000, 70000)])
@pytest.mark.parametrize("reduction", ["token", "sequence"])
def test_policy_over_many_rows_and_sequences(rows, sequences, reduction):
    """One sequence to tens of thousands, empty ones among them, more rows than one block adds up; the formula in 64 bits."""
    from style_transfer_amd.losses import clipped_policy_loss
    vocab = 3
    g = torch.Generator().manual_seed(rows + sequences)
    x, t = logits(rows, vocab, torch.float32, rows, 1.0), torch.randint(0, vocab, (rows,), generator=g)
    t[torch.rand(rows, generator=g) < 0.3] = -100
    cu = torch.cat([torch.tensor([2, rows - 3]), torch.randint(2, rows - 2, (sequences - 1,), generator=g)]).sort().values
    adv, old = rand(1, sequences), torch.full((rows,), -1.0)
    lengths = cu[1:] - cu[:-1]
    of = torch.full((rows,), -1)
    of[2:rows - 3] = torch.repeat_interleave(torch.arange(sequences), lengths)
    keep = (t != -100) & (of >= 0)
    count = torch.zeros(sequences, dtype=torch.float64).index_add_(0, of[keep], torch.ones(int(keep.sum()), dtype=torch.float64))
    w = torch.where(keep, 1 / count[of] / (count > 0).sum() if reduction == "sequence" else 1 / count.sum(), 0.0)
    z = x.double().requires_grad_(True)
    logp = torch.log_softmax(z, 1).gather(1, t.clamp(min=0)[:, None])[:, 0]
    ratio, a = (logp - old.double()).exp(), adv.double()[of]
    each = -torch.minimum(ratio * a, ratio.clamp(0.8, 1.2) * a)
    want = (w * each).sum()
    want.backward()
    leaf = x.cuda().requires_grad_(True)
    got = clipped_policy_loss(leaf, t.cuda(), old.cuda(), adv.cuda(), cu_seqlens=cu.int().cuda(), reduction=reduction)
    got.loss.backward()
    # a row: its logarithm's and its exponential's error, relative to a ratio of at most e; entries: as much of the row's weight
    row = row_error(vocab) * math.e * a.abs()
    close(got.loss, want.detach(), float((w * row).sum()) + 4 * U * float(w @ each.detach().abs()), "loss")
    close(leaf.grad, z.grad, (w * row)[:, None] * 2 + 4 * U * z.grad.abs() + 2.0 ** -126, "gradient")


# ---- distillation -------------------------------------------------------------------------------------------------------------
def teacher(x, k, tau, tail, seed):
    g = torch.Generator().manual_seed(seed)
    n, vocab = x.shape
    idx = torch.stack([torch.randperm(vocab, generator=g)[:k] for _ in range(n)])
    val = x.float().gather(1, idx) + torch.randn(n, k, generator=g)
    if tail:
        val = torch.log_softmax(val / tau, 1) + math.log(0.9)
    return idx, val


def distill_bound(x, idx, val, mask, tau, want, dtype):
    """Elementwise: a row's weight times tau times (q_j + its listed probability + the rest's share), each with the row's error;
    the rest's share divides two sums of the row."""
    half, tiny = HALF[dtype]
    vocab = x.shape[1]
    q = torch.stack([O.row(r, tau)[1] for r in x])
    log2 = q.clamp(min=1e-80).log2().abs()
    w = tau / max(1, x.shape[0] if mask is None else int(mask.sum()))
    fp32 = w * (2 * q + (want / w - q).abs()) * (2 * row_error(vocab) + 40 * U + 4 * log2 * U)
    return (want.abs() + fp32) * half * 1.01 + fp32 + tiny


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("n,vocab,k,tau", [(1, 1, 1, 1.0), (3, 7, 7, 2.0), (6, 1000, 5, 1.0), (5, 2051, 64, 1.5), (3, 8200, 1, 0.5),
                                           (2, 40001, 300, 1.0)])
def test_topk_distill_loss(dtype, tail, n, vocab, k, tau):
    from style_transfer_amd.losses import TopKDistillLoss
    x = logits(n, vocab, dtype, vocab + k)
    idx, val = teacher(x, k, tau, tail, 5)
    mask = None
    if n > 2:
        mask = torch.ones(n, dtype=torch.bool)
        mask[1] = False
        x[1] = math.nan
    if k > 2:
        idx[0, k // 2:] = -1                                  # a shorter list
        idx[-1, 0] = -1
    loss, want = O.distill(torch.where(x.isnan(), 0, x), idx, val, mask, tau, tail)
    leaf = x.cuda().requires_grad_(True)
    got = TopKDistillLoss(tau, tail)(leaf, idx.cuda(), val.cuda(), None if mask is None else mask.cuda())
    close(got, torch.tensor(loss), tau * tau * (2 * row_error(vocab) + 60 * U) + abs(loss) * 4 * U, "loss")
    got.backward()
    x = torch.where(x.isnan(), 0, x)
    close(leaf.grad, want, distill_bound(x, idx, val, mask, tau, want, dtype), "gradient")
    again = TopKDistillLoss(tau, tail)(leaf.detach(), idx.int().cuda(), val.cuda(), None if mask is None else mask.cuda())
    assert torch.equal(again, got.detach())


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("vocab", [300, 9000])
def test_distill_repeated_unused_and_foreign_entries(tail, vocab):
    from style_transfer_amd.losses import topk_distill_loss
    x = logits(6, vocab, torch.float32, 13)
    idx, val = teacher(x, 6, 1.0, tail, 4)
    if tail:
        val = val - math.log(3)                                # listed twice still leaves mass
    idx[0, 3] = idx[0, 1]                                      # a token twice, and three times
    idx[1, [2, 4]] = idx[1, 0].clone()
    idx[2] = -1                                                # no entry
    val[3, :3] = -math.inf                                     # no mass on an entry
    x[4, :] = -math.inf
    x[4, idx[4]] = 1.0                                         # everything off the list is masked: the rest is impossible
    loss, want = O.distill(x[:4], idx[:4], val[:4], None, 1.0, tail)
    leaf = x[:4].cuda().requires_grad_(True)
    got = topk_distill_loss(leaf, idx[:4].cuda(), val[:4].cuda(), tail=tail)
    got.backward()
    close(got, torch.tensor(loss), 2 * row_error(vocab) + 60 * U + abs(loss) * 4 * U, "loss")
    close(leaf.grad, want, distill_bound(x[:4], idx, val, None, 1.0, want, torch.float32), "gradient")
    assert not leaf.grad[2].any() or tail
    leaf = x[4:5].cuda().requires_grad_(True)
    got = topk_distill_loss(leaf, idx[4:5].cuda(), val[4:5].cuda(), tail=tail)
    got.backward()
    assert float(got.detach()) == math.inf if tail else math.isfinite(float(got.detach()))
    assert torch.isfinite(leaf.grad).all()
    idx[5, 2] = vocab                                          # names no token
    leaf = x[5:].cuda().requires_grad_(True)
    got = topk_distill_loss(leaf, idx[5:].cuda(), val[5:].cuda(), tail=tail)
    got.backward()
    assert math.isnan(float(got.detach())) and torch.isnan(leaf.grad).any()
    none = torch.empty(0, vocab, device="cuda", requires_grad=True)
    got = topk_distill_loss(none, torch.empty(0, 3, dtype=torch.long, device="cuda"), torch.empty(0, 3, device="cuda"))
    got.backward()
    assert float(got.detach()) == 0 and none.grad.shape == (0, vocab)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("vocab,k", [(5000, 4096), (300, 500), (60000, 1500)])
def test_distill_long_lists(tail, vocab, k):
    """More entries than a row has threads, or tokens: drawn with repeats."""
    from style_transfer_amd.losses import topk_distill_loss
    x = logits(3, vocab, torch.float32, k)
    idx = torch.randint(0, vocab, (3, k), generator=torch.Generator().manual_seed(vocab))
    idx[1] = torch.where(torch.rand(k, generator=torch.Generator().manual_seed(1)) < 0.5, -1, idx[1])
    val = torch.log_softmax(rand(k, 3, k), 1) - 0.2 if tail else rand(k, 3, k)
    loss, want = O.distill(x, idx, val, None, 1.0, tail)
    leaf = x.cuda().requires_grad_(True)
    got = topk_distill_loss(leaf, idx.cuda(), val.cuda(), tail=tail)
    got.backward()
    # the list's own sums: K / 64 entries a lane where a wave goes through them, as for a row
    more = k / 64 * U
    close(got, torch.tensor(loss), 2 * row_error(vocab) + 60 * U + 4 * more + abs(loss) * 4 * U, "loss")
    q = torch.stack([O.row(r, 1.0)[1] for r in x])
    listed = torch.zeros(3, vocab, dtype=torch.float64)         # what the list subtracts, a token's entries added up
    p = (val.double() if tail else torch.log_softmax(val.double().masked_fill(idx < 0, -math.inf), 1)).exp() * (idx >= 0)
    listed.scatter_add_(1, idx.clamp(min=0), p)
    close(leaf.grad, want, distill_bound(x, idx, val, None, 1.0, want, torch.float32) + (q + listed) / 3 * (4 * more + 40 * U), "gradient")


def test_distill_keeps_what_little_the_rest_holds():
    """The student is sure of a listed token: 1 - sum q has no digit left, the sum off the list has all of them."""
    from style_transfer_amd.losses import topk_distill_loss
    x = torch.full((1, 500), -20.0)
    x[0, 7] = 10.0
    idx, val = torch.tensor([[7]]), torch.tensor([[math.log(0.75)]])
    loss, want = O.distill(x, idx, val, None, 1.0, True)
    leaf = x.cuda().requires_grad_(True)
    got = topk_distill_loss(leaf, idx.cuda(), val.cuda(), tail=True)
    got.backward()
    assert abs(float(got.detach()) - loss) <= 1e-6 * loss
    close(leaf.grad, want, 1e-5 * want.abs(), "gradient")


# ---- every size of row, and rows whose logits are far apart ------------------------------------------------------------------------
#: sizes on both sides of every change of kernel: a wave's rows (4, 8, 16 KB), a block's (32, 64, 128, 256, 320 KB), and beyond
SIZES = [(torch.bfloat16, v) for v in (2040, 2056, 4090, 8191, 8200, 16380, 16390, 32770, 65536, 65550, 131072, 131080, 170001)] + [
    (torch.float32, v) for v in (1023, 1029, 2050, 4095, 8190, 16387, 32769, 65537, 81930, 131072)] + [(torch.float16, 20001), (torch.float16, 140001)]


def far_logits(n, vocab, dtype, seed):
    """Rows whose first vectors say nothing about the rest: masked, tiny, or far below what follows."""
    x = logits(n, vocab, dtype, seed)
    x[1, : vocab // 2] = -math.inf
    x[2] = (x[2].float() * 4 - 60).to(dtype)
    x[2, vocab - 2] = 60.0                                      # 170 bits above the first vectors
    x[3, : vocab - vocab // 3] = torch.finfo(dtype).min
    x[3, vocab // 2] = -3.0
    return x


SIZES += [(torch.bfloat16, 70001), (torch.float32, 40960), (torch.float16, 81921)]       # 140 KB, 160 KB and a little more


@pytest.mark.parametrize("dtype,vocab", SIZES)
def test_policy_rows_of_every_size(dtype, vocab):
    from style_transfer_amd.losses import clipped_policy_loss
    n, tau, ent, kl = 5, 1.1, 0.01, 0.1
    x = far_logits(n, vocab, dtype, vocab)
    t = torch.tensor([[vocab - 1, vocab - 2, vocab - 2, vocab // 2, -100]])
    flat = t.view(-1)
    logp, h, log_q, q = O.token_logprobs(x, flat, tau)
    step = torch.tensor([0.1, -0.1, 0.5, 0.05, 0.0])
    old, ref, adv = logp.float() + step, logp.float() - 0.25, torch.tensor([1.0, -1.0, 0.5, 2.0, 9.0])
    loss, stats, want = O.policy(x, flat, [(0, n)], old, adv, ref, 0.2, 0.2, kl, ent, tau)
    leaf = x.view(1, n, vocab).cuda().requires_grad_(True)
    got = clipped_policy_loss(leaf, t.cuda(), old.view(1, n).cuda(), adv.view(1, n).cuda(), ref.view(1, n).cuda(), kl_coef=kl, entropy_coef=ent,
                              temperature=tau)
    got.loss.backward()
    # old and ref are as far from 0 as the log-probabilities: 2 U of them comes on top of a row's error
    err = row_error(vocab) + 40 * U + 2 * U * float(logp.abs().max())
    close(got.stats, stats, torch.tensor([4 * err, 4 * err, 14 * err, 2 * U]) + stats.abs() * 2 * U, "stats")
    close(got.loss, torch.tensor(loss), 5 * err + 4 * U * float(stats.abs().sum()), "loss")
    w = torch.tensor([0.25] * 4 + [0.0], dtype=torch.float64)
    close(leaf.grad[0], want, grad_bound(want, dtype, log_q, w * (2 * adv.double().abs() + 4 * kl), w * ent, h, tau, extra=err), "gradient")
    with torch.no_grad():
        again = clipped_policy_loss(leaf, t.cuda(), old.view(1, n).cuda(), adv.view(1, n).cuda(), ref.view(1, n).cuda(), kl_coef=kl,
                                    entropy_coef=ent, temperature=tau)
    assert torch.equal(again.loss, got.loss.detach()) and torch.equal(again.stats, got.stats)


@pytest.mark.parametrize("dtype,vocab", SIZES)
@pytest.mark.parametrize("tail", [False, True])
def test_distill_rows_of_every_size(dtype, vocab, tail):
    from style_transfer_amd.losses import topk_distill_loss
    n, k, tau = 5, 70, 1.3
    x = far_logits(n, vocab, dtype, vocab + 1)
    idx, val = teacher(torch.zeros(n, vocab), k, tau, tail, vocab)
    idx[:, 0], idx[:, 1], idx[:, 2] = vocab - 1, vocab // 2, 0  # the last element, a finite one of the masked row, the first
    idx[:, 3:] = torch.where((idx[:, 3:] == vocab - 1) | (idx[:, 3:] == vocab // 2) | (idx[:, 3:] == 0), -1, idx[:, 3:])
    masked = x.gather(1, idx.clamp(min=0).long()) <= torch.finfo(dtype).min
    val = val.masked_fill(masked, -math.inf)                    # the teacher has no mass where the student is masked
    mask = torch.tensor([True, True, True, True, False])
    loss, want = O.distill(x, idx, val, mask, tau, tail)
    leaf = x.cuda().requires_grad_(True)
    got = topk_distill_loss(leaf, idx.cuda(), val.cuda(), mask.cuda(), temperature=tau, tail=tail)
    got.backward()
    # a term p (log p - log q) is off by a row's error and by 8 U of log q, which reaches 250 here
    close(got, torch.tensor(loss), tau * tau * (2 * row_error(vocab) + 60 * U) + abs(loss) * 8 * U, "loss")
    close(leaf.grad, want, distill_bound(x, idx, val, mask, tau, want, dtype), "gradient")


@pytest.mark.parametrize("dtype,vocab", [(torch.float32, 1023), (torch.bfloat16, 8200), (torch.float32, 16387), (torch.float16, 60000),
                                         (torch.float32, 65537), (torch.bfloat16, 170001)])
def test_low_logits_behind_masked_ones(dtype, vocab):
    """Logits far below 0 behind a masked beginning: the first vectors of some waves, or of all, hold nothing to start from."""
    from style_transfer_amd.losses import clipped_policy_loss, topk_distill_loss, token_logprobs
    x = logits(5, vocab, dtype, vocab) - 300.0
    x[0, : vocab // 2] = -math.inf
    x[1, : min(1000, vocab // 2)] = -math.inf
    x[2, vocab // 3:] = -math.inf
    x[3, : vocab - 3] = -math.inf                               # the last elements alone
    x[4, ::2] = -math.inf
    t = torch.tensor([vocab - 1, vocab - 2, 5, vocab - 2, 7])
    logp, h, log_q, q = O.token_logprobs(x, t)
    err = row_error(vocab) + logp.abs() * 2 * U
    leaf = x.cuda().requires_grad_(True)
    got, entropy = token_logprobs(leaf, t.cuda(), return_entropy=True)
    close(got, logp, err, "logp")
    close(entropy, h, (h + 2) * row_error(vocab) + 2 * h * U, "entropy")
    seqs, adv = [(0, 5)], torch.tensor([1.0, -1.0, 2.0, 0.5, -0.5])
    loss, stats, want = O.policy(x, t, seqs, logp.float(), adv, ent=0.1)
    policy = clipped_policy_loss(leaf[None], t[None].cuda(), logp.float()[None].cuda(), adv[None].cuda(), entropy_coef=0.1)
    policy.loss.backward()
    close(policy.stats, stats, 14 * float(err.max()) + stats.abs() * 2 * U, "stats")
    a, b = adv.abs().double() / 5, torch.full((5,), 0.02, dtype=torch.float64)
    close(leaf.grad, want, grad_bound(want, dtype, log_q, a, b, h, extra=2 * float(err.max())), "policy gradient")
    for tail in (False, True):
        idx = torch.tensor([[vocab - 1, vocab - 2], [vocab - 2, vocab - 1], [5, 3], [vocab - 2, vocab - 1], [7, 9]])
        val = torch.tensor([[-0.5, -1.5]]).repeat(5, 1)
        loss, want = O.distill(x, idx, val, None, 1.0, tail)
        leaf.grad = None
        got = topk_distill_loss(leaf, idx.cuda(), val.cuda(), tail=tail)
        got.backward()
        close(got, torch.tensor(loss), 2 * row_error(vocab) + 60 * U + abs(loss) * 8 * U, "loss")
        close(leaf.grad, want, distill_bound(x, idx, val, None, 1.0, want, dtype), "distillation gradient")


@pytest.mark.parametrize("dtype,vocab", [(torch.float32, 2 ** 20), (torch.bfloat16, 2 ** 20), (torch.float16, 2 ** 19 + 3), (torch.float32, 400003)])
@pytest.mark.parametrize("tail", [False, True])
def test_the_largest_vocabularies(dtype, vocab, tail):
    from style_transfer_amd.losses import clipped_policy_loss, topk_distill_loss
    n, k = 3, 40
    x = logits(n, vocab, dtype, vocab)
    idx, val = teacher(x, k, 1.0, tail, 2)
    idx[:, 0], idx[0, 1] = vocab - 1, 0
    loss, want = O.distill(x, idx, val, None, 1.0, tail)
    wide = torch.zeros(n, vocab + 3, dtype=dtype)
    wide[:, 3:] = x                                             # no row begins on 16 bytes
    leaf = wide.cuda()[:, 3:].requires_grad_(True)
    got = topk_distill_loss(leaf, idx.cuda(), val.cuda(), tail=tail)
    got.backward()
    close(got, torch.tensor(loss), 2 * row_error(vocab) + 60 * U + abs(loss) * 4 * U, "loss")
    close(leaf.grad, want, distill_bound(x, idx, val, None, 1.0, want, dtype), "gradient")
    t = torch.tensor([vocab - 1, 0, 77])
    logp, h, log_q, q = O.token_logprobs(x, t)
    loss, stats, want = O.policy(x, t, [(0, n)], logp.float(), torch.ones(n))
    leaf.grad = None
    got = clipped_policy_loss(leaf[None], t[None].cuda(), logp.float()[None].cuda(), torch.ones(1, n).cuda())
    got.loss.backward()
    err = row_error(vocab) + 40 * U
    close(got.stats, stats, 20 * err + stats.abs() * 2 * U, "stats")
    close(leaf.grad, want, grad_bound(want, dtype, log_q, torch.full((n,), 1 / n, dtype=torch.float64), extra=2 * err), "policy gradient")


@pytest.mark.parametrize("dtype,vocab", [(torch.float32, 1000), (torch.bfloat16, 5001), (torch.float32, 20000), (torch.bfloat16, 140000)])
@pytest.mark.parametrize("value", [-2e7, -1e9, -1e10, -3e14, -1e29, 5e10])
def test_rows_of_a_finite_mask(dtype, vocab, value):
    """Rows that hold nothing but a mask's value, or a second one far below it: uniform over the largest, whatever its size."""
    from style_transfer_amd.losses import clipped_policy_loss, topk_distill_loss, token_logprobs
    x = torch.full((3, vocab), value).to(dtype)
    x[1, vocab // 2:] = -math.inf
    x[2, : vocab // 3] = torch.tensor(value).to(dtype) - abs(value) / 8
    t = torch.tensor([vocab - 1, 3, vocab // 2])
    for tau in (1.0, 0.7):
        logp, h, log_q, q = O.token_logprobs(x, t, tau)
        leaf = x.cuda().requires_grad_(True)
        got, entropy = token_logprobs(leaf, t.cuda(), temperature=tau, return_entropy=True)
        close(got, logp, row_error(vocab) + logp.abs() * 2 * U, "logp")
        close(entropy, h, (h + 2) * row_error(vocab) + 2 * h * U, "entropy")
        loss, stats, want = O.policy(x, t, [(0, 3)], logp.float(), torch.ones(3), ent=0.1, tau=tau)
        policy = clipped_policy_loss(leaf[None], t[None].cuda(), logp.float()[None].cuda(), torch.ones(1, 3).cuda(), entropy_coef=0.1, temperature=tau)
        policy.loss.backward()
        err = row_error(vocab) + 24 * U
        close(policy.stats, stats, 14 * err + stats.abs() * 2 * U, "stats")
        third = torch.full((3,), 1 / 3, dtype=torch.float64)
        close(leaf.grad, want, grad_bound(want, dtype, log_q, third, third / 10, h, tau, extra=2 * err), "policy gradient")
        idx, val = torch.tensor([[1, 2], [3, 4], [vocab - 1, vocab - 2]]), torch.tensor([[-0.5, -1.5]]).repeat(3, 1)
        for tail in (False, True):
            loss, want = O.distill(x, idx, val, None, tau, tail)
            leaf.grad = None
            got = topk_distill_loss(leaf, idx.cuda(), val.cuda(), temperature=tau, tail=tail)
            got.backward()
            close(got, torch.tensor(loss), 2 * row_error(vocab) + 60 * U + abs(loss) * 8 * U, "loss")
            close(leaf.grad, want, distill_bound(x, idx, val, None, tau, want, dtype), "distillation gradient")


def test_a_padded_batch_in_place():
    """Rows of a slice at every alignment through the kernels that hold a row: as of a copy, and no other memory is written."""
    from style_transfer_amd import losses
    vocab = 2500
    base = logits(2 * 5, vocab + 9, torch.bfloat16, 2).view(2, 5, vocab + 9).cuda()
    t = labels_for(2 * 3, vocab, 4).view(2, 3).cuda()
    idx, val = teacher(torch.zeros(6, vocab), 9, 1.0, True, 3)
    idx, val, old = idx.view(2, 3, 9).cuda(), val.view(2, 3, 9).cuda(), torch.full((2, 3), -8.0).cuda()
    for off in range(9):
        for fn in (lambda v: losses.clipped_policy_loss(v, t, old, old[:, 0] + 9).loss, lambda v: losses.topk_distill_loss(v, idx, val, tail=True),
                   lambda v: losses.preference_loss(v, t).loss):
            leaf = base.clone().requires_grad_(True)
            view = leaf[:, 1:4, off:off + vocab]
            copy = view.detach().contiguous().requires_grad_(True)
            a, b = fn(view), fn(copy)
            a.backward()
            b.backward()
            assert abs(float(a.detach()) - float(b.detach())) <= 4 * row_error(vocab) * (1 + abs(float(b.detach())))
            inner = leaf.grad[:, 1:4, off:off + vocab].float()
            assert torch.allclose(inner, copy.grad.float(), atol=4 * row_error(vocab), rtol=2 * 2.0 ** -8)
            outer = leaf.grad.clone()
            outer[:, 1:4, off:off + vocab] = 0
            assert not outer.any()


# ---- how they are used --------------------------------------------------------------------------------------------------------
def batch(seed, vocab=700, dtype=torch.float32):
    x = logits(4 * 6, vocab, dtype, seed).view(4, 6, vocab).cuda()
    t = sequence_labels(4, vocab, 2, 6).cuda()
    idx, val = teacher(x.view(-1, vocab).cpu(), 8, 1.0, True, seed)
    return x, t, idx.view(4, 6, 8).cuda(), val.view(4, 6, 8).cuda()


def all_losses(x, t, idx, val, old, ref):
    from style_transfer_amd import losses
    adv = torch.arange(4, device=x.device) * 0.75 - 0.5
    policy = losses.clipped_policy_loss(x, t, old, adv, ref, kl_coef=0.1, entropy_coef=0.01)
    prefer = losses.preference_loss(x, t, (ref * (t != -100)).sum(1))
    distil = losses.topk_distill_loss(x, idx, val, t != -100, tail=True)
    return policy.loss + 0.5 * prefer.loss + 2 * distil + losses.token_logprobs(x, t).sum() * 1e-3


def test_a_training_step_of_all_of_them():
    """Scores, the three losses and one backward pass through their weighted sum: the sum of what each gives alone."""
    from style_transfer_amd import losses
    x, t, idx, val = batch(3)
    with torch.no_grad():
        old = losses.token_logprobs(x, t)
        ref = losses.token_logprobs(x + 0.1 * rand(1, *x.shape).cuda(), t)
    leaf = x.clone().requires_grad_(True)
    all_losses(leaf, t, idx, val, old, ref).backward()
    flat, rows = t.cpu().view(-1), x.cpu().view(-1, x.shape[-1])
    seqs = O.sequences_of(t.cpu())
    adv = (torch.arange(4) * 0.75 - 0.5).repeat_interleave(6)
    keep = flat != -100
    _, _, log_q, q = O.token_logprobs(rows, flat)
    want = O.policy(rows, flat, seqs, old.cpu().view(-1), adv, ref.cpu().view(-1), kl=0.1, ent=0.01)[2]
    want = want + 0.5 * O.preference(rows, flat, seqs, (ref * (t != -100)).sum(1).cpu())[2]
    want = want + 2 * O.distill(rows, idx.cpu().view(-1, 8), val.cpu().view(-1, 8), keep, 1.0, True)[1]
    want = want + O.row_gradient(flat, 1.0, torch.zeros(len(flat)), log_q, q, 1e-3 * keep.double(), torch.zeros(len(flat)))
    got = leaf.grad.cpu().double().view_as(want)
    assert float((got - want).norm() / want.norm()) < 1e-5


def test_gradients_against_differences():
    """The change of each loss along a direction, in 64 bits, is the kernels' gradient along it."""
    from style_transfer_amd import losses
    x, t, idx, val = batch(5, vocab=61)
    rows, flat = x.cpu().view(-1, 61), t.cpu().view(-1)
    seqs, keep = O.sequences_of(t.cpu()), flat != -100
    old, ref = O.token_logprobs(rows, flat)[0].float() + 0.05, O.token_logprobs(rows, flat)[0].float() - 0.2
    adv = rand(9, 24)
    way = rand(11, 24, 61).double()
    cases = [
        (lambda v: losses.preference_loss(v, t, beta=0.5).loss, lambda v: O.preference(v, flat, seqs, beta=0.5)[0]),
        (lambda v: losses.clipped_policy_loss(v, t, old.view(4, 6).cuda(), adv.view(4, 6).cuda(), ref.view(4, 6).cuda(), kl_coef=0.3,
                                              entropy_coef=0.2).loss,
         lambda v: O.policy(v, flat, seqs, old, adv, ref, kl=0.3, ent=0.2)[0]),
        (lambda v: losses.topk_distill_loss(v, idx, val, t != -100, temperature=1.5, tail=True),
         lambda v: O.distill(v, idx.cpu().view(-1, 8), val.cpu().view(-1, 8), keep, 1.5, True)[0]),
        (lambda v: losses.token_logprobs(v, t, return_entropy=True)[1].sum(), lambda v: float(O.token_logprobs(v, flat)[1].sum())),
    ]
    for ours, plain in cases:
        leaf = x.clone().requires_grad_(True)
        ours(leaf).backward()
        step = 1e-4                                             # the difference's own error: step^2 times a third derivative, under 1e-6
        diff = (plain(rows.double() + step * way) - plain(rows.double() - step * way)) / (2 * step)
        along = float((leaf.grad.cpu().double().view(24, 61) * way).sum())
        assert abs(along - diff) <= 1e-4 * float(leaf.grad.norm()) * float(way.norm())


@pytest.mark.parametrize("vocab", [700, 20000])
def test_upstream_gradients_scale_and_repeat(vocab):
    """backward of a weighted loss, and twice through one graph; ``scale`` does the same from inside."""
    from style_transfer_amd import losses
    x, t, idx, val = batch(8, vocab)
    old = losses.token_logprobs(x, t) + 0.1
    adv = rand(2, 4, 6).cuda()
    for fn in (lambda v, s: losses.preference_loss(v, t, scale=s).loss,
               lambda v, s: losses.clipped_policy_loss(v, t, old, adv, entropy_coef=0.1, scale=s).loss,
               lambda v, s: losses.topk_distill_loss(v, idx, val, tail=True, scale=s)):
        leaf = x.clone().requires_grad_(True)
        loss = fn(leaf, 1.0)
        one, = torch.autograd.grad(loss, [leaf], retain_graph=True)
        kept = one.clone()
        # an entry is the sum of up to three products (at a label, and where the entropy's two terms cancel, it is smaller than
        # they are); each differs by a few roundings, and none is more than twice the largest entry of a batch like this one
        tiny = 2 * 8 * U * 3 * float(one.abs().max())
        three, = torch.autograd.grad(3 * loss, [leaf], retain_graph=True)
        again, = torch.autograd.grad(loss, [leaf])
        assert torch.equal(one, kept) and torch.equal(again, kept)       # nobody writes into a gradient that was given away
        assert torch.allclose(three, 3 * one, rtol=8 * U, atol=tiny)
        inside, = torch.autograd.grad(fn(leaf, 3.0), [leaf])
        assert torch.allclose(inside, three, rtol=8 * U, atol=tiny)
        assert abs(float(fn(leaf, 3.0).detach()) - 3 * float(loss.detach())) <= 8 * U * abs(3 * float(loss.detach()))
        loss = fn(leaf, 1.0)
        loss /= 4                                               # a loss is the caller's to change
        quarter, = torch.autograd.grad(loss, [leaf])
        assert torch.allclose(quarter, one / 4, rtol=8 * U, atol=tiny)


def test_without_a_gradient_none_is_made():
    """Under no_grad, or for logits that need none, the value alone: nothing of the logits' size is allocated."""
    from style_transfer_amd import losses
    x, t, idx, val = batch(8, 20000)
    leaf = x.clone().requires_grad_(True)
    old = losses.token_logprobs(x, t)
    for fn in (lambda v: losses.token_logprobs(v, t), lambda v: losses.preference_loss(v, t).loss,
               lambda v: losses.clipped_policy_loss(v, t, old, old + 5).loss, lambda v: losses.topk_distill_loss(v, idx, val, tail=True)):
        for v, mode in ((leaf, torch.no_grad()), (leaf, torch.inference_mode()), (x, torch.enable_grad())):
            with mode:
                torch.cuda.synchronize()
                torch.cuda.reset_peak_memory_stats()
                before = torch.cuda.memory_allocated()
                out = fn(v)
                assert not out.requires_grad and torch.cuda.max_memory_allocated() - before < x.numel()
        assert torch.equal(fn(leaf).detach(), out)


@pytest.mark.parametrize("vocab", [700, 20000])
def test_an_upstream_gradient_that_is_no_number(vocab):
    """It reaches the rows that count and no other: those stay 0."""
    from style_transfer_amd import losses
    x, t, idx, val = batch(5, vocab)
    flat, cu = x.view(24, -1), torch.tensor([0, 6, 12, 15, 20], dtype=torch.int32, device="cuda")
    labels = torch.where(t.view(-1) == -100, 0, t.view(-1))
    old = losses.token_logprobs(flat, labels) + 0.1
    mask = torch.arange(24, device="cuda") < 20
    for fn in (lambda v: losses.preference_loss(v, labels, cu_seqlens=cu).loss,
               lambda v: losses.clipped_policy_loss(v, labels, old, old + 20, cu_seqlens=cu).loss,
               lambda v: losses.topk_distill_loss(v, idx.view(24, -1), val.view(24, -1), mask, tail=True)):
        for up in (math.nan, math.inf):
            leaf = flat.clone().requires_grad_(True)
            (fn(leaf) * up).backward()
            assert not leaf.grad[20:].any() and not torch.isfinite(leaf.grad[:20]).all(1).any()


def test_gradients_beyond_32_bits():
    """Broadcast logits whose gradient rows reach past 2^32 elements: every row as the first of its kind."""
    from style_transfer_amd import losses
    vocab, rows = 40001, 107500
    assert rows * vocab > 2 ** 32
    x = (logits(1, vocab, torch.bfloat16, 3)).cuda()
    t = torch.arange(rows, device="cuda") % 5
    old = torch.full((rows,), -9.0, device="cuda")
    idx, val = (torch.arange(4, device="cuda") * 7).expand(rows, 4).contiguous(), torch.full((rows, 4), -2.0, device="cuda")
    for fn in (lambda v: losses.clipped_policy_loss(v[None], t[None], old[None], old[None] + 10).loss,
               lambda v: losses.topk_distill_loss(v, idx, val, tail=True), lambda v: losses.token_logprobs(v, t).sum()):
        view = x.expand(rows, vocab).detach().requires_grad_(True)
        grad, = torch.autograd.grad(fn(view), [view])
        few = grad[:5].clone()
        assert few.any()
        for first in range(0, rows, 21500):                     # whole groups of five
            part = grad[first:first + 21500].view(-1, 5, vocab)
            assert torch.equal(part, few[None].expand_as(part))
        del grad, part, view


def test_nothing_counts():
    from style_transfer_amd import losses
    x, t, idx, val = batch(8)
    leaf = x.clone().requires_grad_(True)
    got = losses.topk_distill_loss(leaf, idx, val, torch.zeros_like(t, dtype=torch.bool), tail=True)
    got.backward()
    assert float(got.detach()) == 0 and not leaf.grad.any()
    leaf.grad = None
    got = losses.preference_loss(leaf, torch.full_like(t, -100), beta=0.3)
    got.loss.backward()
    assert abs(float(got.loss.detach()) - math.log(2)) < 1e-6 and not leaf.grad.any()


@pytest.mark.parametrize("vocab", [700, 20000])
def test_logits_kept_elsewhere_until_the_backward(vocab):
    """Saved tensors moved to the host and back: the backward reads the copy, whose address and strides are its own."""
    from style_transfer_amd import losses
    x, t, idx, val = batch(6, vocab)
    old = losses.token_logprobs(x, t) + 0.1
    wide = torch.cat([x, x], 2)
    for weight in (1.0, 3.0):
        for fn in (lambda v: losses.token_logprobs(v, t).sum(), lambda v: losses.preference_loss(v, t).loss,
                   lambda v: losses.clipped_policy_loss(v, t, old, old + 9).loss, lambda v: losses.topk_distill_loss(v, idx, val, tail=True)):
            grads = []
            for away in (False, True):
                leaf = wide.clone().requires_grad_(True)
                with torch.autograd.graph.save_on_cpu() if away else torch.enable_grad():
                    loss = weight * fn((leaf * 1)[:, :, 3:vocab + 3])
                other = torch.full_like(wide, math.nan)        # takes the place of what was let go
                loss.backward()
                grads.append(leaf.grad)
                del other
            half = 2 * row_error(vocab)
            assert torch.allclose(grads[0], grads[1], rtol=half, atol=half * float(grads[0].abs().max()))


def test_inside_a_checkpoint():
    """Recomputed in the backward pass, as memory-saving training does: the same gradients."""
    from torch.utils.checkpoint import checkpoint
    x, t, idx, val = batch(7, 5000)
    from style_transfer_amd import losses
    old = losses.token_logprobs(x, t) + 0.1
    grads = []
    for saving in (False, True):
        leaf = x.clone().requires_grad_(True)
        step = lambda v: all_losses(v * 1.5, t, idx, val, old, old - 0.2)  # noqa: E731
        (checkpoint(step, leaf, use_reentrant=False) if saving else step(leaf)).backward()
        grads.append(leaf.grad)
    assert torch.equal(*grads)


def test_no_second_derivative():
    """A graph of the gradient can be asked for; going through it is refused, not answered with 0."""
    from style_transfer_amd import losses
    x, t, idx, val = batch(9)
    old = losses.token_logprobs(x, t)
    for fn in (lambda v: losses.token_logprobs(v, t).sum(), lambda v: losses.preference_loss(v, t).loss,
               lambda v: losses.clipped_policy_loss(v, t, old, old + 9).loss, lambda v: losses.topk_distill_loss(v, idx, val, tail=True)):
        leaf = x.clone().requires_grad_(True)
        plain, = torch.autograd.grad(fn(leaf), [leaf])
        weight = torch.ones((), device="cuda", requires_grad=True)
        for loss, why in ((fn(leaf), "does not require grad"), (weight * fn(leaf), "once_differentiable")):
            grad, = torch.autograd.grad(loss, [leaf], create_graph=True)
            assert torch.equal(grad.detach(), plain)
            with pytest.raises(RuntimeError, match=why):
                grad.sum().backward()


def test_a_changed_input_is_noticed():
    from style_transfer_amd import losses
    x, t, _, _ = batch(8)
    leaf = x.clone().requires_grad_(True)
    y = leaf * 1
    loss = losses.preference_loss(y, t).loss
    y.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("vocab", [700, 20000])
def test_same_numbers_on_every_run_and_stream(vocab):
    from style_transfer_amd import losses
    x, t, idx, val = batch(4, vocab)
    old = losses.token_logprobs(x, t) + 0.1

    def once():
        leaf = x.clone().requires_grad_(True)
        loss = all_losses(leaf, t, idx, val, old, old - 0.2)
        loss.backward()
        return loss.detach(), leaf.grad

    loss, grad = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            a, b = once()
        side.synchronize()
        assert torch.equal(a, loss) and torch.equal(b, grad)


@pytest.mark.parametrize("vocab", [700, 20000])
def test_captured_steps_replay(vocab):
    """Two captured steps with their own inputs, replayed in turn with eager work between: each replay is the eager result."""
    from style_transfer_amd import losses
    steps = []
    for seed in (1, 2):
        x, t, idx, val = batch(seed, vocab)
        old = losses.token_logprobs(x, t) + 0.1
        leaf = x.clone().requires_grad_(True)
        warm = torch.cuda.Stream()
        warm.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(warm):
            torch.autograd.grad(all_losses(leaf, t, idx, val, old, old - 0.2), [leaf])
        torch.cuda.current_stream().wait_stream(warm)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            loss = all_losses(leaf, t, idx, val, old, old - 0.2)
            grad, = torch.autograd.grad(loss, [leaf])
            loss = loss.detach()
        steps.append((graph, leaf, t, idx, val, old, loss, grad))
    for k in range(4):
        for graph, leaf, t, idx, val, old, loss, grad in steps:
            with torch.no_grad():
                leaf.copy_(batch(10 + k, vocab)[0])
            graph.replay()
            torch.cuda.synchronize()
            eager = leaf.detach().clone().requires_grad_(True)
            want = all_losses(eager, t, idx, val, old, old - 0.2)
            want.backward()
            assert torch.equal(loss, want.detach()) and torch.equal(grad, eager.grad)
