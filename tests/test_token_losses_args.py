"""What the losses over rows of logits refuse, before anything is launched (no GPU needed), and their oracle against torch."""
import math

import pytest
import torch

from oracle import token_ops as O


def test_host_tensors_and_wrong_types_are_refused():
    from style_transfer_amd import _lib, losses
    x, t = torch.randn(2, 3, 11), torch.zeros(2, 3, dtype=torch.long)
    calls = [lambda v: losses.token_logprobs(v, t), lambda v: losses.preference_loss(v, t),
             lambda v: losses.clipped_policy_loss(v, t, t.float(), t.float()),
             lambda v: losses.topk_distill_loss(v, t[..., None], t[..., None].float())]
    for call in calls:
        for wrong in (x, x.double(), x.long(), x[0, 0], x[..., :0], x[None]):
            with pytest.raises(_lib.StHipError):
                call(wrong)
        with pytest.raises(TypeError):
            call([1.0])


def _gpu_like(monkeypatch):
    """Host tensors that pass for the GPU's: every check behind the device's runs, and nothing may be launched."""
    from style_transfer_amd import token_losses
    real = token_losses._logits_args

    def args(x):
        if x.stride(-1) != 1 and x.shape[-1] > 1:
            raise token_losses._lib.StHipError("stride")
        return x.data_ptr(), 0, 0, 1, 0, 0, x.shape[-1]

    def never(*_):
        raise AssertionError("launched")

    monkeypatch.setattr(token_losses, "_logits_args", args)
    monkeypatch.setattr(token_losses._lib, "stream_ptr", never)
    monkeypatch.setattr(token_losses, "_on", never)
    return real


@pytest.mark.parametrize("call", [
    lambda L, x, t: L.token_logprobs(x, t[:1]),
    lambda L, x, t: L.token_logprobs(x, t.float()),
    lambda L, x, t: L.token_logprobs(x, t, temperature=0.0),
    lambda L, x, t: L.token_logprobs(x, t, temperature=math.nan),
    lambda L, x, t: L.token_logprobs(x, t, ignore_index=2 ** 31),
    lambda L, x, t: L.token_logprobs(x.transpose(0, 2).contiguous().transpose(0, 2), t),
    lambda L, x, t: L.preference_loss(x[:3], t[:3]),
    lambda L, x, t: L.preference_loss(x, t, beta=0.0),
    lambda L, x, t: L.preference_loss(x, t, kind="other"),
    lambda L, x, t: L.preference_loss(x, t, label_smoothing=0.5),
    lambda L, x, t: L.preference_loss(x, t, kind="ipo", label_smoothing=0.1),
    lambda L, x, t: L.preference_loss(x, t, torch.zeros(3)),
    lambda L, x, t: L.preference_loss(x.flatten(0, 1), t.flatten()),
    lambda L, x, t: L.preference_loss(x, t, cu_seqlens=torch.tensor([0, 3])),
    lambda L, x, t: L.preference_loss(x.flatten(0, 1), t.flatten(), cu_seqlens=torch.tensor([0])),
    lambda L, x, t: L.preference_loss(x.flatten(0, 1), t.flatten(), cu_seqlens=torch.tensor([0.0, 3.0, 6.0])),
    lambda L, x, t: L.clipped_policy_loss(x, t, t.float(), torch.zeros(5)),
    lambda L, x, t: L.clipped_policy_loss(x, t, t, t.float()),
    lambda L, x, t: L.clipped_policy_loss(x, t, t.float(), t.float(), kl_coef=0.1),
    lambda L, x, t: L.clipped_policy_loss(x, t, t.float(), t.float(), clip_low=1.5),
    lambda L, x, t: L.clipped_policy_loss(x, t, t.float(), t.float(), clip_high=-0.1),
    lambda L, x, t: L.clipped_policy_loss(x, t, t.float(), t.float(), reduction="sum"),
    lambda L, x, t: L.topk_distill_loss(x, t, t.float()),
    lambda L, x, t: L.topk_distill_loss(x, t[..., None], t.float()),
    lambda L, x, t: L.topk_distill_loss(x, t[..., None][..., :0], t[..., None][..., :0].float()),
    lambda L, x, t: L.topk_distill_loss(x, t[..., None], t[..., None].float(), t),
    lambda L, x, t: L.topk_distill_loss(x, t[..., None], t[..., None].float(), temperature=-1),
])
def test_what_does_not_fit_is_refused(monkeypatch, call):
    from style_transfer_amd import _lib, losses
    _gpu_like(monkeypatch)
    with pytest.raises(_lib.StHipError):
        call(losses, torch.randn(4, 3, 11), torch.zeros(4, 3, dtype=torch.long))


def test_c_entries_return_errors():
    from style_transfer_amd import _lib
    lib = _lib.load()
    p = 4096                                                   # an address that nobody reads: every call is refused before a launch
    none = (None, 0, 4, 4, 0, 10, 10)
    good = (p, 0, 4, 4, 0, 10, 10)
    labels = (p, 1, -100)
    assert lib.st_token_logprobs_fwd(*none, *labels, 1.0, p, None, None, p, None) == -1 and b"null" in lib.st_last_error()
    assert lib.st_token_logprobs_fwd(*good, None, 1, -100, 1.0, p, None, None, p, None) == -1
    for wrong in ((p, 3, 4, 4, 0, 10, 10), (p, 0, -1, 4, 0, 10, 10), (p, 0, 4, 0, 0, 10, 10), (p, 0, 4, 4, 0, 10, 0), (p, 0, 4, 4, -1, 10, 10),
                  (p + 2, 0, 4, 4, 0, 10, 10), (p, 0, 2 ** 31, 4, 0, 10, 10)):
        assert lib.st_token_logprobs_fwd(*wrong, *labels, 1.0, p, None, None, p, None) == -1, wrong
        assert lib.st_token_logprobs_bwd(*wrong, *labels, 1.0, p, p, None, p, None) == -1, wrong
        assert lib.st_token_loss_bwd(*wrong, *labels, 1.0, p, None, 0, p, None) == -1, wrong
        assert lib.st_distill_loss_bwd(*wrong, p, 1, p, 3, 1.0, 0, p, None, 0, p, None) == -1, wrong
    for tau in (0.0, -1.0, math.inf, math.nan, 1e-60):
        assert lib.st_token_logprobs_fwd(*good, *labels, tau, p, None, None, p, None) == -1
    pref = lambda pairs, kind, beta, eps: lib.st_preference_loss_fwd(*good, *labels, None, pairs, None, kind, 0, beta, eps, 1.0, p, p, None, p, None)  # noqa: E731
    assert pref(1, 0, 0.1, 0.0) == -1                          # 4 rows of 4 are one sequence, not two
    assert pref(0, 0, 0.1, 0.0) == -1
    policy = lambda seqs, low: lib.st_policy_loss_fwd(*good, *labels, 1.0, None, seqs, p, p, 0, None, low, 0.2, 0.0, 0.0, 0, 1.0, p, p, None, None, p, None)  # noqa: E731
    assert policy(2, 0.2) == -1 and policy(1, 1.5) == -1
    assert lib.st_distill_loss_fwd(*good, p, 1, p, 0, None, 1.0, 0, 1.0, p, None, None, p, None) == -1
    assert lib.st_distill_loss_fwd(p, 0, 4, 4, 0, 2 ** 21, 2 ** 21, p, 1, p, 3, None, 1.0, 0, 1.0, p, None, None, p, None) == -1
    assert lib.st_distill_loss_fwd(*good, p, 1, p, 4097, None, 1.0, 0, 1.0, p, None, None, p, None) == -1 and b"4096" in lib.st_last_error()
    many = (p, 0, 2 ** 31 - 1, 2 ** 31 - 1, 0, 10, 10)         # more threads than a launch has
    assert lib.st_token_logprobs_fwd(*many, *labels, 1.0, p, None, None, p, None) == -1 and b"launch" in lib.st_last_error()
    assert lib.st_token_workspace_bytes(0, -1, 10, 0) == 0 and lib.st_token_workspace_bytes(1, 1, 131072, 2) > 0


def test_modules_hold_their_settings():
    from style_transfer_amd.losses import ClippedPolicyLoss, PreferenceLoss, TokenLogProbs, TopKDistillLoss
    assert TokenLogProbs(0.5, -1, True).settings == dict(temperature=0.5, ignore_index=-1, return_entropy=True)
    assert PreferenceLoss(kind="ipo").settings["kind"] == "ipo"
    assert ClippedPolicyLoss(kl_coef=0.1).settings["kl_coef"] == 0.1 and TopKDistillLoss(tail=True).settings["tail"] is True
    for m in (TokenLogProbs(), PreferenceLoss(), ClippedPolicyLoss(), TopKDistillLoss()):
        assert not list(m.parameters())


def test_the_oracle_is_what_torch_computes():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(6, 40, generator=g, dtype=torch.float64).requires_grad_(True)
    t = torch.randint(0, 40, (6,), generator=g)
    t[2] = -100
    keep = (t != -100).double()
    log_q = torch.log_softmax(x / 0.7, 1)
    logp = log_q.gather(1, t.clamp(min=0)[:, None])[:, 0] * keep
    h = -(log_q.exp() * log_q).sum(1) * keep
    want = O.token_logprobs(x.detach(), t, 0.7)
    assert torch.allclose(want[0], logp) and torch.allclose(want[1], h)
    a, b = torch.randn(6, generator=g, dtype=torch.float64) * keep, torch.randn(6, generator=g, dtype=torch.float64) * keep
    grad, = torch.autograd.grad((a * logp + b * h).sum(), [x])
    assert torch.allclose(O.row_gradient(t, 0.7, want[1], want[2], want[3], a, b), grad, atol=1e-12)
    # the three losses' gradients against differences of their own values
    idx, val = torch.stack([torch.randperm(40, generator=g)[:5] for _ in range(6)]), torch.randn(6, 5, generator=g) - 3
    seqs, way = [(0, 2), (2, 3), (3, 4), (4, 6)], torch.randn(6, 40, generator=g, dtype=torch.float64)
    old, adv = logp.detach() - 0.1, torch.randn(6, generator=g)
    for fn in (lambda v: O.preference(v, t, seqs, smoothing=0.1, beta=0.5), lambda v: O.preference(v, t, seqs, kind="ipo", average=True),
               lambda v: O.policy(v, t, seqs, old, adv, old + 0.2, kl=0.2, ent=0.1, tau=0.7, per_sequence=True),
               lambda v: O.distill(v, idx, val, t != -100, 1.5, True), lambda v: O.distill(v, idx, val, None, 1.5, False)):
        v, step = x.detach(), 1e-5
        diff = (fn(v + step * way)[0] - fn(v - step * way)[0]) / (2 * step)
        assert abs(float((fn(v)[-1] * way).sum()) - diff) < 1e-7
