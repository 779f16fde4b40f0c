"""The losses over rows of logits on the host side (no GPU needed): their oracle where differences are infinite, and what their
autograd functions do when nothing is launched."""
import contextlib
import math

import pytest
import torch
import torch.nn.functional as F
from torch.autograd import forward_ad as fwAD

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


class _Nothing:
    """The library with every kernel left out: sizes are small, calls succeed."""

    def __getattr__(self, name):
        return (lambda *_: 256) if name.endswith("bytes") else (lambda *_: 0)


@pytest.fixture
def nothing_runs(monkeypatch):
    """Host tensors that pass for the GPU's, and no launch: what the autograd functions do around the kernels is left."""
    from style_transfer_amd import token_losses

    def args(x):
        rows = x.numel() // x.shape[-1]
        return (x.data_ptr(), 0, rows, x.shape[-2], 0 if x.dim() == 2 else x.stride(0), x.stride(-2), x.shape[-1])

    monkeypatch.setattr(token_losses, "_logits_args", args)
    monkeypatch.setattr(token_losses, "_on", lambda _: contextlib.nullcontext())
    monkeypatch.setattr(token_losses._lib, "load", _Nothing)
    monkeypatch.setattr(token_losses._lib, "stream_ptr", lambda: 0)


X, T = torch.randn(2, 3, 11), torch.zeros(2, 3, dtype=torch.long)
CALLS = {
    "token_logprobs": lambda L, v: L.token_logprobs(v, T).sum(),
    "preference_loss": lambda L, v: L.preference_loss(v, T).loss,
    "clipped_policy_loss": lambda L, v: L.clipped_policy_loss(v, T, T.float(), T.float()).loss,
    "topk_distill_loss": lambda L, v: L.topk_distill_loss(v, T[..., None], T[..., None].float()),
}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("mode", [torch.enable_grad, torch.no_grad])
def test_forward_mode_derivatives_are_refused(nothing_runs, name, mode):
    from style_transfer_amd import losses
    with fwAD.dual_level(), mode():
        assert not CALLS[name](losses, X).requires_grad         # without a tangent a level changes nothing
        with pytest.raises(NotImplementedError):
            CALLS[name](losses, fwAD.make_dual(X, torch.ones_like(X)))


class _NoGradient(torch.autograd.Function):
    @staticmethod
    def forward(ctx, a):
        return a.clone()

    @staticmethod
    def backward(ctx, g):
        return None


@pytest.mark.parametrize("name", CALLS)
def test_a_loss_without_an_upstream_gradient(nothing_runs, name):
    """A node above whose backward gives None: nothing comes from there, and what else reaches the logits does."""
    from style_transfer_amd import losses
    leaf = X.clone().requires_grad_(True)
    (_NoGradient.apply(CALLS[name](losses, leaf * 1)) + leaf.sum()).backward()
    if name != "topk_distill_loss":                             # its kernel gets a gradient of 0, and is not there
        assert torch.equal(leaf.grad, torch.ones_like(X))


@pytest.mark.parametrize("vocab", [2 ** 31, 2 ** 32 + 5])
def test_a_vocabulary_beyond_32_bits_is_refused(vocab):
    """It would reach the kernels as its last 32 bits."""
    from style_transfer_amd import _lib, losses
    x, t = torch.empty(1, vocab, dtype=torch.float16, device="meta"), torch.empty(1, dtype=torch.long, device="meta")
    with pytest.raises(_lib.StHipError, match="at most 2.31 - 1"):
        losses.token_logprobs(x, t)


def test_the_workspace_of_the_largest_vocabulary():
    """500 rows of 2^31 - 1 elements are cut into parts, a thousand are not: no size on the way wraps."""
    from style_transfer_amd import _lib
    lib = _lib.load()
    plain = lib.st_token_workspace_bytes(1, 1024, 1000, 0)
    assert lib.st_token_workspace_bytes(1, 1024, 2 ** 31 - 1, 0) == plain
    assert lib.st_token_workspace_bytes(1, 500, 2 ** 31 - 1, 0) > lib.st_token_workspace_bytes(1, 500, 1000, 0)
