"""Losses over rows of logits, forward and backward on HIP kernels (csrc/token_losses.hip): the labels' log-probabilities,
the preference loss of paired sequences, the clipped policy loss with its KL and entropy terms, and the distillation from a
teacher's top logits.  No counterpart in the reference; they stand beside the loss modules of ``losses``, which exports them.

What they have in common:

* ``logits`` is ``[..., V]`` on the GPU, fp32, bf16 or fp16, with one or two leading dimensions of any stride (a slice
  is read in place) and a last stride of 1.  Gradients flow to the logits alone and have their type; everything else is
  a constant.  Results are fp32.
* ``labels`` (int64 or int32) has the logits' leading shape.  A position whose label is ``ignore_index`` does not count: its
  logits are not read, its results are 0, its gradient is 0.  A label outside ``[0, V)`` makes its row NaN.
* Logits of -inf or of the type's lowest value (a mask) have probability 0.  A row of -inf only has no distribution: its
  log-probability is -inf, its entropy and its gradient are 0.
* Sequences are the rows of ``[B, L, V]`` logits or, with ``cu_seqlens`` (int32, ascending, ``[sequences + 1]``), stretches of
  ``[T, V]`` logits; rows outside all of them do not count and get a zero gradient.
* With nothing that counts a loss is 0.  ``scale`` multiplies a loss and its gradient (a weight, 1 / accumulation steps, a
  static loss scale).
* Derivatives are reverse-mode and of first order: a forward-mode tangent or a second derivative is refused.
* Results do not depend on the run: every sum has a fixed order.
* ``clipped_policy_loss`` and ``topk_distill_loss`` write the gradient of logits that require one in the forward pass, while
  a row is on chip.  A backward pass with an upstream gradient of 1 hands it over; another one (a loss weight outside, a
  dynamic loss scale) computes it again from the logits: pass a known factor as ``scale``.  Until then it is a saved tensor of
  the logits' size beside them, and goes where saved tensors go.  Captured into another graph than its forward pass, a backward
  pass always computes it again.
"""
from __future__ import annotations

import contextlib
from typing import NamedTuple, Optional

import torch
import torch.nn as nn
from torch.autograd import forward_ad as fwAD
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_KINDS = {"sigmoid": 0, "ipo": 1, "hinge": 2}
_REDUCTIONS = {"token": 0, "sequence": 1}
_MOST_VOCAB = 2 ** 31 - 1                                       # an int of the C ABI


class PreferenceOutput(NamedTuple):
    loss: torch.Tensor
    chosen_rewards: torch.Tensor       # beta * (log-probability - reference) of each pair's chosen sequence
    rejected_rewards: torch.Tensor


class PolicyOutput(NamedTuple):
    loss: torch.Tensor
    stats: torch.Tensor                # means of the surrogate, the KL estimate, the entropy, "the clip holds the ratio"


# ---- arguments (checked once a call: a small loss is bound by what happens here) ------------------------------------------------
def _logits_args(x: torch.Tensor):
    """(x, dtype, rows, inner, s_outer, s_inner, vocab) of the C ABI."""
    if not isinstance(x, torch.Tensor):
        raise TypeError("logits: expected a torch.Tensor")
    code, shape = _DTYPES.get(x.dtype), x.shape
    if code is None:
        raise _lib.StHipError(f"logits: expected fp32, bf16 or fp16, got {x.dtype}")
    if len(shape) not in (2, 3) or shape[-1] == 0:
        raise _lib.StHipError(f"logits: expected [T, V] or [B, L, V], got {tuple(shape)}")
    if shape[-1] > _MOST_VOCAB:
        raise _lib.StHipError(f"logits: a vocabulary of {shape[-1]}, at most 2^31 - 1")
    if not x.is_cuda:
        raise _lib.StHipError(f"logits: the HIP hot path needs a tensor on the GPU, got device={x.device} (no CPU fallback)")
    stride = x.stride()
    if stride[-1] != 1 and shape[-1] > 1:
        raise _lib.StHipError(f"logits: the vocabulary's stride is {stride[-1]}, expected 1")
    if len(shape) == 2:
        return x.data_ptr(), code, shape[0], shape[0] or 1, 0, stride[0], shape[1]
    return x.data_ptr(), code, shape[0] * shape[1], shape[1] or 1, stride[0], stride[1], shape[2]


def _whole(t: torch.Tensor, name: str, like: torch.Tensor, shape) -> torch.Tensor:
    """An index tensor beside the logits: int64 or int32, the shape asked for, contiguous."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor")
    if t.dtype is not torch.int64 and t.dtype is not torch.int32:
        raise _lib.StHipError(f"{name}: expected int64 or int32, got {t.dtype}")
    _beside(t, name, like, shape)
    return t.contiguous()


def _floats(t: torch.Tensor, name: str, like: torch.Tensor, shape) -> torch.Tensor:
    """A floating tensor beside the logits, as contiguous fp32."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor")
    if not t.is_floating_point():
        raise _lib.StHipError(f"{name}: expected a floating tensor, got {t.dtype}")
    _beside(t, name, like, shape)
    if t.dtype is torch.float32 and not t.requires_grad and t.is_contiguous():
        return t
    return t.detach().to(torch.float32).contiguous()


def _beside(t, name, like, shape):
    if t.device != like.device:
        raise _lib.StHipError(f"{name}: on {t.device}, the logits are on {like.device}")
    if t.shape != shape:
        raise _lib.StHipError(f"{name}: expected {tuple(shape)}, got {tuple(t.shape)}")


def _label_args(labels: torch.Tensor, ignore_index: int):
    return labels.data_ptr(), int(labels.dtype is torch.int64), ignore_index


def _ignore(ignore_index) -> int:
    ignore_index = int(ignore_index)
    if not -2 ** 31 <= ignore_index < 2 ** 31:
        raise _lib.StHipError(f"ignore_index: {ignore_index} does not fit 32 bits")
    return ignore_index


def _temperature(value) -> float:
    value = float(value)
    if not 0.0 < value < float("inf"):
        raise _lib.StHipError(f"temperature: expected a positive number, got {value}")
    return value


def _sequences(x: torch.Tensor, cu_seqlens: Optional[torch.Tensor]):
    """(number of sequences, cu_seqlens as the kernels read them or None)."""
    if cu_seqlens is None:
        if x.dim() != 3:
            raise _lib.StHipError("[T, V] logits need cu_seqlens: it says where the sequences begin")
        return x.shape[0], None
    if x.dim() != 2:
        raise _lib.StHipError("cu_seqlens goes with [T, V] logits")
    if not isinstance(cu_seqlens, torch.Tensor) or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2:
        raise _lib.StHipError("cu_seqlens: expected a tensor [sequences + 1]")
    cu = _whole(cu_seqlens, "cu_seqlens", x, cu_seqlens.shape).to(torch.int32)
    return cu.numel() - 1, cu


_HERE = contextlib.nullcontext()
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device      # 7 us less in a small loss's backward


def _on(x: torch.Tensor):
    """The logits' device as the current one while a kernel is enqueued on its current stream."""
    if x.get_device() == _current_device():
        return _HERE
    return torch.cuda.device(x.device)


def _f32(x: torch.Tensor, *shape) -> torch.Tensor:
    return x.new_empty(shape, dtype=torch.float32)


def _scratch(x: torch.Tensor, kept: int, work: int):
    """(buffer, address of its first ``kept`` bytes, which a backward pass reads, address of the workspace behind them)."""
    kept = -(-kept // 256) * 256
    buffer = x.new_empty((kept + work + 16,), dtype=torch.uint8)
    at = buffer.data_ptr()
    return buffer, at, at + kept


def _grad_buffer(x: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


# ---- backward passes: on the autograd engine's thread, where every step costs twice (a small loss: 124 -> 100 us with less of them)
def _place(x: torch.Tensor, args):
    """``args`` of the forward pass for the saved logits, which may be a copy elsewhere (saved-tensor hooks): address and strides
    are the copy's own."""
    stride = x.stride()
    if len(stride) == 2:
        return x.data_ptr(), args[1], args[2], args[3], 0, stride[0], args[6]
    return x.data_ptr(), args[1], args[2], args[3], stride[0], stride[1], args[6]


def _backward(fn):
    """A backward pass that cannot be differentiated.  Only where a graph of the gradient is asked for does it need the wrapper
    that says so."""
    wrapped = once_differentiable(fn)

    def backward(ctx, *grads):
        return wrapped(ctx, *grads) if torch.is_grad_enabled() else fn(ctx, *grads)

    return staticmethod(backward)


# ---- log-probabilities ------------------------------------------------------------------------------------------------------
def _logprobs_fwd(x, args, labels, tau, ignore, want_entropy, want_state):
    lib = _lib.load()
    shape = labels.shape
    logp = _f32(x, *shape)
    entropy = _f32(x, *shape) if want_entropy else None
    with _on(x):
        buffer, state, work = _scratch(x, 16 * args[2] if want_state else 0, lib.st_token_workspace_bytes(args[1], args[2], args[6], 0))
        _lib.check(lib.st_token_logprobs_fwd(*args, *_label_args(labels, ignore), tau, logp.data_ptr(), _ptr(entropy),
                                             state if want_state else None, work, _lib.stream_ptr()), "st_token_logprobs_fwd")
    return logp, entropy, buffer


class _TokenLogProbsFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, call):
        args, labels, tau, ignore, want_entropy = call
        logp, entropy, buffer = _logprobs_fwd(x, args, labels, tau, ignore, want_entropy, True)
        ctx.call = args, tau, ignore
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, labels, buffer)
        return (logp, entropy) if want_entropy else logp

    @_backward
    def backward(ctx, g_logp, g_entropy=None):
        if g_logp is None and g_entropy is None:
            return None, None
        x, labels, state = ctx.saved_tensors
        args, tau, ignore = ctx.call
        grad = _grad_buffer(x)
        g_logp = None if g_logp is None else g_logp.contiguous()           # fp32, as the results
        g_entropy = None if g_entropy is None else g_entropy.contiguous()
        with _on(x):
            _lib.check(_lib.load().st_token_logprobs_bwd(*_place(x, args), *_label_args(labels, ignore), tau, state.data_ptr(), _ptr(g_logp), _ptr(g_entropy),
                                                         grad.data_ptr(), _lib.stream_ptr()), "st_token_logprobs_bwd")
        return grad, None


def token_logprobs(logits: torch.Tensor, labels: torch.Tensor, *, temperature: float = 1.0, ignore_index: int = -100,
                   return_entropy: bool = False):
    """``log softmax(logits / temperature)`` at each position's label, fp32 of the labels' shape; with ``return_entropy``
    also the entropy of each position's distribution.  Both are differentiable."""
    args = _logits_args(logits)
    labels = _whole(labels, "labels", logits, logits.shape[:-1])
    tau, ignore = _temperature(temperature), _ignore(ignore_index)
    if _wants_grad(logits):
        return _TokenLogProbsFunction.apply(logits, (args, labels, tau, ignore, bool(return_entropy)))
    logp, entropy, _ = _logprobs_fwd(logits, args, labels, tau, ignore, return_entropy, False)
    return (logp, entropy) if return_entropy else logp


def _wants_grad(x: torch.Tensor) -> bool:
    # a forward-mode tangent: the autograd function refuses it; without one the result would carry none, a derivative of 0
    return (x.requires_grad and torch.is_grad_enabled()) or fwAD.unpack_dual(x).tangent is not None


# ---- the two losses whose rows go through the label's log-probability -------------------------------------------------------------
def _keep(ctx, grad, capture, *tensors):
    """Saves what the backward pass reads, the gradient that the forward kernel wrote among it, so that saved-tensor hooks (the
    host's memory, a checkpoint) reach it too.  ``data``: with a version of its own, since it is given away and may be changed."""
    ctx.given, ctx.capture = False, capture
    ctx.save_for_backward(*tensors, grad.data)


def _capture(lib, stream):
    """The graph that is being captured, 0 outside of a capture, and on the null stream, which cannot be captured."""
    return lib.st_capture_id(stream) if stream else 0


def _take_grad(ctx, x, early, capture):
    """(buffer, 1) the first time: it holds the gradient for an upstream gradient of 1, written by the forward kernel while the
    rows were on chip.  The buffer is given away, so a second backward pass gets a new one, (buffer, 0); as does one that is
    captured without its forward pass, since its replays would find in the buffer what the last of them left."""
    if ctx.given or not early or ctx.capture != capture:
        return _grad_buffer(x), 0
    ctx.given = True
    return early[0].data, 1


def _token_loss_bwd(ctx, gout):
    if gout is None:                                           # a node above has none for the loss
        return None, None
    x, labels, row_grad, *early = ctx.saved_tensors
    args, tau, ignore = ctx.call
    lib = _lib.load()
    with _on(x):
        stream = _lib.stream_ptr()
        grad, for_one = _take_grad(ctx, x, early, _capture(lib, stream))
        _lib.check(lib.st_token_loss_bwd(*_place(x, args), *_label_args(labels, ignore), tau, row_grad.data_ptr(), gout.data_ptr(), for_one,
                                         grad.data_ptr(), stream), "st_token_loss_bwd")
    return grad, None


def _preference_fwd(x, call, need):
    args, labels, ignore, cu, pairs, ref, kind, average, beta, smoothing, scale = call
    lib = _lib.load()
    rows = args[2]
    loss, rewards = _f32(x), _f32(x, 2 * pairs)
    with _on(x):
        buffer, row_grad, work = _scratch(x, 16 * rows if need else 0, lib.st_token_workspace_bytes(args[1], rows, args[6], 2 * pairs))
        _lib.check(lib.st_preference_loss_fwd(*args, *_label_args(labels, ignore), _ptr(cu), pairs, _ptr(ref), kind, average, beta, smoothing,
                                              scale, loss.data_ptr(), rewards.data_ptr(), row_grad if need else None, work,
                                              _lib.stream_ptr()), "st_preference_loss_fwd")
    return loss, rewards, buffer


class _PreferenceFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, call):
        loss, rewards, buffer = _preference_fwd(x, call, True)
        ctx.mark_non_differentiable(rewards)
        ctx.set_materialize_grads(False)
        ctx.call, ctx.given = (call[0], 1.0, call[2]), False
        ctx.save_for_backward(x, call[1], buffer)
        return loss, rewards

    @_backward
    def backward(ctx, gout, _rewards):
        return _token_loss_bwd(ctx, gout)


def preference_loss(logits: torch.Tensor, labels: torch.Tensor, ref_logps: Optional[torch.Tensor] = None, *,
                    cu_seqlens: Optional[torch.Tensor] = None, beta: float = 0.1, kind: str = "sigmoid", label_smoothing: float = 0.0,
                    average: bool = False, ignore_index: int = -100, scale: float = 1.0) -> PreferenceOutput:
    """Preference loss of ``P`` pairs, the mean over them.  Sequences ``0 .. P - 1`` are the chosen ones, ``P .. 2 P - 1`` the
    rejected ones.  With ``L`` the sum of a sequence's label log-probabilities (``average``: their mean) and ``h`` the difference
    of ``L - ref_logps`` (``[2 P]``, default 0) between a pair's two sequences:

    ``kind="sigmoid"``: ``-(1 - label_smoothing) log sigmoid(beta h) - label_smoothing log sigmoid(-beta h)``;
    ``"ipo"``: ``(h - 1 / (2 beta))^2``; ``"hinge"``: ``max(0, 1 - beta h)``.

    Returns ``(loss, chosen_rewards, rejected_rewards)``; the rewards ``beta (L - ref_logps)`` are constants."""
    args = _logits_args(logits)
    labels = _whole(labels, "labels", logits, logits.shape[:-1])
    sequences, cu = _sequences(logits, cu_seqlens)
    if sequences % 2:
        raise _lib.StHipError(f"preference_loss: {sequences} sequences: expected the chosen ones and as many rejected ones behind them")
    if kind not in _KINDS:
        raise _lib.StHipError(f"preference_loss: kind {kind!r}: expected one of {sorted(_KINDS)}")
    beta, label_smoothing, ignore = float(beta), float(label_smoothing), _ignore(ignore_index)
    if not 0.0 < beta < float("inf") or not 0.0 <= label_smoothing < 0.5:
        raise _lib.StHipError(f"preference_loss: beta={beta} label_smoothing={label_smoothing}: expected beta > 0 and 0 <= label_smoothing < 0.5")
    if label_smoothing and kind != "sigmoid":
        raise _lib.StHipError('preference_loss: label_smoothing goes with kind="sigmoid"')
    ref = None if ref_logps is None else _floats(ref_logps, "ref_logps", logits, (sequences,))
    pairs = sequences // 2
    if pairs == 0:
        return PreferenceOutput(_no_loss(logits), _f32(logits, 0), _f32(logits, 0))
    if labels.numel() == 0:                                    # the references alone: one row that does not count, all sequences empty
        labels, cu = labels.new_full((1,), ignore), labels.new_zeros(sequences + 1, dtype=torch.int32)
        logits = torch.cat([logits.reshape(0, logits.shape[-1]), logits.new_zeros(1, logits.shape[-1])])
        args = _logits_args(logits)
    call = (args, labels, ignore, cu, pairs, ref, _KINDS[kind], int(bool(average)), beta, label_smoothing, float(scale))
    loss, rewards = _PreferenceFunction.apply(logits, call) if _wants_grad(logits) else _preference_fwd(logits, call, False)[:2]
    return PreferenceOutput(loss, rewards[:pairs], rewards[pairs:])


def _no_loss(logits: torch.Tensor) -> torch.Tensor:
    """0, connected to logits without rows."""
    return logits.float().sum()


def _policy_fwd(x, call, need):
    args, labels, ignore, tau, cu, sequences, old, adv, ref, low, high, kl, ent, per_sequence, scale = call
    lib = _lib.load()
    rows = args[2]
    loss, stats = _f32(x), _f32(x, 4)
    grad = _grad_buffer(x) if need else None
    with _on(x):
        stream = _lib.stream_ptr()
        buffer, row_grad, work = _scratch(x, 16 * rows if need else 0, lib.st_token_workspace_bytes(args[1], rows, args[6], sequences))
        _lib.check(lib.st_policy_loss_fwd(*args, *_label_args(labels, ignore), tau, _ptr(cu), sequences, old.data_ptr(), adv.data_ptr(),
                                          int(adv.shape != labels.shape), _ptr(ref), low, high, kl, ent, per_sequence, scale,
                                          loss.data_ptr(), stats.data_ptr(), row_grad if need else None, _ptr(grad), work, stream),
                   "st_policy_loss_fwd")
    return loss, stats, grad, buffer, _capture(lib, stream)


class _PolicyFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, call):
        loss, stats, grad, buffer, capture = _policy_fwd(x, call, True)
        ctx.mark_non_differentiable(stats)
        ctx.set_materialize_grads(False)
        ctx.call = call[0], call[3], call[2]
        _keep(ctx, grad, capture, x, call[1], buffer)
        return loss, stats

    @_backward
    def backward(ctx, gout, _stats):
        return _token_loss_bwd(ctx, gout)


def clipped_policy_loss(logits: torch.Tensor, labels: torch.Tensor, old_logps: torch.Tensor, advantages: torch.Tensor,
                        ref_logps: Optional[torch.Tensor] = None, *, cu_seqlens: Optional[torch.Tensor] = None, clip_low: float = 0.2,
                        clip_high: float = 0.2, kl_coef: float = 0.0, entropy_coef: float = 0.0, temperature: float = 1.0,
                        reduction: str = "token", ignore_index: int = -100, scale: float = 1.0) -> PolicyOutput:
    """Clipped policy loss of sampled tokens.  With ``logp`` the label's log-probability, ``r = exp(logp - old_logps)`` and ``A``
    the advantage (the labels' shape: of each position, also where a packed batch has as many sequences as rows; else
    ``[sequences]``: one for all of a sequence), a position's loss is

    ``-min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef (exp(ref - logp) - (ref - logp) - 1) - entropy_coef H``

    and the loss their mean over all positions that count (``reduction="token"``) or over the sequences of the mean over a
    sequence's positions (``"sequence"``; a sequence without any does not count).  ``old_logps`` and ``ref_logps`` have the
    labels' shape.  Without ``ref_logps`` there is no KL term.

    Returns ``(loss, stats)``: ``stats`` holds the same means of the surrogate, the KL estimate, the entropy and of whether the
    clip holds the ratio, as constants."""
    args = _logits_args(logits)
    shape = logits.shape[:-1]
    labels = _whole(labels, "labels", logits, shape)
    sequences, cu = _sequences(logits, cu_seqlens)
    old = _floats(old_logps, "old_logps", logits, shape)
    ref = None if ref_logps is None else _floats(ref_logps, "ref_logps", logits, shape)
    per_row = isinstance(advantages, torch.Tensor) and advantages.shape == shape
    adv = _floats(advantages, "advantages", logits, shape if per_row else (sequences,))
    clip_low, clip_high, kl_coef, entropy_coef = float(clip_low), float(clip_high), float(kl_coef), float(entropy_coef)
    if not 0.0 <= clip_low <= 1.0 or not 0.0 <= clip_high < float("inf"):
        raise _lib.StHipError(f"clipped_policy_loss: clip_low={clip_low} clip_high={clip_high}: expected [0, 1] and >= 0")
    if kl_coef and ref is None:
        raise _lib.StHipError("clipped_policy_loss: kl_coef needs ref_logps")
    if reduction not in _REDUCTIONS:
        raise _lib.StHipError(f"clipped_policy_loss: reduction {reduction!r}: expected one of {sorted(_REDUCTIONS)}")
    tau, ignore = _temperature(temperature), _ignore(ignore_index)
    if labels.numel() == 0:
        return PolicyOutput(_no_loss(logits), torch.zeros(4, device=logits.device))
    call = (args, labels, ignore, tau, cu, sequences, old, adv, ref, clip_low, clip_high, kl_coef, entropy_coef, _REDUCTIONS[reduction],
            float(scale))
    return PolicyOutput(*(_PolicyFunction.apply(logits, call) if _wants_grad(logits) else _policy_fwd(logits, call, False)[:2]))


# ---- distillation -------------------------------------------------------------------------------------------------------------
def _distill_fwd(x, call, need):
    args, idx, val, mask, tau, tail, scale = call
    lib = _lib.load()
    rows = args[2]
    loss = _f32(x)
    grad = _grad_buffer(x) if need else None
    entries = (idx.data_ptr(), int(idx.dtype is torch.int64), val.data_ptr(), idx.shape[-1])
    with _on(x):
        stream = _lib.stream_ptr()
        buffer, row_grad, work = _scratch(x, 32 * rows if need else 0, lib.st_distill_workspace_bytes(rows))
        _lib.check(lib.st_distill_loss_fwd(*args, *entries, _ptr(mask), tau, tail, scale, loss.data_ptr(), row_grad if need else None,
                                           _ptr(grad), work, stream), "st_distill_loss_fwd")
    return loss, grad, buffer, _capture(lib, stream)


class _DistillFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, call):
        loss, grad, buffer, capture = _distill_fwd(x, call, True)
        ctx.call = call[0], call[4], call[5]
        _keep(ctx, grad, capture, x, call[1], call[2], buffer)
        return loss

    @_backward
    def backward(ctx, gout):
        x, idx, val, row_grad, *early = ctx.saved_tensors
        args, tau, tail = ctx.call
        lib = _lib.load()
        with _on(x):
            stream = _lib.stream_ptr()
            grad, for_one = _take_grad(ctx, x, early, _capture(lib, stream))
            _lib.check(lib.st_distill_loss_bwd(*_place(x, args), idx.data_ptr(), int(idx.dtype is torch.int64), val.data_ptr(), idx.shape[-1], tau, tail,
                                               row_grad.data_ptr(), gout.data_ptr(), for_one, grad.data_ptr(), stream), "st_distill_loss_bwd")
        return grad, None


def topk_distill_loss(logits: torch.Tensor, teacher_indices: torch.Tensor, teacher_values: torch.Tensor,
                      mask: Optional[torch.Tensor] = None, *, temperature: float = 1.0, tail: bool = False,
                      scale: float = 1.0) -> torch.Tensor:
    """Distillation from the ``K`` largest logits that a teacher left of each position, ``temperature^2`` times the mean over the
    positions (those where ``mask`` is true) of ``sum_k p_k (log p_k - log q_k)``; ``q`` is the student's softmax of
    ``logits / temperature`` over the whole vocabulary.

    ``teacher_indices`` ``[..., K]`` names the tokens (below 0: an unused entry; the same token twice: the entries add up).
    ``tail=False``: ``teacher_values`` are logits and ``p`` their softmax at ``temperature`` over the list alone.  ``tail=True``:
    they are the teacher's log-probabilities (at ``temperature``, over its whole vocabulary), and all tokens that are not listed
    form one more entry of the sum, with ``1 - sum_k p_k`` and the student's probability of the same tokens.

    At most 2^20 tokens and 4096 entries.  A position with no used entry contributes 0.  An index of ``V`` or more makes its position's
    loss and gradient NaN.  Fill a short list up with -1, not by naming a token again: such a list costs the square of its length (1024
    positions of 32768 tokens: 0.2 ms instead of 0.13 with 256 entries, 28 instead of 0.23 with 4096)."""
    args = _logits_args(logits)
    shape = logits.shape[:-1]
    if not isinstance(teacher_indices, torch.Tensor) or teacher_indices.dim() != logits.dim() or teacher_indices.shape[-1] == 0:
        raise _lib.StHipError("teacher_indices: expected [..., K] with K > 0 and the logits' leading shape")
    entries = (*shape, teacher_indices.shape[-1])
    idx = _whole(teacher_indices, "teacher_indices", logits, entries)
    val = _floats(teacher_values, "teacher_values", logits, entries)
    if mask is not None:
        if not isinstance(mask, torch.Tensor) or mask.dtype is not torch.bool:
            raise _lib.StHipError("mask: expected a bool tensor")
        _beside(mask, "mask", logits, shape)
        mask = mask.contiguous()
    tau = _temperature(temperature)
    if idx.numel() == 0:
        return _no_loss(logits)
    call = (args, idx, val, mask, tau, int(bool(tail)), float(scale))
    return _DistillFunction.apply(logits, call) if _wants_grad(logits) else _distill_fwd(logits, call, False)[0]


# ---- modules ------------------------------------------------------------------------------------------------------------------
class TokenLogProbs(nn.Module):
    """``token_logprobs`` with its settings held."""

    def __init__(self, temperature: float = 1.0, ignore_index: int = -100, return_entropy: bool = False):
        super().__init__()
        self.settings = dict(temperature=_temperature(temperature), ignore_index=_ignore(ignore_index), return_entropy=bool(return_entropy))

    def forward(self, logits, labels):
        return token_logprobs(logits, labels, **self.settings)


class PreferenceLoss(nn.Module):
    """``preference_loss`` with its settings held."""

    def __init__(self, beta: float = 0.1, kind: str = "sigmoid", label_smoothing: float = 0.0, average: bool = False,
                 ignore_index: int = -100, scale: float = 1.0):
        super().__init__()
        self.settings = dict(beta=beta, kind=kind, label_smoothing=label_smoothing, average=average, ignore_index=ignore_index, scale=scale)

    def forward(self, logits, labels, ref_logps=None, cu_seqlens=None):
        return preference_loss(logits, labels, ref_logps, cu_seqlens=cu_seqlens, **self.settings)


class ClippedPolicyLoss(nn.Module):
    """``clipped_policy_loss`` with its settings held."""

    def __init__(self, clip_low: float = 0.2, clip_high: float = 0.2, kl_coef: float = 0.0, entropy_coef: float = 0.0,
                 temperature: float = 1.0, reduction: str = "token", ignore_index: int = -100, scale: float = 1.0):
        super().__init__()
        self.settings = dict(clip_low=clip_low, clip_high=clip_high, kl_coef=kl_coef, entropy_coef=entropy_coef, temperature=temperature,
                             reduction=reduction, ignore_index=ignore_index, scale=scale)

    def forward(self, logits, labels, old_logps, advantages, ref_logps=None, cu_seqlens=None):
        return clipped_policy_loss(logits, labels, old_logps, advantages, ref_logps, cu_seqlens=cu_seqlens, **self.settings)


class TopKDistillLoss(nn.Module):
    """``topk_distill_loss`` with its settings held."""

    def __init__(self, temperature: float = 1.0, tail: bool = False, scale: float = 1.0):
        super().__init__()
        self.settings = dict(temperature=temperature, tail=tail, scale=scale)

    def forward(self, logits, teacher_indices, teacher_values, mask=None):
        return topk_distill_loss(logits, teacher_indices, teacher_values, mask, **self.settings)
