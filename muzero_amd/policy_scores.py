"""Scores of actions under a policy head's logits: log probability, entropy and the best alternatives, with gradient.

The reference reads its policy head through `torch.softmax` and `argmax` alone (src/search/expansion.py:26-27,
src/search/simulation.py:36); a learner or a report that asks how likely the recorded moves are, how sure the network
is and what it would rather play needs these values for every row, in one pass over the logits:

    scores = policy_scores(logits, actions, top=3)
    scores.log_prob, scores.entropy              # [...]        differentiable
    scores.top_actions, scores.top_log_probs     # [..., top]   the latter differentiable

`logits` are the values in front of the head's softmax (`PredictionNetwork.policy_logits`), float32, bfloat16 or
float16, of any leading shape; illegal actions carry -inf.  Results are float32.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from muzero_amd import _hip
from muzero_amd._hip import ptr
from muzero_amd._rows import TYPE, check_tensor, in_memory, on_device, refuse_tangent, rows_of, stream_of, workspace

MAX_TOP = 32
_WHOLE = (torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8)


class PolicyScores(NamedTuple):
    log_prob: Optional[torch.Tensor]       # f32[...]       log p(action), None without actions
    entropy: torch.Tensor                  # f32[...]       -sum p log p
    top_actions: Optional[torch.Tensor]    # i64[..., top]  largest logits first, the lowest index among equals; None: top=0
    top_log_probs: Optional[torch.Tensor]  # f32[..., top]


def _forward(logits: torch.Tensor, actions: Optional[torch.Tensor], top: int, want_stats: bool):
    # A small batch is bound by this function: few calls, no helpers.
    T, V = logits.shape
    empty, dev = torch.empty, logits.device
    log_prob = None if actions is None else empty(T, dtype=torch.float32, device=dev)
    entropy = empty(T, dtype=torch.float32, device=dev)
    stats = empty((T, 3), dtype=torch.float32, device=dev) if want_stats else None
    top_actions = top_log_probs = None
    if top:
        top_actions, top_log_probs = empty((T, top), dtype=torch.int64, device=dev), empty((T, top), dtype=torch.float32, device=dev)
    if T > 0:
        lib, kind = _hip.lib(), TYPE[logits.dtype]
        with on_device(logits):
            need = lib.mz_policy_scores_workspace(kind, T, V, top)
            ws = workspace(need, logits) if need else None
            rc = lib.mz_policy_scores(logits.data_ptr(), kind, logits.stride(0) if T > 1 else V,
                                      None if actions is None else actions.data_ptr(), T, V, top,
                                      None if actions is None else log_prob.data_ptr(), entropy.data_ptr(), ptr(stats),
                                      top_actions.data_ptr() if top else None, top_log_probs.data_ptr() if top else None,
                                      ptr(ws), need, stream_of(logits))
            if rc:
                _hip.check(rc, "mz_policy_scores")
    return log_prob, entropy, stats, top_actions, top_log_probs


def _gradient(ctx, g_log_prob, g_entropy, _g_actions, g_top):
    # Runs on autograd's thread for the device, where every Python object it touches comes from another core's cache: few
    # calls, no helpers on the way of the common case.
    logits, actions, stats, top_actions = ctx.saved_tensors
    T, V = logits.shape
    if forward_ad._current_level >= 0:
        for g in (g_log_prob, g_entropy, g_top):
            if g is not None:
                refuse_tangent(g, "the gradient")
    grad = torch.empty((T, V), dtype=logits.dtype, device=logits.device)
    if T > 0:
        g_log_prob = None if g_log_prob is None else in_memory(g_log_prob)
        g_entropy = None if g_entropy is None else in_memory(g_entropy)
        g_top = None if g_top is None else in_memory(g_top)
        args = (logits.data_ptr(), ctx.kind, logits.stride(0) if T > 1 else V, None if actions is None else actions.data_ptr(), T, V,
                0 if g_top is None else g_top.shape[1], stats.data_ptr(), None if top_actions is None else top_actions.data_ptr(),
                None if g_log_prob is None else g_log_prob.data_ptr(), None if g_entropy is None else g_entropy.data_ptr(),
                None if g_top is None else g_top.data_ptr(), grad.data_ptr(), V, stream_of(logits))
        # autograd has made the logits' device the current one
        rc = _hip.lib().mz_policy_scores_backward(*args)
        if rc:
            _hip.check(rc, "mz_policy_scores_backward")
    return grad, None, None


class _PolicyScores(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, actions, top):
        log_prob, entropy, stats, top_actions, top_log_probs = _forward(logits, actions, top, True)
        ctx.save_for_backward(logits, actions, stats, top_actions)
        ctx.set_materialize_grads(False)
        ctx.kind = TYPE[logits.dtype]
        if top:
            ctx.mark_non_differentiable(top_actions)
        return log_prob, entropy, top_actions, top_log_probs

    @staticmethod
    def backward(ctx, *grads):
        # the guard against a second derivative is needed (and paid for) only where a graph of the gradient is built
        return _guarded_gradient(ctx, *grads) if torch.is_grad_enabled() else _gradient(ctx, *grads)


_guarded_gradient = once_differentiable(_gradient)


def policy_scores(logits: torch.Tensor, actions: Optional[torch.Tensor] = None, top: int = 0) -> PolicyScores:
    """Scores of every row of `logits` [..., V].  `actions` (whole numbers, shape [...]): a negative one scores 0 and
    takes no gradient (no action was played there), one of V or more scores NaN.  `top`: 0..32 alternatives.

    The gradient is a reverse-mode one: logits with a forward-mode tangent are refused.
    A row with nothing but -inf has log probabilities -inf, entropy 0 and no gradient; NaN or +inf make their row NaN."""
    check_tensor(logits, "logits")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits need at least one action in their last dimension, not shape {tuple(logits.shape)}")
    lead, V = logits.shape[:-1], logits.shape[-1]
    if not 0 <= top <= min(MAX_TOP, V):
        raise ValueError(f"top={top} must lie in 0..{MAX_TOP} and not exceed the {V} actions")
    if actions is not None:
        if not isinstance(actions, torch.Tensor) or actions.dtype not in _WHOLE:
            raise TypeError("actions must be a tensor of whole numbers")
        if actions.shape != lead:
            raise ValueError(f"actions of shape {tuple(actions.shape)} do not match logits of shape {tuple(logits.shape)}")
        if actions.device != logits.device:
            raise ValueError(f"actions are on {actions.device}, logits on {logits.device}")
        if actions.dtype is not torch.int64 or actions.dim() != 1 or not actions.is_contiguous() or actions.is_neg():
            actions = in_memory(actions.reshape(-1).to(torch.int64))
    rows = rows_of(logits)
    if torch.is_grad_enabled() and rows.requires_grad:
        log_prob, entropy, top_actions, top_log_probs = _PolicyScores.apply(rows, actions, top)
    else:
        log_prob, entropy, _, top_actions, top_log_probs = _forward(rows, actions, top, False)
    if len(lead) != 1:
        entropy = entropy.reshape(lead)
        if log_prob is not None:
            log_prob = log_prob.reshape(lead)
        if top:
            top_actions, top_log_probs = top_actions.reshape(*lead, top), top_log_probs.reshape(*lead, top)
    return PolicyScores(log_prob, entropy, top_actions, top_log_probs)


def score_actions(pred_net, latent: torch.Tensor, actions: Optional[torch.Tensor] = None, top: int = 0) -> PolicyScores:
    """policy_scores of a PredictionNetwork's policy for latents [B, c, h, w]."""
    return policy_scores(pred_net.policy_logits(latent), actions, top)
