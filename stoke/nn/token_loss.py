# -*- coding: utf-8 -*-
"""Losses on token log-probabilities for fine-tuning decoders
(csrc/token_loss.hip).

* ``token_logprobs``        -- log-probability of given tokens under logits
                               (scoring with an old or reference model, or
                               any loss of one's own: it has a gradient),
* ``fused_policy_loss``     -- clipped policy loss with a KL term,
* ``fused_preference_loss`` -- paired preference loss.

They take logits as ``fused_cross_entropy`` does: ``[..., V]`` with int64
targets, positions with ``ignore_index`` (or a target out of range) ignored.
Ignored positions are not read, whatever their logits hold, and get zero
gradient.  bf16, fp16 and fp32 GPU logits run the HIP kernels: one pass over
the logits forward, one pass and the write of the gradient backward, no fp32
copy.  CPU tensors and float64 take the same formulas in torch.
"""

import torch

from stoke import ops


def _native(logits: torch.Tensor):
    """The extension where its kernels take the call (it checks the
    arguments as ``_check`` does), None for the torch formulas."""
    if logits.is_cuda and logits.dtype != torch.float64:
        return ops._require_ext()
    return None


def _check(logits, targets, what):
    if not logits.is_floating_point() or logits.dim() < 2 \
            or logits.shape[-1] < 1:
        raise ValueError(
            f"Stoke -- {what} takes floating logits [..., V], got "
            f"{logits.dtype} {tuple(logits.shape)}"
        )
    if targets.dtype != torch.int64 or targets.device != logits.device \
            or targets.shape != logits.shape[:-1]:
        raise ValueError(
            f"Stoke -- {what} takes int64 targets of the logits' shape "
            f"without the vocabulary on their device, got {targets.dtype} "
            f"{tuple(targets.shape)} for logits {tuple(logits.shape)}"
        )


def _per_token(v, targets, what):
    """Constant values for each token, broadcast where a size is 1."""
    if v.requires_grad:
        raise ValueError(
            f"Stoke -- {what} is a constant of the loss; detach() it"
        )
    if not v.is_floating_point() or v.device != targets.device \
            or v.dim() != targets.dim() or any(
                a not in (1, b) for a, b in zip(v.shape, targets.shape)):
        raise ValueError(
            f"Stoke -- {what} must hold floating values for targets "
            f"{tuple(targets.shape)} (sizes of 1 broadcast) on their "
            f"device, got {v.dtype} {tuple(v.shape)}"
        )
    return v.expand(targets.shape)


def _eager_logprobs(logits, targets, ignore_index):
    """(log-probabilities in float64 with zeros where ignored, live)."""
    live = (targets != ignore_index) & (targets >= 0) \
        & (targets < logits.shape[-1])
    # ignored rows are left out before any arithmetic: a NaN in them stays
    # out of the gradient too
    rows = torch.log_softmax(logits[live].double(), -1)
    picked = rows.gather(-1, targets[live][:, None])[:, 0]
    lp = torch.zeros(targets.shape, dtype=torch.float64,
                     device=logits.device)
    return lp.masked_scatter(live, picked), live


def _result_dtype(logits):
    return torch.float64 if logits.dtype == torch.float64 else torch.float32


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor,
                   ignore_index: int = -100) -> torch.Tensor:
    """log softmax(logits)[targets] in fp32, 0 at ignored positions.

    logits: [..., V]; targets: [...] int64.
    """
    ext = _native(logits)
    if ext is not None:
        return ext.token_logprobs(logits, targets, ignore_index)
    _check(logits, targets, "token_logprobs")
    lp, _ = _eager_logprobs(logits, targets, ignore_index)
    return lp.to(_result_dtype(logits))


def fused_policy_loss(logits: torch.Tensor, actions: torch.Tensor,
                      old_logprobs: torch.Tensor, advantages: torch.Tensor,
                      ref_logprobs: torch.Tensor = None,
                      clip_low: float = 0.2, clip_high: float = 0.2,
                      kl_coef: float = 0.0,
                      ignore_index: int = -100) -> torch.Tensor:
    """Clipped policy loss with a KL term, mean over non-ignored tokens.

    With lp = log softmax(logits)[actions], rho = exp(lp - old_logprobs) and
    d = ref_logprobs - lp a token's loss is::

        -min(rho * A, clip(rho, 1 - clip_low, 1 + clip_high) * A)
        + kl_coef * (exp(d) - d - 1)

    logits: [..., V]; actions: [...] int64; the other tensors hold a value
    for each token (sizes of 1 broadcast, e.g. advantages [B, 1]) and are
    constants.  At a ratio on the clip the gradient flows.  Without any
    token left the loss and its gradient are 0.  ``ref_logprobs`` is
    required where ``kl_coef`` is not 0.
    """
    ext = _native(logits)
    if ext is not None:
        return ext.policy_loss(logits, actions, old_logprobs, advantages,
                               ref_logprobs, clip_low, clip_high, kl_coef,
                               ignore_index)
    _check(logits, actions, "fused_policy_loss")
    if not (0 <= clip_low <= 1 and clip_high >= 0 and kl_coef >= 0):
        raise ValueError(
            "Stoke -- fused_policy_loss takes 0 <= clip_low <= 1, "
            f"clip_high >= 0 and kl_coef >= 0, got {clip_low}, {clip_high}, "
            f"{kl_coef}"
        )
    if kl_coef != 0 and ref_logprobs is None:
        raise ValueError("Stoke -- kl_coef needs ref_logprobs")
    old = _per_token(old_logprobs, actions, "old_logprobs")
    adv = _per_token(advantages, actions, "advantages")
    lp, live = _eager_logprobs(logits, actions, ignore_index)
    lp, adv = lp[live], adv[live].double()
    rho = (lp - old[live].double()).exp()
    free, held = rho * adv, rho.clamp(1 - clip_low, 1 + clip_high) * adv
    # torch.minimum halves the gradient where both are the same
    tok = -torch.where(free > held, held, free)
    if kl_coef != 0:
        ref = _per_token(ref_logprobs, actions, "ref_logprobs")
        d = ref[live].double() - lp
        # a token that the policy rules out costs inf: not inf - inf
        tok = tok + kl_coef * torch.where(
            d == float("inf"), d, d.exp() - d - 1)
    return (tok.sum() / max(1, tok.numel())).to(_result_dtype(logits))


def fused_preference_loss(logits: torch.Tensor, targets: torch.Tensor,
                          ref_logprobs: torch.Tensor, beta: float = 0.1,
                          label_smoothing: float = 0.0,
                          ignore_index: int = -100,
                          return_rewards: bool = True):
    """Paired preference loss; returns ``(loss, rewards)``, or the loss alone
    with ``return_rewards=False``, as ``Stoke(loss=...)`` takes it.

    logits: [2P, S, V] and targets [2P, S]: the P chosen sequences, then the
    P rejected ones in the same order.  ref_logprobs: [2P, S], the reference
    model's ``token_logprobs``.  A sequence's reward is beta * sum(lp - ref)
    over its non-ignored tokens (``rewards`` [2P] fp32, without gradient);
    with h = reward(chosen) - reward(rejected) a pair's loss is::

        -(1 - label_smoothing) * log sigmoid(h)
        - label_smoothing * log sigmoid(-h)

    and the loss the mean over the pairs.
    """
    ext = _native(logits)
    if ext is not None:
        loss, rewards = ext.preference_loss(
            logits, targets, ref_logprobs, beta, label_smoothing, ignore_index)
        return (loss, rewards) if return_rewards else loss
    _check(logits, targets, "fused_preference_loss")
    if logits.dim() != 3 or logits.shape[0] % 2 or logits.shape[0] == 0:
        raise ValueError(
            "Stoke -- fused_preference_loss takes logits [2P, S, V] (chosen, "
            f"then rejected), got {tuple(logits.shape)}"
        )
    if not (beta > 0 and 0 <= label_smoothing <= 0.5):
        raise ValueError(
            "Stoke -- fused_preference_loss takes beta > 0 and "
            f"0 <= label_smoothing <= 0.5, got {beta}, {label_smoothing}"
        )
    ref = _per_token(ref_logprobs, targets, "ref_logprobs")
    lp, live = _eager_logprobs(logits, targets, ignore_index)
    gap = torch.where(live, lp - ref.double().masked_fill(~live, 0.0), 0.0)
    rewards = beta * gap.sum(-1)
    good, bad = rewards.chunk(2)
    h = good - bad
    ls = torch.nn.functional.logsigmoid
    loss = -(1 - label_smoothing) * ls(h)
    if label_smoothing != 0:  # a margin of +inf: not 0 * inf
        loss = loss - label_smoothing * ls(-h)
    dt = _result_dtype(logits)
    loss = loss.mean().to(dt)
    return (loss, rewards.detach().to(dt)) if return_rewards else loss
