"""Operators over the logits of a token policy (``csrc/token_kernels.cu``): log-probabilities and entropies, the clipped
policy loss with a KL term and an entropy bonus, and the preference loss over pairs of sequences.

The surrogate is PPO's (:func:`tt_rsl_rl_b200.algorithms.ppo.clipped_surrogate_loss`), the policy a softmax over a
vocabulary instead of a Gaussian. Logits are ``[rows, V]`` or ``[batch, rows, V]`` in float32, bfloat16 or float16 with
any row strides (``logits[:, :-1]`` is taken as it is) and contiguous columns; every other input is per row and float32.
A row counts if its ``mask`` is not zero and its token lies in ``[0, V)``: the logits of no other row are read, its
outputs and its gradient are zero. Columns at ``-inf`` have probability zero; a counted row without any finite column
gives NaN, as the formulas do. Gradients go to the logits alone: every other input is a constant.

Each loss comes in two forms. ``*_loss`` is differentiable: it keeps a few numbers per row, and ``backward`` reads the
logits once more. ``*_loss_grad`` returns the loss together with the gradient of the logits (in their type), without
autograd; it can be captured in a CUDA graph and is the faster one. On CPU tensors the same formulas run as PyTorch
operations. CUDA logits with a forward-mode tangent are refused.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import ext

KL_ESTIMATORS = {"k1": 1, "k2": 2, "k3": 3}
PREFERENCE_LOSSES = {"sigmoid": 0, "hinge": 1, "ipo": 2}


class TokenPolicyLoss(NamedTuple):
    """``loss`` and the weighted means that make it up (scalars), ``logp`` of each row's token."""

    loss: torch.Tensor
    surrogate: torch.Tensor
    kl: torch.Tensor
    entropy: torch.Tensor
    clip_fraction: torch.Tensor
    logp: torch.Tensor


class PreferenceLoss(NamedTuple):
    """``loss`` (mean over pairs), ``beta`` times the log-ratios of the chosen and rejected sequences ``[pairs]``, the
    sequences' log-probabilities ``[2 pairs]`` and ``logp`` of each row's token."""

    loss: torch.Tensor
    chosen_rewards: torch.Tensor
    rejected_rewards: torch.Tensor
    seq_logps: torch.Tensor
    logp: torch.Tensor


# ---- checks shared by the CUDA and the CPU path -------------------------------------------------------------------------
def _finite(name: str, value: float) -> float:
    value = float(value)
    if not math.isfinite(value):
        raise ValueError(f"{name} must be finite, got {value}")
    return value


def _refuse_capture(name: str) -> None:
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{name} with gradients cannot be captured in a CUDA graph (autograd's accumulation may run on "
                           f"another stream); capture {name}_grad instead" if name != "token_logprobs" else
                           "token_logprobs with gradients cannot be captured in a CUDA graph; capture "
                           "token_policy_loss_grad or preference_loss_grad instead")


def _check_cpu(logits: torch.Tensor, tokens: torch.Tensor, mask: torch.Tensor | None, temperature: float, **rows) -> None:
    """The refusals of the CUDA entry points, for CPU tensors."""
    if logits.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    if logits.dim() not in (2, 3):
        raise ValueError(f"logits must be [rows, V] or [batch, rows, V], got {tuple(logits.shape)}")
    if logits.shape[-1] == 0:
        raise ValueError("logits need at least one column")
    if logits.shape[-1] > 1 and logits.stride(-1) != 1:
        raise ValueError("the columns of logits must be contiguous")
    if tokens.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"tokens must be int64 or int32, got {tokens.dtype}")
    if mask is not None and mask.dtype not in (torch.bool, torch.uint8, torch.float32):
        raise TypeError(f"mask must be bool, uint8 or float32, got {mask.dtype}")
    for name, x in (rows | {"tokens": tokens, "mask": mask}).items():
        if x is None:
            continue
        if name not in ("tokens", "mask") and x.dtype != torch.float32:
            raise TypeError(f"{name} must be float32, got {x.dtype}")
        if x.device != logits.device:
            raise ValueError(f"{name} must be on the device of the logits")
        if x.shape != logits.shape[:-1]:
            raise ValueError(f"{name} must have the shape {tuple(logits.shape[:-1])}, got {tuple(x.shape)}")
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"temperature must lie in [1e-6, 1e6], got {temperature}")


def _constant(x: torch.Tensor | None) -> torch.Tensor | None:
    return None if x is None else x.detach()


# ---- log-probabilities ----------------------------------------------------------------------------------------------------
def _row_weights(logits, tokens, mask) -> torch.Tensor:
    """Weights of the rows; zero where the token lies outside the vocabulary. Masks of bytes select (any value but zero)."""
    inside = (tokens >= 0) & (tokens < logits.shape[-1])
    if mask is None:
        return inside.float()
    return torch.where(inside, mask if mask.dtype == torch.float32 else (mask != 0).float(), 0.0)


def _logprobs_torch(logits, tokens, weights, temperature):
    counted = weights != 0
    # rows that do not count take part with zeros, so that nothing of them (NaN included) reaches a gradient
    # in 64 bits: a quotient by a small temperature would round the columns' differences away
    z = torch.where(counted[..., None], logits.double(), 0.0) / temperature
    log_p = torch.log_softmax(z, -1)
    tok = tokens.long().clamp(0, logits.shape[-1] - 1)
    logp = log_p.gather(-1, tok[..., None])[..., 0]
    dead = log_p == float("-inf")
    entropy = -(log_p.exp() * log_p.masked_fill(dead, 0.0)).sum(-1)
    return torch.where(counted, logp, 0.0).float(), torch.where(counted, entropy, 0.0).float()


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, mask: torch.Tensor | None = None,
                   temperature: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """``(logp, entropy)`` of each row, float32: the log-probability of its token under
    ``softmax(logits / temperature)`` and that distribution's entropy. Differentiable by the logits. ``mask`` only says
    which rows count: a float mask weighs neither the results nor their gradients."""
    if not logits.is_cuda:
        _check_cpu(logits, tokens, mask, temperature)
        return _logprobs_torch(logits, tokens, _row_weights(logits, tokens, mask), temperature)
    if logits.requires_grad and torch.is_grad_enabled():
        _refuse_capture("token_logprobs")
        return tuple(ext().token_logprobs_autograd(logits, tokens, mask, temperature))
    logp, entropy, _ = ext().token_logprobs(logits, tokens, mask, temperature)
    return logp, entropy


# ---- clipped policy loss ----------------------------------------------------------------------------------------------------
def _policy_settings(ref_logp, clip_param, clip_high, kl_coef, kl_estimator, entropy_coef, reduction):
    if kl_estimator not in KL_ESTIMATORS:
        raise ValueError(f"kl_estimator must be one of {list(KL_ESTIMATORS)}, got {kl_estimator!r}")
    if reduction not in ("mean", "sum"):
        raise ValueError(f"reduction must be 'mean' or 'sum', got {reduction!r}")
    if clip_high is None:
        clip_high = clip_param
    if not math.isfinite(clip_param + clip_high + kl_coef + entropy_coef):
        raise ValueError(f"clip_param, clip_high, kl_coef and entropy_coef must be finite, got {clip_param}, {clip_high}, "
                         f"{kl_coef} and {entropy_coef}")
    if clip_param < 0.0 or clip_high < 0.0:
        raise ValueError(f"clip_param and clip_high must not be negative, got {clip_param} and {clip_high}")
    if kl_coef != 0.0 and ref_logp is None:
        raise ValueError("kl_coef needs ref_logp")
    return 1.0 - clip_param, 1.0 + clip_high, kl_coef, KL_ESTIMATORS[kl_estimator], entropy_coef, reduction == "mean"


def _policy_torch(logits, tokens, old, adv, ref, mask, lo, hi, kl_coef, kl_kind, entropy_coef, mean, temperature):
    old, adv, ref, mask = map(_constant, (old, adv, ref, mask))
    w = _row_weights(logits, tokens, mask)
    counted = w != 0
    logp, entropy = _logprobs_torch(logits, tokens, w, temperature)
    neg_adv = torch.where(counted, -adv, 0.0)
    with torch.no_grad():
        ratio = torch.exp(torch.where(counted, logp - old, 0.0))
        free, cut = neg_adv * ratio, neg_adv * ratio.clamp(lo, hi)
        open_ = (free > cut) | free.isnan() | ((ratio >= lo) & (ratio <= hi))
    # a clipped ratio passes no gradient, an infinite one neither
    moving = torch.where(open_, logp, logp.detach())
    surrogate = torch.where(open_, neg_adv * torch.exp(torch.where(counted, moving - old, 0.0)), cut)
    kl = torch.zeros_like(logp)
    if ref is not None:
        d = torch.where(counted, ref - logp, 0.0)
        kl = -d if kl_kind == 1 else 0.5 * d * d if kl_kind == 2 else torch.expm1(d) - d
    total = w.double().sum()
    inv = torch.where(total != 0, 1.0 / total, 0.0)

    def summed(x):
        return (w.double() * torch.where(counted, x, 0.0).double()).sum()

    loss = summed(surrogate) - entropy_coef * summed(entropy)
    if kl_coef != 0.0:
        loss = loss + kl_coef * summed(kl)
    stats = [(inv * summed(x)).float().detach() for x in (surrogate, kl, entropy, (cut > free).float())]
    return TokenPolicyLoss((loss * inv if mean else loss).float(), *stats, logp.detach())


def token_policy_loss(logits: torch.Tensor, tokens: torch.Tensor, old_logp: torch.Tensor, advantages: torch.Tensor, *,
                      ref_logp: torch.Tensor | None = None, mask: torch.Tensor | None = None, clip_param: float = 0.2,
                      clip_high: float | None = None, kl_coef: float = 0.0, kl_estimator: str = "k3",
                      entropy_coef: float = 0.0, temperature: float = 1.0, reduction: str = "mean") -> TokenPolicyLoss:
    """Clipped policy loss of a token policy, differentiable by the logits.

    With ``r = exp(logp - old_logp)``, ``w`` the mask (weights) and ``d = ref_logp - logp``, the loss is the weighted mean
    (``reduction="sum"``: the weighted sum) over rows of

        ``max(-A r, -A clamp(r, 1 - clip_param, 1 + clip_high)) + kl_coef kl - entropy_coef H``

    where ``kl`` is ``-d`` (``"k1"``), ``d^2 / 2`` (``"k2"``) or ``exp(d) - d - 1`` (``"k3"``). ``clip_high`` defaults to
    ``clip_param``. The other members of the result are weighted means and carry no gradient. If no row counts, loss and
    gradient are zero."""
    settings = _policy_settings(ref_logp, clip_param, clip_high, kl_coef, kl_estimator, entropy_coef, reduction)
    if not logits.is_cuda:
        _check_cpu(logits, tokens, mask, temperature, old_logp=old_logp, advantages=advantages, ref_logp=ref_logp)
        return _policy_torch(logits, tokens, old_logp, advantages, ref_logp, mask, *settings, temperature)
    if logits.requires_grad and torch.is_grad_enabled():
        _refuse_capture("token_policy_loss")
        return TokenPolicyLoss(*ext().token_policy_loss_autograd(
            logits, tokens, old_logp, advantages, ref_logp, mask, *settings[:5], temperature, settings[5]))
    parts = ext().token_policy_loss(logits, tokens, old_logp, advantages, ref_logp, mask, *settings[:5], temperature,
                                    settings[5], False, 1.0, None)
    return TokenPolicyLoss(*parts[:5], parts[6])


def _split_scale(grad_scale):
    if isinstance(grad_scale, torch.Tensor):
        return 1.0, grad_scale
    return _finite("grad_scale", grad_scale), None


def token_policy_loss_grad(logits: torch.Tensor, tokens: torch.Tensor, old_logp: torch.Tensor,
                           advantages: torch.Tensor, *, ref_logp: torch.Tensor | None = None,
                           mask: torch.Tensor | None = None, clip_param: float = 0.2, clip_high: float | None = None,
                           kl_coef: float = 0.0, kl_estimator: str = "k3", entropy_coef: float = 0.0,
                           temperature: float = 1.0, reduction: str = "mean",
                           grad_scale: float | torch.Tensor = 1.0) -> tuple[TokenPolicyLoss, torch.Tensor]:
    """:func:`token_policy_loss` and the gradient of ``grad_scale`` times the loss by the logits, in the logits' type
    (``logits.backward(grad)`` continues from there). ``grad_scale``: a number, or one float32 on the device; a loss
    scale keeps float16 gradients in range."""
    settings = _policy_settings(ref_logp, clip_param, clip_high, kl_coef, kl_estimator, entropy_coef, reduction)
    scale, scale_device = _split_scale(grad_scale)
    if not logits.is_cuda:
        return _grad_torch(token_policy_loss, logits, grad_scale, tokens, old_logp, advantages, ref_logp=ref_logp,
                           mask=mask, clip_param=clip_param, clip_high=clip_high, kl_coef=kl_coef,
                           kl_estimator=kl_estimator, entropy_coef=entropy_coef, temperature=temperature,
                           reduction=reduction)
    parts = ext().token_policy_loss(logits, tokens, old_logp, advantages, ref_logp, mask, *settings[:5], temperature,
                                    settings[5], True, scale, scale_device)
    return TokenPolicyLoss(*parts[:5], parts[6]), parts[7]


def _grad_torch(loss_fn, logits, grad_scale, *args, **kwargs):
    with torch.enable_grad():
        z = logits.detach().requires_grad_()
        result = loss_fn(z, *args, **kwargs)
        grad, = torch.autograd.grad(result.loss * grad_scale, z)
    return result._replace(loss=result.loss.detach()), grad


# ---- preference loss ---------------------------------------------------------------------------------------------------------
def _preference_settings(beta, label_smoothing, loss_type, average):
    if loss_type not in PREFERENCE_LOSSES:
        raise ValueError(f"loss_type must be one of {list(PREFERENCE_LOSSES)}, got {loss_type!r}")
    beta, label_smoothing = _finite("beta", beta), _finite("label_smoothing", label_smoothing)
    if beta <= 0.0:
        raise ValueError(f"beta must be positive, got {beta}")
    if not 0.0 <= label_smoothing <= 0.5:
        raise ValueError(f"label_smoothing must lie in [0, 0.5], got {label_smoothing}")
    if label_smoothing and loss_type != "sigmoid":
        raise ValueError("label_smoothing belongs to loss_type 'sigmoid'")
    return beta, label_smoothing, PREFERENCE_LOSSES[loss_type], bool(average)


def _preference_torch(logits, tokens, ref, offsets, mask, beta, smoothing, kind, average, temperature):
    ref, mask = _constant(ref), _constant(mask)
    w = _row_weights(logits, tokens, mask)
    if logits.dim() == 2 and offsets is not None and offsets.dim() == 1 and offsets.numel():
        # rows before the first and behind the last sequence get no gradient, whatever they hold
        row, ends = torch.arange(len(w)), offsets.long()
        logits = torch.where(((row >= ends[0]) & (row < ends[-1]))[:, None], logits, logits.detach())
    logp, _ = _logprobs_torch(logits, tokens, w, temperature)
    weighted = (w * logp).double()
    if logits.dim() == 3:
        if offsets is not None:
            raise ValueError("offsets belong to packed logits [rows, V]; [sequences, rows, V] has none")
        sums, counts = weighted.sum(1), w.double().sum(1)
    else:
        if offsets is None:
            raise ValueError("packed logits [rows, V] need the offsets of their sequences")
        if offsets.dtype not in (torch.int64, torch.int32):
            raise TypeError(f"offsets must be int64 or int32, got {offsets.dtype}")
        if offsets.dim() != 1 or offsets.numel() < 1:
            raise ValueError("offsets must be [sequences + 1]")
        at = offsets.long().clamp(0, len(w)).tolist()
        if any(a > b for a, b in zip(at[:-1], at[1:])):
            raise ValueError("offsets must not decrease")
        parts = [(weighted[a:b].sum(), w[a:b].double().sum()) for a, b in zip(at[:-1], at[1:])]
        sums, counts = (torch.stack(x) for x in zip(*parts)) if parts else (weighted[:0], weighted[:0])
    if len(sums) % 2:
        raise ValueError(f"sequences 2 k and 2 k + 1 form a pair: their number must be even, got {len(sums)}")
    if ref is not None:
        if ref.dtype != torch.float32:
            raise TypeError(f"ref_logps must be float32, got {ref.dtype}")
        if ref.shape != sums.shape:
            raise ValueError("ref_logps must be [sequences] on the device of the logits")
    lp = torch.where(counts != 0, sums / torch.where(counts != 0, counts, 1.0), 0.0) if average else sums
    rewards = beta * (lp if ref is None else lp - ref.double())
    h = rewards[0::2] - rewards[1::2]
    if kind == 0:
        log_sigmoid = torch.nn.functional.logsigmoid
        losses = -(1.0 - smoothing) * log_sigmoid(h)
        if smoothing:  # an infinite loss of the other side without a weight would leave a NaN
            losses = losses - smoothing * log_sigmoid(-h)
    elif kind == 1:
        losses = torch.relu(1.0 - h)
    else:
        losses = (h / beta - 0.5 / beta) ** 2
    loss = losses.mean().float() if len(losses) else losses.sum().float()
    rewards = rewards.detach().float()
    return PreferenceLoss(loss, rewards[0::2], rewards[1::2], lp.detach().float(), logp.detach())


def preference_loss(logits: torch.Tensor, tokens: torch.Tensor, ref_logps: torch.Tensor | None = None, *,
                    offsets: torch.Tensor | None = None, mask: torch.Tensor | None = None, beta: float = 0.1,
                    label_smoothing: float = 0.0, loss_type: str = "sigmoid", average: bool = False,
                    temperature: float = 1.0) -> PreferenceLoss:
    """Loss over pairs of sequences, the even ones chosen and the odd ones (their successors) rejected, differentiable
    by the logits.

    A sequence's log-probability is the weighted sum (``average=True``: mean) of its rows' ``logp``, summed in 64 bits.
    ``[sequences, rows, V]`` logits hold one sequence per batch entry; packed ``[rows, V]`` logits come with ``offsets``
    ``[sequences + 1]``, non-decreasing row numbers on the same device (values outside ``[0, rows]`` are clamped; rows
    before the first and behind the last sequence get a zero gradient; where they decrease, CPU tensors raise an error, and
    on CUDA, where the host does not wait for them, loss, rewards and gradients are NaN). ``ref_logps`` are the sequences'
    log-probabilities under the reference (None: zero). With ``h`` the difference of ``beta (logp - ref)``, a pair's loss
    is ``-(1 - s) log sigmoid(h) - s log sigmoid(-h)`` (``"sigmoid"``, ``s`` the label smoothing), ``max(0, 1 - h)``
    (``"hinge"``) or ``(h / beta - 1 / (2 beta))^2`` (``"ipo"``)."""
    settings = _preference_settings(beta, label_smoothing, loss_type, average)
    if not logits.is_cuda:
        _check_cpu(logits, tokens, mask, temperature)
        return _preference_torch(logits, tokens, ref_logps, offsets, mask, *settings, temperature)
    if logits.requires_grad and torch.is_grad_enabled():
        _refuse_capture("preference_loss")
        return PreferenceLoss(*ext().preference_loss_autograd(logits, tokens, ref_logps, offsets, mask, *settings,
                                                              temperature))
    parts = ext().preference_loss(logits, tokens, ref_logps, offsets, mask, *settings, temperature, False, 1.0, None)
    return PreferenceLoss(*parts[:5])


def preference_loss_grad(logits: torch.Tensor, tokens: torch.Tensor, ref_logps: torch.Tensor | None = None, *,
                         offsets: torch.Tensor | None = None, mask: torch.Tensor | None = None, beta: float = 0.1,
                         label_smoothing: float = 0.0, loss_type: str = "sigmoid", average: bool = False,
                         temperature: float = 1.0,
                         grad_scale: float | torch.Tensor = 1.0) -> tuple[PreferenceLoss, torch.Tensor]:
    """:func:`preference_loss` and the gradient of ``grad_scale`` times the loss by the logits, in the logits' type."""
    settings = _preference_settings(beta, label_smoothing, loss_type, average)
    scale, scale_device = _split_scale(grad_scale)
    if not logits.is_cuda:
        return _grad_torch(preference_loss, logits, grad_scale, tokens, ref_logps, offsets=offsets, mask=mask, beta=beta,
                           label_smoothing=label_smoothing, loss_type=loss_type, average=average,
                           temperature=temperature)
    *parts, grad = ext().preference_loss(logits, tokens, ref_logps, offsets, mask, *settings, temperature, True, scale,
                                         scale_device)
    return PreferenceLoss(*parts), grad
