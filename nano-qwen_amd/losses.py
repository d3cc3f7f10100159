"""What a model is trained with, on the kernels: from its logits to a scalar loss.

``token_logprobs`` gives the log-probability of each label; ``preference_loss`` and
``policy_loss`` take such log-probabilities, those of a reference or an earlier policy
and a mask, and give a scalar.  Each has its gradient as a kernel.  They serve the
reference's preference and policy training (its training/ loops), which composes the
same formulas from tensor operations.

A pass over the operands instead of one per tensor operation; no atomics, so a call
gives the same bits each time.  Host tensors raise, since there is no CPU path;
gradients of gradients raise, as they do for the attention kernels.
"""

from __future__ import annotations

import math
from contextlib import nullcontext
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib, ops

__all__ = ["token_logprobs", "preference_loss", "policy_loss"]

IGNORE_INDEX = -100

_KINDS = {"sigmoid": _lib.NQ_PREF_SIGMOID, "hinge": _lib.NQ_PREF_HINGE, "ipo": _lib.NQ_PREF_IPO}


def _on(t: torch.Tensor):
    """A launch goes to the current device: make it the operands'."""
    return nullcontext() if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


def _first_order(backward):
    """``once_differentiable`` where a graph of the backward is recorded; without its host time
    (~10 us) where none is."""
    guarded = once_differentiable(backward)

    def call(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return call


def _check_devices(*ts: Optional[torch.Tensor]) -> None:
    ops._require_device(*ts)
    devices = {t.device for t in ts if t is not None}
    if len(devices) > 1:
        raise ValueError(f"the operands lie on different devices: {sorted(map(str, devices))}")


def _workspace(nbytes: int, device) -> Optional[torch.Tensor]:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _check_temperature(temperature: float) -> float:
    t = float(temperature)
    if not (t > 0 and math.isfinite(t)):
        raise ValueError(f"temperature must be positive and finite, got {temperature}")
    return t


def _check_labels(labels: torch.Tensor, rows_shape) -> torch.Tensor:
    if labels.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"labels must be int64 or int32, got {labels.dtype}")
    if tuple(labels.shape) != tuple(rows_shape):
        raise ValueError(f"labels {tuple(labels.shape)} must hold one label per row {tuple(rows_shape)}")
    return labels.to(torch.int64).contiguous()


# ---------------------------------------------------------------------------
# Log-probabilities of labels
# ---------------------------------------------------------------------------

def _rows_2d(x: torch.Tensor):
    """(x, B, S, batch stride, row stride): x as B sequences of S rows, copied only if its
    leading axes do not fold into two or its last axis is not contiguous."""
    V = x.shape[-1]
    if x.stride(-1) != 1 and V > 1:
        x = x.contiguous()
    if x.dim() == 1:
        return x, 1, 1, 0, 0
    if x.dim() == 2:
        return x, 1, x.shape[0], 0, x.stride(0)
    if x.dim() > 3:
        try:
            v = x.view(-1, *x.shape[-2:])
        except RuntimeError:
            v = x.contiguous().view(-1, *x.shape[-2:])
        x = v
    return x, x.shape[0], x.shape[1], x.stride(0), x.stride(1)


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, temperature: float, ignore_index: int):
        x, B, S, bs, rs = _rows_2d(logits)
        V = x.shape[-1]
        out = torch.empty(labels.shape, dtype=torch.float32, device=x.device)
        stats = torch.empty(B * S, 2, dtype=torch.float32, device=x.device)
        lib = _lib.load()
        ws = _workspace(lib.nq_token_logprobs_workspace_bytes(B * S, V), x.device)
        with _on(x):
            _lib.check(lib.nq_token_logprobs(ops._ptr(x), bs, rs, ops._ptr(labels), ops._ptr(out), ops._ptr(stats),
                                             ops._ptr(ws), ws.numel() if ws is not None else 0, B, S, V, ops._code(x),
                                             temperature, ignore_index, ops._stream(x)), "nq_token_logprobs")
        ctx.save_for_backward(logits, labels, stats)
        ctx.temperature, ctx.ignore_index = temperature, ignore_index
        return out

    @staticmethod
    @_first_order
    def backward(ctx, dy):
        logits, labels, stats = ctx.saved_tensors
        x, B, S, bs, rs = _rows_2d(logits)
        dy = dy.contiguous()
        dx = torch.empty(logits.shape, dtype=x.dtype, device=x.device)
        with _on(x):
            _lib.check(_lib.load().nq_token_logprobs_bwd(
                ops._ptr(x), bs, rs, ops._ptr(labels), ops._ptr(stats), ops._ptr(dy), ops._ptr(dx), B, S, x.shape[-1],
                ops._code(x), ctx.temperature, ctx.ignore_index, ops._stream(x)), "nq_token_logprobs_bwd")
        return dx, None, None, None


def token_logprobs(logits: torch.Tensor, labels: torch.Tensor, *, temperature: float = 1.0,
                   ignore_index: int = IGNORE_INDEX) -> torch.Tensor:
    """log softmax(logits / temperature) at each row's label, fp32 and shaped like ``labels``.

    logits: (..., V) bf16 or fp32, any strides (copied only where the last axis is not
    contiguous or more than two leading axes do not fold); labels: (...) int64 or int32.
    A label equal to ``ignore_index`` gives 0 and no gradient, and its row is not read.
    Any other label outside [0, V) gives NaN, and so do its gradients: labels on the
    device are not read back.  A row of -inf, one with NaN and one with +inf give NaN, as
    log_softmax does.

    To leave out a sequence's last position pad the labels with ``ignore_index`` rather
    than slice the logits: the gradient of a slice is a second pass over all of them.
    """
    _check_devices(logits, labels)
    ops._code(logits)
    if logits.dim() == 0 or logits.shape[-1] == 0:
        raise ValueError(f"logits need a last axis of at least one element, got shape {tuple(logits.shape)}")
    labels = _check_labels(labels, logits.shape[:-1])
    temperature = _check_temperature(temperature)
    if labels.numel() == 0:
        return logits.sum(-1).float()  # empty, with logits' place in the graph
    return _TokenLogprobs.apply(logits, labels, temperature, int(ignore_index))


# ---------------------------------------------------------------------------
# Losses over tokens' log-probabilities
# ---------------------------------------------------------------------------

def _token_rows(t: Optional[torch.Tensor], name: str, shape) -> Optional[torch.Tensor]:
    """(B, S) fp32 rows with contiguous tokens, of (B, S) or (B,)."""
    if t is None:
        return None
    if t.dtype not in ops._DTYPES:
        raise TypeError(f"{name} must be float32 or bfloat16, got {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} {tuple(t.shape)} must be shaped like its log-probabilities {tuple(shape)}")
    return _rows(t.float() if t.dtype != torch.float32 else t)


def _rows(t: torch.Tensor) -> torch.Tensor:
    t = t if t.dim() == 2 else t[:, None]
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


def _mask_rows(mask: Optional[torch.Tensor], name: str, shape) -> Optional[torch.Tensor]:
    if mask is None:
        return None
    if tuple(mask.shape) != tuple(shape):
        raise ValueError(f"{name} {tuple(mask.shape)} must be shaped like its log-probabilities {tuple(shape)}")
    return _rows(mask if mask.dtype in (torch.bool, torch.uint8) else mask != 0)


def _pitch(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.stride(0)


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, chosen, rejected, ref_chosen, ref_rejected, chosen_mask, rejected_mask, kind: int, beta: float,
                smoothing: float, average: bool):
        (B, Sc), Sr, dev = chosen.shape, rejected.shape[1], chosen.device
        new = torch.empty
        loss = new((), dtype=torch.float32, device=dev)
        reward_c, reward_r = (new(B, dtype=torch.float32, device=dev) for _ in range(2))
        coef = new(2, B, dtype=torch.float32, device=dev)
        lib = _lib.load()
        ws = _workspace(lib.nq_preference_loss_workspace_bytes(B), dev)
        p = ops._ptr
        with _on(chosen):
            _lib.check(lib.nq_preference_loss(
                p(chosen), _pitch(chosen), p(rejected), _pitch(rejected), p(ref_chosen), _pitch(ref_chosen),
                p(ref_rejected), _pitch(ref_rejected), p(chosen_mask), _pitch(chosen_mask), p(rejected_mask),
                _pitch(rejected_mask), p(loss), p(reward_c), p(reward_r), p(coef), p(ws), ws.numel(), B, Sc, Sr, kind,
                beta, smoothing, int(average), ops._stream(chosen)), "nq_preference_loss")
        ctx.save_for_backward(coef, chosen_mask, rejected_mask)
        ctx.lens = Sc, Sr
        ctx.mark_non_differentiable(reward_c, reward_r)
        ctx.set_materialize_grads(False)  # no zeros for the rewards' gradients
        return loss, reward_c, reward_r

    @staticmethod
    @_first_order
    def backward(ctx, dloss, *_):
        if dloss is None:
            return (None,) * 10
        coef, chosen_mask, rejected_mask = ctx.saved_tensors
        (Sc, Sr), B = ctx.lens, coef.shape[1]
        dc, dr = (torch.empty(B, S, dtype=torch.float32, device=coef.device) if need else None
                  for S, need in zip((Sc, Sr), ctx.needs_input_grad))
        p = ops._ptr
        with _on(coef):
            _lib.check(_lib.load().nq_preference_loss_bwd(
                p(coef), p(dloss), p(chosen_mask), _pitch(chosen_mask), p(rejected_mask), _pitch(rejected_mask), p(dc),
                p(dr), B, Sc, Sr, ops._stream(coef)), "nq_preference_loss_bwd")
        return dc, dr, None, None, None, None, None, None, None, None


def preference_loss(chosen: torch.Tensor, rejected: torch.Tensor, ref_chosen: Optional[torch.Tensor] = None,
                    ref_rejected: Optional[torch.Tensor] = None, *, chosen_mask: Optional[torch.Tensor] = None,
                    rejected_mask: Optional[torch.Tensor] = None, beta: float = 0.1, label_smoothing: float = 0.0,
                    kind: str = "sigmoid", average: bool = False
                    ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Preference loss over B pairs of sequences: (loss, chosen rewards, rejected rewards).

    chosen, rejected: log-probabilities under the policy, (B, Sc) and (B, Sr) per token or
    (B,) per sequence, fp32 (bf16 is converted); ref_chosen, ref_rejected: those of the
    reference model, shaped alike, or None for none.  The masks (bool; other types count
    as != 0) keep tokens; what a masked token holds has no effect.  With d the sum of
    policy - reference over a sequence's kept tokens (``average``: their mean, 0 if there
    are none) and h = beta (d_chosen - d_rejected), ``kind`` selects a pair's loss:

      "sigmoid"  -(1 - label_smoothing) log s(h) - label_smoothing log s(-h)
      "hinge"    max(0, 1 - h)
      "ipo"      (d_chosen - d_rejected - 1 / (2 beta))^2

    The loss is the mean over pairs, a scalar with gradients for chosen and rejected (the
    references get none); the rewards, beta d, are (B,) without gradient.
    """
    _check_devices(chosen, rejected, ref_chosen, ref_rejected, chosen_mask, rejected_mask)
    if kind not in _KINDS:
        raise ValueError(f"kind must be one of {sorted(_KINDS)}, got {kind!r}")
    if not (beta > 0 and math.isfinite(beta)):
        raise ValueError(f"beta must be positive and finite, got {beta}")
    if not 0 <= label_smoothing < 0.5 or (label_smoothing and kind != "sigmoid"):
        raise ValueError("label_smoothing is for the sigmoid loss, from 0 to under 1/2, "
                         f"got {label_smoothing} with {kind!r}")
    for name, t in (("chosen", chosen), ("rejected", rejected)):
        if t.dim() not in (1, 2):
            raise ValueError(f"{name} must be (B, S) or (B,), got shape {tuple(t.shape)}")
    if chosen.shape[0] != rejected.shape[0] or chosen.shape[0] == 0:
        raise ValueError(f"chosen and rejected must hold the same number of sequences, at least one, "
                         f"got {chosen.shape[0]} and {rejected.shape[0]}")
    sc, sr = chosen.shape, rejected.shape
    return _PreferenceLoss.apply(
        _token_rows(chosen, "chosen", sc), _token_rows(rejected, "rejected", sr),
        _token_rows(_detached(ref_chosen), "ref_chosen", sc), _token_rows(_detached(ref_rejected), "ref_rejected", sr),
        _mask_rows(chosen_mask, "chosen_mask", sc), _mask_rows(rejected_mask, "rejected_mask", sr),
        _KINDS[kind], float(beta), float(label_smoothing), bool(average))


def _detached(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return t.detach() if t is not None and t.requires_grad else t


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, lp, old, ref, adv, mask, low: float, high: float, kl_coef: float, mean_of_means: bool):
        (B, S), dev = lp.shape, lp.device
        loss, kl, clipped = (torch.empty((), dtype=torch.float32, device=dev) for _ in range(3))
        weight = torch.empty(B, dtype=torch.float32, device=dev)
        lib = _lib.load()
        ws = _workspace(lib.nq_policy_loss_workspace_bytes(B, S), dev)
        ctx.save_for_backward(lp, old, ref, adv, mask, weight)
        ctx.clip = low, high, kl_coef
        p = ops._ptr
        with _on(lp):
            _lib.check(lib.nq_policy_loss(
                *_policy_operands(lp, old, ref, adv, mask), p(loss), p(kl), p(clipped), p(weight), p(ws), ws.numel(),
                B, S, low, high, kl_coef, int(mean_of_means), ops._stream(lp)), "nq_policy_loss")
        ctx.mark_non_differentiable(kl, clipped)
        ctx.set_materialize_grads(False)
        return loss, kl, clipped

    @staticmethod
    @_first_order
    def backward(ctx, dloss, *_):
        if dloss is None:
            return (None,) * 9
        lp, old, ref, adv, mask, weight = ctx.saved_tensors
        B, S = lp.shape
        grad = torch.empty(B, S, dtype=torch.float32, device=lp.device)
        p = ops._ptr
        with _on(lp):
            _lib.check(_lib.load().nq_policy_loss_bwd(
                *_policy_operands(lp, old, ref, adv, mask), p(weight), p(dloss), p(grad), B, S, *ctx.clip,
                ops._stream(lp)), "nq_policy_loss_bwd")
        return grad, None, None, None, None, None, None, None, None


def _policy_operands(lp, old, ref, adv, mask):
    p = ops._ptr
    return (p(lp), _pitch(lp), p(old), _pitch(old), p(ref), _pitch(ref), p(adv), adv.stride(0), int(adv.dim() == 2),
            p(mask), _pitch(mask))


def policy_loss(logprobs: torch.Tensor, old_logprobs: torch.Tensor, advantages: torch.Tensor, *,
                ref_logprobs: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
                clip_low: float = 0.2, clip_high: Optional[float] = None, kl_coef: float = 0.0,
                reduction: str = "token") -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Clipped policy loss with a KL term over B sequences of tokens: (loss, kl, clipped).

    logprobs, old_logprobs, ref_logprobs: (B, S) log-probabilities of the sampled tokens
    under the policy, the policy that sampled them and a reference (needed with
    ``kl_coef``), fp32 (bf16 is converted).  advantages: (B,) per sequence or (B, S).  The
    mask (bool; other types count as != 0) keeps tokens; what a masked token holds has no
    effect.  Per kept token, with r = exp(logprobs - old_logprobs) and q = ref - logprobs:

      -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef (exp(q) - q - 1)

    ``clip_high`` defaults to ``clip_low``.  ``reduction``: "token", the mean over all kept
    tokens, or "sequence", the mean over the B sequences of each one's mean (0 for one
    without kept tokens).  Returns the loss, a scalar with a gradient for logprobs alone;
    and, without gradient, the kept tokens' mean of exp(q) - q - 1 (0 without a reference)
    and the share of them that the clip decides.
    """
    _check_devices(logprobs, old_logprobs, advantages, ref_logprobs, mask)
    if logprobs.dim() != 2 or logprobs.shape[0] == 0:
        raise ValueError(f"logprobs must be (B, S) with at least one sequence, got shape {tuple(logprobs.shape)}")
    clip_high = clip_low if clip_high is None else clip_high
    if not 0 <= clip_low <= 1 or not (clip_high >= 0 and math.isfinite(clip_high)) or not math.isfinite(kl_coef):
        raise ValueError("clip_low must lie in [0, 1], clip_high be at least 0 and all finite, "
                         f"got {clip_low}, {clip_high} and kl_coef {kl_coef}")
    if kl_coef and ref_logprobs is None:
        raise ValueError("kl_coef needs ref_logprobs")
    if reduction not in ("token", "sequence"):
        raise ValueError(f"reduction must be 'token' or 'sequence', got {reduction!r}")
    shape = logprobs.shape
    adv = _detached(advantages)
    if adv.dim() == 1:
        adv = _token_rows(adv, "advantages", shape[:1])[:, 0]
    else:
        adv = _token_rows(adv, "advantages", shape)
    return _PolicyLoss.apply(
        _token_rows(logprobs, "logprobs", shape), _token_rows(_detached(old_logprobs), "old_logprobs", shape),
        _token_rows(_detached(ref_logprobs), "ref_logprobs", shape), adv, _mask_rows(mask, "mask", shape),
        float(clip_low), float(clip_high), float(kl_coef), reduction == "sequence")
