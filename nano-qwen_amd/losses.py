"""What a model is trained with, on the kernels: from its hidden states to a scalar loss.

``token_logprobs`` gives the log-probability of each label, ``linear_logprobs`` the same from
the last hidden states and the LM head without the logits; ``preference_loss`` and
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
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib, ops

__all__ = ["token_logprobs", "linear_logprobs", "preference_loss", "policy_loss"]

IGNORE_INDEX = -100

_PROXY = torch._C._TorchDispatchModeKey.PROXY
_is_tracing, _dispatch_mode = torch._C._is_tracing, torch._C._get_dispatch_mode
_before_dispatch = torch._ops.mode_stack_state_for_pre_dispatch()  # get(0): the proxy mode there

_KINDS = {"sigmoid": _lib.NQ_PREF_SIGMOID, "hinge": _lib.NQ_PREF_HINGE, "ipo": _lib.NQ_PREF_IPO}


# The device takes less than the host for most of these calls, and the backward's Python runs
# on autograd's own thread, where it takes some three times as long as alone: what needs no
# gradient goes round autograd or through it as one tuple, and little stands around a launch.

def _launch(t: torch.Tensor, fn, name: str, *args) -> None:
    """fn(*args, stream) on t's device (a launch goes to the current one).

    A recording of tensor operations (``torch.jit.trace``, ``make_fx``) holds the outputs'
    allocation and not the launch, and its replays would return what the memory holds: it is
    refused.  ``torch.compile`` breaks its graph here and calls the kernel as it is."""
    if _is_tracing() or _dispatch_mode(_PROXY) is not None or _before_dispatch.get(0) is not None:
        raise RuntimeError(f"{name}: a trace of tensor operations cannot hold the kernels of the losses")
    index = t.get_device()
    args += (torch._C._cuda_getCurrentRawStream(index),)
    if index == torch._C._cuda_getDevice():
        rc = fn(*args)
    else:
        with torch.cuda.device(index):
            rc = fn(*args)
    if rc:
        _lib.check(rc, name)


def _first_order(backward):
    """``once_differentiable`` where a graph of the backward is recorded; without its host time
    (~10 us) where none is."""
    guarded = once_differentiable(backward)

    def call(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return call


def _takes_gradient(*ts: torch.Tensor) -> bool:
    """Whether autograd has a part in the call (forward mode: it refuses it)."""
    if torch.is_grad_enabled():
        for t in ts:
            if t.requires_grad:
                return True
    return ops._forward_ad._current_level >= 0


def _check_devices(first: torch.Tensor, *others: Optional[torch.Tensor]) -> None:
    index = first.get_device()  # -1: on the host
    for t in others:
        if t is not None and t.get_device() != index:
            ops._require_device(first, t)
            raise ValueError(f"the operands lie on different devices: {first.device} and {t.device}")
    if index < 0 or not first.is_cuda:
        ops._require_device(first)


def _memory(t: torch.Tensor) -> int:
    """An operand's pointer, of a tensor that its memory says all of."""
    pointer = t.data_ptr()
    if pointer == 0 and t.numel():
        # distributed, functionalized and other wrapped tensors: a kernel would take the null
        # pointer of an optional operand for one left out
        raise TypeError(f"the kernels need tensors with memory of their own, got {type(t).__name__} without")
    if t.is_neg():  # the imaginary part of a conjugate: its memory holds the opposite
        raise TypeError("the kernels read a tensor's memory as it is: give resolve_neg() of a negative view")
    return pointer


def _check_temperature(temperature: float) -> float:
    t = float(temperature)
    if not (t > 0 and math.isfinite(t)):
        raise ValueError(f"temperature must be positive and finite, got {temperature}")
    return t


def _check_labels(labels: torch.Tensor, rows_shape) -> torch.Tensor:
    if labels.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"labels must be int64 or int32, got {labels.dtype}")
    if labels.shape != rows_shape:
        raise ValueError(f"labels {tuple(labels.shape)} must hold one label per row {tuple(rows_shape)}")
    if labels.dtype != torch.int64:
        labels = labels.to(torch.int64)
    return labels if labels.is_contiguous() else labels.contiguous()


# ---------------------------------------------------------------------------
# Log-probabilities of labels
# ---------------------------------------------------------------------------

def _rows_2d(x: torch.Tensor):
    """(x, B, S, batch stride, row stride): x as B sequences of S rows, copied only if its
    leading axes do not fold into two or its last axis is not contiguous.  The stride of an
    axis of one is anything, and 0 here."""
    V = x.shape[-1]
    if x.stride(-1) != 1 and V > 1:
        x = x.contiguous()
    if x.dim() == 1:
        return x, 1, 1, 0, 0
    if x.dim() == 2:
        return x, 1, x.shape[0], 0, x.stride(0) if x.shape[0] > 1 else 0
    if x.dim() > 3:
        try:
            v = x.view(-1, *x.shape[-2:])
        except RuntimeError:
            v = x.contiguous().view(-1, *x.shape[-2:])
        x = v
    B, S = x.shape[:2]
    return x, B, S, x.stride(0) if B > 1 else 0, x.stride(1) if S > 1 else 0


def _token_forward(logits, labels, temperature: float, ignore_index: int):
    x, B, S, bs, rs = _rows_2d(logits)
    V = x.shape[-1]
    out = x.new_empty(labels.shape, dtype=torch.float32)
    stats = x.new_empty((B * S, 2), dtype=torch.float32)
    lib = _lib.load()
    nbytes = lib.nq_token_logprobs_workspace_bytes(B * S, V)
    ws = x.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    tail = (B, S, V, ops._code(x), temperature, ignore_index)
    _launch(x, lib.nq_token_logprobs, "nq_token_logprobs", _memory(x), bs, rs, _memory(labels), out.data_ptr(),
            stats.data_ptr(), ops._ptr(ws), nbytes, *tail)
    return out, stats, tail


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, rest):
        out, stats, ctx.tail = _token_forward(logits, *rest)
        ctx.save_for_backward(logits, rest[0], stats)
        return out

    @staticmethod
    @_first_order
    def backward(ctx, dy):
        logits, labels, stats = ctx.saved_tensors
        x, _, _, bs, rs = _rows_2d(logits)
        dy = dy.resolve_neg().contiguous()
        dx = x.new_empty(logits.shape)
        _launch(x, _lib.load().nq_token_logprobs_bwd, "nq_token_logprobs_bwd", ops._ptr(x), bs, rs, ops._ptr(labels),
                ops._ptr(stats), ops._ptr(dy), ops._ptr(dx), *ctx.tail)
        return dx, None


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
    if logits.dtype not in ops._DTYPES:
        ops._code(logits)
    if logits.dim() == 0 or not 0 < logits.shape[-1] < 2 ** 31:
        raise ValueError(f"logits need a last axis of 1 to 2^31 - 1 elements, got shape {tuple(logits.shape)}")
    labels = _check_labels(labels, logits.shape[:-1])
    temperature = _check_temperature(temperature)
    if labels.numel() == 0:
        return logits.sum(-1).float()  # empty, with logits' place in the graph
    rest = labels, temperature, int(ignore_index)
    return _TokenLogprobs.apply(logits, rest) if _takes_gradient(logits) else _token_forward(logits, *rest)[0]


def _linear_forward(hidden, weight, labels, temperature: float, ignore_index: int, keep: bool):
    x, w, B, S, bs, rs = _head_operands(hidden, weight)
    V, H = w.shape
    out = x.new_empty(labels.shape, dtype=torch.float32)
    stats = x.new_empty((B * S, 2), dtype=torch.float32)
    lib = _lib.load()
    nkept = lib.nq_linear_logprobs_kept_bytes(B * S, V, H) if keep else 0
    kept = x.new_empty(nkept, dtype=torch.uint8) if nkept else None
    nbytes = lib.nq_linear_logprobs_workspace_bytes(B * S, V, H)
    ws = x.new_empty(nbytes, dtype=torch.uint8)
    _launch(x, lib.nq_linear_logprobs, "nq_linear_logprobs", _memory(x), bs, rs, _memory(w), _memory(labels),
            out.data_ptr(), stats.data_ptr(), ops._ptr(kept), nkept, ws.data_ptr(), nbytes, B, S, V, H, temperature,
            ignore_index)
    return out, stats, kept


class _LinearLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, rest):
        out, stats, kept = _linear_forward(hidden, weight, *rest)
        ctx.save_for_backward(hidden, weight, rest[0], stats, kept)
        ctx.tail = rest[1:3]
        return out

    @staticmethod
    @_first_order
    def backward(ctx, dy):
        hidden, weight, labels, stats, kept = ctx.saved_tensors
        x, w, B, S, bs, rs = _head_operands(hidden, weight)
        V, H = w.shape
        dy = dy.resolve_neg().contiguous()
        dh = x.new_empty(hidden.shape) if ctx.needs_input_grad[0] else None
        dw = w.new_empty((V, H)) if ctx.needs_input_grad[1] else None
        lib = _lib.load()
        nbytes = lib.nq_linear_logprobs_bwd_workspace_bytes(B * S, V, H)
        ws = x.new_empty(nbytes, dtype=torch.uint8)
        _launch(x, lib.nq_linear_logprobs_bwd, "nq_linear_logprobs_bwd", x.data_ptr(), bs, rs, w.data_ptr(),
                labels.data_ptr(), stats.data_ptr(), ops._ptr(kept), 0 if kept is None else kept.numel(),
                dy.data_ptr(), ops._ptr(dh), ops._ptr(dw), ws.data_ptr(), nbytes, B, S, V, H, *ctx.tail)
        return dh, dw, None


def _head_operands(hidden: torch.Tensor, weight: torch.Tensor):
    """(hidden, weight, B, S, batch stride, row stride), copied where rows are not 16-byte aligned."""
    x, B, S, bs, rs = _rows_2d(hidden)
    if bs % 8 or rs % 8 or x.data_ptr() % 16:
        x, B, S, bs, rs = _rows_2d(hidden.contiguous().clone() if hidden.is_contiguous() else hidden.contiguous())
    w = weight.contiguous()
    return x, w if w.data_ptr() % 16 == 0 else w.clone(), B, S, bs, rs


def linear_logprobs(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, *, temperature: float = 1.0,
                    ignore_index: int = IGNORE_INDEX, recompute: bool = False) -> torch.Tensor:
    """``token_logprobs(hidden @ weight.T, labels)`` without the logits, fp32 and shaped like ``labels``.

    hidden: (..., H) bf16 hidden states, rows at any strides; weight: (V, H) bf16, an LM
    head's; H a multiple of 8, at most 2^20; at most 2^24 rows and entries.  Logits are held
    in fp32 and never stored; the backward forms their gradient in bf16, a range of the
    vocabulary at a time (at most 1 GiB up to 2^21 rows, 512 bytes a row beyond), and gives
    hidden and weight gradients summed in fp32.  Rows whose label is ``ignore_index`` take no part in the products.  Labels outside
    [0, V) give NaN, and so do their row's and the weight's gradients.

    A call with a gradient keeps the softmax's numerators for it, in bf16, 2 bytes for each
    entry of each row, where that is faster (widths from 256, more than 64 rows) and at most
    4 GiB; otherwise, and with ``recompute``, it keeps two numbers a row and the backward
    repeats the first product (about a fifth slower).

    An fp32 head goes through its logits:
    ``token_logprobs(F.linear(hidden, weight), labels)``.
    """
    _check_devices(hidden, weight, labels)
    if hidden.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise TypeError(f"hidden and weight must be bfloat16, got {hidden.dtype} and {weight.dtype}; "
                        "token_logprobs takes the logits of other types")
    if hidden.dim() == 0 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"hidden {tuple(hidden.shape)} must be (..., H) and weight {tuple(weight.shape)} (V, H)")
    V, H = weight.shape
    if V == 0 or H == 0 or H % 8 or H > _HEAD_WIDEST:
        raise ValueError("the kernels take at least one entry and widths that are multiples of 8, up to 2^20, "
                         f"got {V} and {H}")
    labels = _check_labels(labels, hidden.shape[:-1])
    temperature = _check_temperature(temperature)
    if labels.numel() == 0:
        return torch.nn.functional.linear(hidden, weight)[..., 0].float()  # empty, with its place in the graph
    if labels.numel() > _HEAD_MOST or V > _HEAD_MOST:
        raise ValueError(f"at most 2^24 rows and entries in one call, got {labels.numel()} and {V}")
    rest = labels, temperature, int(ignore_index)
    if _takes_gradient(hidden, weight):
        return _LinearLogprobs.apply(hidden, weight, (*rest, not recompute))
    return _linear_forward(hidden, weight, *rest, False)[0]


_HEAD_MOST = 1 << 24
_HEAD_WIDEST = 1 << 20
_MOST_SEQUENCES = 1 << 30  # well within the C entries' int, to which ctypes cuts a larger number without a word


# ---------------------------------------------------------------------------
# Losses over tokens' log-probabilities
# ---------------------------------------------------------------------------

def _token_rows(t: Optional[torch.Tensor], name: str, shape) -> Optional[torch.Tensor]:
    """(B, S) fp32 rows with contiguous tokens, of (B, S) or (B,)."""
    if t is None:
        return None
    if t.dtype != torch.float32:
        if t.dtype != torch.bfloat16:
            raise TypeError(f"{name} must be float32 or bfloat16, got {t.dtype}")
        t = t.float()
    if t.shape != shape:
        raise ValueError(f"{name} {tuple(t.shape)} must be shaped like its log-probabilities {tuple(shape)}")
    return _rows(t)


def _rows(t: torch.Tensor) -> torch.Tensor:
    if t.dim() == 1:
        return t[:, None]
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


def _mask_rows(mask: Optional[torch.Tensor], name: str, shape) -> Optional[torch.Tensor]:
    if mask is None:
        return None
    if mask.shape != shape:
        raise ValueError(f"{name} {tuple(mask.shape)} must be shaped like its log-probabilities {tuple(shape)}")
    return _rows(mask if mask.dtype in (torch.bool, torch.uint8) else mask != 0)


def _with_pitch(*ts: Optional[torch.Tensor]):
    """Pointer and row stride of each."""
    args = ()
    for t in ts:
        args += (None, 0) if t is None else (_memory(t), t.stride(0))
    return args


def _saved_pitch(*ts: Optional[torch.Tensor]):
    """The same of what a forward took."""
    args = ()
    for t in ts:
        args += (None, 0) if t is None else (t.data_ptr(), t.stride(0))
    return args


def _preference_forward(chosen, rejected, rest):
    """(loss, coef); rest: the rewards, which it writes, the references, the masks and the numbers."""
    reward_c, reward_r, ref_chosen, ref_rejected, chosen_mask, rejected_mask, kind, beta, smoothing, average = rest
    B, Sc = chosen.shape
    loss, coef = chosen.new_empty(()), chosen.new_empty((2, B))
    lib = _lib.load()
    nbytes = lib.nq_preference_loss_workspace_bytes(B)
    ws = chosen.new_empty(nbytes, dtype=torch.uint8)
    _launch(chosen, lib.nq_preference_loss, "nq_preference_loss",
            *_with_pitch(chosen, rejected, ref_chosen, ref_rejected, chosen_mask, rejected_mask), loss.data_ptr(),
            reward_c.data_ptr(), reward_r.data_ptr(), coef.data_ptr(), ws.data_ptr(), nbytes, B, Sc,
            rejected.shape[1], kind, beta, smoothing, average)
    return loss, coef


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, chosen, rejected, rest):
        loss, coef = _preference_forward(chosen, rejected, rest)
        ctx.save_for_backward(coef, rest[4], rest[5])
        ctx.sizes = *chosen.shape, rejected.shape[1]
        return loss

    @staticmethod
    @_first_order
    def backward(ctx, dloss):
        coef, chosen_mask, rejected_mask = ctx.saved_tensors
        B, Sc, Sr = ctx.sizes
        need, dloss = ctx.needs_input_grad, dloss.resolve_neg()
        dc = coef.new_empty((B, Sc)) if need[0] else None
        dr = coef.new_empty((B, Sr)) if need[1] else None
        _launch(coef, _lib.load().nq_preference_loss_bwd, "nq_preference_loss_bwd", coef.data_ptr(), dloss.data_ptr(),
                *_saved_pitch(chosen_mask, rejected_mask), ops._ptr(dc), ops._ptr(dr), B, Sc, Sr)
        return dc, dr, None


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

    The loss is the mean over pairs (at most 2^30), a scalar with gradients for chosen and rejected (the
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
    if chosen.shape[0] > _MOST_SEQUENCES:
        raise ValueError(f"at most 2^30 sequences in one call, got {chosen.shape[0]}")
    sc, sr = chosen.shape, rejected.shape
    chosen, rejected = _token_rows(chosen, "chosen", sc), _token_rows(rejected, "rejected", sr)
    rewards = chosen.new_empty(sc[0]), chosen.new_empty(sc[0])
    rest = (*rewards, _token_rows(_detached(ref_chosen), "ref_chosen", sc),
            _token_rows(_detached(ref_rejected), "ref_rejected", sr), _mask_rows(chosen_mask, "chosen_mask", sc),
            _mask_rows(rejected_mask, "rejected_mask", sr), _KINDS[kind], float(beta), float(label_smoothing),
            int(bool(average)))
    if _takes_gradient(chosen, rejected):
        return (_PreferenceLoss.apply(chosen, rejected, rest), *rewards)
    return (_preference_forward(chosen, rejected, rest)[0], *rewards)


def _detached(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return t.detach() if t is not None and t.requires_grad else t


def _policy_forward(lp, rest):
    """(loss, weight); rest: kl and clipped, which it writes, the other operands and the numbers."""
    kl, clipped, old, ref, adv, mask, low, high, kl_coef, mean_of_means = rest
    B, S = lp.shape
    loss, weight = lp.new_empty(()), lp.new_empty(B)
    lib = _lib.load()
    nbytes = lib.nq_policy_loss_workspace_bytes(B, S)
    ws = lp.new_empty(nbytes, dtype=torch.uint8)
    _launch(lp, lib.nq_policy_loss, "nq_policy_loss", *_with_pitch(lp, old, ref, adv), adv.dim() - 1,
            *_with_pitch(mask), loss.data_ptr(), kl.data_ptr(), clipped.data_ptr(), weight.data_ptr(),
            ws.data_ptr(), nbytes, B, S, low, high, kl_coef, mean_of_means)
    return loss, weight


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, lp, rest):
        loss, weight = _policy_forward(lp, rest)
        ctx.save_for_backward(lp, *rest[2:6], weight)
        ctx.tail = *lp.shape, *rest[6:9]
        return loss

    @staticmethod
    @_first_order
    def backward(ctx, dloss):
        lp, old, ref, adv, mask, weight = ctx.saved_tensors
        grad, dloss = weight.new_empty(lp.shape), dloss.resolve_neg()
        _launch(weight, _lib.load().nq_policy_loss_bwd, "nq_policy_loss_bwd", *_saved_pitch(lp, old, ref, adv),
                adv.dim() - 1, *_saved_pitch(mask), weight.data_ptr(), dloss.data_ptr(), grad.data_ptr(), *ctx.tail)
        return grad, None


def policy_loss(logprobs: torch.Tensor, old_logprobs: torch.Tensor, advantages: torch.Tensor, *,
                ref_logprobs: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
                clip_low: float = 0.2, clip_high: Optional[float] = None, kl_coef: float = 0.0,
                reduction: str = "token") -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Clipped policy loss with a KL term over B sequences (at most 2^30) of tokens: (loss, kl, clipped).

    logprobs, old_logprobs, ref_logprobs: (B, S) log-probabilities of the sampled tokens
    under the policy, the policy that sampled them and a reference (needed with
    ``kl_coef``), fp32 (bf16 is converted).  advantages: (B,) per sequence or (B, S).  The
    mask (bool; other types count as != 0) keeps tokens; what a masked token holds has no
    effect.  Per kept token, with r = exp(logprobs - old_logprobs) and q = ref - logprobs:

      -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef (exp(q) - q - 1)

    and where A is 0 the KL term alone, however large r.  ``clip_high`` defaults to ``clip_low``.  ``reduction``: "token", the mean over all kept
    tokens, or "sequence", the mean over the B sequences of each one's mean (0 for one
    without kept tokens).  Returns the loss, a scalar with a gradient for logprobs alone;
    and, without gradient, the kept tokens' mean of exp(q) - q - 1 (0 without a reference)
    and the share of them that the clip decides.
    """
    _check_devices(logprobs, old_logprobs, advantages, ref_logprobs, mask)
    if logprobs.dim() != 2 or logprobs.shape[0] == 0:
        raise ValueError(f"logprobs must be (B, S) with at least one sequence, got shape {tuple(logprobs.shape)}")
    if logprobs.shape[0] > _MOST_SEQUENCES:
        raise ValueError(f"at most 2^30 sequences in one call, got {logprobs.shape[0]}")
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
        if adv.dtype != torch.float32 or adv.shape[0] != shape[0]:
            adv = _token_rows(adv, "advantages", shape[:1])[:, 0]
    else:
        adv = _token_rows(adv, "advantages", shape)
    lp = _token_rows(logprobs, "logprobs", shape)
    stats = lp.new_empty(()), lp.new_empty(())
    rest = (*stats, _token_rows(_detached(old_logprobs), "old_logprobs", shape),
            _token_rows(_detached(ref_logprobs), "ref_logprobs", shape), adv, _mask_rows(mask, "mask", shape),
            float(clip_low), float(clip_high), float(kl_coef), int(reduction == "sequence"))
    if _takes_gradient(lp):
        return (_PolicyLoss.apply(lp, rest), *stats)
    return (_policy_forward(lp, rest)[0], *stats)
