"""Losses over a model's logits.

``lm_loss``: next-token cross-entropy for the training step, loss and logit gradient in one pass over the bf16 logits
(C ABI ``wkv6_softmax_xent_bf16``).  ``lm_loss(logits, targets)`` equals
``torch.nn.functional.cross_entropy(logits.float().view(-1, V), targets.view(-1))`` (mean over all tokens) and its
gradient when every target lies in [0, V); a row whose target lies outside that range contributes zero loss and zero
gradient and still counts in the mean's denominator (on both the fused path and the library path), without the fp32 copy of the logits, the stored log-probabilities and the separate backward pass.

The gradient is written over the logits inside the forward call: the logits tensor must not be used afterwards
(the output layer's own backward needs only its input, so a model may pass its logits straight in).

``token_log_probs``, ``policy_loss`` and ``preference_loss``: log-probabilities of given tokens and the losses of training from
sampled or compared answers.  They leave the logits alone, take bf16, fp16 and fp32 logits of any vocabulary, and compute in fp32.
Tokens that ``mask`` leaves out, and those whose target lies outside [0, V), do not count: their logits are not read, their
log-probability is 0 and their gradient zeros.  A row that counts and holds a NaN or +inf, or nothing but -inf, gives NaN.
Temperatures of at least 1e-30 and finite logits of any size are computed as written; forward-mode derivatives are refused.
Forward and backward can be captured into a CUDA graph; as with every backward pass, no eager graph of the same leaves may be alive then.
"""
from __future__ import annotations

import ctypes
import math

import torch

from ._lib import Policy, Preference, TokenLogits, check, lib
from .ops import _DT, _check_cuda, _check_tangents, _native, _ptr, _stream


class _LMLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets):
        V = logits.shape[-1]
        z = logits.detach().view(-1, V)
        rows = z.shape[0]
        assert targets.numel() == rows and targets.dtype == torch.int64
        tg = targets.reshape(-1).contiguous()
        loss_rows = torch.empty((rows,), dtype=torch.float32, device=z.device)
        with torch.cuda.device(z.device):
            check(lib.wkv6_softmax_xent_bf16(rows, V, _ptr(z), _ptr(tg), 1.0 / max(rows, 1), _ptr(loss_rows), _stream(z.device)))
        ctx.save_for_backward(z)          # now holds d(mean loss)/d(logits)
        ctx.shape = logits.shape
        return loss_rows.mean()

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        (g,) = ctx.saved_tensors
        scale = grad_out.resolve_neg().to(torch.float32)
        with torch.cuda.device(g.device):      # in place: the buffer is this function's own; nothing moves for a factor of 1
            check(lib.wkv6_scale_bf16(g.numel(), _ptr(g), _ptr(scale), _stream(g.device)))
        torch.autograd.graph.increment_version(g)      # a second backward would scale it again: autograd refuses that
        return g.view(ctx.shape), None


def lm_loss(logits: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
    """Mean cross-entropy of bf16 ``logits`` [..., V] against int64 ``targets`` [...]; overwrites ``logits``."""
    V = logits.shape[-1]
    if logits.dtype != torch.bfloat16 or V % 8 or V > 65536 or not logits.is_contiguous() or logits.is_neg():
        # same definition as the fused kernel: rows whose target lies outside [0, V) give zero loss and gradient,
        # and the mean runs over all rows
        z, t = logits.float().reshape(-1, V), targets.reshape(-1)
        valid = (t >= 0) & (t < V)
        per_row = torch.nn.functional.cross_entropy(z, t.clamp(0, V - 1), reduction="none") * valid
        return per_row.sum() / max(z.shape[0], 1)
    _check_cuda(logits, targets)
    return _LMLoss.apply(logits, targets.resolve_neg())


def _check_targets(logits, targets, mask, temperature):
    """What all operators on given tokens ask of their arguments."""
    _check_cuda(logits, targets, mask)
    if logits.dtype not in _DT:
        raise TypeError(f"logits must be bf16, fp16 or fp32, not {logits.dtype}")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError("logits must have a vocabulary axis: [..., V] with V >= 1")
    if targets.dtype != torch.int64:
        raise TypeError(f"targets must be int64, not {targets.dtype}")
    if targets.shape != logits.shape[:-1]:
        raise ValueError(f"targets {tuple(targets.shape)} do not fit logits {tuple(logits.shape)}")
    if mask is not None:
        if mask.dtype != torch.bool:
            raise TypeError(f"mask must be bool, not {mask.dtype}")
        if mask.shape != targets.shape:
            raise ValueError(f"mask {tuple(mask.shape)} does not fit targets {tuple(targets.shape)}")
    for t in (targets, mask):
        if t is not None and t.device != logits.device:
            raise ValueError("logits, targets and mask must be on one device")
    if not (temperature >= 1e-30 and math.isfinite(temperature)):
        raise ValueError("temperature must be at least 1e-30 and finite")
    if targets.numel() >= 2 ** 31 or logits.shape[-1] > 2 ** 30:
        raise ValueError("more than 2^31 - 1 tokens, or 2^30 entries of the vocabulary")


def _as_stored(*ts):
    """Tensors that are what their memory holds and no more: lazy negations are carried out, tangents refused."""
    _check_tangents(*ts)
    return tuple(None if t is None else t.resolve_neg() for t in ts)


def _per_token(t, name, targets, strided=False):
    """A constant that goes with every token, in fp32; dense, or (strided) with strides for the sequence and the token."""
    _check_cuda(t)
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} is a constant of the loss: pass it without requires_grad (detach it)")
    if not t.is_floating_point():
        raise TypeError(f"{name} must be floating point, not {t.dtype}")
    if t.shape != targets.shape:
        raise ValueError(f"{name} {tuple(t.shape)} does not fit targets {tuple(targets.shape)}")
    if t.device != targets.device:
        raise ValueError(f"{name} must be on the logits' device")
    t = _as_stored(t)[0].detach().to(torch.float32)
    return t if strided and t.dim() > 0 and (t.dim() <= 2 or t.is_contiguous()) else t.contiguous()


def _sequences(t):
    """[S, T] of a tensor whose axes are tokens: the last one runs along a sequence."""
    return t.shape[:-1].numel() if t.dim() > 1 else 1, t.shape[-1] if t.dim() > 0 else 1


def _rows(logits, targets, mask, temperature):
    """The C ABI's description of the logits' rows, and the tensors it points into."""
    S, T = _sequences(targets)
    V = logits.shape[-1]
    z = logits.detach().reshape(S, T, V)
    if (V > 1 and z.stride(2) != 1) or (T > 1 and z.stride(1) <= 0) or (S > 1 and z.stride(0) <= 0):
        z = z.contiguous()
    targets = targets.contiguous()
    mask = None if mask is None else mask.contiguous()
    p = TokenLogits()
    p.S, p.T, p.V, p.dtype, p.temperature = S, T, V, _DT[z.dtype], temperature
    p.row_stride = z.stride(1) if T > 1 else 0
    p.seq_stride = z.stride(0) if S > 1 else 0
    p.logits, p.targets, p.mask = z.data_ptr(), targets.data_ptr(), 0 if mask is None else mask.data_ptr()
    return p, (z, targets, mask)


def _logit_gradient(ctx, coefficient, per_sequence, factor=None, unless_one=False, out=None):
    logits, targets, mask, stat = ctx.saved_tensors[:4]
    p, held = _rows(logits, targets, mask, ctx.temperature)
    g = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device) if out is None else out
    with torch.cuda.device(g.device):
        check(lib.wkv6_token_log_probs_backward(p, _ptr(stat), _ptr(coefficient), per_sequence, _ptr(factor), unless_one, _ptr(g),
                                                _stream(g.device)))
    return g


def _log_probs(logits, targets, mask, temperature, want_stat):
    p, held = _rows(logits, targets, mask, temperature)
    lp = torch.empty(targets.shape, dtype=torch.float32, device=logits.device)
    stat = torch.empty((*targets.shape, 2), dtype=torch.float32, device=logits.device) if want_stat else None
    with torch.cuda.device(lp.device):
        check(lib.wkv6_token_log_probs(p, _ptr(lp), _ptr(stat), _stream(lp.device)))
    return lp, stat


class _TokenLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, mask, temperature):
        lp, stat = _log_probs(logits, targets, mask, temperature, True)
        ctx.save_for_backward(logits, targets, mask, stat)
        ctx.temperature = temperature
        return lp

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        return _logit_gradient(ctx, _as_stored(grad)[0].to(torch.float32).contiguous(), 0), None, None, None


def token_log_probs(logits: torch.Tensor, targets: torch.Tensor, mask: torch.Tensor | None = None, *,
                    temperature: float = 1.0) -> torch.Tensor:
    """log softmax(logits / temperature) at the given tokens: fp32 of the shape of ``targets`` (int64), for logits [*targets.shape, V].
    ``mask``: bool of the same shape, True where a token counts.  Differentiable with respect to the logits."""
    lp = _native.token_log_probs(logits, targets, mask, temperature)
    if lp is not None:
        return lp
    _check_targets(logits, targets, mask, temperature)
    logits, targets, mask = _as_stored(logits, targets, mask)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _TokenLogProbs.apply(logits, targets, mask, temperature)
    return _log_probs(logits, targets, mask, temperature, False)[0]


_REDUCTIONS = {"mean": 0, "sequence_mean": 1, "sum": 2}


def _policy(logits, targets, mask, temperature, consts, numbers, reduction, want_grad):
    p, held = _rows(logits, targets, mask, temperature)
    dev = logits.device
    c = Policy()
    c.advantages, c.old_log_probs, c.ref_log_probs = (0 if t is None else t.data_ptr() for t in consts)
    d = consts[0].dim()                       # more than two: dense
    c.advantage_row_stride = consts[0].stride(-1) if d in (1, 2) else 1
    c.advantage_seq_stride = consts[0].stride(0) if d == 2 else p.T
    c.clip_low, c.clip_high, c.kl_coef, c.scale = numbers
    c.reduction = reduction
    loss = torch.empty((), dtype=torch.float32, device=dev)
    lp = torch.empty(targets.shape, dtype=torch.float32, device=dev)
    coefficient = torch.empty_like(lp)
    stat = torch.empty((*targets.shape, 2), dtype=torch.float32, device=dev) if want_grad else None
    g = torch.empty(logits.shape, dtype=logits.dtype, device=dev) if want_grad else None
    nbytes = lib.wkv6_policy_loss_workspace_bytes(p.S, p.T, reduction)
    ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        check(lib.wkv6_policy_loss(p, c, _ptr(loss), _ptr(lp), _ptr(stat), _ptr(coefficient), _ptr(g), _ptr(ws), nbytes, _stream(dev)))
    return loss, lp, stat, coefficient, g


class _PolicyLoss(torch.autograd.Function):
    """The forward leaves the gradient for a loss that is the end of the graph.  Where another factor arrives, the backward runs again,
    or is captured into a CUDA graph that the forward is not part of, it is formed anew from the logits (the first one belongs to
    whoever received it, and a replay must not find it as the last one left it)."""

    @staticmethod
    def forward(ctx, logits, targets, mask, temperature, consts, numbers, reduction):
        loss, lp, stat, coefficient, ctx.g = _policy(logits, targets, mask, temperature, consts, numbers, reduction, True)
        ctx.save_for_backward(logits, targets, mask, stat, coefficient)
        ctx.temperature, ctx.capture = temperature, lib.wkv6_capture_id(_stream(lp.device))
        ctx.mark_non_differentiable(lp)
        ctx.set_materialize_grads(False)
        return loss, lp

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, _):
        if grad is None:
            return (None,) * 7
        g, ctx.g = ctx.g, None
        if g is not None and lib.wkv6_capture_id(_stream(g.device)) != ctx.capture:
            g = None
        g = _logit_gradient(ctx, ctx.saved_tensors[4], 0, _as_stored(grad)[0].to(torch.float32), g is not None, g)
        return g, None, None, None, None, None, None


def policy_loss(logits: torch.Tensor, targets: torch.Tensor, advantages: torch.Tensor, old_log_probs: torch.Tensor, *,
                ref_log_probs: torch.Tensor | None = None, mask: torch.Tensor | None = None, clip_low: float = 0.2,
                clip_high: float = 0.2, kl_coef: float = 0.0, temperature: float = 1.0, reduction: str = "mean",
                scale: float = 1.0):
    """Clipped policy loss of sampled tokens, and their log-probabilities: (loss, log_probs).

    With lp = ``token_log_probs(logits, targets, mask)``, ratio = exp(lp - old_log_probs) and d = ref_log_probs - lp, a token's loss is
    ``-min(ratio * A, clamp(ratio, 1 - clip_low, 1 + clip_high) * A) + kl_coef * (exp(d) - d - 1)``.
    ``advantages``, ``old_log_probs``, ``ref_log_probs`` (needed with a KL term only): floating point of the shape of ``targets``,
    [..., T]; they are constants.
    ``reduction``: "mean" over all tokens that count, "sequence_mean" (mean over each sequence's tokens, then over the sequences; one
    without a token adds 0), "sum".  Without any token the loss is 0.
    ``scale`` multiplies the loss and its gradient.  The logit gradient is computed along with the loss, in one pass, for a loss that
    is the end of the graph: a factor applied to the loss afterwards costs a second pass, one given here does not.
    ``log_probs`` carries no gradient."""
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {', '.join(_REDUCTIONS)}, not {reduction!r}")
    if not (0.0 <= clip_low <= 1.0 and clip_high >= 0.0):
        raise ValueError("clip_low must lie in [0, 1] and clip_high must not be negative")
    if not (kl_coef >= 0.0 and math.isfinite(kl_coef) and math.isfinite(scale)):
        raise ValueError("kl_coef must be finite and not negative, scale finite")
    if kl_coef > 0.0 and ref_log_probs is None:
        raise ValueError("a KL term needs ref_log_probs")
    out = _native.policy_loss(logits, targets, mask, advantages, old_log_probs, ref_log_probs, temperature, clip_low, clip_high, kl_coef,
                              scale, _REDUCTIONS[reduction])
    if out is not None:
        return out
    _check_targets(logits, targets, mask, temperature)
    logits, targets, mask = _as_stored(logits, targets, mask)
    consts = (_per_token(advantages, "advantages", targets, strided=True), _per_token(old_log_probs, "old_log_probs", targets),
              _per_token(ref_log_probs, "ref_log_probs", targets) if ref_log_probs is not None else None)
    args = (logits, targets, mask, temperature, consts, (clip_low, clip_high, kl_coef, scale), _REDUCTIONS[reduction])
    if torch.is_grad_enabled() and logits.requires_grad:
        return _PolicyLoss.apply(*args)
    return _policy(*args, False)[:2]


def _preference(logits, targets, mask, ref, numbers, average, want_grad):
    lp, stat = _log_probs(logits, targets, mask, 1.0, want_grad)
    p, held = _rows(logits, targets, mask, 1.0)
    dev = logits.device
    c = Preference()
    c.ref_log_probs = 0 if ref is None else ref.data_ptr()
    c.beta, c.label_smoothing, c.margin, c.scale = numbers
    c.average = average
    loss = torch.empty((), dtype=torch.float32, device=dev)
    seq, coefficient = (torch.empty((p.S,), dtype=torch.float32, device=dev) for _ in range(2))
    nbytes = lib.wkv6_preference_loss_workspace_bytes(p.S)
    ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        check(lib.wkv6_preference_loss(p, _ptr(lp), c, _ptr(loss), _ptr(seq), _ptr(coefficient), _ptr(ws), nbytes, _stream(dev)))
    return loss, seq, stat, coefficient


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, mask, ref, numbers, average):
        loss, seq, stat, coefficient = _preference(logits, targets, mask, ref, numbers, average, True)
        ctx.save_for_backward(logits, targets, mask, stat, coefficient)
        ctx.temperature = 1.0
        ctx.mark_non_differentiable(seq)
        ctx.set_materialize_grads(False)
        return loss, seq

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, _):
        if grad is None:
            return (None,) * 6
        return _logit_gradient(ctx, ctx.saved_tensors[4], 1, _as_stored(grad)[0].to(torch.float32)), None, None, None, None, None


def preference_loss(logits: torch.Tensor, targets: torch.Tensor, ref_log_probs: torch.Tensor | None = None,
                    mask: torch.Tensor | None = None, *, beta: float = 0.1, label_smoothing: float = 0.0, margin: float = 0.0,
                    average: bool = False, scale: float = 1.0):
    """Loss of paired log ratios, and the sequences' log-probabilities: (loss, sequence_log_probs).

    ``logits`` [2P, T, V], ``targets`` and ``mask`` [2P, T]: sequence i < P is preferred to sequence P + i.  With L the sum (``average``:
    the mean) of a sequence's ``token_log_probs`` and R = ``ref_log_probs`` [2P], the same of a reference model (None: zeros),
    D = beta * ((L_i - R_i) - (L_j - R_j)) - margin, and the loss is the mean over the pairs of
    ``-(1 - label_smoothing) * log sigmoid(D) - label_smoothing * log sigmoid(-D)``, times ``scale``.
    A sequence without a token that counts has L = 0; without a pair the loss is 0.
    ``sequence_log_probs`` [2P] carries no gradient (rewards: beta * (L - R))."""
    if targets.dim() != 2 or targets.shape[0] % 2:
        raise ValueError(f"targets must be [2P, T], the preferred sequences first, not {tuple(targets.shape)}")
    if not (math.isfinite(beta) and beta > 0.0 and math.isfinite(margin) and math.isfinite(scale)):
        raise ValueError("beta must be positive and finite, margin and scale finite")
    if not 0.0 <= label_smoothing < 1.0:
        raise ValueError("label_smoothing must lie in [0, 1)")
    out = _native.preference_loss(logits, targets, mask, ref_log_probs, beta, label_smoothing, margin, scale, bool(average))
    if out is not None:
        return out
    _check_targets(logits, targets, mask, 1.0)
    logits, targets, mask = _as_stored(logits, targets, mask)
    ref = None if ref_log_probs is None else _per_token(ref_log_probs, "ref_log_probs", targets[:, 0] if targets.shape[1] else targets.sum(1))
    args = (logits, targets, mask, ref, (beta, label_smoothing, margin, scale), bool(average))
    if torch.is_grad_enabled() and logits.requires_grad:
        return _PreferenceLoss.apply(*args)
    return _preference(*args, False)[:2]
