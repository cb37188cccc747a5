"""AdamW for the training step: one launch per parameter type updates all tensors of a model (C ABI ``wkv6_adamw_step``).

``AdamW`` is a ``torch.optim.Optimizer``; ``adamw_step`` is the update behind it, on lists of tensors.  What they add to the
framework's optimizer: moments in fp32 whatever the parameters' type (a bf16 moment cannot follow beta2 = 0.999: a step changes it by
less than half its last bit), moments in 8 bits (2.03 bytes per value instead of 8), and stochastic rounding of bf16 parameters, which
keeps the updates that are smaller than half a parameter's last bit on average, without an fp32 copy of the parameters.
"""
from __future__ import annotations

import bisect
import math

import torch

from ._lib import AdamWConfig, AdamWTensor, check, lib
from .ops import _DT, _check_cuda, _check_tangents, _native, _ptr, _stream

BLOCK = 256      # values that share a scale where states have 8 bits
BETA1 = 0.94     # the largest with 8 bits: above 17/18, first moments without gradients would never fall


def _check_eps(eps):
    fp32 = torch.finfo(torch.float32)
    if not (eps == 0.0 or fp32.tiny <= eps <= fp32.max):
        raise ValueError(f"eps must be 0 or a normal fp32 number, not {eps}")


def _check_beta1(state_bits, beta1):
    if state_bits == 8 and beta1 > BETA1:
        raise ValueError(f"states in 8 bits take beta1 up to {BETA1}, not {beta1}: first moments are rounded to nearest and would not move")


def _spans(ts):
    return sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in ts if t.numel())


def _overlap(written, grads):
    """Whether a tensor shares memory with one that is written.  Gradients may share it among themselves."""
    spans = _spans(written)
    if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
        return True
    for a, b in _spans(grads):
        i = bisect.bisect_left(spans, (b, b))          # the first that begins at or behind its end
        if i and spans[i - 1][1] > a:
            return True
    return False


def _check_lists(params, grads, exp_avgs, exp_avg_sqs, m_scales, v_scales):
    if (m_scales is None) != (v_scales is None):
        raise ValueError("states in 8 bits need the scales of both moments")
    lists = [l for l in (params, grads, exp_avgs, exp_avg_sqs, m_scales, v_scales) if l is not None]
    if any(len(l) != len(params) for l in lists):
        raise ValueError("all lists must have one tensor per parameter")
    if not params:
        return
    state = torch.float32 if m_scales is None else torch.float8_e4m3fn
    dev = params[0].device
    for l in lists:
        _check_cuda(*l)
        _check_tangents(*l)
    for i, p in enumerate(params):
        if p.dtype not in (torch.bfloat16, torch.float32):
            raise TypeError(f"parameter {i} must be bf16 or fp32, not {p.dtype}")
        if grads[i].dtype != p.dtype:
            raise TypeError(f"gradient {i} must be {p.dtype} as its parameter, not {grads[i].dtype}")
        for t in (exp_avgs[i], exp_avg_sqs[i]):
            if t.dtype != state:
                raise TypeError(f"the moments of parameter {i} must be {state}, not {t.dtype}")
        for t in (grads[i], exp_avgs[i], exp_avg_sqs[i]):
            if t.numel() != p.numel():
                raise ValueError(f"parameter {i} has {p.numel()} values, its gradient or a moment {t.numel()}")
        if m_scales is not None:
            for t in (m_scales[i], v_scales[i]):
                if t.dtype != torch.float32 or t.numel() != -(-p.numel() // BLOCK):
                    raise ValueError(f"the scales of parameter {i} must be fp32, one per {BLOCK} values")
        for l in lists:
            if l[i].device != dev:
                raise ValueError("all tensors must be on one device")
            if l[i].layout != torch.strided or not l[i].is_contiguous():
                raise ValueError(f"tensor {i} of a list is not contiguous")
            if l[i].is_neg():
                raise ValueError(f"tensor {i} of a list is lazily negated: what is written in place has to be what its memory holds")
    if _overlap([t for l in lists if l is not grads for t in l], grads):
        raise ValueError("parameters, moments and scales must not share memory, nor with gradients")


def _device_value(t, dtype, name, dev):
    if t.dtype != dtype or t.numel() != 1 or t.device != dev:
        raise ValueError(f"{name} must be one {dtype} value on the parameters' device")
    _check_tangents(t)
    if t.is_neg():
        raise ValueError(f"{name} is lazily negated: it is read where it lies")
    return t.data_ptr()


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, *, exp_avg_scales=None, exp_avg_sq_scales=None, step, lr=1e-3,
               betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, seed: int = 0, stochastic_rounding: bool = True,
               grad_scale: torch.Tensor | None = None, first_index: int = 0) -> None:
    """One AdamW step over lists of tensors, in place: m <- beta1 m + (1 - beta1) g, v <- beta2 v + (1 - beta2) g^2,
    p <- p (1 - lr weight_decay) - lr / (1 - beta1^t) m / (sqrt(v / (1 - beta2^t)) + eps), all in fp32.

    ``params``: bf16 or fp32, contiguous, both types in one list if need be; ``grads`` of their types.
    ``exp_avgs``, ``exp_avg_sqs``: fp32; or, with ``exp_avg_scales`` and ``exp_avg_sq_scales`` (fp32, one per 256 values counted from the
    tensor's first), float8_e4m3fn codes: m = code * scale, sqrt(v) = code * scale.  New states are zeros in either form.  With 8 bits ``betas[0]`` is at most 0.94: m is rounded
    to nearest, and what changes it by less than half a code's step (3 to 6 %) is lost.
    ``step``: t of this step, counted from 1; an int, or one int64 value on the device (a captured step reads it at every replay, an
    int would stay what it was).  ``lr``: a float, or one fp32 value on the device.
    ``grad_scale``: one fp32 value on the device that multiplies the gradients (clipping, loss scaling).
    ``stochastic_rounding``: bf16 parameters are rounded up or down with the probabilities that keep their mean, else to nearest.  The
    random bits (also of 8-bit states) follow from ``seed`` and the step (the lowest 32 bits of either), and the tensor's and the value's
    positions: the tensor's is its place in the list plus ``first_index``."""
    params, grads, exp_avgs, exp_avg_sqs = list(params), list(grads), list(exp_avgs), list(exp_avg_sqs)
    m_scales = None if exp_avg_scales is None else list(exp_avg_scales)
    v_scales = None if exp_avg_sq_scales is None else list(exp_avg_sq_scales)
    if _native.adamw_step(params, grads, exp_avgs, exp_avg_sqs, m_scales, v_scales, step, lr, betas[0], betas[1], eps, weight_decay, seed,
                          bool(stochastic_rounding), grad_scale, first_index):
        return
    grads = [g.resolve_neg() for g in grads]
    _check_lists(params, grads, exp_avgs, exp_avg_sqs, m_scales, v_scales)
    if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
        raise ValueError("betas must lie in [0, 1)")
    _check_beta1(32 if m_scales is None else 8, betas[0])
    _check_eps(eps)
    if not math.isfinite(weight_decay):
        raise ValueError("weight_decay must be finite")
    if not params:
        return
    if not 0 <= first_index <= 2 ** 31 - len(params):
        raise ValueError("a tensor's place in the list plus first_index must lie in [0, 2^31)")
    dev = params[0].device
    c = AdamWConfig()
    c.state_bits, c.stochastic, c.seed = 32 if m_scales is None else 8, bool(stochastic_rounding), seed
    c.beta1, c.beta2, c.eps, c.weight_decay = *betas, eps, weight_decay
    if isinstance(step, torch.Tensor):
        c.step_device = _device_value(step, torch.int64, "step", dev)
    else:
        if _capturing(dev):
            raise ValueError("a captured step needs its number on the device: an int would be the same at every replay")
        if not 1 <= step < 2 ** 63:
            raise ValueError("steps are counted from 1, in 64 bits")
        c.step = step
    if isinstance(lr, torch.Tensor):
        c.lr_device = _device_value(lr, torch.float32, "lr", dev)
    else:
        if not math.isfinite(lr):
            raise ValueError("lr must be finite")
        c.lr = lr
    if grad_scale is not None:
        c.grad_scale = _device_value(grad_scale, torch.float32, "grad_scale", dev)
    none = [None] * len(params)
    with torch.cuda.device(dev), torch.no_grad():
        for dtype in (torch.bfloat16, torch.float32):
            which = [i for i, p in enumerate(params) if p.dtype == dtype]
            if not which:
                continue
            table = (AdamWTensor * len(which))()
            for e, i in zip(table, which):
                e.p, e.g, e.m, e.v = params[i].data_ptr(), grads[i].data_ptr(), exp_avgs[i].data_ptr(), exp_avg_sqs[i].data_ptr()
                if m_scales is not None:
                    e.m_scale, e.v_scale = m_scales[i].data_ptr(), v_scales[i].data_ptr()
                e.n, e.index = params[i].numel(), first_index + i
            c.dtype = _DT[dtype]
            check(lib.wkv6_adamw_step(c, len(which), table, _stream(dev)))
    for l in (params, exp_avgs, exp_avg_sqs, m_scales or (), v_scales or ()):
        for t in l:
            if not t.is_inference():
                torch.autograd.graph.increment_version(t)


def _capturing(dev):
    with torch.cuda.device(dev):
        return torch.cuda.is_current_stream_capturing()


class AdamW(torch.optim.Optimizer):
    """AdamW over bf16 and fp32 parameters on CUDA devices, each group's in one launch per type (see ``adamw_step``).

    ``state_bits``: 32 (fp32 moments) or 8 (e4m3 codes and a scale per 256 values; ``betas[0]`` up to 0.94).  ``stochastic_rounding``, ``seed``: how bf16
    parameters are rounded.  ``lr`` may be a tensor (one fp32 value on the parameters' device).
    ``grad_scale``: an attribute, None or one fp32 value on the device that multiplies the gradients of the next steps.
    ``capturable``: the step number is kept on the device (one per group), so that ``step`` can be captured into a CUDA graph; every
    parameter that gets gradients must then get them from its group's first step on.  A float ``lr`` stays in a captured step as it was.
    A group whose ``capturable`` is set or cleared later goes on from its step; that next step has to lie outside of a capture.
    ``state_dict`` holds the moments in their own types; ``load_state_dict`` keeps them (parameters do not lend them theirs)."""

    grad_scale = None       # of the class: copies and unpickled optimizers do not go through __init__

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, *, state_bits: int = 32,
                 stochastic_rounding: bool = True, seed: int = 0, capturable: bool = False):
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32")
        if not isinstance(lr, torch.Tensor) and not (math.isfinite(lr) and lr >= 0.0):
            raise ValueError("lr must be finite and not negative")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError("betas must lie in [0, 1)")
        _check_eps(eps)
        if not (math.isfinite(weight_decay) and weight_decay >= 0.0):
            raise ValueError("weight_decay must be finite and not negative")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      stochastic_rounding=stochastic_rounding, seed=seed, capturable=capturable, step=None))

    def add_param_group(self, param_group):
        settings = {**self.defaults, **param_group}
        _check_beta1(settings["state_bits"], settings["betas"][0])
        super().add_param_group(param_group)

    def _state_of(self, p, group):
        s = self.state[p]
        if not s:
            if group["capturable"] and group["step"] is not None:
                raise RuntimeError("a capturable group's parameters must have gradients from its first step on")
            if p.is_cuda and _capturing(p.device):
                raise RuntimeError("take a first step before the capture: new states would be zeroed at every replay")
            if group["state_bits"] == 32:
                s["exp_avg"], s["exp_avg_sq"] = (torch.zeros(p.shape, dtype=torch.float32, device=p.device) for _ in range(2))
            else:
                for key in ("exp_avg", "exp_avg_sq"):
                    s[key] = torch.zeros(p.shape, dtype=torch.float8_e4m3fn, device=p.device)
                    s[key + "_scale"] = torch.zeros(-(-p.numel() // BLOCK), dtype=torch.float32, device=p.device)
            s["step"] = 0
        return s

    @staticmethod
    def _leave_capturable(group, state):
        """A group that is capturable no longer goes on from its number on the device."""
        if _capturing(group["step"].device):
            raise RuntimeError("a group that is capturable no longer has to take its next step outside of the capture")
        at = int(group["step"])
        for p in group["params"]:
            if state.get(p):
                state[p]["step"] = at
        group["step"] = None

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        first = 0
        for group in self.param_groups:
            if group["step"] is not None and not group["capturable"]:
                self._leave_capturable(group, self.state)
            # parameters of one launch: on one device, and at one step (a parameter that had no gradient before is behind)
            batches = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("AdamW does not take sparse gradients")
                s = self._state_of(p, group)
                batches.setdefault((p.device, s["step"]), []).append((p, s))
            if group["capturable"] and batches:
                if len(batches) > 1:
                    raise RuntimeError("a capturable group's parameters must be on one device")
                if group["step"] is None:
                    dev, at = next(iter(batches))
                    if _capturing(dev):
                        raise RuntimeError("take a first step before the capture: a new step number would be set back at every replay")
                    group["step"] = torch.full((), at, dtype=torch.int64, device=dev)
                group["step"].add_(1)
            for (_, at), batch in batches.items():      # one batch where the number is on the device
                ps, ss = [p for p, _ in batch], [s for _, s in batch]
                scales = ([s[k + "_scale"] for s in ss] for k in ("exp_avg", "exp_avg_sq")) if group["state_bits"] == 8 else (None, None)
                m_scales, v_scales = scales
                try:
                    adamw_step(ps, [p.grad.contiguous() for p in ps], [s["exp_avg"] for s in ss], [s["exp_avg_sq"] for s in ss],
                               exp_avg_scales=m_scales, exp_avg_sq_scales=v_scales,
                               step=group["step"] if group["capturable"] else at + 1, lr=group["lr"], betas=group["betas"], eps=group["eps"],
                               weight_decay=group["weight_decay"], seed=group["seed"], stochastic_rounding=group["stochastic_rounding"],
                               grad_scale=self.grad_scale, first_index=first)
                except Exception:
                    if group["capturable"]:
                        group["step"].sub_(1)      # refused: not a step
                    raise
                if not group["capturable"]:
                    for s in ss:
                        s["step"] = at + 1
                first += len(ps)
        return loss

    def load_state_dict(self, state_dict):
        # between the hooks: behind those that make a state dict of another one, before those that look at what was loaded
        seen = []
        hooks = (self.register_load_state_dict_pre_hook(lambda _, d: seen.append(d)),
                 self.register_load_state_dict_post_hook(lambda _: self._own_types(seen[0]), prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    def _own_types(self, state_dict):
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        own = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(saved, own):
            for key, x in state_dict["state"].get(i, {}).items():
                self.state[p][key] = x.detach().to(p.device, copy=True) if isinstance(x, torch.Tensor) else x
        for group in self.param_groups:
            for key in ("step", "lr"):
                if isinstance(group[key], torch.Tensor) and group["params"]:
                    group[key] = group[key].to(group["params"][0].device, copy=True)
