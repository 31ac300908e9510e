"""Optimizer operators on the device: the global gradient norm, clipping by it, and an Adam step
that applies the clipping factor while it reads the gradients.

The reference trains with ``torch.optim.Adam`` and does not clip (fno_ns/train_official.py:56-154);
these are what ``fno_train`` uses where a run asks for clipping or the fused step.  Gradients may be
float32, bfloat16, float16 or complex64 (a spectral weight's, taken as its real and imaginary
parts), in any mix and of any size.  Calls run on the current stream of the tensors' device,
synchronise nothing and can be captured in a CUDA graph; results are bitwise repeatable.  Tensors with a
forward-mode tangent are refused.  A failed check raises RuntimeError.
"""

from __future__ import annotations

import math

import torch

import _scx
from spectral_conv_ext import _check

_scx_torch = _scx.torch_binding()
_dense, _overlaps_itself = _scx_torch.dense, _scx_torch.overlaps_itself


def _number(value, name: str) -> float:
    value = float(value)
    _check(value >= 0.0, name, " must not be negative, got ", value)
    return value


def grad_norm(tensors) -> torch.Tensor:
    """The 2-norm over all elements of all ``tensors`` (an iterable of CUDA tensors, or one), as a
    0-d float32 tensor on their device.  The sum is held in 64 bits.  Differentiable, any number of
    times (the gradient of zeros is zero).  Without tensors: 0 on the CPU, as
    torch.nn.utils.get_total_norm gives."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not tensors:
        return torch.tensor(0.0)
    return _scx_torch.grad_norm(tensors)


def clip_grads_(grads, max_norm: float) -> torch.Tensor:
    """Multiplies every tensor of ``grads`` in place by min(1, max_norm / (norm + 1e-6)), norm
    their global 2-norm before clipping, which is returned (0-d float32 on their device, detached).
    A norm that is not finite propagates as in torch.nn.utils.clip_grad_norm_.  No two tensors may
    share memory."""
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    max_norm = _number(max_norm, "max_norm")
    if not grads:
        return torch.tensor(0.0)
    return _scx_torch.clip_grads(grads, max_norm)


def clip_grad_norm_(parameters, max_norm: float) -> torch.Tensor:
    """Clips the gradients of ``parameters`` by their global 2-norm, as
    torch.nn.utils.clip_grad_norm_ does; parameters without a gradient, and repeats of one, are
    passed over.  Returns the norm before clipping."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else parameters
    return clip_grads_([p.grad for p in dict.fromkeys(parameters) if p.grad is not None], max_norm)


def adam_step_(params, grads, exp_avgs, exp_avg_sqs, steps, *, lr, betas=(0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 0.0, decoupled: bool = False, max_norm: float | None = None,
               total_norm: torch.Tensor | None = None) -> torch.Tensor | None:
    """One Adam step over lists of tensors, in place (the update of torch.optim.Adam, or of AdamW
    with ``decoupled``).

    params       float32, bfloat16, float16 or complex64 CUDA tensors, dense, none sharing memory
    grads        like params (type and shape), left as they are; none shares memory with what is written
    exp_avgs, exp_avg_sqs   the moments: float32 (complex64 for complex params), whatever the
                 params' type, of the params' shape and strides
    steps        0-d float32 CUDA tensors, one per parameter, counted up by the call (so a replayed
                 CUDA graph advances)
    lr           a number, or a 0-d float32 CUDA tensor that the kernels read
    max_norm     clip: the gradients enter multiplied by min(1, max_norm / (norm + 1e-6)), norm
                 their global 2-norm, which the call returns; with ``total_norm`` (0-d float32), by
                 that norm instead (several groups, several ranks)
    """
    params, grads, exp_avgs, exp_avg_sqs, steps = (list(v) for v in (params, grads, exp_avgs, exp_avg_sqs, steps))
    n = len(params)
    _check(len(grads) == n and len(exp_avgs) == n and len(exp_avg_sqs) == n and len(steps) == n,
           "params, grads, exp_avgs, exp_avg_sqs and steps must have the same length")
    clip = max_norm is not None
    _check(clip or total_norm is None, "total_norm needs max_norm")
    max_norm = _number(max_norm, "max_norm") if clip else 0.0
    beta1, beta2 = (float(b) for b in betas)
    _check(0.0 <= beta1 < 1.0 and 0.0 <= beta2 < 1.0, "betas must be in [0, 1), got ", betas)
    eps, weight_decay = _number(eps, "eps"), _number(weight_decay, "weight_decay")
    if n == 0:
        return total_norm if total_norm is not None else (torch.tensor(0.0) if clip else None)
    on_device = isinstance(lr, torch.Tensor) and lr.is_cuda
    rate = 0.0 if on_device else float(lr)
    _check(math.isfinite(rate) and rate >= 0.0, "lr must be finite and not negative, got ", lr)
    return _scx_torch.adam_step(params, grads, exp_avgs, exp_avg_sqs, steps, rate, lr if on_device else None, beta1,
                                beta2, eps, weight_decay, bool(decoupled), max_norm if clip else None, total_norm)


class FusedAdam(torch.optim.Optimizer):
    """Adam (AdamW with ``decoupled_weight_decay``) on ``adam_step_``: one call per parameter
    group, with ``max_norm`` clipping the gradients by the global norm over all groups on their
    way into the update (``p.grad`` is not changed).  ``last_norm`` is that norm, a 0-d tensor on
    the device, after a step (without any gradient 0 on the CPU, as ``clip_grad_norm_`` gives).

    State and options carry torch.optim.Adam's names, so state dicts go both ways (``step`` on the
    device, as torch's ``fused`` and ``capturable`` forms keep it; moments are float32 for bfloat16
    and float16 parameters, and stay so through load_state_dict).  ``lr`` may be a 0-d float32 CUDA
    tensor, which a captured step reads at each replay.  A parameter's first step, which makes its
    state, is refused in a capture."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.0, *,
                 decoupled_weight_decay: bool = False, max_norm: float | None = None):
        self.max_norm = None if max_norm is None else _number(max_norm, "max_norm")
        self.last_norm = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                                      decoupled_weight_decay=decoupled_weight_decay))

    def __getstate__(self):
        return {**super().__getstate__(), "max_norm": self.max_norm, "last_norm": self.last_norm}

    def __setstate__(self, state):
        super().__setstate__(state)
        for group in self.param_groups:
            group.setdefault("decoupled_weight_decay", False)
            _check(not group.get("amsgrad") and not group.get("maximize"),
                   "FusedAdam has no amsgrad or maximize form")

    @staticmethod
    def _moment(p: torch.Tensor, value: torch.Tensor | None = None) -> torch.Tensor:
        kind = torch.complex64 if p.is_complex() else torch.float32
        new = torch.zeros_like(p, dtype=kind, memory_format=torch.preserve_format, requires_grad=False)
        return new if value is None else new.copy_(value)

    def load_state_dict(self, state_dict) -> None:
        # the base class casts moments to their parameter's type: they are taken over from the source, which is
        # what the caller's hooks have made of it, before the caller's own hooks on the result
        source = []
        hooks = [self.register_load_state_dict_pre_hook(lambda _, given: source.append(given)),
                 self.register_load_state_dict_post_hook(lambda _: self._keep_moments(source[-1]), prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    @torch.no_grad()
    def _keep_moments(self, state_dict) -> None:
        ours = [p for g in self.param_groups for p in g["params"]]
        theirs = [i for g in state_dict["param_groups"] for i in g["params"]]
        for p, i in zip(ours, theirs):
            saved = state_dict["state"].get(i)
            if saved:
                self.state[p].update(step=torch.as_tensor(saved["step"]).to(p.device, torch.float32, copy=True),
                                     exp_avg=self._moment(p, saved["exp_avg"]),
                                     exp_avg_sq=self._moment(p, saved["exp_avg_sq"]))

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        work = []
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None]
            for p in params:
                state = self.state[p]
                if not state:
                    _check(not (p.is_cuda and torch.cuda.is_current_stream_capturing()),
                           "a parameter's first step has to run before it is captured: its zero moments and count "
                           "would be made again at every replay")
                    state["step"] = torch.zeros((), dtype=torch.float32, device=p.device)
                    state["exp_avg"] = self._moment(p)
                    state["exp_avg_sq"] = self._moment(p)
            if params:
                work.append((group, params))
        total = None
        if not work:
            self.last_norm = None if self.max_norm is None else torch.tensor(0.0)
        if self.max_norm is not None and len(work) > 1:
            total = grad_norm([p.grad for _, params in work for p in params])
        for group, params in work:
            states = [self.state[p] for p in params]
            self.last_norm = adam_step_(
                params, [p.grad for p in params], [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states],
                [s["step"] for s in states], lr=group["lr"], betas=group["betas"], eps=group["eps"],
                weight_decay=group["weight_decay"], decoupled=group["decoupled_weight_decay"], max_norm=self.max_norm,
                total_norm=total)
        return loss
