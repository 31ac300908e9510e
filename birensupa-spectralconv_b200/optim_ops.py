"""Optimizer operators on the device: the global gradient norm, clipping by it, and an Adam step
that applies the clipping factor while it reads the gradients.

The reference trains with ``torch.optim.Adam`` and does not clip (fno_ns/train_official.py:56-154);
these are what ``fno_train`` uses where a run asks for clipping or the fused step.  Gradients may be
float32, bfloat16, float16 or complex64 (a spectral weight's, taken as its real and imaginary
parts), in any mix and of any size.  Calls run on the current stream of the tensors' device,
synchronise nothing and can be captured in a CUDA graph; results are bitwise repeatable.  A failed
check raises RuntimeError.
"""

from __future__ import annotations

import math
from array import array
from itertools import chain
from operator import attrgetter

import torch

import _scx
from spectral_conv_ext import _check

# element type codes of include/scx.h, and how many such elements one tensor element is
_CODES = {torch.float32: (0, 1), torch.bfloat16: (1, 1), torch.float16: (2, 1), torch.complex64: (0, 2)}


def _dense(t: torch.Tensor) -> bool:
    """Whether the elements of t fill one run of memory, in whatever order, each once."""
    if t.is_contiguous():
        return True
    expect = 1
    for stride, size in sorted((st, sz) for sz, st in zip(t.shape, t.stride()) if sz != 1):
        if stride != expect:
            return False
        expect *= size
    return True


def _overlaps_itself(t: torch.Tensor) -> bool:
    reach = 0
    for stride, size in sorted((st, sz) for sz, st in zip(t.shape, t.stride()) if sz > 1):
        if stride <= reach:
            return True
        reach += stride * (size - 1)
    return False


_dtype, _shape, _layout = attrgetter("dtype"), attrgetter("shape"), attrgetter("layout")
_device_index, _is_contiguous = torch.Tensor.get_device, torch.Tensor.is_contiguous


def _check_tensors(tensors: list, name: str) -> torch.device:
    """One CUDA device, strided layout, known element types."""
    index = tensors[0].get_device()
    if index < 0 or set(map(_device_index, tensors)) != {index} or not _CODES.keys() >= set(map(_dtype, tensors)):
        device = tensors[0].device
        for t in tensors:
            _check(t.device.type == "cuda", name, " must be CUDA tensors")
            _check(t.dtype in _CODES, name, " must be float32, bfloat16, float16 or complex64, got ", t.dtype)
            _check(t.device == device, name, " must be on one device")
    _check(all([layout is torch.strided for layout in map(_layout, tensors)]), name, " must not be sparse")
    return torch.device("cuda", index)


def _pointers(tensors) -> array:
    return array("Q", map(torch.Tensor.data_ptr, tensors))


def _described(tensors) -> tuple[array, array]:
    """(element counts, element types) of a list for the C calls."""
    kinds = [_CODES[d] for d in map(_dtype, tensors)]
    return (array("q", [n * k[1] for n, k in zip(map(torch.Tensor.numel, tensors), kinds)]),
            array("i", [k[0] for k in kinds]))


def _address(values: array) -> int:
    return values.buffer_info()[0]


def _workspace(nbytes: int, device: torch.device) -> torch.Tensor:
    # a block of its own per call: calls on other streams and captured graphs share nothing
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def _changed(*lists) -> None:
    """Tells autograd (and whoever caches by version) that the kernels wrote these tensors."""
    torch.autograd.graph.increment_version(chain(*lists))


def _number(value, name: str) -> float:
    value = float(value)
    _check(value >= 0.0, name, " must not be negative, got ", value)
    return value


def grad_norm(tensors) -> torch.Tensor:
    """The 2-norm over all elements of all ``tensors`` (an iterable of CUDA tensors, or one), as a
    0-d float32 tensor on their device.  The sum is held in 64 bits.  Without tensors: 0 on the
    CPU, as torch.nn.utils.get_total_norm gives."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not tensors:
        return torch.tensor(0.0)
    device = _check_tensors(tensors, "tensors")
    if not all(map(_is_contiguous, tensors)):
        tensors = [t if _dense(t) else t.contiguous() for t in tensors]
    pointers = _pointers(tensors)
    counts, kinds = _described(tensors)
    n = len(tensors)
    norm = torch.empty((), dtype=torch.float32, device=device)
    with _scx.device_guard(device):
        ws = _workspace(_scx.lib.scx_grad_norm_workspace_size(n), device)
        _scx.check(_scx.lib.scx_grad_norm(n, _address(pointers), _address(counts), _address(kinds), norm.data_ptr(),
                                          ws.data_ptr(), ws.numel(), _scx.stream_of(device)), "scx_grad_norm")
    return norm


@torch.no_grad()
def clip_grads_(grads, max_norm: float) -> torch.Tensor:
    """Multiplies every tensor of ``grads`` in place by min(1, max_norm / (norm + 1e-6)), norm
    their global 2-norm before clipping, which is returned (0-d float32 on their device).  A norm
    that is not finite propagates as in torch.nn.utils.clip_grad_norm_.  No two tensors may share
    memory."""
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    max_norm = _number(max_norm, "max_norm")
    if not grads:
        return torch.tensor(0.0)
    device = _check_tensors(grads, "grads")
    flat = grads
    if not all(map(_is_contiguous, grads)):
        _check(not any(_overlaps_itself(g) for g in grads), "grads must not be expanded tensors")
        flat = [g if _dense(g) else g.contiguous() for g in grads]
    pointers = _pointers(flat)
    counts, kinds = _described(flat)
    n = len(flat)
    norm = torch.empty((), dtype=torch.float32, device=device)
    with _scx.device_guard(device):
        ws = _workspace(_scx.lib.scx_grad_norm_workspace_size(n), device)
        _scx.check(_scx.lib.scx_grad_clip(n, _address(pointers), _address(counts), _address(kinds), max_norm,
                                          norm.data_ptr(), ws.data_ptr(), ws.numel(), _scx.stream_of(device)),
                   "scx_grad_clip")
    if flat is not grads:
        for g, f in zip(grads, flat):
            if f is not g:
                g.copy_(f)
    _changed(grads)
    return norm


def clip_grad_norm_(parameters, max_norm: float) -> torch.Tensor:
    """Clips the gradients of ``parameters`` by their global 2-norm, as
    torch.nn.utils.clip_grad_norm_ does; parameters without a gradient, and repeats of one, are
    passed over.  Returns the norm before clipping."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else parameters
    return clip_grads_([p.grad for p in dict.fromkeys(parameters) if p.grad is not None], max_norm)


def _same_layout(t: torch.Tensor, p: torch.Tensor) -> bool:
    return (t.is_contiguous() and p.is_contiguous()) or all(
        a == b for a, b, size in zip(t.stride(), p.stride(), p.shape) if size > 1)


_MOMENTS = {torch.float32: torch.float32, torch.bfloat16: torch.float32, torch.float16: torch.float32,
            torch.complex64: torch.complex64}


def _checked_lists(params, grads, exp_avgs, exp_avg_sqs, steps, device: torch.device) -> list:
    """Checks an Adam step's lists; returns the gradients, those of another layout than their
    parameter's (or lazily conjugated or negated) copied to it."""
    kinds, shapes = list(map(_dtype, params)), list(map(_shape, params))
    moments = [_MOMENTS[k] for k in kinds]
    _check(list(map(_dtype, grads)) == kinds and list(map(_shape, grads)) == shapes
           and all([layout is torch.strided for layout in map(_layout, grads)]),
           "a gradient must have its parameter's type and shape")
    _check(list(map(_dtype, exp_avgs)) == moments and list(map(_dtype, exp_avg_sqs)) == moments
           and list(map(_shape, exp_avgs)) == shapes and list(map(_shape, exp_avg_sqs)) == shapes,
           "moments must be float32 (complex64 for a complex parameter), of their parameter's shape")
    _check(set(map(_dtype, steps)) == {torch.float32} and set(map(torch.Tensor.numel, steps)) == {1},
           "steps must be single float32 values")
    _check(set(map(_device_index, chain(grads, exp_avgs, exp_avg_sqs, steps))) == {device.index},
           "gradients, moments and steps must be on the params' device")
    if torch.complex64 in kinds:
        _check(not any(map(torch.Tensor.is_conj, chain(params, exp_avgs, exp_avg_sqs))),
               "params and moments must not be conjugate views")
    _check(not any(map(torch.Tensor.is_neg, chain(params, exp_avgs, exp_avg_sqs))),
           "params and moments must not be negated views")
    copied = [g.is_conj() or g.is_neg() for g in grads]
    if not all(map(_is_contiguous, chain(params, grads, exp_avgs, exp_avg_sqs))):
        for p, m, v in zip(params, exp_avgs, exp_avg_sqs):
            _check(_dense(p) and _same_layout(m, p) and _same_layout(v, p),
                   "params must be dense, and moments of their params' strides")
        copied = [c or not _same_layout(g, p) for c, g, p in zip(copied, grads, params)]
    if any(copied):
        grads = [torch.empty_like(p).copy_(g) if c else g for c, g, p in zip(copied, grads, params)]
    return grads


@torch.no_grad()
def adam_step_(params, grads, exp_avgs, exp_avg_sqs, steps, *, lr, betas=(0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 0.0, decoupled: bool = False, max_norm: float | None = None,
               total_norm: torch.Tensor | None = None) -> torch.Tensor | None:
    """One Adam step over lists of tensors, in place (the update of torch.optim.Adam, or of AdamW
    with ``decoupled``).

    params       float32, bfloat16, float16 or complex64 CUDA tensors, dense, none sharing memory
    grads        like params (type and shape), left as they are
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
    device = _check_tensors(params, "params")
    rate, rate_ptr = lr, None
    if isinstance(lr, torch.Tensor):
        if lr.is_cuda:
            _check(lr.dtype == torch.float32 and lr.numel() == 1 and lr.device == device,
                   "lr must be a number or one float32 value on the params' device")
            rate, rate_ptr = 0.0, lr.data_ptr()
        else:
            rate = float(lr)
    _check(math.isfinite(rate) and rate >= 0.0, "lr must be finite and not negative, got ", lr)
    if total_norm is not None:
        _check(total_norm.dtype == torch.float32 and total_norm.numel() == 1 and total_norm.device == device,
               "total_norm must be one float32 value on the params' device")
    grads = _checked_lists(params, grads, exp_avgs, exp_avg_sqs, steps, device)
    arrays = [_pointers(v) for v in (params, grads, exp_avgs, exp_avg_sqs, steps)]
    counts, kinds = _described(params)
    norm = torch.empty((), dtype=torch.float32, device=device) if clip and total_norm is None else None
    with _scx.device_guard(device):
        ws = _workspace(_scx.lib.scx_adam_workspace_size(n), device)
        _scx.check(_scx.lib.scx_adam_step(
            n, *[_address(a) for a in arrays], _address(counts), _address(kinds), rate, rate_ptr, beta1, beta2, eps,
            weight_decay, int(decoupled), max_norm, total_norm.data_ptr() if total_norm is not None else None,
            norm.data_ptr() if norm is not None else None, ws.data_ptr(), ws.numel(), _scx.stream_of(device)),
            "scx_adam_step")
    _changed(params, exp_avgs, exp_avg_sqs, steps)
    return norm if total_norm is None else total_norm


class FusedAdam(torch.optim.Optimizer):
    """Adam (AdamW with ``decoupled_weight_decay``) on ``adam_step_``: one call per parameter
    group, with ``max_norm`` clipping the gradients by the global norm over all groups on their
    way into the update (``p.grad`` is not changed).  ``last_norm`` is that norm, a 0-d tensor on
    the device, after a step.

    State and options carry torch.optim.Adam's names, so state dicts go both ways (``step`` on the
    device, as torch's ``fused`` and ``capturable`` forms keep it; moments are float32 for bfloat16
    and float16 parameters, and stay so through load_state_dict).  ``lr`` may be a 0-d float32 CUDA
    tensor, which a captured step reads at each replay."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.0, *,
                 decoupled_weight_decay: bool = False, max_norm: float | None = None):
        self.max_norm = None if max_norm is None else _number(max_norm, "max_norm")
        self.last_norm = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                                      decoupled_weight_decay=decoupled_weight_decay))

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

    @torch.no_grad()
    def load_state_dict(self, state_dict) -> None:
        super().load_state_dict(state_dict)
        # the base class casts moments to their parameter's type: take them over from the source
        ours = [p for g in self.param_groups for p in g["params"]]
        theirs = [i for g in state_dict["param_groups"] for i in g["params"]]
        for p, i in zip(ours, theirs):
            saved = state_dict["state"].get(i)
            if saved:
                self.state[p] = {"step": torch.as_tensor(saved["step"]).to(p.device, torch.float32, copy=True),
                                 "exp_avg": self._moment(p, saved["exp_avg"]),
                                 "exp_avg_sq": self._moment(p, saved["exp_avg_sq"])}

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
                    state["step"] = torch.zeros((), dtype=torch.float32, device=p.device)
                    state["exp_avg"] = self._moment(p)
                    state["exp_avg_sq"] = self._moment(p)
            if params:
                work.append((group, params))
        total = None
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
