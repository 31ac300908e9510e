"""The norms after and before a block, fused with the block's gate, residual scale and residual
addition, on the device and differentiable:

    r = x + scale * act(gate) * post(y)        the residual stream after the block whose output is y
    n = pre(r)                                 the input of the next block

``post`` and ``pre`` normalise each position over its channels (RMSNorm or LayerNorm).  The
reference's layers have no residual stream (fno_ns/model.py:87-134); ``fno_model.ResidualFNO2d``
is built on this operator.  Fields [B, C, ...] (``dim=1``, the layout of every map here) and tokens
[..., C] (``dim=-1``); float32, bfloat16 and float16.  Calls run on the current stream of x's device,
synchronise nothing and can be captured in a CUDA graph; results, gradients included, are bitwise
repeatable.  A failed check raises RuntimeError.
"""

from __future__ import annotations

import ctypes
import math

import torch

import _scx
from spectral_conv_ext import _check

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_KINDS = {"rms": 0, "layer": 1}
_ACTIVATIONS = {"none": 0, "sigmoid": 1, "silu": 2}


def _ptr(t: torch.Tensor | None) -> int | None:
    return t.data_ptr() if t is not None else None


def _tensors(x, y, gate, post_weight, post_bias, pre_weight, pre_bias, scale, r=None, n=None, stats=None):
    return _scx.ResidualNormTensors(x.data_ptr(), _ptr(y), _ptr(gate), _ptr(post_weight), _ptr(post_bias),
                                    _ptr(pre_weight), _ptr(pre_bias), _ptr(scale), _ptr(r), _ptr(n), _ptr(stats))


def _forward(config, x, y, gate, vectors, keep_stats: bool):
    """(r or None, n or None, stats or None) of contiguous inputs."""
    r = torch.empty_like(x) if y is not None else None
    n = torch.empty_like(x) if config.pre_norm else None
    stats = None
    if keep_stats:
        stats = torch.empty(4, config.batch * config.length, dtype=torch.float32, device=x.device)
    with _scx.device_guard(x.device):
        t = _tensors(x, y, gate, *vectors, r, n, stats)
        _scx.check(_scx.lib.scx_residual_norm_fwd(ctypes.addressof(config), ctypes.addressof(t),
                                                  _scx.stream_of(x.device)), "scx_residual_norm_fwd")
    return r, n, stats


class ResidualNormFunction(torch.autograd.Function):
    """Autograd form of ``residual_norm``.  Keeps the inputs and four statistics per position; r is
    recomputed in the backward."""

    @staticmethod
    def forward(ctx, config, x, y, gate, post_weight, post_bias, pre_weight, pre_bias, scale):
        r, n, stats = _forward(config, x, y, gate, (post_weight, post_bias, pre_weight, pre_bias, scale), True)
        ctx.config = config
        ctx.save_for_backward(x, y, gate, post_weight, post_bias, pre_weight, pre_bias, scale, stats)
        ctx.set_materialize_grads(False)
        # without y, r is x: returned from here so that its gradient joins n's before the rounding
        return (x if y is None else r), n

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dr, dn):
        x, y, gate, *vectors, stats = ctx.saved_tensors
        none = (None,) * 9
        if dr is None and dn is None:
            return none
        if x.numel() == 0:
            return (None, *[torch.zeros_like(t) if t is not None and need else None
                            for t, need in zip((x, y, gate, *vectors), ctx.needs_input_grad[1:])])
        dr = dr.contiguous() if dr is not None else None
        dn = dn.contiguous() if dn is not None else None
        grads = [torch.empty_like(t) if t is not None and need else None
                 for t, need in zip((x, y, gate, *vectors), ctx.needs_input_grad[1:])]
        config = ctx.config
        dx, dy, dgate, d_post_w, d_post_b, d_pre_w, d_pre_b, d_scale = grads
        with _scx.device_guard(x.device):
            nbytes = _scx.lib.scx_residual_norm_bwd_workspace_size(ctypes.addressof(config))
            ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
            t = _tensors(x, y, gate, *vectors, stats=stats)
            g = _scx.ResidualNormGrads(_ptr(dr), _ptr(dn), _ptr(dx), _ptr(dy), _ptr(dgate), _ptr(d_post_w),
                                       _ptr(d_post_b), _ptr(d_pre_w), _ptr(d_pre_b), _ptr(d_scale))
            _scx.check(_scx.lib.scx_residual_norm_bwd(ctypes.addressof(config), ctypes.addressof(t),
                                                      ctypes.addressof(g), ws.data_ptr(), nbytes,
                                                      _scx.stream_of(x.device)), "scx_residual_norm_bwd")
        return (None, *grads)


def residual_norm(x: torch.Tensor, y: torch.Tensor | None = None, *, pre_weight: torch.Tensor | None = None,
                  pre_bias: torch.Tensor | None = None, post_weight: torch.Tensor | None = None,
                  post_bias: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                  gate_activation: str = "none", scale: torch.Tensor | float | None = None, kind: str = "rms",
                  eps: float = 1e-5, dim: int = 1, post_norm: bool = True, pre_norm: bool = True):
    """(r, n) of the formulas above; differentiable in every tensor.

    x       the residual stream, a float32, bfloat16 or float16 CUDA tensor with its channels on
            ``dim`` (1, or -1 for the last)
    y       the block's output, like x; None: r is x and n = pre(x), the norm in front of a first block
    gate    None, a gate per element (x's shape), or one per sample and channel, [x.shape[0], C], which
            is broadcast over the positions; of x's type.  ``gate_activation``: none, sigmoid or silu
    scale   None, a number, or a vector [C]
    pre_weight, pre_bias, post_weight, post_bias, scale   [C], all float32 or all of x's type; None:
            ones and zeros
    kind    "rms": v / sqrt(mean(v^2) + eps); "layer": the same of v less its mean
    post_norm=False   adds y without the norm after the block; pre_norm=False   n is None

    Tensors that are not contiguous are copied first.  Statistics and sums are float32; r and n are
    rounded once, n from the unrounded r.
    """
    shape, dtype, device = x.shape, x.dtype, x.device
    rank = len(shape)
    # the messages are only put together on failure: a single-token call is as long as its checks
    if rank < 2:
        _check(False, "x must have at least 2 dimensions, got ", tuple(shape))
    if dim != 1 and dim != -1 and dim != rank - 1:
        _check(False, "dim must be 1 or -1, got ", dim)
    _check(x.is_cuda, "x must be a CUDA tensor")
    if dtype not in _TYPES:
        _check(False, "x must be float32, bfloat16 or float16, got ", dtype)
    if kind not in _KINDS:
        _check(False, "kind must be 'rms' or 'layer', got ", kind)
    if gate_activation not in _ACTIVATIONS:
        _check(False, "gate_activation must be 'none', 'sigmoid' or 'silu', got ", gate_activation)
    eps = float(eps)
    if not 0.0 <= eps < math.inf:
        _check(False, "eps must be finite and not negative, got ", eps)
    last = dim != 1 or rank == 2
    channels = shape[-1] if last else shape[1]
    if not 0 < channels <= 262144:
        _check(False, "x must have 1 to 262144 channels, got ", channels)
    if y is None:
        _check(gate is None and scale is None and post_weight is None and post_bias is None,
               "gate, scale, post_weight and post_bias need y")
        _check(pre_norm, "nothing to compute: no y and no pre_norm")
    elif y.shape != shape or y.dtype != dtype or y.device != device:
        _check(False, "y must have x's shape, type and device")
    _check(post_norm or (post_weight is None and post_bias is None), "post_weight and post_bias need post_norm")
    _check(pre_norm or (pre_weight is None and pre_bias is None), "pre_weight and pre_bias need pre_norm")
    batch = shape[0]
    length = x.numel() // (batch * channels) if batch else 0
    number = 1.0
    if scale is not None and not isinstance(scale, torch.Tensor):
        number, scale = float(scale), None
        if not math.isfinite(number):
            _check(False, "scale must be finite, got ", number)
    mode = 0
    if gate is not None:
        _check(gate.dtype == dtype and gate.device == device, "gate must have x's type and device")
        mode = 2 if gate.shape == shape else 1
        if mode == 1 and gate.shape != (batch, channels):
            _check(False, "gate must have the shape of x or ", (batch, channels), ", got ", tuple(gate.shape))
    wide = None
    vectors = (post_weight, post_bias, pre_weight, pre_bias, scale)
    for v in vectors:
        if v is not None:
            if v.shape != (channels,) or v.device != device:
                _check(False, "weights, biases and scale must be [", channels, "] on x's device")
            if v.dtype is not wide:
                _check(wide is None and (v.dtype is torch.float32 or v.dtype is dtype),
                       "weights, biases and scale must all be float32 or all of x's type")
                wide = v.dtype
    config = _scx.ResidualNormConfig(batch, length, channels, last, _TYPES[dtype],
                                     _TYPES[wide or torch.float32], _KINDS[kind], mode,
                                     _ACTIVATIONS[gate_activation], bool(post_norm), bool(pre_norm), eps, number)
    wanted = torch.is_grad_enabled() and any([t is not None and t.requires_grad for t in (x, y, gate, *vectors)])
    args = [t if t is None or t.is_contiguous() else t.contiguous() for t in (x, y, gate, *vectors)]
    if wanted:
        return ResidualNormFunction.apply(config, *args)
    r, n, _ = _forward(config, args[0], args[1], args[2], args[3:], False)
    return (x if y is None else r), n
