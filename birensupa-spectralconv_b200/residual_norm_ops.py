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

import math

import torch

import _scx
from spectral_conv_ext import _check

_scx_torch = _scx.torch_binding()
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_KINDS = {"rms": 0, "layer": 1}
_ACTIVATIONS = {"none": 0, "sigmoid": 1, "silu": 2}


def residual_norm(x: torch.Tensor, y: torch.Tensor | None = None, *, pre_weight: torch.Tensor | None = None,
                  pre_bias: torch.Tensor | None = None, post_weight: torch.Tensor | None = None,
                  post_bias: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                  gate_activation: str = "none", scale: torch.Tensor | float | None = None, kind: str = "rms",
                  eps: float = 1e-5, dim: int = 1, post_norm: bool = True, pre_norm: bool = True):
    """(r, n) of the formulas above; differentiable once in every tensor, in reverse mode (a tensor with a
    forward-mode tangent is refused).

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
    options = [batch, length, channels, last, _TYPES[dtype], _TYPES[wide or torch.float32], _KINDS[kind], mode,
               _ACTIVATIONS[gate_activation], bool(post_norm), bool(pre_norm)]
    return _scx_torch.residual_norm(options, eps, number, x, y, gate, *vectors)
