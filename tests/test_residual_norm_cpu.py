"""CPU: refusals of the residual-norm entry points, at the C ABI and in the Python layer."""

from __future__ import annotations

import ctypes

import pytest
import torch

import _scx
import residual_norm_ops

INVALID = 1  # cudaErrorInvalidValue


def _config(**more):
    base = dict(batch=2, length=3, channels=8, channels_last=1, dtype=0, weight_dtype=0, kind=0, gate_mode=0, gate_act=0,
                post_norm=1, pre_norm=1, eps=1e-5, scale=1.0)
    return _scx.ResidualNormConfig(**{**base, **more})


def _tensors(**more):
    return _scx.ResidualNormTensors(**{**dict(x=256, y=512, r=1024, n=2048, stats=4096), **more})


def _fwd(config, tensors):
    return _scx.lib.scx_residual_norm_fwd(ctypes.byref(config), ctypes.byref(tensors), None)


@pytest.mark.parametrize("bad", [
    dict(batch=-1), dict(length=-1), dict(channels=0), dict(channels=(1 << 18) + 1), dict(batch=1 << 41), dict(length=1 << 41),
    dict(batch=1 << 30, length=1 << 30), dict(channels_last=2), dict(dtype=3), dict(weight_dtype=1), dict(kind=2),
    dict(gate_mode=3), dict(gate_act=-1), dict(eps=-1.0), dict(eps=float("nan")), dict(scale=float("inf")),
])
def test_configurations_refused(bad):
    assert _fwd(_config(**bad), _tensors()) == INVALID
    assert _scx.lib.scx_residual_norm_bwd_workspace_size(ctypes.byref(_config(**bad))) == 0


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(x=258), dict(y=513), dict(r=None), dict(n=None), dict(r=1026), dict(stats=4097),
    dict(pre_weight=257), dict(scale=1023),
])
def test_addresses_refused(bad):
    assert _fwd(_config(), _tensors(**bad)) == INVALID


def test_gate_address_needed():
    assert _fwd(_config(gate_mode=1), _tensors()) == INVALID


def test_null_structs_and_empty_calls():
    lib = _scx.lib
    assert lib.scx_residual_norm_fwd(None, ctypes.byref(_tensors()), None) == INVALID
    assert lib.scx_residual_norm_fwd(ctypes.byref(_config()), None, None) == INVALID
    assert _fwd(_config(batch=0), _tensors()) == 0
    assert lib.scx_residual_norm_bwd_workspace_size(None) == 0
    assert lib.scx_residual_norm_bwd_workspace_size(ctypes.byref(_config(length=0))) == 0


@pytest.mark.parametrize("bad", ["workspace", "size", "stats", "dx", "empty"])
def test_backward_refused(bad):
    config = _config(batch=0) if bad == "empty" else _config()
    t = _tensors(stats=None) if bad == "stats" else _tensors()
    g = _scx.ResidualNormGrads(dr=8192, dx=8193 if bad == "dx" else 16384)
    need = _scx.lib.scx_residual_norm_bwd_workspace_size(ctypes.byref(_config()))
    assert need > 0
    ws = ctypes.c_void_p(4097 if bad == "workspace" else 4096)
    size = need - 1 if bad == "size" else need
    assert _scx.lib.scx_residual_norm_bwd(ctypes.byref(config), ctypes.byref(t), ctypes.byref(g), ws, size, None) == INVALID


@pytest.mark.parametrize("config, y, grads", [
    (dict(), None, dict(dy=512)), (dict(), None, dict(d_scale=512)), (dict(), None, dict(d_post_weight=512)),
    (dict(), 512, dict(dgate=512)), (dict(post_norm=0), 512, dict(d_post_bias=512)),
    (dict(pre_norm=0), 512, dict(dn=512)), (dict(pre_norm=0), 512, dict(d_pre_weight=512)),
])
def test_gradients_of_what_is_not_there_are_refused(config, y, grads):
    c = _config(**config)
    need = _scx.lib.scx_residual_norm_bwd_workspace_size(ctypes.byref(c))
    g = _scx.ResidualNormGrads(dr=8192, dx=16384, **grads)
    assert _scx.lib.scx_residual_norm_bwd(ctypes.byref(c), ctypes.byref(_tensors(y=y)), ctypes.byref(g),
                                          ctypes.c_void_p(4096), need, None) == INVALID


def test_python_refusals():
    op = residual_norm_ops.residual_norm
    x = torch.zeros(2, 4, 3)
    for args, kwargs, text in [
        ((torch.zeros(4),), {}, "dimensions"), ((x,), dict(dim=0), "dim"), ((x,), {}, "CUDA"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            op(*args, **kwargs)


def test_the_binding_formats_its_messages():
    """Numbers in a message go through the C++ runtime's streams, which have to be torch's."""
    import _scx_torch

    with pytest.raises(RuntimeError, match="11 options, got 2"):
        _scx_torch.residual_norm([1, 2], 0.0, 1.0, torch.zeros(2, 2), None, None, None, None, None, None, None)


class _Cuda(torch.Tensor):
    """A host tensor that claims to be on the device, for the checks behind that one."""

    is_cuda = property(lambda self: True)


@pytest.mark.parametrize("change, text", [
    (dict(kind="group"), "kind"), (dict(gate_activation="tanh"), "gate_activation"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(y=None, scale=2.0), "need y"), (dict(y=None, pre_norm=False), "nothing"),
    (dict(post_norm=False, post_weight=torch.ones(4)), "post_norm"), (dict(pre_norm=False, pre_bias=torch.ones(4)), "pre_norm"),
    (dict(scale=float("nan")), "scale"), (dict(y=torch.zeros(2, 4, 2)), "y must"), (dict(y=torch.zeros(2, 4, 3).half()), "y must"),
    (dict(gate=torch.zeros(2, 3)), "gate"), (dict(gate=torch.zeros(2, 4).half()), "gate"), (dict(gate=torch.zeros(2, 4, 1)), "gate"),
    (dict(pre_weight=torch.ones(3)), "weights"), (dict(pre_weight=torch.ones(4).double()), "all"),
    (dict(x=torch.zeros(2, 4, 3).double()), "float32"), (dict(x=torch.zeros(2, 0, 3)), "channels"),
])
def test_python_refusals_behind_the_device_check(change, text):
    args = dict(x=torch.zeros(2, 4, 3), y=torch.zeros(2, 4, 3))
    args.update(change)
    x = args.pop("x").as_subclass(_Cuda)
    with pytest.raises(RuntimeError, match=text):
        residual_norm_ops.residual_norm(x, args.pop("y"), **args)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("gate", ["none", "sample", "full"])
@pytest.mark.parametrize("act", ["none", "sigmoid", "silu"])
@pytest.mark.parametrize("post", [True, False])
def test_reference_formulas_against_autograd(kind, gate, act, post):
    """The hand-derived gradients that the GPU tests compare with, against torch autograd in 64 bits."""
    from residual_norm_reference import reference

    g = torch.Generator().manual_seed(0)
    rand = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    B, L, C, eps, number = 2, 5, 6, 1e-3, -0.7
    t = {"x": rand(B, L, C), "y": rand(B, L, C), "post_weight": rand(C), "post_bias": rand(C), "pre_weight": rand(C),
         "pre_bias": rand(C), "scale": rand(C)}
    if not post:
        t["post_weight"] = t["post_bias"] = None
    t["gate"] = {"none": None, "sample": rand(B, 1, C), "full": rand(B, L, C)}[gate]
    dr, dn = rand(B, L, C), rand(B, L, C)
    got = reference(t["x"], t["y"], t["gate"], t, kind=kind, act=act, eps=eps, number=number, post=post, dr=dr, dn=dn)
    leaves = {k: v.clone().requires_grad_(True) for k, v in t.items() if v is not None}

    def norm(v, w, b):
        if kind == "layer":
            v = v - v.mean(-1, keepdim=True)
        return v / (v.square().mean(-1, keepdim=True) + eps).sqrt() * w + b

    z = norm(leaves["y"], leaves["post_weight"], leaves["post_bias"]) if post else leaves["y"]
    a = 1.0
    if gate != "none":
        a = {"none": lambda v: v, "sigmoid": torch.sigmoid, "silu": torch.nn.functional.silu}[act](leaves["gate"])
    r = leaves["x"] + number * leaves["scale"] * a * z
    n = norm(r, leaves["pre_weight"], leaves["pre_bias"])
    grads = torch.autograd.grad((r, n), list(leaves.values()), (dr, dn))
    torch.testing.assert_close(got["r"][0], r.detach(), rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(got["n"][0], n.detach(), rtol=1e-12, atol=1e-12)
    for k, v in zip(leaves, grads):
        torch.testing.assert_close(got["d_" + k][0].reshape(v.shape), v, rtol=1e-10, atol=1e-10)
