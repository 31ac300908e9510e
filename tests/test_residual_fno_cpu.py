"""CPU: the residual FNO's construction, its host path and its refusals."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest
import torch

import fno_model


@pytest.mark.parametrize("gate", ["none", "element", "sample"])
@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_host_path_and_gradients(gate, norm):
    torch.manual_seed(0)
    model = fno_model.ResidualFNO2d(modes1=3, modes2=3, width=6, n_layers=2, in_channels=2, gate=gate, norm=norm)
    x = torch.randn(2, 2, 8, 10)
    y = model(x, use_supa=False)
    assert y.shape == (2, 1, 8, 10) and bool(torch.isfinite(y).all())
    y.square().sum().backward()
    for name, p in model.named_parameters():
        assert p.grad is not None and bool(torch.isfinite(torch.view_as_real(p.grad) if p.is_complex() else p.grad).all()), name


def test_refusals():
    with pytest.raises(ValueError, match="gate"):
        fno_model.ResidualFNO2d(gate="channel")
    with pytest.raises(ValueError, match="norm"):
        fno_model.ResidualFNO2d(norm="batch")
    with pytest.raises(ValueError, match="layer"):
        fno_model.ResidualFNO2d(n_layers=0)
    model = fno_model.ResidualFNO2d(modes1=3, modes2=3, width=6, n_layers=1, in_channels=2)
    with pytest.raises(ValueError, match="x must be"):
        model(torch.zeros(2, 3, 8, 8), use_supa=False)
    with pytest.raises(RuntimeError, match="CUDA"):
        model.forward_autograd(torch.zeros(2, 2, 8, 8))
    with pytest.raises(RuntimeError, match="CUDA"):
        model.forward_device(torch.zeros(2, 2, 8, 8))


def test_without_the_torch_binding():
    """libscx.so alone (make lib) serves everything but the operators of the binding, which say what is missing."""
    code = """
import sys
sys.modules["_scx_torch"] = None  # an import of it fails as where it was not built
import fno_model, fno_train, torch
x = torch.zeros(1, 2, 8, 8)
small = dict(modes1=3, modes2=3, width=6, n_layers=4, in_channels=2)
assert fno_model.FNO2d(**small)(x, use_supa=False).shape == (1, 1, 8, 8)
assert fno_model.ResidualFNO2d(**small)(x, use_supa=False).shape == (1, 1, 8, 8)
for name in ("optim_ops", "residual_norm_ops"):
    try:
        __import__(name)
    except ImportError as e:
        assert "_scx_torch.so" in str(e) and "make -C" in str(e), str(e)
    else:
        raise AssertionError(name)
"""
    path = str(Path(fno_model.__file__).resolve().parent)
    done = subprocess.run([sys.executable, "-c", code], cwd=path, capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
