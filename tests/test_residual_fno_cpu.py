"""CPU: the residual FNO's construction, its host path and its refusals."""

from __future__ import annotations

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
