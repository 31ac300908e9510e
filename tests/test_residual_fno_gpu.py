"""GPU: the operators together, as training runs them: the residual FNO on the device against its
host path (outputs and every gradient), optimizer steps with the clipping folded in against
torch.optim.Adam with torch's clipping, and the training command."""

from __future__ import annotations

import copy
import json

import pytest
import torch

import fno_model
import fno_train
import optim_ops
import scx_data

pytestmark = pytest.mark.gpu


def _real(t):
    return torch.view_as_real(t) if t.is_complex() else t


def _rel(ref, got):
    ref, got = _real(ref.detach()).double().cpu(), _real(got.detach()).double().cpu()
    return float((got - ref).norm() / ref.norm().clamp_min(1e-30))


def _model(gate="element", norm="rms", **more):
    torch.manual_seed(0)
    sizes = dict(modes1=12, modes2=12, width=32, n_layers=4, in_channels=10)
    return fno_model.ResidualFNO2d(**{**sizes, **more}, gate=gate, norm=norm)


def _loss(model, x, y, host=False):
    pred = model(x, use_supa=False) if host else model.forward_autograd(x)
    return torch.norm(pred - y) / torch.norm(y)


@pytest.mark.parametrize("gate, norm", [("none", "rms"), ("element", "rms"), ("sample", "layer"), ("element", "layer")])
def test_forward_and_gradients_match_the_host_path(gate, norm, cuda_device):
    """To the framework's own bound of 1e-4, each gradient relative to its own norm floored at 1e-3 of
    the whole gradient's."""
    ref = _model(gate, norm)
    dev = copy.deepcopy(ref).to(cuda_device)
    x, y = scx_data.fno_pairs_device(2, seed=5, device=cuda_device)
    assert _rel(ref(x.cpu(), use_supa=False), dev.forward_autograd(x)) <= 1e-4
    assert _rel(dev.forward_device(x), dev.forward_autograd(x)) <= 1e-5
    assert _rel(dev(x), dev.forward_device(x).cpu()) == 0.0
    _loss(ref, x.cpu(), y.cpu(), host=True).backward()
    _loss(dev, x, y).backward()
    total = sum(float(_real(p.grad).double().square().sum()) for p in ref.parameters()) ** 0.5
    for (name, p), q in zip(ref.named_parameters(), dev.parameters()):
        a, b = _real(p.grad).double(), _real(q.grad).double().cpu()
        assert float((a - b).norm()) <= 1e-4 * max(float(a.norm()), 1e-3 * total), name


@pytest.mark.parametrize("shape", [(1, 10, 48, 40), (3, 10, 33, 31)])
def test_other_grids_and_depths(shape, cuda_device):
    ref = _model(modes1=8, modes2=8, width=20, n_layers=6)
    dev = copy.deepcopy(ref).to(cuda_device)
    x = torch.randn(shape, generator=torch.Generator().manual_seed(3))
    assert _rel(ref(x, use_supa=False), dev.forward_device(x.to(cuda_device))) <= 1e-4


def test_fused_steps_follow_torch_adam_with_clipping(cuda_device):
    """Five steps on the same batches.  Both sides round in float32, differently; Adam divides by
    sqrt(v), so that a gradient's relative error e moves a parameter by up to lr e per step, and
    signs of near-zero gradients differ by up to 2 lr: the means are held to 1e-2 of a step."""
    start = _model().to(cuda_device)
    x, y = scx_data.fno_pairs_device(8, seed=6, device=cuda_device)
    lr, limit = 1e-3, 0.05
    ours, theirs = copy.deepcopy(start), copy.deepcopy(start)
    opt = optim_ops.FusedAdam(ours.parameters(), lr=lr, weight_decay=1e-4, max_norm=limit)
    ref = torch.optim.Adam(theirs.parameters(), lr=lr, weight_decay=1e-4)
    for k in range(5):
        batch = slice(k % 4 * 2, k % 4 * 2 + 2)
        for model, o in ((ours, opt), (theirs, ref)):
            o.zero_grad()
            _loss(model, x[batch], y[batch]).backward()
            if o is ref:
                norm = torch.nn.utils.clip_grad_norm_(theirs.parameters(), limit)
            o.step()
        assert abs(float(opt.last_norm) - float(norm)) <= 1e-3 * float(norm)
    for (name, p), q, s in zip(ours.named_parameters(), theirs.parameters(), start.parameters()):
        moved = float((_real(q) - _real(s)).detach().abs().mean())
        assert float((_real(p) - _real(q)).detach().abs().mean()) <= 1e-2 * 5 * lr, name
        assert moved > 0.0, name


def test_the_one_call_forward_sees_a_fused_step(cuda_device):
    """FNO2d.forward_device keeps device copies of its weights by their versions."""
    torch.manual_seed(0)
    model = fno_model.FNO2d().to(cuda_device)
    x, y = scx_data.fno_pairs_device(2, seed=7, device=cuda_device)
    before = model.forward_device(x)
    opt = optim_ops.FusedAdam(model.parameters(), lr=1e-2)
    _loss(model, x, y).backward()
    opt.step()
    after = model.forward_device(x)
    assert _rel(model.forward_autograd(x), after) <= 1e-4 and _rel(before, after) > 1e-3


@pytest.mark.parametrize("fused", [False, True])
def test_training_loop(fused, tmp_path, cuda_device):
    x, y = scx_data.fno_pairs_device(6, seed=8, device=cuda_device)
    model = _model(n_layers=3).to(cuda_device)
    out = fno_train.train(model, x[:4], y[:4], x[4:], y[4:], epochs=2, batch_size=2, max_grad_norm=0.5, fused_adam=fused,
                          checkpoint=str(tmp_path / "best.pt"), log=lambda *_: None)
    assert out["steps"] == 4 and all(e["grad_norm"] > 0.0 for e in out["history"])
    saved = torch.load(tmp_path / "best.pt")
    _model(n_layers=3).load_state_dict(saved["model"])


def test_training_command(capsys, cuda_device):
    fno_train.main(["--epochs", "1", "--n-train", "4", "--n-test", "2", "--batch-size", "2", "--modes", "8", "--layers", "5",
                    "--residual", "sample", "--norm", "layer", "--fused-adam", "--max-grad-norm", "1.0"])
    text = capsys.readouterr().out
    assert json.loads(text[text.index("{"):])["steps"] == 2


def test_a_captured_training_step(cuda_device):
    """Forward, backward and the fused step of the residual FNO in one CUDA graph: replays do what
    eager steps do, bit for bit."""
    x, y = scx_data.fno_pairs_device(2, seed=9, device=cuda_device)
    start = _model(n_layers=2).to(cuda_device)

    def make():
        model = copy.deepcopy(start)
        return model, optim_ops.FusedAdam(model.parameters(), lr=1e-3, max_norm=0.1)

    def step(model, opt):
        grads = torch.autograd.grad(_loss(model, x, y), list(model.parameters()))
        for p, g in zip(model.parameters(), grads):
            p.grad = g
        opt.step()

    eager, opt_e = make()
    for _ in range(4):
        step(eager, opt_e)
    model, opt = make()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(model, opt)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(model, opt)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(_real(p), _real(q)) for p, q in zip(model.parameters(), eager.parameters()))


@pytest.mark.parametrize("gate", ["element", "sample"])
def test_a_model_on_the_host_runs_on_the_device(gate, cuda_device):
    """model(x) as FNO2d's: weights held on the host are copied for the call and stay where they are."""
    model = _model(gate)
    there = copy.deepcopy(model).to(cuda_device)
    x = torch.randn(2, 10, 32, 32)
    want = there.forward_device(x.to(cuda_device)).cpu()
    for given in (x, x.to(cuda_device)):
        got = model(given)
        assert not got.is_cuda and torch.equal(got, want)
    assert all(not p.is_cuda for p in model.parameters())
    with torch.no_grad():
        model.first_weight.mul_(2.0)
        there.first_weight.mul_(2.0)
    assert torch.equal(model(x), there.forward_device(x.to(cuda_device)).cpu())
    model.prepare_supa_eval()
    assert all(p.is_cuda for p in model.parameters()) and torch.equal(model(x), there(x))
