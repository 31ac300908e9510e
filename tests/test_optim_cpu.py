"""CPU: refusals of the gradient norm, clipping and Adam entry points, at the C ABI and in the
Python layer, and the host-side logic that needs no device."""

from __future__ import annotations

import copy
import ctypes
import pickle

import pytest
import torch

import _scx
import optim_ops

INVALID = 1  # cudaErrorInvalidValue


def _ptrs(*values):
    return (ctypes.c_void_p * len(values))(*values)


def _counts(*values):
    return (ctypes.c_longlong * len(values))(*values)


def _types(*values):
    return (ctypes.c_int * len(values))(*values)


WS = ctypes.c_void_p(4096)
NORM = ctypes.c_void_p(256)


def _norm(n=1, ptrs=_ptrs(512), counts=_counts(8), types=_types(0), norm=NORM, ws=WS, size=1 << 20):
    return _scx.lib.scx_grad_norm(n, ptrs, counts, types, norm, ws, size, None)


def _clip(n=1, ptrs=_ptrs(512), counts=_counts(8), types=_types(0), max_norm=1.0, norm=NORM, ws=WS, size=1 << 20):
    return _scx.lib.scx_grad_clip(n, ptrs, counts, types, max_norm, norm, ws, size, None)


@pytest.mark.parametrize("bad", [
    dict(n=-1), dict(ptrs=None), dict(counts=None), dict(types=None), dict(norm=None), dict(ws=None),
    dict(ws=ctypes.c_void_p(4097)), dict(norm=ctypes.c_void_p(258)), dict(size=64), dict(counts=_counts(-1)),
    dict(types=_types(3)), dict(types=_types(-1)), dict(ptrs=_ptrs(514)), dict(ptrs=_ptrs(None)),
    dict(ptrs=_ptrs(513), types=_types(1)), dict(counts=_counts(1 << 41)),
])
def test_norm_and_clip_refuse(bad):
    assert _norm(**bad) == INVALID
    assert _clip(**bad) == INVALID


@pytest.mark.parametrize("max_norm", [-1.0, float("nan")])
def test_clip_refuses_the_limit(max_norm):
    assert _clip(max_norm=max_norm) == INVALID


def test_clip_refuses_shared_memory():
    assert _clip(n=2, ptrs=_ptrs(512, 512), counts=_counts(8, 8), types=_types(0, 0)) == INVALID
    assert _clip(n=2, ptrs=_ptrs(540, 512), counts=_counts(8, 8), types=_types(0, 0)) == INVALID


def _adam(n=1, p=_ptrs(1024), g=_ptrs(2048), m=_ptrs(4096), v=_ptrs(5120), t=_ptrs(6144), counts=_counts(8),
          types=_types(0), lr=1e-3, lr_device=None, b1=0.9, b2=0.999, eps=1e-8, wd=0.0, max_norm=1.0, given=None,
          norm=NORM, ws=WS, size=1 << 20):
    return _scx.lib.scx_adam_step(n, p, g, m, v, t, counts, types, lr, lr_device, b1, b2, eps, wd, 0, max_norm, given,
                                  norm, ws, size, None)


@pytest.mark.parametrize("bad", [
    dict(n=-1), dict(p=None), dict(g=None), dict(m=None), dict(v=None), dict(t=None), dict(t=_ptrs(None)),
    dict(t=_ptrs(6146)), dict(counts=None), dict(types=None), dict(types=_types(7)), dict(lr=float("nan")),
    dict(b1=1.0), dict(b2=-0.1), dict(b2=1.0), dict(eps=-1.0), dict(wd=float("inf")), dict(max_norm=-1.0),
    dict(given=ctypes.c_void_p(512)), dict(ws=None), dict(size=128), dict(p=_ptrs(1026)),
    dict(m=_ptrs(1024)), dict(v=_ptrs(1040)), dict(t=_ptrs(1028)), dict(norm=ctypes.c_void_p(257)),
])
def test_adam_refuses(bad):
    assert _adam(**bad) == INVALID


def test_workspace_sizes():
    assert _scx.lib.scx_grad_norm_workspace_size(-1) == 0 and _scx.lib.scx_adam_workspace_size(-1) == 0
    one = _scx.lib.scx_grad_norm_workspace_size(1)
    assert one > 0 and _scx.lib.scx_grad_norm_workspace_size(10_000) > one
    assert _scx.lib.scx_adam_workspace_size(100) >= one + 800


def test_python_refusals():
    t = torch.zeros(4)
    with pytest.raises(RuntimeError, match="CUDA"):
        optim_ops.grad_norm([t])
    with pytest.raises(RuntimeError, match="CUDA"):
        optim_ops.clip_grads_([t], 1.0)
    with pytest.raises(RuntimeError, match="max_norm"):
        optim_ops.clip_grads_([t], -1.0)
    with pytest.raises(RuntimeError, match="max_norm"):
        optim_ops.clip_grads_([t], float("nan"))
    with pytest.raises(RuntimeError, match="CUDA"):
        optim_ops.adam_step_([t], [t], [t], [t], [t], lr=1e-3)
    with pytest.raises(RuntimeError, match="same length"):
        optim_ops.adam_step_([t], [], [t], [t], [t], lr=1e-3)
    with pytest.raises(RuntimeError, match="betas"):
        optim_ops.adam_step_([t], [t], [t], [t], [t], lr=1e-3, betas=(1.0, 0.9))
    with pytest.raises(RuntimeError, match="total_norm"):
        optim_ops.adam_step_([t], [t], [t], [t], [t], lr=1e-3, total_norm=t)
    with pytest.raises(RuntimeError, match="max_norm"):
        optim_ops.FusedAdam([torch.nn.Parameter(t)], max_norm=-2.0)


def test_empty_lists():
    assert float(optim_ops.grad_norm([])) == 0.0
    assert float(optim_ops.clip_grads_([], 1.0)) == 0.0
    assert float(optim_ops.clip_grad_norm_([torch.nn.Parameter(torch.zeros(2))], 1.0)) == 0.0
    assert optim_ops.adam_step_([], [], [], [], [], lr=1e-3) is None


def test_dense_and_overlap():
    t = torch.zeros(4, 6, 5)
    assert optim_ops._dense(t) and optim_ops._dense(t.permute(2, 0, 1)) and optim_ops._dense(t[1:3])
    assert not optim_ops._dense(t[:, 1:3]) and not optim_ops._dense(t[..., ::2]) and not optim_ops._dense(t[:1, :1].expand(4, 6, 5))
    assert optim_ops._overlaps_itself(t[:1].expand(4, 6, 5)) and not optim_ops._overlaps_itself(t[:, 1:3])
    assert optim_ops._overlaps_itself(torch.zeros(16).as_strided((3, 4), (1, 2)))


def test_state_dict_of_torch_adam_loads_and_keeps_float32_moments():
    p = torch.nn.Parameter(torch.zeros(3, dtype=torch.bfloat16))
    ours = optim_ops.FusedAdam([p], lr=1e-3)
    m = torch.full((3,), 1.0 + 2.0**-20)
    state = {"state": {0: {"step": 7, "exp_avg": m, "exp_avg_sq": m * m}},
             "param_groups": [{"lr": 5e-4, "betas": (0.8, 0.9), "eps": 1e-7, "weight_decay": 0.1, "amsgrad": False,
                               "maximize": False, "params": [0]}]}
    ours.load_state_dict(state)
    got = ours.state[p]
    assert got["exp_avg"].dtype == torch.float32 and torch.equal(got["exp_avg"], m) and float(got["step"]) == 7.0
    assert ours.param_groups[0]["lr"] == 5e-4 and ours.param_groups[0]["decoupled_weight_decay"] is False
    back = torch.optim.Adam([torch.nn.Parameter(torch.zeros(3))], lr=1e-3)
    back.load_state_dict(ours.state_dict())
    assert float(back.state_dict()["state"][0]["step"]) == 7.0
    state["param_groups"][0]["amsgrad"] = True
    with pytest.raises(RuntimeError, match="amsgrad"):
        ours.load_state_dict(state)


def test_a_copied_or_pickled_optimizer_still_clips():
    ours = optim_ops.FusedAdam([torch.nn.Parameter(torch.zeros(3))], lr=1e-3, max_norm=0.5, decoupled_weight_decay=True)
    for other in (copy.deepcopy(ours), pickle.loads(pickle.dumps(ours))):
        assert other.max_norm == 0.5 and other.last_norm is None
        assert other.param_groups[0]["decoupled_weight_decay"] is True
        other.step()  # no gradients: nothing to do, and nothing missing


def test_a_step_without_gradients_leaves_no_old_norm():
    ours = optim_ops.FusedAdam([torch.nn.Parameter(torch.zeros(3))], lr=1e-3, max_norm=0.5)
    ours.last_norm = torch.tensor(7.0)
    ours.step()
    assert float(ours.last_norm) == 0.0


def test_a_step_on_the_host_is_refused():
    p = torch.nn.Parameter(torch.ones(2))
    p.grad = torch.ones(2)
    with pytest.raises(RuntimeError, match="params must be CUDA"):
        optim_ops.FusedAdam([p]).step()


def test_load_state_dict_hooks_see_and_change_what_is_loaded():
    p = torch.nn.Parameter(torch.zeros(3, dtype=torch.bfloat16))
    ours = optim_ops.FusedAdam([p], lr=1e-3)
    m = torch.full((3,), 1.0 + 2.0**-20)
    groups = [{"lr": 5e-4, "betas": (0.8, 0.9), "eps": 1e-7, "weight_decay": 0.1, "params": [0]}]
    state = {"state": {0: {"step": 7, "exp_avg": m, "exp_avg_sq": m * m, "note": 5}}, "param_groups": groups}
    other = {"state": {0: {"step": 9, "exp_avg": 2 * m, "exp_avg_sq": m, "note": 5}}, "param_groups": groups}
    seen = []
    before = ours.register_load_state_dict_pre_hook(lambda opt, given: other)
    after = ours.register_load_state_dict_post_hook(lambda opt: seen.append(opt.state[p]["exp_avg"].clone()))
    ours.load_state_dict(state)
    got = ours.state[p]
    assert torch.equal(got["exp_avg"], 2 * m) and torch.equal(got["exp_avg_sq"], m) and float(got["step"]) == 9.0
    assert got["note"] == 5 and got["exp_avg"].dtype == torch.float32
    assert len(seen) == 1 and torch.equal(seen[0], 2 * m)
    before.remove()
    after.remove()
    ours.load_state_dict(state)
    assert torch.equal(ours.state[p]["exp_avg"], m) and len(seen) == 1
    assert not ours._optimizer_load_state_dict_pre_hooks and not ours._optimizer_load_state_dict_post_hooks


@pytest.mark.parametrize("address", [1024, 1000, 1052, 4096, 4124, 5116, 6144, 6116])
def test_adam_refuses_gradients_in_what_it_writes(address):
    """32 bytes at `address`, against params at 1024, moments at 4096 and 5120 and the count at 6144."""
    assert _adam(g=_ptrs(address)) == INVALID
