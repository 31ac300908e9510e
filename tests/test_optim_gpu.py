"""GPU: the global gradient norm, clipping and the Adam step against the formulas in 64 bits.

Tolerances count roundings.  u(t) = finfo(t).eps / 2 is one rounding to type t.
* norm: 64-bit sums (their own error, n 2^-53, is below 2^-30 here), one rounding to float32:
  |got - N| <= 1.01 u(f32) N.
* clip: the factor is rounded once to float32, the product once to float32 and once to t:
  |got - g c| <= (2 u(f32) + u(t)) |g c| (1.01), plus half the smallest number of t.
* Adam, all in float32 until p is rounded to t.  g' takes 2 roundings for c g and one for the decay
  (on the sum of the magnitudes); m = b1 m + r1 g' takes at most 2 more on each term (constant,
  product or sum): |dm| <= 6 u (|b1 m| + r1 |g'|_mag).  v likewise, with g' squared: relative 10 u.
  The update k m / (sqrt(v) q + eps): relative u(f32) (k, product, root, q, fma, quotient and half of
  v's 10) <= 12 u, plus m's own error through it; p: one rounding to float32 of the decayed sum and
  one to t.
"""

from __future__ import annotations

import math
import random

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import optim_ops

pytestmark = pytest.mark.gpu

U32 = torch.finfo(torch.float32).eps / 2


def _u(t):
    return torch.finfo(torch.float32 if t == torch.complex64 else t).eps / 2


def _real(t):
    return torch.view_as_real(t.resolve_conj()) if t.is_complex() else t


def _f64(t):
    return _real(t.detach().clone()).double()


def _norm64(tensors):
    return math.sqrt(sum(float(_f64(t).square().sum()) for t in tensors))


def _randn(shape, dtype, dev, g, scale=1.0):
    if dtype == torch.complex64:
        return torch.view_as_complex(torch.randn(*shape, 2, device=dev, generator=g) * scale)
    return (torch.randn(*shape, device=dev, generator=g) * scale).to(dtype)


def _gen(dev, seed=0):
    return torch.Generator(device=dev).manual_seed(seed)


def _check_norm(got, tensors):
    n = _norm64(tensors)
    assert got.shape == () and got.dtype == torch.float32
    assert abs(float(got) - n) <= 1.01 * U32 * n, (float(got), n)


def _check_clipped(grads, before, max_norm):
    n = math.sqrt(sum(float(b.square().sum()) for b in before))
    c = min(1.0, max_norm / (n + 1e-6))
    for g, b in zip(grads, before):
        want = b * c
        t = torch.float32 if g.is_complex() else g.dtype
        bound = 1.01 * ((2 * U32 + _u(t)) * want.abs()) + torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2
        assert bool(((_f64(g) - want).abs() <= bound).all())


SIZES = [[1], [7], [1023, 1, 1025], [4096], [0, 5, 0], [262144 + 3, 17, 2, 99991], [1_500_001, 3, 800_000]]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.complex64])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_norm_and_clip(sizes, dtype, cuda_device):
    g = _gen(cuda_device, len(sizes))
    grads = [_randn((n,), dtype, cuda_device, g, 10.0 ** (-k)) for k, n in enumerate(sizes)]
    before = [_f64(t) for t in grads]
    total = optim_ops.grad_norm(grads)
    _check_norm(total, grads)
    for factor in (2.0, 0.37):  # a limit above the norm leaves every bit as it was
        kept = [t.clone() for t in grads]
        got = optim_ops.clip_grads_(grads, factor * float(total))
        assert torch.equal(got, total)
        if factor > 1.0:
            assert all(torch.equal(a, b) for a, b in zip(kept, grads))
        else:
            _check_clipped(grads, before, factor * float(total))


@pytest.mark.parametrize("count", [31, 32, 33, 448, 449, 1000])
def test_many_tensors_of_mixed_types(count, cuda_device):
    rng = random.Random(count)
    g = _gen(cuda_device, count)
    kinds = [torch.float32, torch.bfloat16, torch.float16, torch.complex64]
    grads = [_randn((rng.randint(0, 3000),), rng.choice(kinds), cuda_device, g, 10.0 ** rng.uniform(-3, 0))
             for _ in range(count)]
    before = [_f64(t) for t in grads]
    _check_norm(optim_ops.grad_norm(grads), grads)
    limit = 0.5 * _norm64(grads)
    _check_norm_value = float(optim_ops.clip_grads_(grads, limit))
    assert abs(_check_norm_value - 2.0 * limit) <= 4 * U32 * limit
    _check_clipped(grads, before, limit)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [1, 3, 5])
def test_views_off_the_vector_alignment(offset, dtype, cuda_device):
    """Views at odd offsets of one buffer: neighbours keep their values."""
    g = _gen(cuda_device, offset)
    flat = _randn((40_000,), dtype, cuda_device, g)
    views = [flat[offset:offset + 9001], flat[10_000 + offset:10_000 + offset + 3], flat[20_001:39_000]]
    before, rest = [_f64(v) for v in views], flat.clone()
    limit = 0.25 * _norm64(views)
    optim_ops.clip_grads_(views, limit)
    _check_clipped(views, before, limit)
    mask = torch.ones(40_000, dtype=torch.bool, device=cuda_device)
    for a, n in ((offset, 9001), (10_000 + offset, 3), (20_001, 18_999)):
        mask[a:a + n] = False
    assert torch.equal(flat[mask], rest[mask])


def test_strides(cuda_device):
    g = _gen(cuda_device)
    base = _randn((24, 40, 6), torch.float32, cuda_device, g)
    grads = [base.clone().permute(2, 0, 1), base.clone()[:, 3:17], base.clone()[..., ::2],
             torch.randn(5, 6, dtype=torch.complex64, device=cuda_device, generator=g).conj()]
    before = [_f64(t) for t in grads]
    _check_norm(optim_ops.grad_norm(grads), grads)
    limit = 0.4 * _norm64(grads)
    optim_ops.clip_grads_(grads, limit)
    _check_clipped(grads, before, limit)
    row = torch.randn(1, 8, device=cuda_device)
    _check_norm(optim_ops.grad_norm([row.expand(5, 8)]), [row.expand(5, 8)])
    with pytest.raises(RuntimeError, match="expanded"):
        optim_ops.clip_grads_([row.expand(5, 8)], 1.0)
    with pytest.raises(RuntimeError):
        optim_ops.clip_grads_([row, row], 1.0)


@pytest.mark.parametrize("value", [1e30, 1e-30, 3e38])
def test_norms_whose_squares_leave_float32(value, cuda_device):
    for dtype in (torch.float32, torch.bfloat16):
        t = torch.full((5,), value, device=cuda_device).to(dtype)
        want = _norm64([t])
        got = float(optim_ops.grad_norm([t]))
        if want < torch.finfo(torch.float32).max:
            assert abs(got - want) <= 1.01 * U32 * want
        else:
            assert got == math.inf


def test_non_finite_gradients_follow_torch(cuda_device):
    for bad in (math.inf, -math.inf, math.nan):
        grads = [torch.randn(3000, device=cuda_device), torch.randn(5, device=cuda_device)]
        grads[0][1234] = bad
        params = [torch.nn.Parameter(t.clone()) for t in grads]
        for p, t in zip(params, grads):
            p.grad = t.clone()
        want = torch.nn.utils.clip_grad_norm_(params, 1.0)
        got = optim_ops.clip_grads_(grads, 1.0)
        assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))
        for p, t in zip(params, grads):
            assert torch.equal(p.grad.nan_to_num(7.0), t.nan_to_num(7.0))


def test_zero_gradients_and_zero_limit(cuda_device):
    grads = [torch.zeros(100, device=cuda_device), torch.randn(9, device=cuda_device)]
    optim_ops.clip_grads_(grads, 0.0)
    assert not grads[1].any()
    assert float(optim_ops.clip_grads_(grads, 1.0)) == 0.0


def test_clip_grad_norm_of_parameters(cuda_device):
    a, b, c = (torch.nn.Parameter(torch.randn(50, device=cuda_device)) for _ in range(3))
    a.grad, b.grad = torch.randn(50, device=cuda_device), torch.randn(50, device=cuda_device)
    before, version = [_f64(a.grad), _f64(b.grad)], a.grad._version
    n = _norm64([a.grad, b.grad])
    got = optim_ops.clip_grad_norm_([a, b, c, a], 0.5 * n)
    assert abs(float(got) - n) <= 1.01 * U32 * n
    _check_clipped([a.grad, b.grad], before, 0.5 * n)
    assert a.grad._version > version


def test_repeatable(cuda_device):
    g = _gen(cuda_device)
    grads = [_randn((n,), torch.float32, cuda_device, g) for n in (700_001, 33, 90_000)]
    assert len({float(optim_ops.grad_norm(grads)) for _ in range(5)}) == 1


# ------------------------------------------------------------------------------- Adam


def _adam_state(shapes, dtype, dev, g, moments=True):
    real = torch.complex64 if dtype == torch.complex64 else torch.float32
    params = [_randn(s, dtype, dev, g, 0.3) for s in shapes]
    grads = [_randn(s, dtype, dev, g, 10.0 ** (-k % 4)) for k, s in enumerate(shapes)]
    m = [_randn(s, real, dev, g, 0.1 if moments else 0.0) for s in shapes]
    v = [_randn(s, real, dev, g, 0.1 if moments else 0.0) for s in shapes]
    for t in v:
        _real(t).square_()
    return params, grads, m, v


def _check_adam(params, m, v, before, *, step, lr, betas, eps, wd, decoupled, c):
    b1, b2 = betas
    for p, mm, vv, (p0, g0, m0, v0) in zip(params, m, v, before):
        t = torch.float32 if p.is_complex() else p.dtype
        g = c * g0 + (0.0 if decoupled else wd) * p0
        gmag = (c * g0).abs() + (0.0 if decoupled else wd) * p0.abs()
        m1 = b1 * m0 + (1 - b1) * g
        v1 = b2 * v0 + (1 - b2) * g * g
        k, q = lr / (1 - b1**step), 1 / math.sqrt(1 - b2**step)
        den = v1.sqrt() * q + eps
        upd = k * m1 / den
        shrink = lr * wd if decoupled else 0.0
        p1 = p0 - shrink * p0 - upd
        tiny = 2.0**-149
        dm = 6 * U32 * ((b1 * m0).abs() + (1 - b1) * gmag) + 2 * tiny
        # g' may cancel (decay against gradient): its error, 3 u |g'|_mag, enters v through 2 g' dg'
        dg = 3 * U32 * gmag + tiny
        dv = 10 * U32 * v1 + (1 - b2) * (2 * g.abs() * dg + dg * dg) + 4 * tiny
        root = v1.sqrt()
        droot = torch.where(v1 > 4 * dv, dv / root.clamp_min(1e-300), (v1 + dv).sqrt() - (v1 - dv).clamp_min(0).sqrt())
        dupd = 12 * U32 * upd.abs() + k * dm / den + upd.abs() * (droot * q / (den - droot * q).clamp_min(1e-300))
        dp = 1.05 * dupd + U32 * (p1.abs() + 2 * shrink * p0.abs()) + _u(t) * (p1.abs() + dupd) + 2 * torch.finfo(t).smallest_normal * torch.finfo(t).eps
        assert bool(((_f64(mm) - m1).abs() <= 1.05 * dm).all())
        assert bool(((_f64(vv) - v1).abs() <= 1.05 * dv).all())
        assert bool(((_f64(p) - p1).abs() <= dp).all()), float(((_f64(p) - p1).abs() / dp).max())


SHAPES = [[(1,)], [(5,), (1025,), (0,)], [(300, 7), (64,), (33, 31, 9)], [(1_000_003,), (12,), (70_001,)]]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.complex64])
@pytest.mark.parametrize("shapes", SHAPES, ids=str)
@pytest.mark.parametrize("form", ["plain", "decay", "decoupled", "clip", "clip_decay"])
def test_adam_step(shapes, dtype, form, cuda_device):
    g = _gen(cuda_device, 3)
    params, grads, m, v = _adam_state(shapes, dtype, cuda_device, g)
    before = [tuple(_f64(t) for t in ts) for ts in zip(params, grads, m, v)]
    kept = [t.clone() for t in grads]
    steps = [torch.full((), 6.0, device=cuda_device) for _ in params]
    n = _norm64(grads)
    max_norm = 0.3 * n if "clip" in form else None
    wd = 0.01 if "dec" in form else 0.0
    hyper = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8)
    got = optim_ops.adam_step_(params, grads, m, v, steps, weight_decay=wd, decoupled=form == "decoupled",
                               max_norm=max_norm, **hyper)
    if max_norm is None:
        assert got is None
    else:
        _check_norm(got, grads)
    assert all(torch.equal(a, b) for a, b in zip(kept, grads)) and all(float(s) == 7.0 for s in steps)
    c = min(1.0, max_norm / (n + 1e-6)) if max_norm else 1.0
    _check_adam(params, m, v, before, step=7, wd=wd, decoupled=form == "decoupled", c=c, **hyper)


def test_adam_from_the_first_step_and_other_hyperparameters(cuda_device):
    g = _gen(cuda_device, 4)
    params, grads, m, v = _adam_state([(999,), (128, 3)], torch.float32, cuda_device, g, moments=False)
    grads[0][:100] = 0.0  # zero gradients and zero moments: no update
    before = [tuple(_f64(t) for t in ts) for ts in zip(params, grads, m, v)]
    steps = [torch.zeros((), device=cuda_device), torch.zeros((), device=cuda_device)]
    hyper = dict(lr=0.1, betas=(0.0, 0.5), eps=1e-3)
    optim_ops.adam_step_(params, grads, m, v, steps, **hyper)
    assert torch.equal(params[0][:100].double(), before[0][0][:100])
    _check_adam(params, m, v, before, step=1, wd=0.0, decoupled=False, c=1.0, **hyper)


@pytest.mark.parametrize("count", [32, 33, 450])
def test_adam_over_many_tensors_with_their_own_steps(count, cuda_device):
    rng = random.Random(count)
    g = _gen(cuda_device, count)
    shapes = [(rng.randint(1, 900),) for _ in range(count)]
    params, grads, m, v = _adam_state(shapes, torch.float32, cuda_device, g)
    before = [tuple(_f64(t) for t in ts) for ts in zip(params, grads, m, v)]
    at = [float(rng.randint(0, 50)) for _ in range(count)]
    steps = [torch.full((), t, device=cuda_device) for t in at]
    n = _norm64(grads)
    hyper = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8)
    got = optim_ops.adam_step_(params, grads, m, v, steps, max_norm=0.5 * n, **hyper)
    _check_norm(got, grads)
    for k in range(count):
        assert float(steps[k]) == at[k] + 1
        _check_adam(params[k:k + 1], m[k:k + 1], v[k:k + 1], before[k:k + 1], step=at[k] + 1, wd=0.0, decoupled=False,
                    c=0.5 * n / (n + 1e-6), **hyper)


def test_adam_views_and_strides(cuda_device):
    """Buckets whose views sit at different offsets per list, transposed parameters, a gradient of
    other strides, a conjugate gradient."""
    g = _gen(cuda_device, 5)
    hyper = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8)
    flat = [torch.randn(9000, device=cuda_device, generator=g) for _ in range(4)]
    flat[3].square_()
    views = [[f[o:o + 7001]] for f, o in zip(flat, (1, 2, 3, 1))]
    base = [torch.randn(30, 50, device=cuda_device, generator=g) for _ in range(4)]
    base[3].square_()
    views = [a + [b.t()] for a, b in zip(views, base)]
    views[1][1] = base[1].reshape(50, 30).clone()  # contiguous, where its parameter is transposed
    conj = [torch.randn(77, dtype=torch.complex64, device=cuda_device, generator=g) for _ in range(4)]
    torch.view_as_real(conj[3]).square_()
    conj[1] = conj[1].conj()
    params, grads, m, v = ([*a, b] for a, b in zip(views, conj))
    before = [tuple(_f64(t) for t in ts) for ts in zip(params, grads, m, v)]
    edge = flat[0][0].item()
    steps = [torch.zeros((), device=cuda_device) for _ in params]
    optim_ops.adam_step_(params, grads, m, v, steps, **hyper)
    _check_adam(params, m, v, before, step=1, wd=0.0, decoupled=False, c=1.0, **hyper)
    assert flat[0][0].item() == edge
    with pytest.raises(RuntimeError, match="dense"):
        t = torch.randn(8, 8, device=cuda_device)[:, :4]
        optim_ops.adam_step_([t], [t], [t], [t], [steps[0]], lr=1e-3)
    with pytest.raises(RuntimeError):
        optim_ops.adam_step_(params[:1] * 2, grads[:1] * 2, m[:1] * 2, v[:1] * 2, steps[:2], lr=1e-3)
    with pytest.raises(RuntimeError):
        optim_ops.adam_step_(params, grads, m, v, [steps[0]] * 3, lr=1e-3)
    with pytest.raises(RuntimeError, match="type"):
        optim_ops.adam_step_(params[:1], [grads[0].double()], m[:1], v[:1], steps[:1], lr=1e-3)


def test_adam_decay_below_half_a_step_of_p_is_kept(cuda_device):
    """lr wd = 2e-8 is less than half a step of p: it has to join the update before the rounding."""
    p = torch.full((64,), 1.5, device=cuda_device)
    zeros = torch.zeros_like(p)
    m = torch.linspace(0.0, 1.2e-7, 64, device=cuda_device)
    before = [tuple(_f64(t) for t in (p, zeros, m, torch.ones_like(p)))]
    v, step = torch.ones_like(p), torch.full((), 1e6, device=cuda_device)
    hyper = dict(lr=1.0, betas=(0.9, 0.999), eps=0.0)
    optim_ops.adam_step_([p], [zeros], [m], [v], [step], weight_decay=2e-8, decoupled=True, **hyper)
    _check_adam([p], [m], [v], before, step=1e6 + 1, wd=2e-8, decoupled=True, c=1.0, **hyper)


def test_adam_with_a_given_norm_and_a_device_rate(cuda_device):
    g = _gen(cuda_device, 6)
    params, grads, m, v = _adam_state([(5000,), (17,)], torch.float32, cuda_device, g)
    before = [tuple(_f64(t) for t in ts) for ts in zip(params, grads, m, v)]
    steps = [torch.zeros((), device=cuda_device) for _ in params]
    total, lr = torch.full((), 20.0, device=cuda_device), torch.full((), 0.25, device=cuda_device)
    got = optim_ops.adam_step_(params, grads, m, v, steps, lr=lr, weight_decay=0.125, decoupled=True, max_norm=5.0,
                               total_norm=total)
    assert got is total
    _check_adam(params, m, v, before, step=1, lr=0.25, betas=(0.9, 0.999), eps=1e-8, wd=0.125, decoupled=True,
                c=5.0 / (20.0 + 1e-6))


# ------------------------------------------------------------------- streams, graphs, optimizer


def test_two_streams_and_two_graphs(cuda_device):
    """Calls on two streams, and two captured graphs replayed in turn, keep apart."""
    g = _gen(cuda_device, 7)
    lists = [[_randn((200_000,), torch.float32, cuda_device, g, s) for _ in range(3)] for s in (1.0, 5.0)]
    want = [_norm64(t) for t in lists]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                got[k].append(optim_ops.grad_norm(lists[k]))
    torch.cuda.synchronize()
    for k in (0, 1):
        assert all(abs(float(x) - want[k]) <= 1.01 * U32 * want[k] for x in got[k])
    graphs, outs = [], []
    for t in lists:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(optim_ops.clip_grads_(t, 1.0))
        graphs.append(graph)
    fresh = [[t.clone() for t in ts] for ts in lists]
    for _ in range(3):
        for k in (0, 1):
            for t, f in zip(lists[k], fresh[k]):
                t.copy_(f)
            graphs[k].replay()
    torch.cuda.synchronize()
    for k in (0, 1):
        assert abs(float(outs[k]) - want[k]) <= 1.01 * U32 * want[k]
        _check_clipped(lists[k], [_f64(t) for t in fresh[k]], 1.0)


def test_captured_adam_step_advances(cuda_device):
    g = _gen(cuda_device, 8)
    params, grads, m, v = _adam_state([(3000,), (40, 40)], torch.float32, cuda_device, g)
    other = [[t.clone() for t in ts] for ts in (params, grads, m, v)]
    steps = [torch.zeros((), device=cuda_device) for _ in params]
    steps2 = [torch.zeros((), device=cuda_device) for _ in params]
    optim_ops.adam_step_(params, grads, m, v, steps, lr=1e-2, max_norm=1.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        optim_ops.adam_step_(params, grads, m, v, steps, lr=1e-2, max_norm=1.0)
    for _ in range(3):
        graph.replay()
    for _ in range(4):
        optim_ops.adam_step_(*other, steps2, lr=1e-2, max_norm=1.0)
    assert float(steps[0]) == 4.0
    assert all(torch.equal(a, b) for a, b in zip(params + m + v, other[0] + other[2] + other[3]))


def test_fused_adam_follows_torch_adam(cuda_device):
    """Groups, a scheduler, clipping over all groups, a parameter that has no gradient at first, and
    the state dict both ways: five steps against torch.optim.Adam in 64 bits, whose own 64-bit error
    is nil here; each of our steps adds at most the single step's error, so 5 steps stay within
    1e-6 of lr-sized moves."""
    g = _gen(cuda_device, 9)
    init = [_randn(s, torch.float32, cuda_device, g) for s in ((40, 30), (30,), (9, 5))]
    data = [[_randn(t.shape, torch.float32, cuda_device, g) for t in init] for _ in range(5)]
    ours = [torch.nn.Parameter(t.clone()) for t in init]
    ref = [torch.nn.Parameter(t.double()) for t in init]
    groups = lambda ps: [{"params": ps[:2]}, {"params": ps[2:], "lr": 5e-3, "weight_decay": 0.1}]  # noqa: E731
    opt = optim_ops.FusedAdam(groups(ours), lr=1e-2, max_norm=3.0)
    opt_ref = torch.optim.Adam(groups(ref), lr=1e-2)
    scheds = [torch.optim.lr_scheduler.CosineAnnealingLR(o, T_max=5) for o in (opt, opt_ref)]
    for k, batch in enumerate(data):
        for p, q, d in zip(ours, ref, batch):
            skip = k == 0 and p is ours[1]
            p.grad, q.grad = (None, None) if skip else (d.clone(), d.double())
        n = torch.nn.utils.clip_grad_norm_(ref, 3.0)
        opt.step()
        opt_ref.step()
        for s in scheds:
            s.step()
        assert abs(float(opt.last_norm) - float(n)) <= 1.01 * U32 * float(n)
        if k == 2:
            state = opt.state_dict()
            opt = optim_ops.FusedAdam(groups(ours), lr=1.0, max_norm=3.0)
            opt.load_state_dict(state)
            scheds[0].optimizer = opt
            for grp, old in zip(opt.param_groups, state["param_groups"]):
                assert grp["lr"] == old["lr"]
    for p, q in zip(ours, ref):
        assert float((p.detach().double() - q.detach()).abs().max()) <= 1e-6
        assert opt.state[p]["step"].item() == opt_ref.state[q]["step"].item()


def test_versions_move_with_the_step(cuda_device):
    """Caches keyed by a parameter's version (the device copies of the FNO weights) see the step."""
    p = torch.nn.Parameter(torch.ones(10, device=cuda_device))
    p.grad = torch.ones_like(p)
    opt = optim_ops.FusedAdam([p], lr=0.1)
    version = p._version
    opt.step()
    assert p._version > version and float(p.detach()[0]) < 1.0


def test_more_than_2_31_values(cuda_device):
    """One tensor past 32-bit offsets, zero but for its ends, beside a small one."""
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of device memory")
    n = (1 << 31) + 12_345
    big = torch.zeros(n, dtype=torch.bfloat16, device=cuda_device)
    big[:100], big[-100:] = 3.0, 4.0
    small = torch.full((5,), 2.0, device=cuda_device)
    want = math.sqrt(100 * 9 + 100 * 16 + 5 * 4)
    assert abs(float(optim_ops.grad_norm([big, small])) - want) <= 1.01 * U32 * want
    p = torch.full((n,), 1.0, dtype=torch.bfloat16, device=cuda_device)
    m, v = torch.zeros(n, device=cuda_device), torch.zeros(n, device=cuda_device)
    step = torch.zeros((), device=cuda_device)
    optim_ops.adam_step_([p], [big], [m], [v], [step], lr=0.25, max_norm=want / 2)
    assert float(m[-1]) > 0.0 and float(m[100]) == 0.0 and float(p[n // 2]) == 1.0
    assert float(p[0]) == float(p[-1]) == 0.75 and float(p[-101]) == 1.0  # a first step moves by lr
    optim_ops.clip_grads_([big, small], want / 2)
    assert float(big[0]) == 1.5 and float(big[-1]) == 2.0 and float(big[-101]) == 0.0 and float(small[0]) == 1.0


def test_only_empty_tensors(cuda_device):
    empty = [torch.zeros(0, device=cuda_device), torch.zeros(3, 0, dtype=torch.complex64, device=cuda_device)]
    assert float(optim_ops.grad_norm(empty)) == 0.0 and float(optim_ops.clip_grads_(empty, 1.0)) == 0.0
    steps = [torch.zeros((), device=cuda_device) for _ in empty]
    got = optim_ops.adam_step_(empty, empty, empty, empty, steps, lr=1.0, max_norm=1.0)
    assert float(got) == 0.0 and [float(s) for s in steps] == [1.0, 1.0]


def test_forward_derivatives_are_refused(cuda_device):
    t, one = torch.ones(5, device=cuda_device), torch.ones(5, device=cuda_device)
    with fwAD.dual_level():
        dual = fwAD.make_dual(t, one)
        with pytest.raises(RuntimeError, match="forward-mode"):
            optim_ops.grad_norm([one, dual])
        with pytest.raises(RuntimeError, match="forward-mode"):
            optim_ops.clip_grads_([dual], 1.0)
        step = torch.zeros((), device=cuda_device)
        for k in range(4):
            lists = [[torch.ones(5, device=cuda_device)] for _ in range(4)]
            lists[k] = [dual]
            with pytest.raises(RuntimeError, match="forward-mode"):
                optim_ops.adam_step_(*lists, [step], lr=1.0)
    assert torch.equal(t, one)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.complex64])
def test_the_norm_is_differentiable(dtype, cuda_device):
    """dN/dg = g / N, per component of complex values: N is off by 1.01 u, and the quotient, the product and
    the rounding to the type add one each."""
    g = _gen(cuda_device, 10)
    kinds = [(300, 7), (1,), (0,), (4096 + 3,)]
    grads = [_randn(s, dtype, cuda_device, g).requires_grad_(k != 1) for k, s in enumerate(kinds)]
    grads.append(_randn((6, 8), torch.float32, cuda_device, g).requires_grad_(True))
    views = [*grads[:-1], grads[-1].t()[::2]]  # one that is not dense
    total = optim_ops.grad_norm(views)
    _check_norm(total, views)
    wrt = [t for t in grads if t.requires_grad]
    got = torch.autograd.grad(total, wrt, torch.full_like(total, -1.5))
    n = _norm64(views)
    for t, d in zip(wrt, got):
        assert d.dtype == t.dtype
        value = _f64(t)
        if t is grads[-1]:
            value[:, 1::2] = 0.0
        want = -1.5 * value / n
        bound = (4 * U32 + _u(t.dtype)) * want.abs() + torch.finfo(d.dtype).tiny
        assert bool(((_f64(d) - want).abs() <= bound).all())
    with torch.no_grad():
        assert not optim_ops.grad_norm(views).requires_grad
    zero = torch.zeros(5, device=cuda_device, requires_grad=True)
    (d,) = torch.autograd.grad(optim_ops.grad_norm([zero]), zero)
    assert torch.equal(d, torch.zeros_like(d))


def test_a_penalty_on_the_gradient_norm(cuda_device):
    """f = sum w^3 / 3 has the gradient w^2, N = |w^2| and dN/dw = 2 w^3 / N; then the second derivative of N
    itself, v / N - g (g v) / N^3.  The first takes 4 roundings for w^2, at most 5 for N, 2 for their quotient and
    5 more behind it: 24 u bounds them.  In the second the float32 sum g v adds chains of at most 40: 64 u of the
    terms' magnitudes."""
    g = _gen(cuda_device, 11)
    w = _randn((1000,), torch.float32, cuda_device, g).requires_grad_(True)
    (grad,) = torch.autograd.grad((w**3).sum() / 3, w, create_graph=True)
    (got,) = torch.autograd.grad(optim_ops.grad_norm([grad]), w)
    w64 = _f64(w)
    want = 2 * w64**3 / w64.square().norm()
    assert bool(((got.double() - want).abs() <= 24 * U32 * want.abs()).all())
    v = _randn((1000,), torch.float32, cuda_device, g)
    (first,) = torch.autograd.grad(optim_ops.grad_norm([w]), w, create_graph=True)
    (second,) = torch.autograd.grad(first, w, v)
    n, v64 = w64.norm(), v.double()
    want = v64 / n - w64 * (w64 * v64).sum() / n**3
    size = v64.abs() / n + w64.abs() * (w64 * v64).abs().sum() / n**3
    assert bool(((second.double() - want).abs() <= 64 * U32 * size).all())



LONG = [1, 4097, 2047, 4095, 8193, 2048, 12287, 4096, 2049, 8188, 8191, 3, 8192, 12288, 4100, 2052, 17_000_003, 8196, 0, 4099]


def _long_list(dtype, dev, g, scale=1.0, square=False):
    """Views with gaps between them of one buffer, each list's neighbours at other alignments: more than
    16.8M float32 values, beside tensors around the counts that a block has in flight (1024 vectors of 4,
    twice that, and 512)."""
    wide = 2 if dtype == torch.complex64 else 1
    sizes = [n if n < 1 << 20 else n // wide for n in LONG]
    flat = torch.randn(wide * (sum(sizes) + len(sizes)), device=dev, generator=g) * scale
    if square:
        flat.square_()
    buffer = torch.view_as_complex(flat.view(-1, 2)) if wide == 2 else flat
    views, at = [], 0
    for n in sizes:
        views.append(buffer[at:at + n])
        at += n + 1
    return flat, views


@pytest.mark.parametrize("dtype", [torch.float32, torch.complex64])
def test_long_lists_norm(dtype, cuda_device):
    """Ones in a run of the list at a time, zeros elsewhere: a vector that is lost or taken twice changes the
    norm by more than 2^-19 of it."""
    flat, views = _long_list(dtype, cuda_device, _gen(cuda_device, 12))
    _check_norm(optim_ops.grad_norm(views), views)
    edges = list(range(0, flat.numel(), 1_000_003)) + [flat.numel()]
    for a, b in zip(edges, edges[1:]):
        flat.zero_()
        flat[a:b] = 1.0
        _check_norm(optim_ops.grad_norm(views), views)
    flat.fill_(math.nan)  # the gaps are not read
    for v in views:
        v.fill_(0.0)
    assert float(optim_ops.grad_norm(views)) == 0.0


@pytest.mark.parametrize("dtype", [torch.float32, torch.complex64])
def test_long_lists_clip(dtype, cuda_device):
    flat, views = _long_list(dtype, cuda_device, _gen(cuda_device, 13))
    before, rest = [_f64(v) for v in views], flat.clone()
    limit = 0.37 * _norm64(views)
    got = optim_ops.clip_grads_(views, limit)
    assert abs(float(got) - limit / 0.37) <= 1.01 * U32 * float(got)
    _check_clipped(views, before, limit)
    for v in views:
        v.zero_()
    kept = flat != 0
    assert int(kept.sum()) >= 15 and torch.equal(flat[kept], rest[kept])


@pytest.mark.parametrize("dtype", [torch.float32, torch.complex64])
@pytest.mark.parametrize("clip", [False, True])
def test_long_lists_adam(clip, dtype, cuda_device):
    g = _gen(cuda_device, 14)
    flats, lists = zip(*(_long_list(dtype, cuda_device, g, s, k == 3) for k, s in enumerate((0.3, 1.0, 0.1, 0.1))))
    params, grads, m, v = lists
    before = [tuple(_f64(t) for t in ts) for ts in zip(params, grads, m, v)]
    rest = [f.clone() for f in flats]
    steps = [torch.full((), 6.0, device=cuda_device) for _ in params]
    n = _norm64(grads)
    hyper = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8)
    optim_ops.adam_step_(params, grads, m, v, steps, max_norm=0.3 * n if clip else None, **hyper)
    assert torch.equal(flats[1], rest[1]) and all(float(s) == 7.0 for s in steps)
    _check_adam(params, m, v, before, step=7, wd=0.0, decoupled=False, c=0.3 * n / (n + 1e-6) if clip else 1.0, **hyper)
    for k in (0, 2, 3):
        for t in lists[k]:
            t.zero_()
        kept = flats[k] != 0
        assert int(kept.sum()) >= 15 and torch.equal(flats[k][kept], rest[k][kept])


@pytest.mark.parametrize("decay, decoupled", [(0.0, False), (0.0, True), (0.01, True)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rate_on_device", [False, True])
def test_infinite_parameters_stay_as_in_torch(rate_on_device, dtype, decay, decoupled, cuda_device):
    """A parameter held at an infinity (a masked entry) keeps it, and its moments are those of its gradient.
    The others agree to the roundings: in float32 3 updates of 0.125 by 24 u and 6 of p; in bfloat16 torch's moments
    are rounded too, 3 updates by 2^-6 and 6 halves of a step 2^-7 of p."""
    p = torch.linspace(-1.0, 1.0, 40, device=cuda_device).to(dtype)
    p[3], p[20], p[38] = -math.inf, math.inf, -math.inf
    grad = torch.randn(40, device=cuda_device, generator=_gen(cuda_device, 15)).to(dtype)
    grad[20] = 0.0
    ours, ref = torch.nn.Parameter(p.clone()), torch.nn.Parameter(p.clone())
    ours.grad, ref.grad = grad.clone(), grad.clone()
    lr = torch.full((), 0.125, device=cuda_device) if rate_on_device else 0.125
    kind = torch.optim.AdamW if decoupled else torch.optim.Adam
    opt = optim_ops.FusedAdam([ours], lr=lr, weight_decay=decay, decoupled_weight_decay=decoupled)
    opt_ref = kind([ref], lr=0.125, weight_decay=decay)
    for _ in range(3):
        opt.step()
        opt_ref.step()
    for k in (3, 20, 38):
        assert float(ours.detach()[k]) == float(ref.detach()[k]) == float(p[k])
    assert bool(torch.isfinite(opt.state[ours]["exp_avg"]).all()) and bool(torch.isfinite(opt.state[ours]["exp_avg_sq"]).all())
    rest = torch.isfinite(p)
    torch.testing.assert_close(ours.detach()[rest], ref.detach()[rest], rtol=0.0,
                               atol=1e-5 if dtype == torch.float32 else 0.05)


def test_the_last_norm_is_of_the_last_step(cuda_device):
    p = torch.nn.Parameter(torch.ones(4, device=cuda_device))
    opt = optim_ops.FusedAdam([p], lr=1e-2, max_norm=1.0)
    p.grad = torch.full_like(p, 2.0)
    opt.step()
    assert float(opt.last_norm) == 4.0
    opt.zero_grad()
    opt.step()  # without a gradient: as clip_grad_norm_ gives then
    assert float(opt.last_norm) == 0.0


def test_a_first_step_is_not_captured(cuda_device):
    """Its zero moments and count would be made again at every replay."""
    p = torch.nn.Parameter(torch.ones(4, device=cuda_device))
    p.grad = torch.ones_like(p)
    opt = optim_ops.FusedAdam([p], lr=0.5)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before it is captured"):
        with torch.cuda.graph(graph):
            opt.step()
    assert not opt.state[p] and bool((p.detach() == 1.0).all())
    del graph
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    graph.replay()
    graph.replay()
    assert float(opt.state[p]["step"]) == 3.0


def test_tracing_is_refused(cuda_device):
    """A trace would keep the outputs' allocation and not the kernels."""
    x = torch.randn(8, device=cuda_device)
    for call in (lambda a: optim_ops.grad_norm([a]), lambda a: optim_ops.clip_grads_([a.clone()], 1.0)):
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(call, x, check_trace=False)


def test_adam_lists_beside_one_another(cuda_device):
    """Parameter, gradient and moments one behind the other in one buffer, in either order."""
    for order in ((0, 1, 2, 3), (3, 2, 1, 0), (1, 0, 3, 2)):
        flat = torch.randn(4 * 1001, device=cuda_device, generator=_gen(cuda_device, 16)).abs()
        lists = [[flat[1001 * k:1001 * (k + 1)]] for k in order]
        before = [tuple(_f64(t[0]) for t in lists)]
        step = torch.zeros((), device=cuda_device)
        hyper = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8)
        optim_ops.adam_step_(*lists, [step], **hyper)
        _check_adam(lists[0], lists[2], lists[3], before, step=1, wd=0.0, decoupled=False, c=1.0, **hyper)
        with pytest.raises(RuntimeError):
            optim_ops.adam_step_(lists[0], [flat[500:1501]], lists[2], lists[3], [step], **hyper)
