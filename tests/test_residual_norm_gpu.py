"""GPU: the residual-norm operator against its formulas in 64 bits (tests/residual_norm_reference.py
has the bounds and how they are derived), forward and backward, in both layouts."""

from __future__ import annotations

import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import _scx
from residual_norm_ops import residual_norm
from residual_norm_reference import like, reference, rows_of, within

pytestmark = pytest.mark.gpu

VECTORS = ("post_weight", "post_bias", "pre_weight", "pre_bias", "scale")


def _inputs(shape, dim, dtype, dev, *, gate="none", vectors=VECTORS, wide=True, seed=0, mean=0.3):
    g = torch.Generator(device=dev).manual_seed(seed)
    C = shape[1] if dim == 1 else shape[-1]
    rand = lambda s, m=0.0, d=1.0: (torch.randn(*s, device=dev, generator=g) * d + m)  # noqa: E731
    t = {"x": rand(shape, 0.0, 1.5).to(dtype), "y": rand(shape, mean, 0.7).to(dtype), "gate": None}
    if gate == "full":
        t["gate"] = rand(shape).to(dtype)
    elif gate == "sample":
        t["gate"] = rand((shape[0], C)).to(dtype)
    for k in VECTORS:
        t[k] = rand((C,), 0.0 if "bias" in k else 1.0, 0.2).to(torch.float32 if wide else dtype) if k in vectors else None
    return t, rand(shape).to(dtype), rand(shape).to(dtype)


def _gate_rows(t, dim):
    gate = t["gate"]
    if gate is None:
        return None
    return rows_of(gate, dim) if gate.shape == t["x"].shape else gate.detach().double()[:, None, :]


def _expected(t, dim, dr=None, dn=None, **options):
    return reference(rows_of(t["x"], dim), rows_of(t["y"], dim) if t["y"] is not None else None, _gate_rows(t, dim), t,
                     dr=rows_of(dr, dim) if dr is not None else None, dn=rows_of(dn, dim) if dn is not None else None,
                     **options)


def _compare(name, got, want, t, dim):
    value, bound = want
    if name in ("r", "n", "d_x", "d_y") or (name == "d_gate" and t["gate"].shape == t["x"].shape):
        value, bound = like(value, t["x"].shape, dim), like(bound, t["x"].shape, dim)
    elif name == "d_gate":
        value, bound = value[:, 0], bound[:, 0]
    assert got.shape == value.shape, name
    assert within(got, value, bound), (name, float((got.detach().double() - value).abs().max()))


def _run(t, dim, dr, dn, *, kind="rms", act="none", eps=1e-5, number=None, post=True, pre=True, train=True, skip=()):
    """Forward without gradients, then forward and backward, each output compared."""
    names = [k for k in ("x", "y", "gate", *VECTORS) if t[k] is not None]
    kwargs = dict(kind=kind, gate_activation=act, eps=eps, dim=dim, post_norm=post, pre_norm=pre)
    if number is not None:
        kwargs["scale"] = number
    args = lambda s: {**{k: s[k] for k in ("gate", *VECTORS) if s[k] is not None}, **kwargs}  # noqa: E731
    want = _expected(t, dim, dr, dn, kind=kind, act=act, eps=eps, number=1.0 if number is None else number, post=post,
                     pre=pre)
    with torch.no_grad():
        r, n = residual_norm(t["x"], t["y"], **args(t))
    if t["y"] is None:
        assert r is t["x"]
    else:
        _compare("r", r, want["r"], t, dim)
    if pre:
        _compare("n", n, want["n"], t, dim)
    else:
        assert n is None
    if not train:
        return
    leaves = {k: (v.detach().clone().requires_grad_(k not in skip) if v is not None else None) for k, v in t.items()}
    r2, n2 = residual_norm(leaves["x"], leaves["y"], **args(leaves))
    assert torch.equal(r2, r) and (n2 is None or torch.equal(n2, n))
    outs = [(o, d) for o, d in ((r2, dr), (n2, dn)) if o is not None and d is not None]
    wrt = [k for k in names if k not in skip]
    grads = torch.autograd.grad([o for o, _ in outs], [leaves[k] for k in wrt], [d for _, d in outs], allow_unused=True)
    for k, got in zip(wrt, grads):
        if "d_" + k not in want:
            assert got is None or not got.any(), k
            continue
        _compare("d_" + k, got, want["d_" + k], t, dim)


TOKENS = [(1, 1), (1, 1, 8), (2, 3, 7), (5, 33), (3, 17, 100), (1, 2, 4096), (2, 2, 5001), (4, 9, 1025), (7, 40, 64),
          (1, 3, 16384), (1, 1, 20000), (33, 2, 48), (2, 700, 16), (3, 5, 8192), (2, 3, 2, 36), (2, 600, 4104), (1, 2, 12000), (2, 3, 2050), (1, 5, 7001),
          (2, 350, 2100), (2, 350, 3001), (1, 500, 6004), (1, 500, 2304), (2, 300, 1002)]
FIELDS = [(2, 4, 1, 1), (1, 5, 3, 5), (3, 32, 8, 16), (2, 36, 9, 7), (2, 200, 5, 13), (1, 64, 32, 32), (2, 32, 70),
          (4, 1, 31), (1, 513, 40), (2, 20, 12, 12, 4), (20, 32, 4), (1, 32, 64, 64), (3, 24, 100, 7), (2, 1100, 33), (1, 96, 36), (3, 40, 5, 8), (2, 300, 64), (1, 75, 41), (1, 130, 9),
          (2, 256, 20, 20), (2, 768, 16, 20), (2, 1024, 300), (2, 700, 15, 17), (1, 1023, 333)]
SHAPES = [(s, -1) for s in TOKENS] + [(s, 1) for s in FIELDS]
GATES = [("none", "none"), ("sample", "sigmoid"), ("full", "silu")]


@pytest.mark.parametrize("gate, act", GATES)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape, dim", SHAPES, ids=str)
def test_forward_and_backward(shape, dim, dtype, kind, gate, act, cuda_device):
    if gate == "sample" and dim == -1 and len(shape) == 2:
        gate = "full"  # one position per sample
    t, dr, dn = _inputs(shape, dim, dtype, cuda_device, gate=gate)
    _run(t, dim, dr, dn, kind=kind, act=act)


@pytest.mark.parametrize("shape, dim", [((3, 19, 40), -1), ((2, 32, 8, 12), 1), ((2, 33, 5, 3), 1), ((2, 5, 2048), -1)], ids=str)
@pytest.mark.parametrize("act", ["none", "sigmoid", "silu"])
@pytest.mark.parametrize("gate", ["sample", "full"])
def test_gates(gate, act, shape, dim, cuda_device):
    t, dr, dn = _inputs(shape, dim, torch.float32, cuda_device, gate=gate, seed=1)
    t["gate"] *= 8.0  # saturated on both sides
    _run(t, dim, dr, dn, kind="layer", act=act)


def test_the_sigmoid_over_its_range(cuda_device):
    """x = 0 and y = 1 without norms: r is the activation itself.  Within 10 roundings of the value where
    that is a normal number, below the smallest of them otherwise; the ends and NaN as they are."""
    g = torch.cat([torch.linspace(-95.0, 95.0, 200_003), torch.linspace(-1.0, 1.0, 100_001),
                   torch.tensor([float("inf"), float("-inf"), float("nan"), 0.0, -0.0, 3e38, -3e38, 1e-40])]).to(cuda_device)
    g = g[:g.numel() // 4 * 4].view(-1, 4) if g.numel() % 4 else g.view(-1, 4)
    for act in ("sigmoid", "silu"):
        r, _ = residual_norm(torch.zeros_like(g), torch.ones_like(g), gate=g, gate_activation=act, post_norm=False,
                             pre_norm=False, dim=-1)
        s = torch.special.expit(g.double())
        want = s if act == "sigmoid" else g.double() * s
        finite = torch.isfinite(want)
        off = (r.double() - want).abs()[finite]
        # where the sigmoid is below the normal numbers it may be zero
        small = torch.where(s < 1.2e-38, want.abs(), 0 * s)[finite]
        assert bool((off <= 10 * 2.0**-24 * want.abs()[finite] + small + 1.2e-38).all())
        assert torch.equal(torch.isnan(r)[~finite], torch.isnan(want)[~finite])


@pytest.mark.parametrize("dim", [1, -1])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_the_sigmoid_of_every_two_byte_gate(dtype, dim, cuda_device):
    """All 65536 gates, as above.  The exponent t = -g log2(e) of a two-byte gate is rounded once and log2(e) is
    off by 0.22 roundings: 1.25 |g| roundings of exp(-g), of which exp(-g) / (1 + exp(-g)) reaches the sigmoid; r
    is rounded once to the type, half a step of the value or of the numbers below the normal ones."""
    bits = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16)
    g = bits.view(dtype).view(16, 64, 64).to(cuda_device)
    half = torch.finfo(dtype).eps / 2
    for act in ("sigmoid", "silu"):
        r, _ = residual_norm(torch.zeros_like(g), torch.ones_like(g), gate=g, gate_activation=act, post_norm=False,
                             pre_norm=False, dim=dim)
        wide = g.double()
        s = torch.special.expit(wide)
        want = s if act == "sigmoid" else wide * s
        finite = torch.isfinite(want)
        small = torch.where(s < 1.2e-38, want.abs(), 0 * s)
        near = want.abs() * (1 + (11 + 1.25 * (-wide).clamp(0, 1e39)) * 2.0**-24)  # no 0 * inf
        bound = near - want.abs() + near * half + torch.finfo(dtype).tiny * half + small
        assert ((r.double() - want).abs() <= bound)[finite].all()
        # infinities and NaN as they are: silu of -inf is -inf times 0
        assert torch.equal(r[~finite].isnan(), want[~finite].isnan())
        assert torch.equal(r.isinf(), want.isinf())



@pytest.mark.parametrize("shape, dim", [((3, 19, 40), -1), ((2, 32, 8, 12), 1), ((1, 2, 3000), -1), ((1, 9, 6000), -1),
                                        ((1, 9, 5002), -1), ((2, 700, 12), 1)], ids=str)
@pytest.mark.parametrize("option", ["no_vectors", "narrow", "number", "no_post", "no_pre", "no_y", "only_dr", "only_dn",
                                    "frozen_vectors", "frozen_y", "frozen_x", "sample_frozen", "weights_only"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_options(option, dtype, shape, dim, cuda_device):
    gate = "none" if option == "no_y" else "sample" if option == "sample_frozen" else "full"
    vectors = {"no_vectors": (), "no_post": ("pre_weight", "pre_bias", "scale"), "no_pre": ("post_weight", "post_bias"),
               "no_y": ("pre_weight", "pre_bias"), "number": ("post_weight", "pre_weight")}.get(option, VECTORS)
    t, dr, dn = _inputs(shape, dim, dtype, cuda_device, gate=gate, vectors=vectors, wide=option != "narrow", seed=2)
    if option == "no_y":
        t["y"] = None
    skip = {"frozen_vectors": VECTORS, "frozen_y": ("y",), "frozen_x": ("x",), "sample_frozen": ("gate", "x"),
            "weights_only": ("x", "y", "gate")}.get(option, ())
    _run(t, dim, None if option == "only_dn" else dr, None if option in ("only_dr", "no_pre") else dn, kind="layer",
         act="sigmoid" if gate != "none" else "none", number=-0.3 if option == "number" else None,
         post=option != "no_post", pre=option != "no_pre", skip=skip)


@pytest.mark.parametrize("shape, dim", [((2, 6, 32), -1), ((2, 32, 4, 4), 1)], ids=str)
def test_extremes(shape, dim, cuda_device):
    """Zero rows (only eps under the root), constant rows, large offsets, eps 0."""
    t, dr, dn = _inputs(shape, dim, torch.float32, cuda_device, seed=3)
    t["y"].zero_()
    _run(t, dim, dr, dn, kind="rms")
    t["y"].fill_(3.0)
    _run(t, dim, dr, dn, kind="layer", train=False)
    t, dr, dn = _inputs(shape, dim, torch.float32, cuda_device, seed=4, mean=50.0)
    _run(t, dim, dr, dn, kind="layer", eps=0.0)


def test_non_finite_rows_stay_to_themselves(cuda_device):
    for dim, shape in ((-1, (4, 5, 48)), (1, (2, 32, 8, 8))):
        t, _, _ = _inputs(shape, dim, torch.float32, cuda_device, seed=5)
        clean = residual_norm(t["x"], t["y"], dim=dim)
        bad = t["y"].clone()
        bad[(1, 2, 7) if dim == -1 else (1, 7, 3, 4)] = float("nan")
        bad[(2, 0, 3) if dim == -1 else (0, 7, 0, 1)] = float("inf")
        got = residual_norm(t["x"], bad, dim=dim)
        hit = torch.zeros(shape, dtype=torch.bool, device=cuda_device)
        if dim == -1:
            hit[1, 2] = hit[2, 0] = True
        else:
            hit[1, :, 3, 4] = hit[0, :, 0, 1] = True
        for a, b in zip(clean, got):
            assert torch.equal(a[~hit], b[~hit]) and bool(torch.isnan(b[hit]).any())


def test_layouts_strides_and_offsets(cuda_device):
    """Transposed, sliced and expanded inputs and gradients, and bases off the vector alignment."""
    dev = cuda_device
    for dim, shape in ((-1, (3, 10, 40)), (1, (3, 40, 10))):
        t, dr, dn = _inputs(shape, dim, torch.float32, dev, gate="full", seed=6)
        want = residual_norm(t["x"], t["y"], gate=t["gate"], dim=dim, pre_weight=t["pre_weight"])
        moved = {k: t[k].transpose(1, 2).contiguous().transpose(1, 2) for k in ("x", "y", "gate")}
        wide = torch.empty(80, device=dev)
        wide[::2] = t["pre_weight"]
        got = residual_norm(moved["x"], moved["y"], gate=moved["gate"], dim=dim, pre_weight=wide[::2])
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        flat = torch.empty(3 * t["x"].numel() + 9, device=dev)
        for k, name in enumerate(("x", "y", "gate")):
            v = flat[k * t["x"].numel() + 2 * k + 1:][:t["x"].numel()].view(shape)
            v.copy_(t[name])
            moved[name] = v
        off = torch.empty(41, device=dev)[1:]
        off.copy_(t["pre_weight"])
        leaf = moved["x"].detach().requires_grad_(True)
        r, n = residual_norm(leaf, moved["y"], gate=moved["gate"], dim=dim, pre_weight=off)
        for a, b in zip(want, (r, n)):
            torch.testing.assert_close(a, b, rtol=2e-6, atol=2e-6)  # another order of the channel sums: 11 U of values below 4
        (r.sum() + n.sum()).backward()  # expanded gradients
        ones = torch.ones_like(t["x"])
        t["x"].requires_grad_(True)
        out = residual_norm(t["x"], t["y"], gate=t["gate"], dim=dim, pre_weight=t["pre_weight"])
        (g,) = torch.autograd.grad(out, t["x"], (ones, ones))
        torch.testing.assert_close(leaf.grad, g, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("weight_offset", [1, 2, 4])
@pytest.mark.parametrize("offset", [1, 2, 6])
@pytest.mark.parametrize("channels", [40, 1002])
def test_two_byte_tokens_off_the_vector_alignment(channels, offset, weight_offset, cuda_device):
    """Inputs, gradients and fp32 weights that start some elements into their buffers."""
    t, dr, dn = _inputs((2, 33, channels), -1, torch.bfloat16, cuda_device, gate="full", seed=11)

    def moved(v, by):
        room = torch.empty(v.numel() + by, dtype=v.dtype, device=v.device)[by:].view(v.shape)
        return room.copy_(v)

    t = {k: moved(v, weight_offset if k in VECTORS else offset) for k, v in t.items()}
    dr, dn = moved(dr, offset), moved(dn, offset)
    leaves = {k: v.detach().requires_grad_(True) for k, v in t.items()}
    assert all(v.data_ptr() == t[k].data_ptr() for k, v in leaves.items())
    r, n = residual_norm(leaves["x"], leaves["y"], gate=leaves["gate"], gate_activation="silu", kind="layer", dim=-1,
                         **{k: leaves[k] for k in VECTORS})
    want = _expected(t, -1, dr, dn, kind="layer", act="silu", eps=1e-5, number=1.0, post=True, pre=True)
    _compare("r", r, want["r"], t, -1)
    _compare("n", n, want["n"], t, -1)
    grads = torch.autograd.grad((r, n), list(leaves.values()), (dr, dn))
    for k, got in zip(leaves, grads):
        _compare("d_" + k, got, want["d_" + k], t, -1)


def test_a_second_derivative_is_refused(cuda_device):
    x = torch.randn(3, 8, device=cuda_device, requires_grad=True)
    y = torch.randn(3, 8, device=cuda_device, requires_grad=True)
    r, n = residual_norm(x, y)
    gx, gy = torch.autograd.grad((r * r).sum() + (n * n).sum(), (x, y), create_graph=True)
    with pytest.raises(RuntimeError, match="once only"):
        (gx.sum() + gy.sum()).backward()


def test_empty(cuda_device):
    for shape, dim in (((0, 5, 8), -1), ((3, 0, 8), -1), ((0, 8, 4), 1), ((2, 8, 0), 1)):
        x = torch.zeros(shape, device=cuda_device, requires_grad=True)
        w = torch.ones(8, device=cuda_device, requires_grad=True)
        r, n = residual_norm(x, torch.zeros_like(x), pre_weight=w, dim=dim)
        assert r.shape == n.shape == x.shape
        (r.sum() + n.sum()).backward()
        assert x.grad.shape == x.shape and not w.grad.any()


def test_repeatable_and_alone(cuda_device):
    """Bitwise the same on every run, from poisoned memory, on two streams at once."""
    for dim, shape in ((-1, (2, 300, 520)), (1, (3, 36, 33, 20))):
        t, dr, dn = _inputs(shape, dim, torch.float32, cuda_device, gate="sample", seed=7)
        names = [k for k in ("x", "y", "gate", *VECTORS)]
        for k in names:
            t[k].requires_grad_(True)

        def once():
            r, n = residual_norm(t["x"], t["y"], gate=t["gate"], gate_activation="silu", dim=dim,
                                 **{k: t[k] for k in VECTORS})
            return [r, n, *torch.autograd.grad((r, n), [t[k] for k in names], (dr, dn))]

        first = once()
        torch.empty(1 << 24, device=cuda_device).fill_(float("nan"))
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        for _ in range(4):
            for s in streams:
                with torch.cuda.stream(s):
                    again = once()
                s.synchronize()
                assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_gradients_against_differences(cuda_device):
    """Central differences of the operator itself, in float32 with a step of 2^-6: the forward's own
    error is below 2^-20 of outputs below 8, so a difference carries 2^-11, and the truncation is
    h^2/6 times a third derivative of order 10: 2^-10; the directions are unit vectors of 2^-6."""
    for dim, shape in ((-1, (2, 2, 24)), (1, (2, 24, 3))):
        t, dr, dn = _inputs(shape, dim, torch.float32, cuda_device, gate="sample", seed=8)

        def loss(s):
            r, n = residual_norm(s["x"], s["y"], gate=s["gate"], gate_activation="silu", dim=dim, kind="layer",
                                 **{k: s[k] for k in VECTORS})
            return (r.double() * dr).sum() + (n.double() * dn).sum()

        leaves = {k: v.clone().requires_grad_(True) for k, v in t.items()}
        r, n = residual_norm(leaves["x"], leaves["y"], gate=leaves["gate"], gate_activation="silu", dim=dim,
                             kind="layer", **{k: leaves[k] for k in VECTORS})
        grads = torch.autograd.grad((r, n), list(leaves.values()), (dr, dn))
        for k, g in zip(leaves, grads):
            d = torch.randn_like(t[k])
            d /= d.norm()
            step = 2.0**-6
            up, down = ({**t, k: t[k] + s * step * d} for s in (1, -1))
            slope = float((loss(up) - loss(down)) / (2 * step))
            assert abs(slope - float((g * d).sum())) <= 2e-2 * (1 + float(g.norm())), k


def test_captured(cuda_device):
    """Forward and gradients captured in two graphs that are replayed in turn, with new inputs."""
    made = []
    for dim, shape in ((-1, (2, 50, 256)), (1, (2, 32, 16, 16))):
        t, dr, dn = _inputs(shape, dim, torch.float32, cuda_device, gate="sample", seed=9)
        names = list(t)
        leaves = {k: v.clone().requires_grad_(True) for k, v in t.items()}

        def step(s, dim=dim, dr=dr, dn=dn, names=names):
            r, n = residual_norm(s["x"], s["y"], gate=s["gate"], gate_activation="sigmoid", dim=dim,
                                 **{k: s[k] for k in VECTORS})
            return [r, n, *torch.autograd.grad((r, n), [s[k] for k in names], (dr, dn))]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(leaves)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(leaves)
        made.append((graph, leaves, outs, step))
    for _ in range(3):
        for _, leaves, _, _ in made:
            with torch.no_grad():
                for v in leaves.values():
                    v.mul_(0.9)
        for graph, *_ in made:
            graph.replay()
        torch.cuda.synchronize()
        for _, leaves, outs, step in made:
            fresh = {k: v.detach().clone().requires_grad_(True) for k, v in leaves.items()}
            assert all(torch.equal(a, b) for a, b in zip(outs, step(fresh)))


def test_one_position_equals_the_same_position_of_a_batch(cuda_device):
    """Serving one token gives what the whole prompt gave there, to the order of the channel sums."""
    t, _, _ = _inputs((1, 37, 512), -1, torch.float32, cuda_device, seed=10)
    vec = {k: t[k] for k in VECTORS}
    r, n = residual_norm(t["x"], t["y"], dim=-1, **vec)
    one = residual_norm(t["x"][:, 20:21], t["y"][:, 20:21], dim=-1, **vec)
    torch.testing.assert_close(one[0], r[:, 20:21], rtol=2e-5, atol=2e-5)
    torch.testing.assert_close(one[1], n[:, 20:21], rtol=2e-5, atol=2e-5)


def test_other_types_on_the_device_are_refused(cuda_device):
    x = torch.zeros(2, 4, 3, device=cuda_device)
    with pytest.raises(RuntimeError, match="y must"):
        residual_norm(x, torch.zeros(2, 4, 3))
    with pytest.raises(RuntimeError, match="weights"):
        residual_norm(x, pre_weight=torch.ones(4))
    with pytest.raises(RuntimeError, match="float32"):
        residual_norm(x.double())


@pytest.mark.parametrize("dim, shape", [(-1, (2, 551_000, 2048)), (1, (2, 36, 31_000_004)), (1, (1, 33, 66_000_003))], ids=str)
def test_offsets_past_32_bits(dim, shape, cuda_device):
    """Over 2^31 elements, all zeros but the first and the last positions: those give what a tensor of
    their own gives (bitwise, being the same sums in the same order), gradients included."""
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of device memory")
    dev, half = cuda_device, torch.float16
    C = shape[-1] if dim == -1 else shape[1]
    few = 8

    def ends(t):  # the first positions of the first sample and the last of the last one
        return (t[0, :few], t[-1, -few:]) if dim == -1 else (t[0, :, :few], t[-1, :, -few:])

    g = torch.Generator(device=dev).manual_seed(0)
    full, small = {}, {}
    for k in ("x", "y", "dr", "dn"):
        full[k] = torch.zeros(shape, dtype=half, device=dev)
        for part in ends(full[k]):
            part.copy_(torch.randn(part.shape, device=dev, generator=g))
        small[k] = torch.stack(ends(full[k]))
    w = (1.0 + 0.1 * torch.randn(C, device=dev, generator=g))
    got = []
    for t in (full, small):
        x, y, v = t["x"].requires_grad_(True), t["y"].requires_grad_(True), w.clone().requires_grad_(True)
        r, n = residual_norm(x, y, pre_weight=v, post_weight=w, dim=dim)
        got.append((r, n, *torch.autograd.grad((r, n), (x, y, v), (t["dr"], t["dn"]))))
    for a, b in zip(got[0][:4], got[1][:4]):
        assert torch.equal(torch.stack(ends(a.detach())), b.detach())
    torch.testing.assert_close(got[0][4], got[1][4], rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("leaf", [False, True])
def test_a_forward_derivative_is_refused(leaf, cuda_device):
    """A tangent that the kernels cannot carry must not be read as zero, in whatever input it comes and
    whether gradients are recorded or not."""
    t, _, _ = _inputs((3, 5, 8), -1, torch.float32, cuda_device, gate="full")
    with fwAD.dual_level():
        for k, v in t.items():
            dual = {**t, k: fwAD.make_dual(v.clone().requires_grad_(leaf), torch.ones_like(v))}
            x, y = dual.pop("x"), dual.pop("y")
            for mode in (True, False):
                with torch.set_grad_enabled(mode), pytest.raises(RuntimeError, match="forward-mode"):
                    residual_norm(x, y, dim=-1, gate_activation="sigmoid", **dual)
    residual_norm(t.pop("x"), t.pop("y"), dim=-1, **t)


@pytest.mark.parametrize("shape, dim", [((2, 33, 40), -1), ((2, 40, 33), 1), ((2, 20000, 3), 1)], ids=str)
@pytest.mark.parametrize("gate_mode", [0, 1, 2])
def test_weights_of_a_norm_that_is_not_taken_are_not_used(gate_mode, shape, dim, cuda_device):
    """At the C ABI weights and biases may be given with post_norm or pre_norm 0: outputs and gradients are
    those of a call without them."""
    C, length = (shape[1], shape[2]) if dim == 1 else (shape[2], shape[1])
    t, dr, dn = _inputs(shape, dim, torch.float32, cuda_device, gate=["none", "sample", "full"][gate_mode], seed=13)
    for post, pre in ((0, 1), (1, 0), (0, 0)):
        config = _scx.ResidualNormConfig(batch=shape[0], length=length, channels=C, channels_last=int(dim == -1), gate_mode=gate_mode,
                                         gate_act=1, post_norm=post, pre_norm=pre, eps=1e-5, scale=0.5)
        nbytes = _scx.lib.scx_residual_norm_bwd_workspace_size(ctypes.byref(config))
        got = []
        for given in (True, False):
            r, n, dx, dy = (torch.zeros_like(t["x"]) for _ in range(4))
            stats = torch.zeros(4 * shape[0] * length, device=cuda_device)
            dscale = torch.zeros(C, device=cuda_device)
            dgate = torch.zeros_like(t["gate"]) if gate_mode else None
            ws = torch.zeros(nbytes, dtype=torch.uint8, device=cuda_device)
            keep = {k: t[k].data_ptr() for k in ("post_weight", "post_bias") if post or given}
            keep |= {k: t[k].data_ptr() for k in ("pre_weight", "pre_bias") if pre or given}
            tensors = _scx.ResidualNormTensors(x=t["x"].data_ptr(), y=t["y"].data_ptr(), scale=t["scale"].data_ptr(), r=r.data_ptr(),
                                               n=n.data_ptr(), stats=stats.data_ptr(), **keep,
                                               gate=t["gate"].data_ptr() if gate_mode else None)
            grads = _scx.ResidualNormGrads(dr=dr.data_ptr(), dn=dn.data_ptr() if pre else None, dx=dx.data_ptr(),
                                           dy=dy.data_ptr(), d_scale=dscale.data_ptr(),
                                           dgate=dgate.data_ptr() if gate_mode else None)
            stream = torch.cuda.current_stream().cuda_stream
            assert _scx.lib.scx_residual_norm_fwd(ctypes.byref(config), ctypes.byref(tensors), stream) == 0
            assert _scx.lib.scx_residual_norm_bwd(ctypes.byref(config), ctypes.byref(tensors), ctypes.byref(grads),
                                                  ws.data_ptr(), nbytes, stream) == 0
            torch.cuda.synchronize()
            got.append([r, n, dx, dy, dscale] + ([dgate] if gate_mode else []))
        assert all(torch.equal(a, b) for a, b in zip(*got))
        want = _expected({**t, **({} if post else {"post_weight": None, "post_bias": None})}, dim, dr, dn if pre else None,
                         kind="rms", act="sigmoid", eps=1e-5, number=0.5, post=bool(post), pre=bool(pre))
        _compare("r", got[0][0], want["r"], t, dim)
        _compare("d_scale", got[0][4], want["d_scale"], t, dim)
        if gate_mode:
            _compare("d_gate", got[0][5], want["d_gate"], t, dim)


@pytest.mark.parametrize("shape, dim", [((3, 5, 8), -1), ((2, 32, 4, 4), 1), ((1, 1), -1)], ids=str)
def test_negated_views(shape, dim, cuda_device):
    """Tensors whose sign is a bit of the view (as the imaginary part of a conjugate has) and not of the
    values in memory, among the inputs and the incoming gradients."""
    t, dr, dn = _inputs(shape, dim, torch.float32, cuda_device, gate="full", seed=12)
    flipped = {k: torch._neg_view(-v) for k, v in t.items()}
    assert all(v.is_neg() and torch.equal(v, t[k]) for k, v in flipped.items())
    got = []
    for s, d, e in ((t, dr, dn), (flipped, torch._neg_view(-dr), torch._neg_view(-dn))):
        leaves = {k: v.detach().requires_grad_(True) for k, v in s.items()}
        outs = residual_norm(leaves["x"], leaves["y"], gate=leaves["gate"], gate_activation="sigmoid", dim=dim,
                             **{k: leaves[k] for k in VECTORS})
        got.append([*outs, *torch.autograd.grad(outs, list(leaves.values()), (d, e))])
        with torch.no_grad():
            got[-1] += residual_norm(s["x"], s["y"], dim=dim)
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_tracing_is_refused(cuda_device):
    """A trace would keep the outputs' allocation and not the kernel that fills them."""
    x, y = torch.randn(2, 3, 8, device=cuda_device)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda a, b: residual_norm(a, b, dim=-1), (x, y), check_trace=False)
