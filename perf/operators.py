"""Cases of the training-step and block operators: the global gradient norm, clipping, the
Adam step that applies the clipping factor, and the norms before and after a block fused with
the block's gate and residual scale.

With ``own`` false, ``run`` computes a case in elementary torch operations; with ``own`` true
it makes the calls a user makes of ``optim_ops`` and ``residual_norm_ops``.
"""

import math
import random
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
LR, BETA1, BETA2, ADAM_EPS, WEIGHT_DECAY = 2.0e-4, 0.9, 0.999, 1.0e-8, 1.0e-4
NORM_EPS = 1.0e-5


def _package():
    path = str(Path(__file__).resolve().parents[1] / "birensupa-spectralconv_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import optim_ops
    import residual_norm_ops

    return optim_ops, residual_norm_ops


# --------------------------------------------------------------------------- cases


def _fno(name, op, width, modes, tensors, **more):
    return {"name": name, "op": op, "params": "fno", "width": width, "modes": modes, "tensors": tensors,
            "dtype": "float32", **more}


def _block(name, **case):
    base = {"op": "block", "layout": "field", "kind": "rms", "dtype": "float32", "gate": "none", "act": "none",
            "scale": True, "bias": False, "train": False, "lead": 1, "length": 1, "height": 1, "width": 1}
    return {"name": name, **base, **case}


def listed():
    return [
        # the gradient of the FNO-NS model (width 32, modes 12, 4 layers, every parameter): the norm that a
        # training loop logs each step
        _fno("norm_fno_ns", "norm", 32, 12, 22),
        # a logged norm over many bf16 tensors of very different sizes, from single values to millions
        {"name": "norm_ragged_bf16", "op": "norm", "params": "ragged", "tensors": 61, "largest": 9_000_001, "seed": 3,
         "dtype": "bfloat16", "bucket": False},
        # clipping in front of an optimizer: the layers of a width-64, modes-32 FNO, beyond L2
        _fno("clip_fno_w64_m32", "clip", 64, 32, 22),
        # clipping gradients that are views of one flat bucket, as data-parallel training keeps them
        {"name": "clip_bucket", "op": "clip", "params": "ragged", "tensors": 40, "largest": 70_001, "seed": 5,
         "dtype": "float32", "bucket": True},
        # one optimizer step of the FNO-NS model with its lift frozen, the smallest training there is here
        _fno("adam_fno_ns", "adam", 32, 12, 20, clip=True, decoupled=False),
        # one optimizer step of the width-64, modes-32 model
        _fno("adam_fno_w64_m32", "adam", 64, 32, 20, clip=True, decoupled=True),
        # bf16 parameters of very different sizes with fp32 moments, no clipping
        {"name": "adam_ragged_bf16", "op": "adam", "params": "ragged", "tensors": 17, "largest": 4_000_003, "seed": 7,
         "dtype": "bfloat16", "bucket": False, "clip": False, "decoupled": True},
        # serving one token: a block's output joins the residual stream and the next block's input is normed
        _block("block_token_bf16", layout="token", dtype="bfloat16", channels=4096),
        # serving the FNO-NS grid at its batch of 20, one gate per sample and channel
        _block("block_fno_ns", lead=20, channels=32, height=64, width=64, gate="sample", act="sigmoid"),
        # a training pass on the 256 x 256 grid, gated per element: the largest
        _block("block_train_256", lead=16, channels=64, height=256, width=256, gate="full", act="sigmoid", train=True),
        # a training pass on an irregular grid, LayerNorm with biases, one gate per sample and channel
        _block("block_train_irregular", lead=7, channels=36, height=96, width=160, kind="layer", bias=True,
               gate="sample", act="silu", train=True),
        # a training pass over tokens in bf16
        _block("block_train_tokens", layout="token", lead=2, length=4096, channels=2048, dtype="bfloat16",
               gate="full", act="silu", train=True),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "clip", "adam", "block", "block", "block"])
    if op != "block":
        if rng.random() < 0.35:
            case = _fno("", op, rng.choice([16, 20, 24, 32, 36, 48, 64]), rng.randint(5, 32),
                        rng.randint(10, 20 if op == "adam" else 22))
        else:
            case = {"op": op, "params": "ragged", "tensors": rng.randint(1, 19 if op == "adam" else 60),
                    "largest": _log_int(rng, 1000, 5_000_000), "seed": rng.randint(0, 9999),
                    "dtype": rng.choice(["float32", "bfloat16"] if op != "norm" else ["float32", "bfloat16", "float16"]),
                    "bucket": rng.random() < 0.4}
        if op == "adam":
            case.update(clip=rng.random() < 0.6, decoupled=rng.random() < 0.5)
    else:
        case = _block("", kind=rng.choice(["rms", "layer"]), dtype=rng.choice(["float32", "bfloat16", "float16"]),
                      gate=rng.choice(["none", "sample", "full"]), act=rng.choice(["none", "sigmoid", "silu"]),
                      scale=rng.random() < 0.7, bias=rng.random() < 0.4, train=rng.random() < 0.6)
        if rng.random() < 0.5:
            case.update(layout="token", lead=_log_int(rng, 1, 32), channels=_log_int(rng, 8, 8192))
            case["length"] = _log_int(rng, 1, max(1, min(8192, 30_000_000 // (case["lead"] * case["channels"]))))
        else:
            case.update(lead=rng.randint(1, 20), channels=_log_int(rng, 4, 160), height=_log_int(rng, 1, 256))
            room = 30_000_000 // (case["lead"] * case["channels"] * case["height"])
            case["width"] = _log_int(rng, 1, max(1, min(256, room)))
    case.pop("name", None)
    return case


# --------------------------------------------------------------------------- inputs


def _param_shapes(case):
    """[(shape, complex)] of the case's parameters."""
    if case["params"] == "fno":
        w, m = case["width"], case["modes"]
        shapes = [((w, 12), False), ((w,), False)]
        for _ in range(4):
            shapes += [((w, w, m, m), True), ((w, w, m, m), True), ((w, w), False), ((w,), False)]
        shapes += [((128, w), False), ((128,), False), ((1, 128), False), ((1,), False)]
        return shapes[len(shapes) - case["tensors"]:]
    rng = random.Random(case["seed"])
    sizes = [int(round(math.exp(rng.uniform(0.0, math.log(case["largest"]))))) for _ in range(case["tensors"] - 1)]
    sizes.insert(rng.randint(0, len(sizes)), case["largest"])
    return [((n,), False) for n in sizes]


def _count(shapes):
    return sum(math.prod(s) * (2 if c else 1) for s, c in shapes)


def _tensor_list(case, g, dev, scales=None, dtype=None, square=False):
    """One tensor per parameter, normal values times a scale of the tensor's own; views of one
    flat buffer where the case keeps a bucket."""
    dtype = dtype or DTYPES[case["dtype"]]
    shapes = _param_shapes(case)
    sizes = [math.prod(s) * (2 if c else 1) for s, c in shapes]
    flat = torch.randn(sum(sizes), generator=g, device=dev)
    parts = list(flat.split(sizes))
    if scales is not None:
        parts = [p * s for p, s in zip(parts, scales)]
    if square:
        parts = [p * p for p in parts]
    parts = [p.to(dtype) for p in parts]
    parts = list(torch.cat(parts).split(sizes)) if case.get("bucket") else [p.clone() for p in parts]
    return [torch.view_as_complex(p.view(*s, 2)) if c else p.view(s) for p, (s, c) in zip(parts, shapes)]


def _optim_inputs(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    rng = random.Random(seed)
    n = case["tensors"]
    scales = [10.0 ** rng.uniform(-4.0, -1.0) for _ in range(n)]
    grads = _tensor_list(case, g, dev, scales)
    rough = math.sqrt(sum(s * s * t.numel() * (2 if t.is_complex() else 1) for s, t in zip(scales, grads)))
    state = {"case": case, "grads": grads, "max_norm": 0.3 * rough}
    if case["op"] == "adam":
        state["params"] = _tensor_list(case, g, dev, [0.05] * n)
        state["m"] = _tensor_list(case, g, dev, [0.3 * s for s in scales], torch.float32)
        state["v"] = _tensor_list(case, g, dev, scales, torch.float32, square=True)
        # the moments of complex parameters are kept as complex tensors, the squares per component
        state["steps"] = torch.full((n,), float(rng.randint(0, 2000)), device=dev)
        state["step_list"] = list(state["steps"].unbind())
    return state


def _block_shape(case):
    if case["layout"] == "token":
        return (case["lead"], case["length"], case["channels"])
    return (case["lead"], case["channels"], case["height"], case["width"])


def _block_inputs(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    shape, c, dtype = _block_shape(case), case["channels"], DTYPES[case["dtype"]]

    def normal(*s, mean=0.0, std=1.0, to=dtype):
        return torch.randn(*s, generator=g, device=dev).mul_(std).add_(mean).to(to)

    state = {"case": case, "x": normal(*shape, std=1.5), "y": normal(*shape, mean=0.2, std=0.7),
             "pre_weight": normal(c, mean=1.0, std=0.1, to=torch.float32),
             "post_weight": normal(c, mean=1.0, std=0.1, to=torch.float32), "pre_bias": None, "post_bias": None,
             "gate": None, "scale": None}
    if case["bias"]:
        state["pre_bias"] = normal(c, std=0.1, to=torch.float32)
        state["post_bias"] = normal(c, std=0.1, to=torch.float32)
    if case["gate"] == "sample":
        state["gate"] = normal(case["lead"], c)
    elif case["gate"] == "full":
        state["gate"] = normal(*shape)
    if case["scale"]:
        state["scale"] = normal(c, mean=0.5, std=0.1, to=torch.float32)
    if case["train"]:
        state["dr"] = normal(*shape)
        state["dn"] = normal(*shape)
        for k in _leaves(case):
            state[k].requires_grad_(True)
    return state


def _leaves(case):
    names = ["x", "y", "pre_weight", "post_weight"]
    if case["bias"]:
        names += ["pre_bias", "post_bias"]
    if case["gate"] != "none":
        names.append("gate")
    if case["scale"]:
        names.append("scale")
    return names


def prepare(case, seed):
    return (_block_inputs if case["op"] == "block" else _optim_inputs)(case, seed)


# --------------------------------------------------------------------------- the passes


def _real(t):
    return torch.view_as_real(t) if t.is_complex() else t


def _plain_norm(grads):
    return torch.stack([(_real(g).float() * _real(g).float()).sum(dtype=torch.float64) for g in grads]).sum().sqrt().float()


def _plain_scale(g, factor):
    _real(g).copy_(_real(g).float() * factor)


def _plain_clip(grads, max_norm):
    total = _plain_norm(grads)
    factor = torch.clamp(max_norm / (total + 1.0e-6), max=1.0)
    [_plain_scale(g, factor) for g in grads]
    return total


def _plain_adam_one(p, g, m, v, step, factor, decoupled):
    p, g, m, v = _real(p), _real(g), _real(m), _real(v)
    step.add_(1.0)
    p32, g32 = p.float(), g.float() * factor
    if decoupled:
        p32 = p32 * (1.0 - LR * WEIGHT_DECAY)
    else:
        g32 = g32 + WEIGHT_DECAY * p32
    m.copy_(BETA1 * m + (1.0 - BETA1) * g32)
    v.copy_(BETA2 * v + (1.0 - BETA2) * g32 * g32)
    t = step.double()
    size = (LR / (1.0 - BETA1**t)).float()
    root = (1.0 / (1.0 - BETA2**t).sqrt()).float()
    p.copy_(p32 - size * m / (v.sqrt() * root + ADAM_EPS))


def _run_optim(s):
    case = s["case"]
    if case["op"] == "norm":
        if own:
            return _package()[0].grad_norm(s["grads"])
        return _plain_norm(s["grads"])
    if case["op"] == "clip":
        limit = s["max_norm"]
        s["max_norm"] *= 0.999  # a limit that falls from step to step: the next pass over these gradients clips too
        total = _package()[0].clip_grads_(s["grads"], limit) if own else _plain_clip(s["grads"], limit)
        return {"grads": s["grads"], "norm": total}
    limit = s["max_norm"] if case["clip"] else None
    if own:
        total = _package()[0].adam_step_(s["params"], s["grads"], s["m"], s["v"], s["step_list"], lr=LR,
                                         betas=(BETA1, BETA2), eps=ADAM_EPS, weight_decay=WEIGHT_DECAY,
                                         decoupled=case["decoupled"], max_norm=limit)
    else:
        total, factor = None, 1.0
        if limit is not None:
            total = _plain_norm(s["grads"])
            factor = torch.clamp(limit / (total + 1.0e-6), max=1.0)
        [_plain_adam_one(*t, factor, case["decoupled"])
         for t in zip(s["params"], s["grads"], s["m"], s["v"], s["step_list"])]
    out = {"params": s["params"], "m": s["m"], "v": s["v"], "steps": s["steps"]}
    if total is not None:
        out["norm"] = total
    return out


def _plain_channel_norm(t, kind, weight, bias, dim):
    shape = [1] * t.dim()
    shape[dim] = t.shape[dim]
    if kind == "layer":
        t = t - t.mean(dim, keepdim=True)
    t = t / torch.sqrt((t * t).mean(dim, keepdim=True) + NORM_EPS) * weight.view(shape)
    return t + bias.view(shape) if bias is not None else t


def _plain_block(s):
    case = s["case"]
    dim = 1 if case["layout"] == "field" else 2
    x = s["x"].float()
    u = _plain_channel_norm(s["y"].float(), case["kind"], s["post_weight"], s["post_bias"], dim)
    if s["scale"] is not None:
        shape = [1] * x.dim()
        shape[dim] = x.shape[dim]
        u = u * s["scale"].view(shape)
    if s["gate"] is not None:
        a = s["gate"].float()
        if case["act"] != "none":
            sig = 1.0 / (1.0 + torch.exp(-a))
            a = a * sig if case["act"] == "silu" else sig
        if case["gate"] == "sample":
            a = a[:, :, None, None] if dim == 1 else a[:, None, :]
        u = u * a
    r = x + u
    n = _plain_channel_norm(r, case["kind"], s["pre_weight"], s["pre_bias"], dim)
    return r.to(s["x"].dtype), n.to(s["x"].dtype)


def _run_block(s):
    case = s["case"]
    if own:
        r, n = _package()[1].residual_norm(
            s["x"], s["y"], pre_weight=s["pre_weight"], pre_bias=s["pre_bias"], post_weight=s["post_weight"],
            post_bias=s["post_bias"], gate=s["gate"], gate_activation=case["act"], scale=s["scale"],
            kind=case["kind"], eps=NORM_EPS, dim=1 if case["layout"] == "field" else -1)
    else:
        r, n = _plain_block(s)
    out = {"r": r, "n": n}
    if case["train"]:
        names = _leaves(case)
        grads = torch.autograd.grad((r, n), [s[k] for k in names], (s["dr"], s["dn"]))
        out.update({"d_" + k: v for k, v in zip(names, grads)})
    return out


def run(state):
    return (_run_block if state["case"]["op"] == "block" else _run_optim)(state)


# --------------------------------------------------------------------------- the work


def work(case):
    if case["op"] == "block":
        n = math.prod(_block_shape(case))
        e = 4 if case["dtype"] == "float32" else 2
        full = 1 if case["gate"] == "full" else 0
        arrays = 4 + full  # x, y and a gate per element in, r and n out
        if case["train"]:
            arrays += 4 + full  # the gradients of r and n in, those of x, y and the gate out
        sample = 2 * case["lead"] * case["channels"] if case["gate"] == "sample" else 0
        return {"bytes": e * (n * arrays + sample) + 32 * case["channels"], "flops": n * (50 if case["train"] else 16)}
    n = _count(_param_shapes(case))
    e = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "norm":
        return {"bytes": e * n, "flops": 2 * n}
    if case["op"] == "clip":
        return {"bytes": 2 * e * n, "flops": 3 * n}
    return {"bytes": (3 * e + 16) * n, "flops": 16 * n}


# --------------------------------------------------------------------------- 64-bit values


def _f64(t):
    return _real(t.detach()).double()


def _like(values, t):
    return torch.view_as_complex(values.contiguous()) if t.is_complex() else values


def _exact_optim(case, seed):
    s = _optim_inputs(case, seed)
    grads = [_f64(g) for g in s["grads"]]
    total = math.sqrt(sum(float((g * g).sum()) for g in grads))
    if case["op"] == "norm":
        return torch.tensor(total, dtype=torch.float64)
    factor = min(1.0, s["max_norm"] / (total + 1.0e-6))
    if case["op"] == "clip":
        return {"grads": [_like(g * factor, t) for g, t in zip(grads, s["grads"])],
                "norm": torch.tensor(total, dtype=torch.float64)}
    out = {"params": [], "m": [], "v": [], "steps": s["steps"] + 1.0}
    if case["clip"]:
        out["norm"] = torch.tensor(total, dtype=torch.float64)
    else:
        factor = 1.0
    for k, g in enumerate(grads):
        p, m, v = _f64(s["params"][k]), _f64(s["m"][k]), _f64(s["v"][k])
        t = float(s["steps"][k]) + 1.0
        g = factor * g
        if not case["decoupled"]:
            g = g + WEIGHT_DECAY * p
        m = m + (1.0 - BETA1) * (g - m)
        v = v + (1.0 - BETA2) * (g.square() - v)
        mh, vh = m / -math.expm1(t * math.log(BETA1)), v / -math.expm1(t * math.log(BETA2))
        p = p - LR * mh / (vh.sqrt() + ADAM_EPS) - (LR * WEIGHT_DECAY * p if case["decoupled"] else 0.0)
        for name, value in (("params", p), ("m", m), ("v", v)):
            out[name].append(_like(value, s[name][k]))
    return out


def _exact_block(case, seed):
    """Forward and hand-derived gradients in 64 bits, channels moved last."""
    s = _block_inputs(case, seed)
    field, c = case["layout"] == "field", case["channels"]

    def rows(t):
        t = t.detach().double()
        return t.movedim(1, -1).reshape(case["lead"], -1, c) if field else t.reshape(case["lead"], -1, c)

    def back(t):
        shape = _block_shape(case)
        return t.reshape(shape[0], *shape[2:], c).movedim(-1, 1) if field else t.reshape(shape)

    def vec(name, other):
        return s[name].detach().double() if s[name] is not None else torch.full((c,), other, dtype=torch.float64, device="cuda")

    center = 1.0 if case["kind"] == "layer" else 0.0

    def hat(t):
        t = t - center * t.mean(-1, keepdim=True)
        inv = (t.square().mean(-1, keepdim=True) + NORM_EPS).rsqrt()
        return t * inv, inv

    def through(h, inv, d):
        """Gradient of the normalised values' input, given the gradient d of those values."""
        return inv * (d - center * d.mean(-1, keepdim=True) - h * (d * h).mean(-1, keepdim=True))

    x, y = rows(s["x"]), rows(s["y"])
    w_post, b_post = vec("post_weight", 1.0), vec("post_bias", 0.0)
    w_pre, b_pre, scale = vec("pre_weight", 1.0), vec("pre_bias", 0.0), vec("scale", 1.0)
    one = torch.ones((), dtype=torch.float64, device="cuda")
    a, da = one, one
    if s["gate"] is not None:
        gate = rows(s["gate"]) if case["gate"] == "full" else s["gate"].detach().double()[:, None, :]
        sig = torch.special.expit(gate)
        if case["act"] == "none":
            a = gate
        elif case["act"] == "sigmoid":
            a, da = sig, sig * (1.0 - sig)
        else:
            a, da = gate * sig, sig * (1.0 + gate * (1.0 - sig))
    yh, y_inv = hat(y)
    z = yh * w_post + b_post
    r = x + scale * a * z
    rh, r_inv = hat(r)
    out = {"r": back(r), "n": back(rh * w_pre + b_pre)}
    if not case["train"]:
        return out
    dr, dn = rows(s["dr"]), rows(s["dn"])
    total = dr + through(rh, r_inv, dn * w_pre)
    dz = total * scale * a
    sums = {"pre_weight": dn * rh, "pre_bias": dn, "post_weight": dz * yh, "post_bias": dz, "scale": total * a * z}
    out["d_x"], out["d_y"] = back(total), back(through(yh, y_inv, dz * w_post))
    for k in _leaves(case):
        if k in sums:
            out["d_" + k] = sums[k].sum((0, 1))
        elif k == "gate":
            dg = total * scale * z * da
            out["d_gate"] = back(dg) if case["gate"] == "full" else dg.sum(1)
    return out


def exact(case, seed):
    return (_exact_block if case["op"] == "block" else _exact_optim)(case, seed)
