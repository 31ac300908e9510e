"""The residual-norm operator in 64 bits, with a bound on the float32 error of each output.

``reference`` works on [positions-first] rows: x, y, gate broadcast to [B, L, C].  Bounds carry each
rounding forward from the formulas.  U = 2^-24 is one float32 rounding; a sum over the channels adds
chains of at most C/8 + 16 terms per thread and tree, so its relative error (of the sum of
magnitudes) is S = (C/8 + 16) U; a sum over P positions adds chains of at most P/8 + 128.  expf is
within 2 units in the last place, so an activation is within 10 U of its value.
"""

from __future__ import annotations

import torch

U = 2.0**-24


def rows_of(t: torch.Tensor, dim: int) -> torch.Tensor:
    t = t.detach().double()
    if dim == 1 and t.dim() > 2:
        t = t.movedim(1, -1)
    return t.reshape(t.shape[0], -1, t.shape[-1])


def like(rows: torch.Tensor, shape, dim: int) -> torch.Tensor:
    if dim == 1 and len(shape) > 2:
        return rows.reshape(shape[0], *shape[2:], shape[1]).movedim(-1, 1)
    return rows.reshape(shape)


def _mean(t):
    return t.mean(-1, keepdim=True)


def reference(x, y, gate, vec, *, kind, act, eps, number=1.0, post=True, pre=True, dr=None, dn=None):
    """x, y, dr, dn: [B, L, C] float64; gate: None, [B, 1, C] or [B, L, C]; vec: dict of [C] float64 or
    None (post_weight, post_bias, pre_weight, pre_bias, scale).  Returns {name: (value, bound)}."""
    C = x.shape[-1]
    S = (C / 8 + 16) * U
    one = torch.ones((), dtype=torch.float64, device=x.device)
    zero = 0 * one
    center = 1.0 if kind == "layer" else 0.0
    get = lambda k, other: vec[k].double() if vec.get(k) is not None else other  # noqa: E731
    w, b, w2, b2 = get("post_weight", one), get("post_bias", zero), get("pre_weight", one), get("pre_bias", zero)
    scale = get("scale", one) * number

    def hat(v, ev):
        """Normalised v and the bound on it, given the bound on v; also rho and its relative bound."""
        mu = center * _mean(v)
        rho = ((v - mu).square().mean(-1, keepdim=True) + eps).rsqrt()
        emu = center * (S * _mean(v.abs()) + _mean(ev))
        ed = ev + emu + U * (v - mu).abs()
        erho = S / 2 + 6 * U + _mean((v - mu).abs() * ed) * rho * rho + 0.5 * _mean(ed * ed) * rho * rho
        h = (v - mu) * rho
        return h, rho * ed + h.abs() * (erho + 2 * U), rho, erho

    out = {}
    if y is None:
        r, er = x, 0 * x
    else:
        if post:
            h, eh, rho, erho = hat(y, 0 * y)
            z = h * w + b
            ez = w.abs() * eh + 2 * U * ((h * w).abs() + b.abs())
        else:
            h, z, eh, ez, rho, erho = y, y, 0 * y, 0 * y, one, zero
        a, slope, eslope = one, one, zero
        if gate is not None:
            sig = torch.special.expit(gate)
            if act == "none":
                a = gate
            elif act == "sigmoid":
                a, slope, eslope = sig, sig * (1 - sig), 12 * U * sig
            else:
                a, slope, eslope = gate * sig, sig * (1 + gate * (1 - sig)), 16 * U * sig * (1 + gate.abs())
        u = scale * a
        r = x + u * z
        er = u.abs() * ez + 14 * U * (u * z).abs() + U * r.abs()
        out["r"] = (r, er)
    if pre:
        k, ek, rho2, erho2 = hat(r, er)
        out["n"] = (k * w2 + b2, w2.abs() * ek + 2 * U * ((k * w2).abs() + b2.abs()))
    if dr is None and dn is None:
        return out
    P = x.shape[0] * x.shape[1]
    SP = (P / 8 + 128) * U

    def total(v, ev, dims=(0, 1)):
        return v.sum(dims), ev.sum(dims) + SP * v.abs().sum(dims)

    t, et = (dr, 0 * dr) if dr is not None else (0 * x, 0 * x)
    if dn is not None and pre:
        d = dn * w2
        ed = U * d.abs()
        m1, em1 = center * _mean(d), center * (_mean(ed) + S * _mean(d.abs()))
        m2, em2 = _mean(d * k), _mean(ed * k.abs() + d.abs() * ek) + (S + U) * _mean((d * k).abs())
        inner = d - m1 - k * m2
        mag = d.abs() + m1.abs() + (k * m2).abs()
        ei = ed + em1 + k.abs() * em2 + ek * m2.abs() + 4 * U * mag
        t, et = t + rho2 * inner, rho2 * ei + (rho2 * inner).abs() * (erho2 + 2 * U)
        et = et + U * t.abs()
        out["d_pre_weight"] = total(dn * k, dn.abs() * ek + U * (dn * k).abs())
        out["d_pre_bias"] = total(dn, 0 * dn)
    out["d_x"] = (t, et)
    if y is None:
        return out
    dz = t * u
    edz = u.abs() * et + 14 * U * dz.abs()
    if post:
        e = dz * w
        ee = w.abs() * edz + U * e.abs()
        m3, em3 = center * _mean(e), center * (_mean(ee) + S * _mean(e.abs()))
        m4, em4 = _mean(e * h), _mean(ee * h.abs() + e.abs() * eh) + (S + U) * _mean((e * h).abs())
        inner = e - m3 - h * m4
        mag = e.abs() + m3.abs() + (h * m4).abs()
        ei = ee + em3 + h.abs() * em4 + eh * m4.abs() + 4 * U * mag
        out["d_y"] = (rho * inner, rho * ei + (rho * inner).abs() * (erho + 2 * U))
        out["d_post_weight"] = total(dz * h, edz * h.abs() + dz.abs() * eh + U * (dz * h).abs())
        out["d_post_bias"] = total(dz, edz)
    else:
        out["d_y"] = (dz, edz)
    v, ev = t * a * z, (a * z).abs() * et + (t * a).abs() * ez + 14 * U * (t * a * z).abs()
    value, bound = total(v, ev)
    out["d_scale"] = (value * number, bound * abs(number) + 2 * U * (value * number).abs())
    if gate is not None:
        tz, etz = t * z, z.abs() * et + t.abs() * ez + U * (t * z).abs()
        if gate.shape[1] == 1 and x.shape[1] != 1:
            tz, etz = tz.sum(1, keepdim=True), etz.sum(1, keepdim=True) + SP * tz.abs().sum(1, keepdim=True)
        f = scale * slope
        out["d_gate"] = (tz * f, f.abs() * etz + tz.abs() * (scale.abs() * eslope + 4 * U * f.abs()))
    return out


def within(got: torch.Tensor, value: torch.Tensor, bound: torch.Tensor) -> bool:
    """got (of any type) within its bound of value: the float32 bound, one rounding to got's type of
    what was computed, and that type's smallest steps."""
    info = torch.finfo(got.dtype)
    limit = 1.05 * bound * (1 + info.eps) + info.eps / 2 * value.abs() * 1.01 + 2 * info.smallest_normal * info.eps
    return bool(((got.detach().double() - value).abs() <= limit).all())
