"""The dense operators in 64 bits, with a bound of each result's error.

``u`` is half a step of the result's type (finfo.eps / 2).  A kernel may differ from the exact
value by
  * the float32 sum of K products: at most (K + 16) * 2^-23 * sum |a_k b_k| (a rounding or a
    truncation, 2^-23 relative, per addition);
  * phi and phi' in float32: (8 + 2 |z|) * 2^-23 * |z| and (8 + 2 |z|) * 2^-23 * (1 + |z|) (the
    exponential's argument is rounded, 2^-23 |z|, and a handful of float32 operations follow);
  * phi and phi' at a z that is off: |phi'| <= 1.13 and |phi''| <= 0.8 for silu and gelu; relu'
    jumps by 1 where z can change sign;
  * the rounding of what is stored (and of dz, dg, du between the products of a backward pass):
    u relative, plus half the smallest subnormal of the type.
Every bound is an elementwise sum of these terms.
"""
import math

import torch

E23 = 2.0 ** -23
HALF_SUBNORMAL = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}


def half_step(dt):
    return torch.finfo(dt).eps / 2


def stored(v, err, dt):
    """Error of v after rounding to dt, v itself being off by err."""
    return err * (1 + half_step(dt)) + v.abs() * half_step(dt) + HALF_SUBNORMAL[dt]


def phi(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z / math.sqrt(2)))
    return z


def slope(z, act):
    if act == "relu":
        return (z > 0).double()
    if act == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z / math.sqrt(2))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


def product(a, b):
    """a b^T and the bound of its float32 sum."""
    return a @ b.t(), (a.shape[1] + 16) * E23 * (a.abs() @ b.abs().t())


def _phi_err(z, ez, act):
    return ez if act == "none" else 1.13 * ez + (8 + 2 * z.abs()) * E23 * z.abs()


def _slope_err(z, ez, act):
    if act == "none":
        return torch.zeros_like(z)
    if act == "relu":
        return (z.abs() <= ez).double()
    return 0.8 * ez + (8 + 2 * z.abs()) * E23 * (1 + z.abs())


def linear(x, w, bias=None, act="none", scale=None, residual=None, out_dtype=None):
    """(out, bound) for 2-D x."""
    dt = out_dtype or x.dtype
    z, ez = product(x.double(), w.double())
    if bias is not None:
        z = z + bias.double()
        ez = ez + E23 * z.abs()
    y, e = phi(z, act), _phi_err(z, ez, act)
    if scale is not None:
        y, e = y * scale.double(), e * scale.double().abs()
        e = e + E23 * y.abs()
    if residual is not None:
        y = y + residual.double()
        e = e + E23 * y.abs()
    return y, stored(y, e, dt)


def linear_backward(g, x, w, bias=None, act="none", scale=None):
    """Dict of (value, bound) for dx, dw, dbias, dscale."""
    dt = x.dtype
    xd, wd, gd = x.double(), w.double(), g.double()
    z, ez = product(xd, wd)
    if bias is not None:
        z = z + bias.double()
        ez = ez + E23 * z.abs()
    gs = gd if scale is None else gd * scale.double()
    dz = gs * slope(z, act)
    e32 = gs.abs() * _slope_err(z, ez, act) + 4 * E23 * dz.abs()
    exact_copy = act == "none" and scale is None and g.dtype == dt
    e16 = torch.zeros_like(dz) if exact_copy else stored(dz, e32, dt)
    M = x.shape[0]
    got = {}

    def rounded(v, err, t):
        return v, stored(v, err, t)

    v, e = product(dz, wd.t())
    got["dx"] = rounded(v, e + e16 @ wd.abs(), dt)
    v, e = product(dz.t(), xd.t())
    got["dw"] = rounded(v, e + e16.t() @ xd.abs(), w.dtype)
    if bias is not None:
        err = e32.sum(0) + (M + 16) * E23 * dz.abs().sum(0)
        got["dbias"] = rounded(dz.sum(0), err, bias.dtype)
    if scale is not None:
        y = phi(z, act)
        err = (gd.abs() * _phi_err(z, ez, act)).sum(0) + (M + 16) * E23 * (gd * y).abs().sum(0)
        got["dscale"] = rounded((gd * y).sum(0), err, scale.dtype)
    return got


def gated(x, wg, wu, act):
    zg, eg = product(x.double(), wg.double())
    zu, eu = product(x.double(), wu.double())
    y, ey = phi(zg, act), _phi_err(zg, eg, act)
    out = y * zu
    e = ey * (zu.abs() + eu) + y.abs() * eu + E23 * out.abs()
    return out, stored(out, e, x.dtype)


def gated_backward(g, x, wg, wu, act):
    dt = x.dtype
    xd, gd = x.double(), g.double()
    zg, eg = product(xd, wg.double())
    zu, eu = product(xd, wu.double())
    y, s = phi(zg, act), slope(zg, act)
    ey, es = _phi_err(zg, eg, act), _slope_err(zg, eg, act)
    dg, du = gd * zu * s, gd * y
    edg = stored(dg, gd.abs() * (eu * s.abs() + (zu.abs() + eu) * es) + 4 * E23 * dg.abs(), dt)
    edu = stored(du, gd.abs() * ey + 4 * E23 * du.abs(), dt)
    got = {}
    a, ea = product(dg, wg.double().t())
    b, eb = product(du, wu.double().t())
    v = a + b
    got["dx"] = (v, stored(v, 2 * (ea + eb) + edg @ wg.double().abs() + edu @ wu.double().abs(), dt))
    for name, d, ed in (("dw_gate", dg, edg), ("dw_up", du, edu)):
        v, e = product(d.t(), xd.t())
        got[name] = (v, stored(v, e + ed.t() @ xd.abs(), dt))
    return got


def assert_within(actual, value_bound, what=""):
    value, bound = value_bound
    a = actual.detach().double()
    assert a.shape == value.shape, f"{what}: shape {tuple(a.shape)} != {tuple(value.shape)}"
    off = (a - value).abs() - bound
    off = torch.where(torch.isfinite(a), off, torch.full_like(off, math.inf))
    if off.numel():
        k = int(off.argmax())
        worst = float(off.flatten()[k])
        assert worst <= 0, (f"{what}: element {k} is {float(a.flatten()[k]):.9g}, expected {float(value.flatten()[k]):.9g} "
                            f"within {float(bound.flatten()[k]):.3g}")
