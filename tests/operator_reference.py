"""Plain 64-bit forms of the operators and the error each kernel may make, element by element.

The allowances follow from the arithmetic, not from observed errors:

* a product accumulated over k terms in FP32, truncation allowed (u = 2^-23), is off by at most
  (k + 2) u |A||B|;
* a rounding to a format is off by at most half a step, finfo.eps / 2 of the value, or half its smallest
  subnormal;
* the kernels' exponential and reciprocal are the hardware's approximations (2 u and u, and the rounding of the
  exponent, 1.2 |x| u), their normal distribution function is off by (12 + z^2 / 2) u of its smaller side, and an
  activation is a few FP32 operations on them: (8 + 4 |z| + |z|^3) u |z| covers each of them (the cube from gelu_tanh's
  argument; gelu's own error is largest against it at z = 0, where 12 u Phi(-|z|) is 6 u), twice that with |z| + 1 its
  slope; both have slopes below 1.2.
"""

from __future__ import annotations

import math

import torch

U = 2.0 ** -23
DTYPES = {"tf32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def value(x, precision):
    """A product's operand in 64 bits (TF32: rounded to 10 fraction bits, nearest even)."""
    if precision != "tf32":
        return x.double()
    mantissa, exponent = torch.frexp(x.double())
    return torch.ldexp(torch.round(mantissa * 2048.0), exponent - 11)


def half_step(x, precision_dtype):
    info = torch.finfo(precision_dtype)
    return x.abs() * (info.eps / 2) + info.tiny * info.eps / 2


def operand_half_step(x, precision):
    """Half a step of the format in which an intermediate enters a product."""
    return x.abs() * 2.0 ** -11 if precision == "tf32" else half_step(x, DTYPES[precision])


def activation(z, name):
    """(act(z), act'(z)) in 64 bits."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z), (z > 0).double()
    if name == "gelu":
        cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
        return z * cdf, cdf + z * torch.exp(-z * z / 2.0) / math.sqrt(2.0 * math.pi)
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1.0 + z * (1.0 - s))
    c = 2.0 * math.sqrt(2.0 / math.pi)
    s = torch.sigmoid(c * (z + 0.044715 * z ** 3))
    return z * s, s + z * s * (1.0 - s) * c * (1.0 + 3.0 * 0.044715 * z ** 2)


def _activation_error(z):
    return (8.0 + 4.0 * z.abs() + z.abs() ** 3) * z.abs() * U


def _slope_error(z):
    return 2.0 * (8.0 + 4.0 * z.abs() + z.abs() ** 3) * (z.abs() + 1.0) * U


def product(a, b):
    """(a @ b, allowance) in 64 bits."""
    return a @ b, (a.shape[-1] + 2) * U * (a.abs() @ b.abs())


def epilogue(a, b, precision, bias=None, act="none", residual=None):
    """{"out": (value, allowance before its last rounding), "preact": ...}"""
    z, tz = product(value(a, precision), value(b, precision))
    if bias is not None:
        z = z + bias.double()
        tz = tz + U * (z.abs() + bias.double().abs())
    out, _ = activation(z, act)
    tol = tz if act == "none" else 1.2 * tz + _activation_error(z)
    if residual is not None:
        out = out + residual.double()
        tol = tol + U * out.abs()
    return {"out": (out, tol), "preact": (z, tz)}


def epilogue_backward(dout, a, b, precision, preact=None, act="none"):
    d = dout.double()
    if act == "none":
        dz, tdz = value(dout, precision), torch.zeros_like(d)
        raw, traw = d, tdz
    else:
        _, slope = activation(preact.double(), act)
        raw = dz = d * slope
        traw = d.abs() * _slope_error(preact.double()) + U * raw.abs()
        tdz = traw + operand_half_step(raw, precision)
    av, bv = value(a, precision), value(b, precision)
    da, tda = product(dz, bv.T)
    db, tdb = product(av.T, dz)
    m = dout.shape[0]
    return {"da": (da, tda + tdz @ bv.abs().T), "db": (db, tdb + av.abs().T @ tdz),
            "dbias": (raw.sum(0), traw.sum(0) + (m + 2) * U * raw.abs().sum(0))}


def grouped(a, b, offsets, precision, out):
    """Rows of no group keep what `out` held."""
    result, tol = out.double().clone(), torch.zeros_like(out, dtype=torch.float64)
    av, bv = value(a, precision), value(b, precision)
    for g, (lo, hi) in enumerate(zip(offsets[:-1], offsets[1:])):
        if lo < hi:
            result[lo:hi], tol[lo:hi] = product(av[lo:hi], bv[g])
    return result, tol


def grouped_backward(dout, a, b, offsets, precision, da):
    dv, av, bv = value(dout, precision), value(a, precision), value(b, precision)
    result, tol = da.double().clone(), torch.zeros_like(da, dtype=torch.float64)
    db, tdb = torch.zeros_like(bv), torch.zeros_like(bv)
    for g, (lo, hi) in enumerate(zip(offsets[:-1], offsets[1:])):
        if lo < hi:
            result[lo:hi], tol[lo:hi] = product(dv[lo:hi], bv[g].T)
            db[g], tdb[g] = product(av[lo:hi].T, dv[lo:hi])
    return (result, tol), (db, tdb)


def cross_entropy(hidden, weight, labels, precision, ignore=-100):
    z, tz = product(value(hidden, precision), value(weight, precision))
    v = z.shape[1]
    lse = torch.logsumexp(z, 1)
    # The sum's relative error: a chain of at most 256 + v / 256 terms with an exponent's rounding each.
    tlse = tz.amax(1) + (600.0 + v / 128.0 + 8.0 * (z.abs().amax(1) + lse.abs())) * U
    kept = labels != ignore
    index = torch.where(kept, labels, torch.zeros_like(labels)).long()[:, None]
    picked, tpicked = z.gather(1, index)[:, 0], tz.gather(1, index)[:, 0]
    zero = torch.zeros_like(lse)
    loss = torch.where(kept, lse - picked, zero)
    return {"lse": (lse, tlse), "loss": (loss, torch.where(kept, tlse + tpicked + U * (lse.abs() + picked.abs()), zero)),
            "z": (z, tz)}


def cross_entropy_backward(grad, hidden, weight, labels, precision, ignore=-100):
    forward = cross_entropy(hidden, weight, labels, precision, ignore)
    (z, tz), (lse, tlse) = forward["z"], forward["lse"]
    kept = labels != ignore
    scale = torch.where(kept, grad.double(), torch.zeros_like(lse))[:, None]
    p = torch.exp(z - lse[:, None])
    hot = torch.zeros_like(p)
    hot[torch.arange(len(labels), device=p.device)[kept], labels[kept].long()] = 1.0
    dz = scale * (p - hot)
    tp = p * (tz + tlse[:, None] + (8.0 + 4.0 * (z - lse[:, None]).abs()) * U)
    tdz = scale.abs() * (tp + 2 * U * (p + hot)) + operand_half_step(dz, precision) * (scale != 0)
    hv, wv = value(hidden, precision), value(weight, precision)
    dh, tdh = product(dz, wv.T)
    dw, tdw = product(hv.T, dz)
    # dH is added up over pieces of the vocabulary: a few more FP32 sums.
    return {"dhidden": (dh, 1.1 * tdh + tdz @ wv.abs().T), "dweight": (dw, tdw + hv.abs().T @ tdz)}


def assert_within(got, expected, allowance, what):
    """|got - expected| <= allowance + the rounding of got's own format, everywhere."""
    assert tuple(got.shape) == tuple(expected.shape), f"{what}: shape {tuple(got.shape)}"
    assert torch.isfinite(got).all(), f"{what}: {int((~torch.isfinite(got)).sum())} values are not finite"
    bound = allowance + half_step(expected.abs() + allowance, got.dtype)
    excess = (got.double() - expected).abs() - bound
    worst = int(excess.argmax())
    assert float(excess.flatten()[worst]) <= 0.0, (
        f"{what}: element {worst} is {float(got.flatten()[worst])}, expected {float(expected.flatten()[worst])} "
        f"+- {float(bound.flatten()[worst])}; {int((excess > 0).sum())} of {excess.numel()} outside")
