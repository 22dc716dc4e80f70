"""What lies between two blocks of a residual stream, a linear layer with its tail, and rows in 8 bits, in 64 bits, for the tests."""
from __future__ import annotations

import math

import torch


def kept(x):
    """What 8 bits hold of x (..., C), and the byte of each group: the step is the power of two for which a group's largest magnitude rounds to at most 127."""
    c = x.shape[-1]
    wide = torch.nn.functional.pad(x.double(), (0, -c % 32)).unflatten(-1, (-1, 32))
    top = wide.abs().amax(-1, keepdim=True)
    finite = torch.isfinite(wide).all(-1, keepdim=True)
    fraction, exponent = torch.frexp(torch.where(finite, top, 1.0))
    exponent = exponent - 7 + (fraction * 128 >= 127.5)                # of the step
    byte = (exponent + 133).clamp(max=254)
    byte = torch.where((byte < 8) | (top == 0), 0, byte)
    step = torch.ldexp(torch.ones_like(top), byte - 133)
    value = torch.where(byte == 0, 0.0, (wide / step).round().clamp(-127, 127) * step)
    value = torch.where(finite, value, math.nan)
    return value.flatten(-2)[..., :c], torch.where(finite, byte, 255).squeeze(-1).to(torch.uint8)


def shared(table, shape, samples):
    """Rows of a table (groups, L, ...) as the rows of a stream (groups * samples, L, C) take them."""
    if samples == 1:
        return table.double().reshape(*shape[:-1], table.shape[-1])
    t = table.double().reshape(-1, 1, shape[-2], table.shape[-1])
    return t.expand(-1, samples, -1, -1).reshape(*shape[:-1], table.shape[-1])


def over_samples(rows, like, samples):
    """Sums of a stream's rows over the samples that share a row of `like`."""
    if samples == 1:
        return rows.reshape(like.shape[:-1] + rows.shape[-1:])
    l = rows.shape[-2]
    return rows.reshape(-1, samples, l, rows.shape[-1]).sum(1).reshape(like.shape[:-1] + rows.shape[-1:])


def residual(x, u, gate, scale, samples):
    """(r, the sum of its terms' magnitudes)."""
    base = u if x is None else x
    r = torch.zeros(base.shape, dtype=torch.float64, device=base.device)
    size = r.clone()
    if x is not None:
        t = x.double() if scale is None else x.double() * scale.double()
        r, size = r + t, size + t.abs()
    if u is not None:
        t = u.double() if gate is None else u.double() * torch.sigmoid(shared(gate, base.shape, samples))
        r, size = r + t, size + t.abs()
    return r, size


def norm_factor(shape, weight, gate_shift, samples):
    """(m, v) of y = m LayerNorm(r) + v."""
    c = shape[-1]
    if gate_shift is not None:
        t = shared(gate_shift, shape, samples)
        return torch.sigmoid(t[..., :c]), t[..., c:]
    return (1.0 if weight is None else weight.double()), 0.0


def statistics(r, eps):
    r = r.double()
    mean = r.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((r - mean).square().mean(-1, keepdim=True) + eps)
    z = (r - mean) * rstd
    # z is off by the rounding of r - mean, which is relative to |r| + mean |r|
    return z, rstd, rstd * (r.abs() + r.abs().mean(-1, keepdim=True)) + z.abs()


def residual_norm_gradient(dr, dy, r, u, gate, x, scale, weight, gate_shift, samples, eps):
    """{name: (gradient, what bounds its rounding errors: the sums of the magnitudes of its terms)}."""
    shape = r.shape
    t = torch.zeros(shape, dtype=torch.float64, device=r.device) if dr is None else dr.double()
    size = t.abs()
    out = {}
    if dy is not None:
        z, rstd, dz = statistics(r, eps)
        m, _ = norm_factor(shape, weight, gate_shift, samples)
        d = dy.double()
        g = d * m
        t = t + rstd * (g - g.mean(-1, keepdim=True) - z * (g * z).mean(-1, keepdim=True))
        size = size + rstd * (g.abs() + g.abs().mean(-1, keepdim=True) + dz * (g.abs() * z.abs()).mean(-1, keepdim=True)
                              + z.abs() * (g.abs() * dz).mean(-1, keepdim=True))
        if gate_shift is not None:
            slope = (shared(gate_shift, shape, samples)[..., :shape[-1]]).sigmoid()
            slope = slope * (1 - slope)
            pair = lambda a, b: torch.cat((over_samples(a, gate_shift, samples), over_samples(b, gate_shift, samples)), -1)
            out["gate_shift"] = pair(d * z * slope, d), pair(d.abs() * dz * slope, d.abs())
        else:
            rows = lambda a: a.reshape(-1, shape[-1]).sum(0)
            out["weight"], out["bias"] = (rows(d * z), rows(d.abs() * dz)), (rows(d), rows(d.abs()))
    s = 1.0 if gate is None else torch.sigmoid(shared(gate, shape, samples))
    k = 1.0 if scale is None else scale.double()
    out["x"], out["u"] = (t * k, size * abs(k)), (t * s, size * s)
    if gate is not None and u is not None:
        slope = s * (1 - s)
        out["gate"] = over_samples(t * u.double() * slope, gate, samples), over_samples(size * (u.double() * slope).abs(), gate, samples)
    if scale is not None and x is not None:
        out["scale"] = (t * x.double()).reshape(-1, shape[-1]).sum(0), (size * x.double().abs()).reshape(-1, shape[-1]).sum(0)
    return out


FUNCTIONS = {
    None: lambda z: z,
    "sigmoid": torch.sigmoid,
    "silu": lambda z: z * torch.sigmoid(z),
    "gelu": lambda z: 0.5 * z * torch.erfc(-z / math.sqrt(2.0)),
    "relu": torch.relu,
}


def linear(x, w, bias, activation, residual=None, dy=None):
    """(y, dx, dw, db) and z."""
    f = FUNCTIONS[activation]
    with torch.enable_grad():
        x, w = x.double().detach().requires_grad_(), w.double().detach().requires_grad_()
        b = torch.zeros(w.shape[0], dtype=torch.float64, device=w.device) if bias is None else bias.double().detach()
        b.requires_grad_()
        z = x @ w.t() + b
        y = f(z)
        grads = () if dy is None else torch.autograd.grad(y, [x, w, b], dy.double())
    y = y.detach() if residual is None else y.detach() + residual.double()
    return (y, *grads), z.detach()


def slope(z, activation):
    """f'(z).  (1 - sigmoid(z) is sigmoid(-z): the difference has no digits left where a gate is wide open.)"""
    if activation in ("sigmoid", "silu"):
        s, shut = torch.sigmoid(z), torch.sigmoid(-z)
        return s * shut if activation == "sigmoid" else s + z * s * shut
    with torch.enable_grad():
        z = z.detach().requires_grad_()
        return torch.autograd.grad(FUNCTIONS[activation](z).sum(), z)[0]
