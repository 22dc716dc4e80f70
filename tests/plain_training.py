"""The training operators in 64 bits, for the tests."""
from __future__ import annotations

import math

import numpy as np
import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}      # a rounding, relative to the value
U32 = 2.0 ** -24


def layer_norm(x, weight, bias, eps):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    z = (x - mean) / torch.sqrt((x - mean).square().mean(-1, keepdim=True) + eps)
    return z if weight is None else z * weight.double() + (0 if bias is None else bias.double())


def layer_norm_gradient(dy, x, weight, eps):
    """(dx, dweight, dbias) and what bounds their rounding errors: the sums of the magnitudes of their terms."""
    x, dy = x.double(), dy.double()
    c = x.shape[-1]
    x, dy = x.reshape(-1, c), dy.reshape(-1, c)
    mean = x.mean(-1, keepdim=True)
    r = 1.0 / torch.sqrt((x - mean).square().mean(-1, keepdim=True) + eps)
    z = (x - mean) * r
    g = dy if weight is None else dy * weight.double()
    dx = r * (g - g.mean(-1, keepdim=True) - z * (g * z).mean(-1, keepdim=True))
    # z is off by the rounding of x - mean, which is relative to |x| + mean |x|
    dz = r * (x.abs() + x.abs().mean(-1, keepdim=True)) + z.abs()
    size = r * (g.abs() + g.abs().mean(-1, keepdim=True) + dz * (g.abs() * z.abs()).mean(-1, keepdim=True) + z.abs() * (g.abs() * dz).mean(-1, keepdim=True))
    return (dx, (dy * z).sum(0), dy.sum(0)), (size, (dy.abs() * dz).sum(0), dy.abs().sum(0))


def philox(block, offset, seed):
    """Four words for each block number: Philox-4x32-10 (Salmon et al., SC 2011) on Python-sized integers in numpy."""
    low = np.uint64(0xFFFFFFFF)
    block = np.asarray(block, dtype=np.uint64)
    c = [block & low, block >> np.uint64(32), np.full_like(block, offset & 0xFFFFFFFF), np.full_like(block, offset >> 32)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, -1)


def kept(shape, shared_dim, p, rng):
    """The mask as it broadcasts against `shape`."""
    shape = list(shape)
    if shared_dim is not None:
        shape[shared_dim] = 1
    n = math.prod(shape)
    words = philox(np.arange((n + 3) // 4, dtype=np.uint64), rng[1], rng[0]).reshape(-1)[:n]
    return torch.from_numpy(words >= np.uint64(int(p * 2 ** 32 + 0.5))).view(shape)


def feed_forward(x, w_in, w_out):
    return feed_forward_pass(x, w_in, w_out)[0]


def feed_forward_gradient(dy, x, w_in, w_out):
    """(dx, dw_in, dw_out)."""
    return feed_forward_pass(x, w_in, w_out, dy)[1:4]


def feed_forward_pass(x, w_in, w_out, dy=None, operand=0.0, gate=0.0, sums=0.0):
    """(y, dx, dw_in, dw_out) and, for each, what the roundings in between can move it by at the very worst: h, da and db are off by
    `operand` of themselves, by what an error of `gate` in sigmoid(a) makes of them, and by what a, b and dh bring, sums that are off by `sums` of
    their terms' magnitudes (|silu'| < 1.1, |silu''| <= 0.5)."""
    shape, c = x.shape, x.shape[-1]
    x, wi, wo = x.double().reshape(-1, c), w_in.double(), w_out.double()
    a, b = (x @ wi.t()).chunk(2, -1)
    s = torch.sigmoid(a)
    h = a * s * b
    da0, db0 = (sums * (x.abs() @ wi.abs().t())).chunk(2, -1)
    dh_off = operand * h.abs() + gate * (a * b).abs() + 1.1 * b.abs() * da0 + (a * s).abs() * db0
    out, room = [(h @ wo.t()).reshape(shape)], [(dh_off @ wo.abs().t()).reshape(shape)]
    if dy is not None:
        dy = dy.double().reshape(-1, c)
        g = dy @ wo
        dab = torch.cat((g * b * s * (1 + a * (1 - s)), g * a * s), -1)
        off = operand * dab.abs() + gate * torch.cat(((g * b).abs() * (1 + a.abs()), (g * a).abs()), -1)
        dg = sums * (dy.abs() @ wo.abs())
        off = off + torch.cat((1.1 * b.abs() * dg + 1.1 * g.abs() * db0 + 0.5 * (g * b).abs() * da0, (a * s).abs() * dg + 1.1 * g.abs() * da0), -1)
        out += [(dab @ wi).reshape(shape), dab.t() @ x, dy.t() @ h]
        room += [(off @ wi.abs()).reshape(shape), off.t() @ x.abs(), dy.abs().t() @ dh_off]
    return (*out, *room) if dy is not None else (out[0], room[0])
