"""The training operators of the pair and single tracks, at the sizes a training step calls them with, for timing.

One residual update of a pair stack in training is  z <- z + dropout(Transition(z))  with
Transition = LayerNorm -> gated feed-forward; the same parts serve the single track (384 channels), the token transformer (768)
and K-Fold's own trunk (256).  Three operators, each with its backward pass:

  norm   LayerNorm over the channels:  y, and from dy  dx, d weight, d bias
  ffn    gated feed-forward  y = (silu(x Wa^T) * (x Wb^T)) Wo^T  with [Wa; Wb] = w_in, and from dy  dx, d w_in, d w_out
  drop   dropout whose mask comes from a counter-based generator and is never stored, along with the residual sum, the mask
         shared along rows or columns of the pair tensor or by nothing; and from dy  dx

A pass is one forward and one backward call.  The random numbers of the dropout are the words of Philox-4x32-10 (Salmon, Moraes,
Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011): element e of the (unshared) mask takes word e % 4 of block
e / 4, counter = (block, offset) as two 64-bit numbers, key = seed, and is dropped when the word is below p 2^32.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
EPS = 1e-5
EXPANSION = {128: 4, 256: 4, 384: 4, 768: 2}      # hidden channels of a feed-forward per channel, by track


def listed():
    return [
        # The single track of a small crop in float32: all latency.
        {"name": "norm-64x384-f32", "kind": "norm", "rows": 64, "c": 384, "dtype": "f32", "affine": True},
        # The pair tensor of a small protein, an odd token count.
        {"name": "norm-251p-128", "kind": "norm", "rows": 251 * 251, "c": 128, "dtype": "bf16", "affine": True},
        # The trunk's pair tensor at the usual training crop of 384 tokens.
        {"name": "norm-384p-256", "kind": "norm", "rows": 384 * 384, "c": 256, "dtype": "bf16", "affine": True},
        # The token transformer: 768 channels of 48 diffusion samples, LayerNorm without scale and offset, as AdaLN has it.
        {"name": "norm-48x301x768-f32", "kind": "norm", "rows": 48 * 301, "c": 768, "dtype": "f32", "affine": False},
        # The single track's feed-forward: few rows, wide weights.
        {"name": "ffn-331x384", "kind": "ffn", "rows": 331, "c": 384, "pad": 0.0},
        # The pair track: a small protein, the usual crop, and the largest one trained on.
        {"name": "ffn-251p-128", "kind": "ffn", "rows": 251 * 251, "c": 128, "pad": 0.0},
        {"name": "ffn-384p-128", "kind": "ffn", "rows": 384 * 384, "c": 128, "pad": 0.1},
        # The trunk's 256 channels at the usual crop.
        {"name": "ffn-384p-256", "kind": "ffn", "rows": 384 * 384, "c": 256, "pad": 0.05},
        # Dropout of the single track, every element by itself.
        {"name": "drop-301x384", "kind": "drop", "shape": "1,1,301,384", "share": "none", "p": 0.1, "dtype": "f32"},
        # Row-wise and column-wise dropout of the pair track's triangle updates.
        {"name": "drop-251p-128-rows", "kind": "drop", "shape": "1,251,251,128", "share": "rows", "p": 0.25, "dtype": "bf16"},
        {"name": "drop-768p-128-cols", "kind": "drop", "shape": "1,768,768,128", "share": "columns", "p": 0.25, "dtype": "bf16"},
        # Every element of the trunk's pair tensor by itself.
        {"name": "drop-384p-256", "kind": "drop", "shape": "1,384,384,256", "share": "none", "p": 0.15, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "ffn", "ffn", "drop"])
    if kind == "norm":
        c = rng.choice([64, 128, 256, 384, 768, 1024, rng.randint(9, 1024)])
        return {"kind": kind, "rows": _log_int(rng, 1, 384 * 384 * 256 // c), "c": c, "dtype": rng.choice(["bf16", "bf16", "f32"]),
                "affine": rng.random() < 0.8}
    if kind == "ffn":
        c = rng.choice([128, 128, 256, 256, 384, 768])
        rows = _log_int(rng, 16, 384) ** 2 if c <= 256 else _log_int(rng, 1, 6000)
        return {"kind": kind, "rows": rows + rng.randint(0, 7), "c": c, "pad": round(rng.choice([0.0, rng.uniform(0.0, 0.2)]), 3)}
    share = rng.choice(["none", "rows", "columns"])
    n = _log_int(rng, 8, 340 if share == "none" else 640)
    c = rng.choice([64, 128, 128, 256, rng.randint(5, 200)])
    return {"kind": kind, "shape": f"{rng.choice([1, 1, 2]) if n < 200 else 1},{n},{n},{c}", "share": share, "p": round(rng.uniform(0.02, 0.5), 3),
            "dtype": rng.choice(["bf16", "bf16", "f32"])}


# ------------------------------------------------------------------------------------------------ inputs
def _normal(gen, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device=DEVICE, dtype=dtype)


def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    kind, st = case["kind"], {"case": case}
    if kind == "norm":
        rows, c, dt = case["rows"], case["c"], _dtype(case)
        # a residual stream: channels of different offset and spread
        st["x"] = (_normal(gen, rows, c) * (0.5 + 2.0 * torch.rand(c, generator=gen, device=DEVICE)) + _normal(gen, c)).to(dt)
        st["dy"] = (0.02 * _normal(gen, rows, c)).to(dt)
        st["weight"] = 1.0 + 0.1 * _normal(gen, c) if case["affine"] else None
        st["bias"] = 0.1 * _normal(gen, c) if case["affine"] else None
    elif kind == "ffn":
        rows, c = case["rows"], case["c"]
        hidden = c * EXPANSION[c]
        st["x"] = _normal(gen, rows, c).to(torch.bfloat16)
        st["dy"] = (0.02 * _normal(gen, rows, c)).to(torch.bfloat16)
        if int(case["pad"] * rows):
            st["dy"][rows - int(case["pad"] * rows):] = 0        # padding: nothing comes back through the masked loss
        st["w_in"] = (_normal(gen, 2 * hidden, c) * c ** -0.5).to(torch.bfloat16)
        st["w_out"] = (_normal(gen, c, hidden) * hidden ** -0.5).to(torch.bfloat16)
    else:
        shape, dt = _shape(case), _dtype(case)
        st["x"], st["residual"] = _normal(gen, *shape).to(dt), _normal(gen, *shape).to(dt)
        st["dy"] = (0.02 * _normal(gen, *shape)).to(dt)
        st["rng"] = _stream(seed)
    return st


def _shape(case):
    return tuple(int(v) for v in case["shape"].split(","))


def _stream(seed):
    """(seed, offset) of the case's generator, 63 and 40 bits of the case's seed."""
    s = (int(seed) * 0x5851F42D4C957F2D + 0x14057B7EF767814F) % (1 << 63)
    return s, (s >> 7) % (1 << 40)


def _shared_dim(case):
    return {"none": None, "rows": -3, "columns": -2}[case["share"]]


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_norm(x, weight, bias, dy):
    x32, d = x.float(), dy.float()
    xc = x32 - x32.mean(-1, keepdim=True)
    rstd = torch.rsqrt(xc.square().mean(-1, keepdim=True) + EPS)
    xhat = xc * rstd
    y = xhat if weight is None else xhat * weight + bias
    g = d if weight is None else d * weight
    dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    out = {"y": y.to(x.dtype), "dx": dx.to(x.dtype)}
    if weight is not None:
        out["dweight"], out["dbias"] = (d * xhat).sum(0), d.sum(0)
    return out


def _plain_ffn(x, w_in, w_out, dy):
    x32, d, wi, wo = x.float(), dy.float(), w_in.float(), w_out.float()
    a, b = (x32 @ wi.t()).chunk(2, -1)
    s = 1.0 / (1.0 + torch.exp(-a))
    silu = a * s
    h = silu * b
    y = h @ wo.t()
    dh = d @ wo
    dab = torch.cat((dh * b * (s + silu * (1.0 - s)), dh * silu), -1)
    return {"y": y.to(x.dtype), "dx": (dab @ wi).to(x.dtype), "dw_in": (dab.t() @ x32).to(w_in.dtype), "dw_out": (d.t() @ h).to(w_out.dtype)}


def _plain_words(n, stream):
    """The first n words of the stream, int64."""
    low = 0xFFFFFFFF
    block = torch.arange((n + 3) // 4, device=DEVICE, dtype=torch.int64)
    (seed, offset) = stream
    c0, c1, c2, c3 = block & low, block >> 32, torch.full_like(block, offset & low), torch.full_like(block, offset >> 32)
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (p1 >> 32 & low) ^ c1 ^ k0, p1 & low, (p0 >> 32 & low) ^ c3 ^ k1, p0 & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack((c0, c1, c2, c3), -1).flatten()[:n]


def _plain_drop(x, p, stream, shared_dim, residual=None):
    shape = list(x.shape)
    if shared_dim is not None:
        shape[shared_dim] = 1
    kept = (_plain_words(math.prod(shape), stream) >= int(p * 4294967296.0 + 0.5)).view(shape)
    out = torch.where(kept, x.float() * (1.0 / (1.0 - p)), 0.0)
    return (out if residual is None else residual.float() + out).to(x.dtype)


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    case, x, dy = state["case"], state["x"], state["dy"]
    if own:
        from kfold_b200 import functional as F
        if case["kind"] == "norm":
            y = F.layer_norm(x, state["weight"], state["bias"], EPS)
            dx, dweight, dbias = F.layer_norm_backward(dy, x, state["weight"], EPS, need_bias=state["bias"] is not None)
            return {"y": y, "dx": dx} if dweight is None else {"y": y, "dx": dx, "dweight": dweight, "dbias": dbias}
        if case["kind"] == "ffn":
            y = F.gated_feed_forward(x, state["w_in"], state["w_out"])
            dx, dw_in, dw_out = F.gated_feed_forward_backward(dy, x, state["w_in"], state["w_out"])
            return {"y": y, "dx": dx, "dw_in": dw_in, "dw_out": dw_out}
        share = _shared_dim(case)
        return {"y": F.dropout(x, case["p"], state["rng"], shared_dim=share, residual=state["residual"]),
                "dx": F.dropout(dy, case["p"], state["rng"], shared_dim=share)}
    if case["kind"] == "norm":
        return _plain_norm(x, state["weight"], state["bias"], dy)
    if case["kind"] == "ffn":
        return _plain_ffn(x, state["w_in"], state["w_out"], dy)
    share = _shared_dim(case)
    return {"y": _plain_drop(x, case["p"], state["rng"], share, state["residual"]), "dx": _plain_drop(dy, case["p"], state["rng"], share)}


def work(case):
    """x and dy read, y and dx written (the dropout reads the residual too); weights read and their gradients written."""
    if case["kind"] == "norm":
        n, size = case["rows"] * case["c"], 4 if case["dtype"] == "f32" else 2
        # statistics 4 and y 3 operations an element, the gradient's two sums and itself 9, the weights' gradients 3
        return {"bytes": 4 * n * size + (16 * case["c"] if case["affine"] else 0), "flops": 19 * n}
    if case["kind"] == "ffn":
        rows, c = case["rows"], case["c"]
        weights = 3 * c * c * EXPANSION[c]
        # forward one product with every weight, backward two (hidden channels that a backward pass computes again are not counted)
        return {"bytes": 2 * (4 * rows * c + 2 * weights), "flops": 2 * rows * (3 * weights)}
    n, size = math.prod(_shape(case)), 4 if case["dtype"] == "f32" else 2
    return {"bytes": 5 * n * size, "flops": 3 * n}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_norm(st):
    x, dy = st["x"].double(), st["dy"].double()
    n = x.shape[-1]
    mean = x.sum(-1, keepdim=True) / n
    sigma = torch.sqrt(((x - mean) ** 2).sum(-1, keepdim=True) / n + EPS)
    z = (x - mean) / sigma
    out = {}
    if st["weight"] is None:
        out["y"], g = z, dy
    else:
        out["y"], g = torch.addcmul(st["bias"].double(), z, st["weight"].double()), dy * st["weight"].double()
    # the Jacobian of z is (I - 1 1^T / n - z z^T / n) / sigma
    out["dx"] = (g - g.sum(-1, keepdim=True) / n - z * ((z * g).sum(-1, keepdim=True) / n)) / sigma
    if st["weight"] is not None:
        out["dweight"], out["dbias"] = (z * dy).sum(0), dy.sum(0)
    return out


def _exact_ffn(st):
    w_in, w_out = st["w_in"].double(), st["w_out"].double()
    hidden = w_out.shape[1]
    wa, wb = w_in[:hidden], w_in[hidden:]
    rows = st["x"].shape[0]
    out = {"y": [], "dx": [], "dw_in": torch.zeros_like(w_in), "dw_out": torch.zeros_like(w_out)}
    for r in range(0, rows, 16384):
        x, dy = st["x"][r:r + 16384].double(), st["dy"][r:r + 16384].double()
        u, v = x @ wa.T, x @ wb.T
        gate = torch.sigmoid(u)
        out["y"].append((u * gate * v) @ w_out.T)
        dh = dy @ w_out
        du, dv = dh * v * gate * (1 + u * (1 - gate)), dh * u * gate
        out["dx"].append(du @ wa + dv @ wb)
        out["dw_in"][:hidden] += du.T @ x
        out["dw_in"][hidden:] += dv.T @ x
        out["dw_out"] += dy.T @ (u * gate * v)
    out["y"], out["dx"] = torch.cat(out["y"]), torch.cat(out["dx"])
    return out


def _exact_kept(case, seed):
    """Truth values of the mask, from the generator's definition on unsigned integers."""
    shape = list(_shape(case))
    if case["share"] != "none":
        shape[{"rows": 1, "columns": 2}[case["share"]]] = 1
    n = math.prod(shape)
    key, offset = _stream(seed)
    mask32, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    ctr = np.zeros((4, -(-n // 4)), dtype=np.uint64)
    ctr[0] = np.arange(ctr.shape[1], dtype=np.uint64)
    ctr[1], ctr[0] = ctr[0] >> half, ctr[0] & mask32
    ctr[2], ctr[3] = offset % (1 << 32), offset // (1 << 32)
    keys = [key % (1 << 32), key // (1 << 32)]
    for _ in range(10):
        a, b = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
        ctr = np.stack(((b >> half) ^ ctr[1] ^ np.uint64(keys[0]), b & mask32, (a >> half) ^ ctr[3] ^ np.uint64(keys[1]), a & mask32))
        keys = [(keys[0] + 0x9E3779B9) % (1 << 32), (keys[1] + 0xBB67AE85) % (1 << 32)]
    words = ctr.T.reshape(-1)[:n]
    return torch.from_numpy(words >= np.uint64(math.floor(case["p"] * 2 ** 32 + 0.5))).view(shape)


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "norm":
        return _exact_norm(st)
    if case["kind"] == "ffn":
        return _exact_ffn(st)
    kept = _exact_kept(case, seed).to(DEVICE)
    zero = torch.zeros((), dtype=torch.float64, device=DEVICE)
    grown = lambda t: torch.where(kept, t.double() / (1 - case["p"]), zero)
    return {"y": st["residual"].double() + grown(st["x"]), "dx": grown(st["dy"])}
