"""Operators around the conditioned and pair blocks in training, at the sizes a training step calls them with, for timing.

Three operators, each with its backward pass:

  step    what lies between two blocks of a residual stream x: the block's output u is gated and added, and the stream is normalised for the
          next block.  r = x + sigmoid(gate) u;  y = sigmoid(g) LayerNorm(r) + v with [g | v] = gate_shift, or weight LayerNorm(r) + bias.
          gate and gate_shift are projections of the conditioning, shared by all diffusion samples of a complex, or a sample's own.
          From dr, dy:  dx, du, dgate, d gate_shift (summed over the samples that share them), d weight, d bias.
  linear  y = f(x W^T + b) (+ residual), f one of nothing, sigmoid, silu, gelu, relu; from dy  dx, dW, db.
  keep    activations kept for the backward pass in 8 bits: 32 neighbouring channels share a power of two, a value is a whole number of
          -127 ... 127 of it.  Written beside the operator that makes them, read by the gradients.

The stream is stored in its type, and what is normalised is the stored value; a backward pass that has kept r in 8 bits normalises what these
stand for.  A pass is one forward and one backward call.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
EPS = 1e-5
GROUP = 32                                        # channels that share a power of two


def listed():
    return [
        # The token transformer (768 channels, conditioning in bf16) on a peptide: one sample, all latency.
        {"name": "step-1x64x768", "kind": "step", "groups": 1, "samples": 1, "tokens": 64, "c": 768, "dtype": "bf16", "norm": "adaptive", "gate": True, "keep": False},
        # Five samples of an odd complex that share their conditioning.
        {"name": "step-5x301x768", "kind": "step", "groups": 1, "samples": 5, "tokens": 301, "c": 768, "dtype": "bf16", "norm": "adaptive", "gate": True, "keep": False},
        # A training step's 48 noise levels of a 384-token crop, each with a conditioning of its own; the stream in float32, as under autocast.
        {"name": "step-48x384x768-mixed", "kind": "step", "groups": 48, "samples": 1, "tokens": 384, "c": 768, "dtype": "mixed", "norm": "adaptive", "gate": True, "keep": False},
        # The same noise levels on one shared conditioning, the stream kept in 8 bits.
        {"name": "step-48x384x768-keep", "kind": "step", "groups": 1, "samples": 48, "tokens": 384, "c": 768, "dtype": "bf16", "norm": "adaptive", "gate": True, "keep": True},
        # The pair tensor between two of its updates: sum and LayerNorm with scale and offset, kept in 8 bits.
        {"name": "step-384p-128-keep", "kind": "step", "groups": 1, "samples": 1, "tokens": 384 * 384, "c": 128, "dtype": "bf16", "norm": "affine", "gate": False, "keep": True},
        # The output gate of the token transformer on a small complex: few rows.
        {"name": "linear-301x384-768-sigmoid", "kind": "linear", "rows": 301, "k": 384, "n": 768, "dtype": "bf16", "act": "sigmoid", "bias": True, "residual": False, "keep": False},
        # Gates and shifts of the adaptive norm for the noise levels of a training step.
        {"name": "linear-48x384x384-1536", "kind": "linear", "rows": 48 * 384, "k": 384, "n": 1536, "dtype": "bf16", "act": "none", "bias": True, "residual": False, "keep": False},
        # The language model's pair features through the first layer of their perceptron.
        {"name": "linear-384p-512-256-gelu", "kind": "linear", "rows": 384 * 384, "k": 512, "n": 256, "dtype": "bf16", "act": "gelu", "bias": True, "residual": False, "keep": False},
        # A projection back onto the pair tensor, its rows kept in 8 bits for the weight's gradient.
        {"name": "linear-251p-128-keep", "kind": "linear", "rows": 251 * 251, "k": 128, "n": 128, "dtype": "bf16", "act": "none", "bias": False, "residual": True, "keep": True},
        # The single conditioning in float32.
        {"name": "linear-331x384-384-f32", "kind": "linear", "rows": 331, "k": 384, "n": 384, "dtype": "f32", "act": "silu", "bias": True, "residual": True, "keep": False},
        # A pair tensor of a small protein, and the trunk's at the usual crop, put away and taken back.
        {"name": "keep-251p-128", "kind": "keep", "rows": 251 * 251, "c": 128, "dtype": "bf16"},
        {"name": "keep-384p-256", "kind": "keep", "rows": 384 * 384, "c": 256, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["step", "step", "step", "linear", "linear", "linear", "keep"])
    if kind == "step":
        adaptive = rng.random() < 0.7
        c = rng.choice([128, 128, 256, 384, 768, 768, rng.randint(9, 1024)])
        groups = rng.choice([1, 1, 2, rng.randint(1, 48)])
        samples = rng.choice([1, 1, 5, rng.randint(2, 48)])
        most = max(1, 14_000_000 // (groups * samples * c))
        return {"kind": kind, "groups": groups, "samples": samples, "tokens": _log_int(rng, 1, most), "c": c, "dtype": rng.choice(["bf16", "bf16", "mixed", "f32"]),
                "norm": "adaptive" if adaptive else "affine", "gate": rng.random() < 0.7, "keep": rng.random() < 0.3}
    if kind == "linear":
        k, n = (8 * _log_int(rng, 4, 128) for _ in range(2))
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        most = (19_000_000_000 if dtype == "bf16" else 4_000_000_000) // (k * n)
        return {"kind": kind, "rows": _log_int(rng, 1, min(most, 70_000_000 // max(k, n))), "k": k, "n": n, "dtype": dtype,
                "act": rng.choice(["none", "none", "sigmoid", "silu", "gelu", "relu"]), "bias": rng.random() < 0.6, "residual": rng.random() < 0.4,
                "keep": rng.random() < 0.3}
    c = rng.choice([64, 128, 128, 256, 384, 768, rng.randint(5, 1500)])
    return {"kind": kind, "rows": _log_int(rng, 1, 36_000_000 // c), "c": c, "dtype": rng.choice(["bf16", "bf16", "f32"])}


# ------------------------------------------------------------------------------------------------ inputs
def _types(case):
    """(type of the residual stream, type of what the blocks compute in)."""
    return {"bf16": (torch.bfloat16, torch.bfloat16), "mixed": (torch.float32, torch.bfloat16), "f32": (torch.float32, torch.float32)}[case["dtype"]]


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    normal = lambda *shape: torch.randn(shape, generator=gen, device=DEVICE)
    stream, act = _types(case)
    st = {"case": case}
    if case["kind"] == "step":
        g, s, l, c = (case[k] for k in ("groups", "samples", "tokens", "c"))
        # a residual stream: channels of different offset and spread
        st["x"] = (normal(g, s, l, c) * (0.5 + 2.0 * torch.rand(c, generator=gen, device=DEVICE)) + normal(c)).to(stream)
        st["u"] = normal(g, s, l, c).to(act)
        st["dr"], st["dy"] = (0.02 * normal(g, s, l, c)).to(stream), (0.02 * normal(g, s, l, c)).to(act)
        st["gate"] = (normal(g, l, c) - 1.0).to(act) if case["gate"] else None
        adaptive = case["norm"] == "adaptive"
        st["gate_shift"] = normal(g, l, 2 * c).to(act) if adaptive else None
        st["weight"], st["bias"] = (None, None) if adaptive else (1.0 + 0.1 * normal(c), 0.1 * normal(c))
    elif case["kind"] == "linear":
        rows, k, n = case["rows"], case["k"], case["n"]
        st["x"] = normal(rows, k).to(act)
        st["w"] = (normal(n, k) * k ** -0.5).to(act)
        st["bias"] = 0.5 * normal(n) if case["bias"] else None
        st["residual"] = normal(rows, n).to(act) if case["residual"] else None
        st["dy"] = (0.02 * normal(rows, n)).to(act)
    else:
        rows, c = case["rows"], case["c"]
        st["x"] = (normal(rows, c) * (0.5 + 2.0 * torch.rand(c, generator=gen, device=DEVICE)) + normal(c)).to(act)
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_kept(x):
    """What 8 bits a value hold of x, in 32 bits: the step of a group is the power of two for which its largest magnitude rounds to at most 127."""
    c = x.shape[-1]
    wide = torch.nn.functional.pad(x.float(), (0, -c % GROUP)).unflatten(-1, (-1, GROUP))
    top = wide.abs().amax(-1, keepdim=True)
    step = torch.exp2(torch.floor(torch.log2(top.double())) - 6.0)
    step = torch.where(top >= 127.5 * step, 2.0 * step, step).float()
    return torch.where(top > 0, torch.round(wide / step) * step, 0.0).flatten(-2)[..., :c]


def _plain_step(st):
    case, x, u, gate, gs = st["case"], st["x"].float(), st["u"].float(), st["gate"], st["gate_shift"]
    stream, act = _types(case)
    dy = st["dy"].float()
    sg = None if gate is None else 1.0 / (1.0 + torch.exp(-gate.float().unsqueeze(1)))
    r = (x + (u if sg is None else sg * u)).to(stream)

    def norm(t):
        tc = t - t.mean(-1, keepdim=True)
        rstd = torch.rsqrt(tc.square().mean(-1, keepdim=True) + EPS)
        return tc * rstd, rstd

    if gs is None:
        m, v = st["weight"], st["bias"]
    else:
        m, v = gs.float().unsqueeze(1).chunk(2, -1)
        m = 1.0 / (1.0 + torch.exp(-m))
    z, rstd = norm(r.float())
    out = {"r": r, "y": (m * z + v).to(act)}
    if case["keep"]:
        kept = _plain_kept(r)
        out["kept"] = kept.to(stream)
        z, rstd = norm(kept)
    gz = dy * m
    total = st["dr"].float() + rstd * (gz - gz.mean(-1, keepdim=True) - z * (gz * z).mean(-1, keepdim=True))
    out["dx"] = total.to(stream)
    out["du"] = (total if sg is None else sg * total).to(act)
    if sg is not None:
        out["dgate"] = ((total * u).sum(1, keepdim=True) * sg * (1.0 - sg)).squeeze(1).to(act)
    if gs is None:
        out["dweight"], out["dbias"] = (dy * z).sum((0, 1, 2)), dy.sum((0, 1, 2))
    else:
        out["dgate_shift"] = torch.cat(((dy * z).sum(1) * (m * (1.0 - m)).squeeze(1), dy.sum(1)), -1).to(act)
    return out


def _plain_activation(z, act):
    """f(z) and f'(z)."""
    if act == "none":
        return z, None
    if act == "relu":
        return torch.where(z > 0, z, 0.0), (z > 0).to(z.dtype)
    if act == "gelu":
        phi = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    s = 1.0 / (1.0 + torch.exp(-z))
    return (s, s * (1.0 - s)) if act == "sigmoid" else (z * s, s * (1.0 + z * (1.0 - s)))


def _plain_linear(st):
    case, x, w, dy = st["case"], st["x"].float(), st["w"].float(), st["dy"].float()

    def before(t):
        z = t @ w.t()
        return z if st["bias"] is None else z + st["bias"]

    y, slope = _plain_activation(before(x), case["act"])
    out = {"y": (y if st["residual"] is None else y + st["residual"].float()).to(st["x"].dtype)}
    if case["keep"]:
        x = _plain_kept(st["x"])
        if slope is not None:
            slope = _plain_activation(before(x), case["act"])[1]
    dz = dy if slope is None else dy * slope
    out["dx"], out["dw"] = (dz @ w).to(st["x"].dtype), (dz.t() @ x).to(st["w"].dtype)
    if st["bias"] is not None:
        out["dbias"] = dz.sum(0)
    return out


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if own:
        from kfold_b200 import functional as F
        if case["kind"] == "keep":
            return {"kept": F.expand(F.compress(state["x"]))}
        if case["kind"] == "linear":
            x, w, bias, act = state["x"], state["w"], state["bias"], None if case["act"] == "none" else case["act"]
            y = F.fused_linear(x, w, bias, activation=act, residual=state["residual"])
            dx, dw, db = F.fused_linear_backward(state["dy"], F.compress(x) if case["keep"] else x, w, bias, activation=act)
            return {"y": y, "dx": dx, "dw": dw} if bias is None else {"y": y, "dx": dx, "dw": dw, "dbias": db}
        gate, about = state["gate"], dict(gate=state["gate"], weight=state["weight"], gate_shift=state["gate_shift"], samples=case["samples"], eps=EPS)
        r, y, *kept = F.residual_norm(state["x"], state["u"], bias=state["bias"], compress=case["keep"], **about)
        g = F.residual_norm_backward(state["dr"], state["dy"], kept[0] if kept else r, state["u"], **about)
        out = {"r": r, "y": y, "dx": g.x, "du": g.u}
        if kept:
            out["kept"] = F.expand(kept[0])
        if gate is not None:
            out["dgate"] = g.gate
        return out | ({"dweight": g.weight, "dbias": g.bias} if state["gate_shift"] is None else {"dgate_shift": g.gate_shift})
    if case["kind"] == "step":
        return _plain_step(state)
    return _plain_linear(state) if case["kind"] == "linear" else {"kept": _plain_kept(state["x"]).to(state["x"].dtype)}


def work(case):
    """What comes in read once and what goes out written once.  A value kept in 8 bits, with its share of a group's power of two, is 33 / 32 bytes."""
    size = {"bf16": (2, 2), "mixed": (4, 2), "f32": (4, 4)}[case["dtype"]]
    kept = 33 / 32
    if case["kind"] == "keep":
        n = case["rows"] * case["c"]
        return {"bytes": int(n * (2 * size[1] + 2 * kept)), "flops": 6 * n}
    if case["kind"] == "linear":
        rows, k, n, s = case["rows"], case["k"], case["n"], size[1]
        # forward x and W, y (and the residual); backward dy, x and W again, dx and dW
        total = s * (rows * (2 * k + 2 * n + (n if case["residual"] else 0)) + 3 * k * n) + (s * rows * k if not case["keep"] else 2 * kept * rows * k)
        return {"bytes": int(total + (12 * n if case["bias"] else 0)), "flops": 6 * rows * k * n}
    g, s, l, c = (case[k] for k in ("groups", "samples", "tokens", "c"))
    n, table = g * s * l * c, g * l * c
    # forward x, u -> r, y; backward dr, dy, r -> dx, du, and u where its gate has a gradient
    total = n * (4 * size[0] + 4 * size[1]) + (n * size[1] if case["gate"] else 0) + n * (2 * kept + 2 * size[0] if case["keep"] else size[0])
    total += size[1] * table * ((3 if case["gate"] else 0) + (6 if case["norm"] == "adaptive" else 0))
    return {"bytes": int(total), "flops": 40 * n}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_kept(x):
    """Whole numbers of a group's power of two, which comes from the largest magnitude's fraction and exponent."""
    c = x.shape[-1]
    full = torch.zeros(*x.shape[:-1], -(-c // GROUP) * GROUP, dtype=torch.float64, device=x.device)
    full[..., :c] = x
    full = full.view(*x.shape[:-1], -1, GROUP)
    fraction, exponent = torch.frexp(full.abs().max(-1, keepdim=True).values)      # fraction in [0.5, 1)
    exponent = exponent - 7 + (fraction * 128.0 >= 127.5)
    return torch.ldexp(torch.round(torch.ldexp(full, -exponent)), exponent).reshape(*x.shape[:-1], -1)[..., :c]


def _exact_step(st):
    case = st["case"]
    leaf = lambda name: None if st[name] is None else st[name].double().requires_grad_()
    x, u, gate, gs, weight, bias = (leaf(k) for k in ("x", "u", "gate", "gate_shift", "weight", "bias"))
    r = x + (u if gate is None else torch.sigmoid(gate)[:, None] * u)
    stored = r.detach().to(st["x"].dtype).double()

    def normed(t):
        t = (t - t.mean(-1, keepdim=True)) / torch.sqrt(t.var(-1, unbiased=False, keepdim=True) + EPS)
        if gs is None:
            return t * weight + bias
        return torch.sigmoid(gs[:, None, ..., :case["c"]]) * t + gs[:, None, ..., case["c"]:]

    out = {"r": r.detach(), "y": normed(stored).detach()}
    if case["keep"]:
        out["kept"] = stored = _exact_kept(stored)
    stored.requires_grad_()
    params = [weight, bias] if gs is None else [gs]
    through, *rest = torch.autograd.grad(normed(stored), [stored, *params], st["dy"].double())
    wanted = {"dx": x, "du": u} | ({} if gate is None else {"dgate": gate})
    out |= dict(zip(wanted, torch.autograd.grad(r, list(wanted.values()), st["dr"].double() + through)))
    out |= dict(zip(("dweight", "dbias") if gs is None else ("dgate_shift",), rest))
    if case["keep"]:
        out["kept"] = out["kept"].detach()
    return out


def _exact_linear(st):
    case, x0 = st["case"], st["x"].double()
    f = {"none": lambda t: t, "sigmoid": torch.sigmoid, "relu": torch.relu, "silu": lambda t: t * torch.sigmoid(t),
         "gelu": lambda t: 0.5 * t * torch.erfc(-t / math.sqrt(2.0))}[case["act"]]
    x, w = (_exact_kept(x0) if case["keep"] else x0.clone()).requires_grad_(), st["w"].double().requires_grad_()
    bias = None if st["bias"] is None else st["bias"].double().requires_grad_()
    layer = lambda t: f(t @ w.T if bias is None else torch.addmm(bias, t, w.T))
    with torch.no_grad():
        out = {"y": layer(x0) if st["residual"] is None else layer(x0) + st["residual"]}
    wanted = {"dx": x, "dw": w} | ({} if bias is None else {"dbias": bias})
    return out | dict(zip(wanted, torch.autograd.grad(layer(x), list(wanted.values()), st["dy"].double())))


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "keep":
        return {"kept": _exact_kept(st["x"].double())}
    return _exact_step(st) if case["kind"] == "step" else _exact_linear(st)
