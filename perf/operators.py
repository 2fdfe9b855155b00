"""Performance cases of the dense-layer operators that a trained update rule is made of.

* ``norm``: layer norm over the rows' last axis, with the row statistics its adjoint reads;
* ``norm_adjoint``: the gradients of its input, scale and shift;
* ``linear``: a matrix product with bias, activation and residual, and the preactivation where it is kept;
* ``linear_adjoint``: the gradients of its input, weights and bias through the activation.

``rows`` are particles (of every system and step in a batch) or samples. Sizes are those of the library's
update rules (66 or 123 features, 128 or 256 hidden units, 18 or 27 outputs, 4,096 to 65,536 particles), and
generic wide layers. Inputs are rows of features whose channels have offsets and scales of their own, weights
are N(0, 1 / in), adjoints N(0, 0.05).
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ACTIVATIONS = ("identity", "relu", "gelu", "silu")
# the largest listed cases' products of sizes, which bound the drawn ones
MOST_NORM, MOST_LINEAR, MOST_ADJOINT = 1 << 27, 1 << 38, 1 << 37


def listed():
    return [
        # the features of one small system (the library's own benchmark size): the smallest call
        dict(name="norm_4k", op="norm", type="f32", rows=4096, width=66, pad=0, shift=True),
        # activations of a wide layer, 32,768 rows: the largest pass over memory
        dict(name="norm_wide", op="norm", type="bf16", rows=32768, width=4096, pad=0, shift=True),
        # the features of the headline system of 65,536 particles, backward
        dict(name="norm_adjoint_64k", op="norm_adjoint", type="f32", rows=65536, width=66, pad=0, shift=True),
        # an odd width inside a wider buffer, in half precision
        dict(name="norm_adjoint_odd", op="norm_adjoint", type="f16", rows=5003, width=1023, pad=5, shift=True),
        # a training batch of a wide layer, backward
        dict(name="norm_adjoint_wide", op="norm_adjoint", type="bf16", rows=16384, width=4096, pad=0, shift=True),
        # the update rule's first layer over the headline system, forward, its preactivation kept for training
        dict(name="linear_64k", op="linear", type="f32", rows=65536, inputs=66, outputs=128, activation="relu",
             bias=True, residual=False, keep=True, pad=0),
        # one row through a square layer with a residual, as a served model answers: latency and weight bandwidth
        dict(name="linear_one", op="linear", type="bf16", rows=1, inputs=4096, outputs=4096, activation="identity",
             bias=True, residual=True, keep=False, pad=0),
        # a batch through a residual layer in full precision
        dict(name="linear_f32", op="linear", type="f32", rows=8192, inputs=1024, outputs=1024,
             activation="identity", bias=True, residual=True, keep=False, pad=0),
        # the widening layer of a residual block, forward in training
        dict(name="linear_wide", op="linear", type="bf16", rows=16384, inputs=2048, outputs=8192,
             activation="gelu", bias=True, residual=False, keep=True, pad=0),
        # the update rule's first layer over the headline system, backward: a long sum for few weights
        dict(name="linear_adjoint_64k", op="linear_adjoint", type="f32", rows=65536, inputs=66, outputs=128,
             activation="relu", bias=True, pad=0),
        # odd sizes in half precision
        dict(name="linear_adjoint_odd", op="linear_adjoint", type="f16", rows=3001, inputs=777, outputs=1111,
             activation="silu", bias=True, pad=3),
        # the widening layer of a residual block, backward
        dict(name="linear_adjoint_wide", op="linear_adjoint", type="bf16", rows=8192, inputs=2048, outputs=8192,
             activation="gelu", bias=True, pad=0),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("norm", "norm_adjoint", "linear", "linear_adjoint"))
    case = dict(op=op, type=rng.choice(("f32", "bf16", "f16")), pad=rng.choice((0, 0, 0, 3, 8)))
    if op.startswith("norm"):
        width = spread(8, 16384)
        most = MOST_NORM // (2 if op == "norm_adjoint" else 1)
        return dict(case, width=width, rows=max(1, min(spread(1, 262144), most // width)),
                    shift=rng.random() < 0.8)
    inputs, outputs = spread(8, 8192), spread(8, 8192)
    most = MOST_LINEAR if op == "linear" else MOST_ADJOINT
    if case["type"] == "f32":
        most //= 8
    rows = max(1, min(spread(1, 65536), most // (inputs * outputs)))
    case.update(rows=rows, inputs=inputs, outputs=outputs, activation=rng.choice(ACTIVATIONS),
                bias=rng.random() < 0.8)
    if op == "linear":
        case.update(residual=rng.random() < 0.5, keep=rng.random() < 0.5 and case["activation"] != "identity")
    return case


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = TYPES[case["type"]]
    rows, norm = case["rows"], case["op"].startswith("norm")
    width = case["width"] if norm else case["inputs"]

    def normal(*shape, scale=1.0, offset=0.0):
        return torch.randn(*shape, generator=g, device="cuda") * scale + offset

    def features():
        scale = torch.rand(width, generator=g, device="cuda") + 0.5
        wide = torch.zeros(rows, width + case["pad"], dtype=dtype, device="cuda")
        wide[:, :width] = normal(rows, width) * scale + 0.3 * normal(width)
        return wide[:, :width]

    s = {"case": case, "x": features()}
    if norm:
        s["gamma"] = normal(width, scale=0.2, offset=1.0).to(dtype) if case["shift"] else None
        s["beta"] = normal(width, scale=0.2).to(dtype) if case["shift"] else None
        if case["op"] == "norm_adjoint":
            s["dy"] = normal(rows, width, scale=0.05).to(dtype)
            x = s["x"].float()
            s["mean"] = x.mean(1)
            s["rstd"] = torch.rsqrt((x - s["mean"][:, None]).square().mean(1) + EPS)
        return s
    outputs = case["outputs"]
    s["weight"] = normal(outputs, width, scale=1.0 / math.sqrt(width)).to(dtype)
    if case["op"] == "linear":
        s["bias"] = normal(outputs, scale=0.1).to(dtype) if case["bias"] else None
        s["residual"] = normal(rows, outputs).to(dtype) if case["residual"] else None
    else:
        s["dy"] = normal(rows, outputs, scale=0.05).to(dtype)
        s["preactivation"] = normal(rows, outputs).to(dtype) if case["activation"] != "identity" else None
    return s


def run(s):
    return _kernels(s) if own else _plain(s)


def _kernels(s):
    from burn_automata_amd import layers

    case = s["case"]
    if case["op"] == "norm":
        r = layers.layer_norm(s["x"], s["gamma"], s["beta"], EPS)
        return {"out": r.out, "mean": r.mean, "rstd": r.rstd}
    if case["op"] == "norm_adjoint":
        r = layers.layer_norm_adjoint(s["dy"], s["x"], s["mean"], s["rstd"], s["gamma"])
        return {"x": r.x, "gamma": r.gamma, "beta": r.beta}
    if case["op"] == "linear":
        r = layers.linear(s["x"], s["weight"], s["bias"], case["activation"], s["residual"], case["keep"])
        return {"out": r.out, "preactivation": r.preactivation}
    r = layers.linear_adjoint(s["dy"], s["x"], s["weight"], s["preactivation"], case["activation"],
                              bias=case["bias"])
    return {"x": r.x, "weight": r.weight, "bias": r.bias}


# ---------------------------------------------------------------- the plain forms, in 32 bits
GELU_A, GELU_B = math.sqrt(2.0 / math.pi), 0.044715


def _activate(z, name):
    if name == "relu":
        return torch.maximum(z, torch.zeros((), device=z.device))
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.tanh(GELU_A * (z + GELU_B * z * z * z)))
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _slope(z, name):
    if name == "relu":
        return (z > 0).float()
    if name == "gelu":
        t = torch.tanh(GELU_A * (z + GELU_B * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * GELU_A * (1.0 + 3.0 * GELU_B * z * z)
    s = 1.0 / (1.0 + torch.exp(-z))
    return s * (1.0 + z * (1.0 - s))


def _plain(s):
    case, x, dtype = s["case"], s["x"].float(), TYPES[s["case"]["type"]]
    if case["op"] == "norm":
        mean = x.sum(1) / x.shape[1]
        centred = x - mean[:, None]
        rstd = 1.0 / torch.sqrt((centred * centred).sum(1) / x.shape[1] + EPS)
        y = centred * rstd[:, None]
        if s["gamma"] is not None:
            y = y * s["gamma"].float() + s["beta"].float()
        return {"out": y.to(dtype), "mean": mean, "rstd": rstd}
    dy = s["dy"].float() if "dy" in s else None
    if case["op"] == "norm_adjoint":
        xhat = (x - s["mean"][:, None]) * s["rstd"][:, None]
        g = dy if s["gamma"] is None else dy * s["gamma"].float()
        dx = s["rstd"][:, None] * (g - g.sum(1, keepdim=True) / x.shape[1]
                                   - xhat * ((g * xhat).sum(1, keepdim=True) / x.shape[1]))
        if s["gamma"] is None:
            return {"x": dx.to(dtype), "gamma": None, "beta": None}
        return {"x": dx.to(dtype), "gamma": (dy * xhat).sum(0).to(dtype), "beta": dy.sum(0).to(dtype)}
    w = s["weight"].float()
    if case["op"] == "linear":
        z = x @ w.t()
        if s["bias"] is not None:
            z = z + s["bias"].float()
        y = _activate(z, case["activation"])
        if s["residual"] is not None:
            y = y + s["residual"].float()
        return {"out": y.to(dtype), "preactivation": z.to(dtype) if case["keep"] else None}
    dz = dy if s["preactivation"] is None else dy * _slope(s["preactivation"].float(), case["activation"])
    return {"x": (dz @ w).to(dtype), "weight": (dz.t() @ x).to(dtype),
            "bias": dz.sum(0).to(dtype) if case["bias"] else None}


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    size, rows = {"f32": 4, "bf16": 2, "f16": 2}[case["type"]], case["rows"]
    if case["op"].startswith("norm"):
        params = 2 * case["width"] if case["shift"] else 0
        if case["op"] == "norm":
            return {"bytes": size * (2 * rows * case["width"] + params) + 8 * rows, "flops": 8 * rows * case["width"]}
        return {"bytes": size * (3 * rows * case["width"] + params * 3 // 2) + 8 * rows,
                "flops": (14 if params else 11) * rows * case["width"]}
    k, n = case["inputs"], case["outputs"]
    if case["op"] == "linear":
        whole = 1 + case["residual"] + case["keep"]
        return {"bytes": size * (rows * k + n * k + whole * rows * n + case["bias"] * n), "flops": 2 * rows * k * n}
    whole = 1 + (case["activation"] != "identity")
    return {"bytes": size * (2 * rows * k + 2 * n * k + whole * rows * n + case["bias"] * n),
            "flops": 4 * rows * k * n}


# ---------------------------------------------------------------- the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    if case["op"].startswith("norm"):
        gamma = torch.ones(case["width"], dtype=torch.float64, device="cuda") if s["gamma"] is None else s["gamma"].double()
        var, mean = torch.var_mean(x, dim=1, correction=0)
        rstd = (var + EPS).pow(-0.5)
        if case["op"] == "norm":
            y = torch.addcmul(torch.zeros_like(gamma) if s["beta"] is None else s["beta"].double(),
                              (x - mean.unsqueeze(1)) * rstd.unsqueeze(1), gamma)
            return {"out": y, "mean": mean, "rstd": rstd}
        out = {"x": torch.empty_like(x), "gamma": torch.zeros_like(gamma), "beta": s["dy"].double().sum(0)}
        step = max(1, (1 << 25) // case["width"])
        for at in range(0, case["rows"], step):  # by reverse differentiation of the definition
            leaf = x[at:at + step].clone().requires_grad_()
            scale = gamma.clone().requires_grad_()
            v, m = torch.var_mean(leaf, dim=1, correction=0, keepdim=True)
            y = (leaf - m) / (v + EPS).sqrt() * scale
            out["x"][at:at + step], dgamma = torch.autograd.grad(y, (leaf, scale), s["dy"][at:at + step].double())
            out["gamma"] += dgamma
        return out if case["shift"] else {"x": out["x"], "gamma": None, "beta": None}
    act = {"identity": lambda v: v, "relu": torch.nn.functional.relu, "silu": torch.nn.functional.silu,
           "gelu": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}[case["activation"]]
    if case["op"] == "linear":
        z = torch.nn.functional.linear(x, s["weight"].double(), None if s["bias"] is None else s["bias"].double())
        y = act(z)
        return {"out": y if s["residual"] is None else y + s["residual"].double(),
                "preactivation": z if case["keep"] else None}
    dz = s["dy"].double()
    if s["preactivation"] is not None:
        z = s["preactivation"].double().requires_grad_()
        dz, = torch.autograd.grad(act(z), z, dz)
    return {"x": torch.mm(dz, s["weight"].double()), "weight": torch.mm(dz.T.contiguous(), x),
            "bias": torch.ones(case["rows"], dtype=torch.float64, device="cuda") @ dz if case["bias"] else None}
