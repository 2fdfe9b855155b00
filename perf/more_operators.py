"""Performance cases of the operators that a mixture of update rules is made of, each particle using few of many
rules.

* ``route``: scores of the experts, the best ``top_k`` of each row and their weights, and the plan that sorts the
  rows' entries by expert;
* ``route_adjoint``: the gradient of the router's logits from those of the weights;
* ``linear``: each expert's linear layer over its slots of the plan, from rows (gathered) or from slots;
* ``linear_adjoint``: the gradients of its input, weights and bias through the activation;
* ``combine``: the weighted sum of each row's slots, added to a residual;
* ``combine_adjoint``: the gradients of the slots and of the weights.

``rows`` are particles (of every system and step in a batch) or samples, S = rows * top_k slots. Sizes are those of
the library's update rules (66 features, 128 hidden units, 18 outputs, 4,096 to 65,536 particles), and generic wide
layers. Logits are N(0, 1) with offsets that make some experts more popular than others (``closed``: a tenth of
the entries and a tenth of the rows are masked); weights are N(0, 1 / in), adjoints N(0, 0.05).
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-20  # of the renormalised weights
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ACTIVATIONS = ("identity", "relu", "gelu", "silu")
# of the largest listed cases, which bound the drawn ones: logits, slots times width, weights, products
MOST_LOGITS, MOST_SLOTS, MOST_WEIGHTS, MOST_LINEAR, MOST_ADJOINT = 1 << 24, 1 << 26, 1 << 26, 1 << 37, 1 << 36


def listed():
    return [
        # a small system (the library's own benchmark size) among a few rules: the smallest call
        dict(name="route_4k", op="route", type="f32", rows=4096, experts=8, top_k=2, scores="softmax", bias=False,
             groups=1, top_groups=1, renormalise=True, closed=False, pad=0),
        # many samples among many experts in groups, balanced by a bias
        dict(name="route_groups", op="route", type="bf16", rows=65536, experts=256, top_k=8, scores="sigmoid",
             bias=True, groups=8, top_groups=4, renormalise=True, closed=False, pad=0),
        # the headline system's router, backward
        dict(name="route_adjoint_64k", op="route_adjoint", type="f32", rows=65536, experts=8, top_k=2,
             scores="softmax", renormalise=True, closed=False, pad=0),
        # many experts, an odd number, some masked, in half precision, backward
        dict(name="route_adjoint_odd", op="route_adjoint", type="f16", rows=20011, experts=123, top_k=5,
             scores="softmax", renormalise=False, closed=True, pad=5),
        # one sample through a wide layer of its experts, as a served model answers: weight bandwidth and latency
        dict(name="linear_one", op="linear", type="bf16", rows=1, experts=32, top_k=4, inputs=2048, outputs=1024,
             activation="silu", bias=True, gather=True, keep=False, closed=False, pad=0),
        # the rules' first layer over the headline system, its preactivation kept for training
        dict(name="linear_64k", op="linear", type="f32", rows=65536, experts=8, top_k=2, inputs=66, outputs=128,
             activation="gelu", bias=True, gather=True, keep=True, closed=False, pad=0),
        # the widening layer of a batch's experts, in training
        dict(name="linear_wide", op="linear", type="bf16", rows=8192, experts=8, top_k=2, inputs=2048, outputs=4096,
             activation="gelu", bias=True, gather=True, keep=True, closed=False, pad=0),
        # the rules' first layer over the headline system, backward: long sums for few weights
        dict(name="linear_adjoint_64k", op="linear_adjoint", type="f32", rows=65536, experts=8, top_k=2, inputs=66,
             outputs=128, activation="gelu", bias=True, gather=True, closed=False, pad=0),
        # odd sizes in half precision, from slots, some rows without an expert
        dict(name="linear_adjoint_odd", op="linear_adjoint", type="f16", rows=1501, experts=7, top_k=3, inputs=777,
             outputs=333, activation="silu", bias=True, gather=False, closed=True, pad=3),
        # the widening layer of a batch's experts, backward
        dict(name="linear_adjoint_wide", op="linear_adjoint", type="bf16", rows=4096, experts=8, top_k=2, inputs=2048,
             outputs=4096, activation="gelu", bias=True, gather=True, closed=False, pad=0),
        # the headline system's particles with the sum of their rules' updates
        dict(name="combine_64k", op="combine", type="f32", rows=65536, experts=8, top_k=2, width=18, weights=True,
             residual=True, closed=False, pad=0),
        # a wide layer's results back to rows, backward
        dict(name="combine_adjoint_wide", op="combine_adjoint", type="bf16", rows=8192, experts=8, top_k=2, width=4096,
             weights=True, closed=False, pad=0),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("route", "route_adjoint", "linear", "linear", "linear_adjoint", "linear_adjoint", "combine",
                     "combine_adjoint"))
    case = dict(op=op, type=rng.choice(("f32", "bf16", "f16")), closed=rng.random() < 0.25,
                pad=rng.choice((0, 0, 0, 3, 8)))
    experts = spread(2, 256)
    top_k = min(experts, rng.randint(1, 8))
    rows = spread(1, 65536)
    if op.startswith("route"):
        case.update(scores=rng.choice(("softmax", "sigmoid")), renormalise=rng.random() < 0.7)
        if op == "route":
            groups = rng.choice([g for g in (1, 1, 2, 3, 4, 8) if g == 1 or experts >= 4 * g])
            experts -= experts % groups
            top_groups = rng.randint(1, groups)
            top_k = min(top_k, experts // groups * top_groups)
            case.update(bias=rng.random() < 0.5, groups=groups, top_groups=top_groups)
        return dict(case, rows=max(1, min(rows, MOST_LOGITS // experts)), experts=experts, top_k=top_k)
    if op.startswith("combine"):
        width = spread(8, 8192)
        case.update(rows=max(1, min(rows, MOST_SLOTS // (width * top_k))), experts=experts, top_k=top_k, width=width,
                    weights=rng.random() < 0.8)
        if op == "combine":
            case.update(residual=rng.random() < 0.5)
        return case
    inputs, outputs = spread(8, 4096), spread(8, 4096)
    experts = max(2, min(experts, MOST_WEIGHTS // (inputs * outputs)))
    top_k = min(experts, top_k)
    most = MOST_LINEAR if op == "linear" else MOST_ADJOINT
    if case["type"] == "f32":
        most //= 8
    rows = max(1, min(rows, most // (inputs * outputs * top_k), MOST_SLOTS // (max(inputs, outputs) * top_k)))
    case.update(rows=rows, experts=experts, top_k=top_k, inputs=inputs, outputs=outputs,
                activation=rng.choice(ACTIVATIONS), bias=rng.random() < 0.8, gather=rng.random() < 0.6)
    if op == "linear":
        case.update(keep=rng.random() < 0.5 and case["activation"] != "identity")
    return case


# ---------------------------------------------------------------- what a program has in hand
def _sorted(entries, experts):
    """The plan of the entries' experts [rows, k] (-1: none)."""
    keys = torch.where(entries < 0, experts, entries.long()).reshape(-1)
    order = torch.sort(keys, stable=True)[1]
    slots = torch.empty_like(order)
    slots[order] = torch.arange(order.numel(), device="cuda")
    offsets = torch.zeros(experts + 1, dtype=torch.int64, device="cuda")
    offsets.scatter_add_(0, (keys + 1).clamp_max(experts), (keys < experts).long())
    return offsets.cumsum(0).int(), order.int(), slots.int().reshape(entries.shape)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = TYPES[case["type"]]
    rows, experts, k, op = case["rows"], case["experts"], case["top_k"], case["op"]

    def normal(*shape, scale=1.0, offset=0.0):
        return torch.randn(*shape, generator=g, device="cuda") * scale + offset

    def padded(t):
        wide = torch.zeros(t.shape[0], t.shape[1] + case["pad"], dtype=dtype, device="cuda")
        wide[:, :t.shape[1]] = t
        return wide[:, :t.shape[1]]

    logits = normal(rows, experts) + normal(experts, scale=0.5)
    if case["closed"]:
        shut = torch.rand(rows, experts, generator=g, device="cuda") < 0.1
        shut |= torch.rand(rows, 1, generator=g, device="cuda") < 0.1
        logits = torch.where(shut, -math.inf, logits)
    s = {"case": case}
    if op == "route":
        s["logits"] = padded(logits)
        s["bias"] = normal(experts, scale=0.02) if case["bias"] else None
        return s
    logits = logits.to(dtype).float()
    best, chosen = (t[:, :k] for t in torch.sort(logits, dim=1, descending=True, stable=True))
    chosen = torch.where(best == -math.inf, -1, chosen).int()
    if op == "route_adjoint":
        s.update(logits=padded(logits), experts=chosen, weights_adjoint=normal(rows, k, scale=0.05))
        return s
    s["offsets"], s["order"], s["slots"] = _sorted(chosen, experts)
    slots = rows * k
    if op.startswith("combine"):
        width = case["width"]
        s["y"] = padded(normal(slots, width))
        s["weights"] = torch.softmax(best.clamp_min(-30.0), dim=1) if case["weights"] else None
        if op == "combine":
            s["residual"] = normal(rows, width).to(dtype) if case["residual"] else None
        else:
            s["out_adjoint"] = normal(rows, width, scale=0.05).to(dtype)
        return s
    s["bounds"] = s["offsets"].tolist()  # the plain form's loop over the experts
    inputs, outputs = case["inputs"], case["outputs"]
    s["x"] = padded(normal(rows if case["gather"] else slots, inputs))
    s["weight"] = normal(experts, outputs, inputs, scale=1.0 / math.sqrt(inputs)).to(dtype)
    if op == "linear":
        s["bias"] = normal(experts, outputs, scale=0.1).to(dtype) if case["bias"] else None
    else:
        s["out_adjoint"] = normal(slots, outputs, scale=0.05).to(dtype)
        s["preactivation"] = normal(slots, outputs).to(dtype) if case["activation"] != "identity" else None
    return s


def run(s):
    return _kernels(s) if own else _plain(s)


def _kernels(s):
    from burn_automata_amd import experts

    case = s["case"]
    if case["op"] == "route":
        r = experts.route(s["logits"], case["top_k"], case["scores"], s["bias"], case["groups"], case["top_groups"],
                          case["renormalise"])
        return {"experts": r.experts, "weights": r.weights, "offsets": r.plan.offsets, "order": r.plan.order,
                "slots": r.plan.slots}
    if case["op"] == "route_adjoint":
        return {"logits": experts.route_adjoint(s["weights_adjoint"], s["logits"], s["experts"], case["scores"],
                                                case["renormalise"])}
    plan = experts.Plan(s["offsets"], s["order"], s["slots"])
    if case["op"] == "combine":
        return {"out": experts.combine(s["y"], plan, s["weights"], s["residual"])}
    if case["op"] == "combine_adjoint":
        r = experts.combine_adjoint(s["out_adjoint"], s["y"], plan, s["weights"])
        return {"y": r.y, "weights": r.weights}
    if case["op"] == "linear":
        r = experts.linear(s["x"], s["weight"], plan, s["bias"], case["activation"], case["gather"], case["keep"])
        return {"out": r.out, "preactivation": r.preactivation}
    r = experts.linear_adjoint(s["out_adjoint"], s["x"], s["weight"], plan, s["preactivation"], case["activation"],
                               case["gather"], bias=case["bias"])
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


def _scores(logits, name):
    if name == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-logits))
    most = logits.amax(1, keepdim=True)
    e = torch.exp(logits - torch.where(most == -math.inf, 0.0, most))
    return e / e.sum(1, keepdim=True).clamp_min(torch.finfo(e.dtype).tiny)


def _plain_route(s):
    case = s["case"]
    rows, experts, k, groups = case["rows"], case["experts"], case["top_k"], case["groups"]
    logits = s["logits"].double()  # the order of the experts' keys is that of 64 bits
    keys = scores = logits
    if s["bias"] is not None or groups > 1:
        scores = _scores(logits, case["scores"])
    if s["bias"] is not None:
        scores = scores + s["bias"].double()
        keys = scores = torch.where(logits == -math.inf, -math.inf, scores)
    if groups > 1:
        open_ = torch.where(logits == -math.inf, -math.inf, scores).reshape(rows, groups, -1)
        best = torch.sort(open_, dim=2, descending=True)[0][:, :, :2]
        total = torch.where(best == -math.inf, 0.0, best).sum(2)
        total = torch.where(best[:, :, 0] == -math.inf, -math.inf, total)
        kept = torch.sort(total, dim=1, descending=True, stable=True)[1][:, :case["top_groups"]]
        allowed = torch.zeros(rows, groups, dtype=torch.bool, device="cuda").scatter_(1, kept, True)
        keys = torch.where(allowed[:, :, None], keys.reshape(rows, groups, -1), -math.inf).reshape(rows, experts)
    best, chosen = (t[:, :k] for t in torch.sort(keys, dim=1, descending=True, stable=True))
    weights = torch.gather(_scores(s["logits"].float(), case["scores"]), 1, chosen)
    weights = torch.where(best == -math.inf, 0.0, weights)
    if case["renormalise"]:
        weights = weights / (weights.sum(1, keepdim=True) + EPS)
    chosen = torch.where(best == -math.inf, -1, chosen).int()
    offsets, order, slots = _sorted(chosen, experts)
    return {"experts": chosen, "weights": weights, "offsets": offsets, "order": order, "slots": slots}


def _plain_route_adjoint(s):
    case = s["case"]
    p = _scores(s["logits"].float(), case["scores"])
    at = s["experts"].long().clamp_min(0)
    live = (s["experts"] >= 0).float()
    g = s["weights_adjoint"] * live
    chosen = torch.gather(p, 1, at) * live
    if case["renormalise"]:
        total = chosen.sum(1, keepdim=True) + EPS
        g = (g - (g * chosen).sum(1, keepdim=True) / total) / total * live
    dense = torch.zeros_like(p).scatter_add_(1, at, g)
    if case["scores"] == "sigmoid":
        d = dense * p * (1.0 - p)
    else:
        d = p * (dense - (g * chosen).sum(1, keepdim=True))
    return {"logits": d.to(TYPES[case["type"]])}


def _plain(s):
    case, dtype = s["case"], TYPES[s["case"]["type"]]
    if case["op"] == "route":
        return _plain_route(s)
    if case["op"] == "route_adjoint":
        return _plain_route_adjoint(s)
    k = case["top_k"]
    live = (s["slots"] < s["offsets"][-1]).float()  # [rows, k]
    if case["op"] == "combine":
        part = s["y"].float()[s["slots"].long()]
        w = live if s["weights"] is None else s["weights"] * live
        out = (part * w[:, :, None]).sum(1)
        if s["residual"] is not None:
            out = out + s["residual"].float()
        return {"out": out.to(dtype)}
    if case["op"] == "combine_adjoint":
        dout = s["out_adjoint"].float()
        w = live if s["weights"] is None else s["weights"] * live
        rows = (s["order"] // k).long()
        dy = dout[rows] * w.reshape(-1)[s["order"].long()][:, None]
        if s["weights"] is None:
            return {"y": dy.to(dtype), "weights": None}
        dots = (s["y"].float()[s["slots"].long()] * dout[:, None, :]).sum(2) * live
        return {"y": dy.to(dtype), "weights": dots}
    x, bounds = s["x"].float(), s["bounds"]
    slots, n, inputs = case["rows"] * k, case["outputs"], case["inputs"]
    rows = (s["order"] // k).long()
    if case["gather"]:
        x = x[rows]
    if case["op"] == "linear":
        z = torch.zeros(slots, n, device="cuda")
        for e in range(case["experts"]):
            a, b = bounds[e], bounds[e + 1]
            if b > a:
                z[a:b] = x[a:b] @ s["weight"][e].float().t()
                if s["bias"] is not None:
                    z[a:b] += s["bias"][e].float()
        return {"out": _activate(z, case["activation"]).to(dtype),
                "preactivation": z.to(dtype) if case["keep"] else None}
    dz = s["out_adjoint"].float()
    if s["preactivation"] is not None:
        dz = dz * _slope(s["preactivation"].float(), case["activation"])
    dx = torch.zeros(slots, inputs, device="cuda")
    dw = torch.zeros(case["experts"], n, inputs, device="cuda")
    db = torch.zeros(case["experts"], n, device="cuda")
    for e in range(case["experts"]):
        a, b = bounds[e], bounds[e + 1]
        if b > a:
            dx[a:b] = dz[a:b] @ s["weight"][e].float()
            dw[e] = dz[a:b].t() @ x[a:b]
            db[e] = dz[a:b].sum(0)
    if case["gather"]:
        dx = (dx[s["slots"].long()] * live[:, :, None]).sum(1)
    return {"x": dx.to(dtype), "weight": dw.to(dtype), "bias": db.to(dtype) if case["bias"] else None}


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    size, rows, k, experts = {"f32": 4, "bf16": 2, "f16": 2}[case["type"]], case["rows"], case["top_k"], case["experts"]
    slots = rows * k
    if case["op"] == "route":
        return {"bytes": size * rows * experts + 4 * experts * case["bias"] + 16 * slots + 4 * (experts + 1),
                "flops": 10 * rows * experts}
    if case["op"] == "route_adjoint":
        return {"bytes": 2 * size * rows * experts + 8 * slots, "flops": 10 * rows * experts}
    if case["op"] == "combine":
        return {"bytes": size * case["width"] * (slots + rows * (1 + case["residual"])) + 4 * slots * (1 + case["weights"]),
                "flops": 2 * slots * case["width"]}
    if case["op"] == "combine_adjoint":
        w = case["weights"]
        return {"bytes": size * case["width"] * (slots * (1 + w) + rows) + 4 * slots * (1 + 2 * w),
                "flops": (3 if w else 1) * slots * case["width"]}
    n, m = case["outputs"], case["inputs"]
    used = min(experts, slots)  # experts whose weights are read
    x = size * m * (rows if case["gather"] else slots)
    if case["op"] == "linear":
        return {"bytes": x + size * (used * n * (m + case["bias"]) + slots * n * (1 + case["keep"])) + 4 * slots,
                "flops": 2 * slots * m * n}
    whole = 1 + (case["activation"] != "identity")
    return {"bytes": 2 * x + size * (n * m * (used + experts) + experts * n * case["bias"] + whole * slots * n) + 4 * slots,
            "flops": 4 * slots * m * n}


# ---------------------------------------------------------------- the definitions, in 64 bits
def _exact_weights(logits, chosen, case):
    """The weights of the chosen experts [rows, k] (-1: none), differentiable."""
    if case["scores"] == "sigmoid":
        p = torch.sigmoid(logits)
    else:
        none = (logits == -math.inf).all(1, keepdim=True)
        p = torch.softmax(logits.masked_fill(none, 0.0), dim=1)
    picked = p.gather(1, chosen.long().clamp_min(0)).masked_fill(chosen < 0, 0.0)
    return picked / (picked.sum(1, keepdim=True) + EPS) if case["renormalise"] else picked


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "route":
        return {"experts": None, "weights": _exact_weights(s["logits"].double(), _plain_route(s)["experts"], case),
                "offsets": None, "order": None, "slots": None}
    if case["op"] == "route_adjoint":  # by reverse differentiation of the definition
        leaf = s["logits"].double()
        finite = leaf != -math.inf
        leaf = leaf.requires_grad_()
        w = _exact_weights(leaf, s["experts"], case)
        d, = torch.autograd.grad((w * s["weights_adjoint"].double()).sum(), leaf)
        return {"logits": torch.where(finite, d, 0.0)}
    rows, k, experts, dev = case["rows"], case["top_k"], case["experts"], "cuda"
    # slots' experts and rows, from the plan
    slot = torch.arange(rows * k, device=dev)
    expert = torch.searchsorted(s["offsets"][1:].contiguous().long(), slot, right=True)  # `experts`: none
    row, live = torch.div(s["order"].long(), k, rounding_mode="floor"), expert < experts
    if case["op"].startswith("combine"):
        w = torch.ones(rows * k, dtype=torch.float64, device=dev) if s["weights"] is None else s["weights"].double().reshape(-1)
        w = w[s["order"].long()] * live
        if case["op"] == "combine":
            out = torch.zeros(rows, case["width"], dtype=torch.float64, device=dev) if s["residual"] is None else s["residual"].double()
            return {"out": out.index_add(0, row, s["y"].double() * w.unsqueeze(1))}
        dout = s["out_adjoint"].double().index_select(0, row)
        dots = torch.zeros(rows * k, dtype=torch.float64, device=dev)
        dots[s["order"].long()] = (s["y"].double() * dout).sum(1).masked_fill(~live, 0.0)
        return {"y": dout.mul(w.unsqueeze(1)), "weights": None if s["weights"] is None else dots.reshape(rows, k)}
    act = {"identity": lambda v: v, "relu": torch.nn.functional.relu, "silu": torch.nn.functional.silu,
           "gelu": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}[case["activation"]]
    n, m = case["outputs"], case["inputs"]
    of = [(expert == e).nonzero()[:, 0] for e in range(experts)]
    at = (lambda i: row[i]) if case["gather"] else (lambda i: i)
    if case["op"] == "linear":
        out = torch.zeros(rows * k, n, dtype=torch.float64, device=dev)
        z = torch.zeros_like(out) if case["keep"] else None
        for e, i in enumerate(of):
            if i.numel():
                v = torch.nn.functional.linear(s["x"][at(i)].double(), s["weight"][e].double(),
                                               None if s["bias"] is None else s["bias"][e].double())
                out[i] = act(v)
                if z is not None:
                    z[i] = v
        return {"out": out, "preactivation": z}
    dz = s["out_adjoint"].double()
    if s["preactivation"] is not None:
        z = s["preactivation"].double().requires_grad_()
        dz, = torch.autograd.grad(act(z), z, dz)
    dx = torch.zeros(rows if case["gather"] else rows * k, m, dtype=torch.float64, device=dev)
    dw = torch.zeros(experts, n, m, dtype=torch.float64, device=dev)
    db = torch.zeros(experts, n, dtype=torch.float64, device=dev)
    for e, i in enumerate(of):
        if i.numel():
            dx.index_add_(0, at(i), torch.mm(dz[i], s["weight"][e].double()))
            dw[e] = torch.mm(dz[i].T.contiguous(), s["x"][at(i)].double())
            db[e] = torch.ones(i.numel(), dtype=torch.float64, device=dev) @ dz[i]
    return {"x": dx, "weight": dw, "bias": db if case["bias"] else None}
