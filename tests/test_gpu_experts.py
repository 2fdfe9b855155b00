"""The layers of a mixture of update rules against their definitions in 64 bits.

Tolerances, elementwise, from rounding alone. u is the unit roundoff of the array's type (f32 2^-24, bf16 2^-8, f16
2^-11) and e = 2^-24 that of the f32 sums. A sum of K products in any order is within (K + 8) e times the sum of their
absolute values. A score is within S = (|l - max| + 32) e of itself: the rounded difference in the exponent, an
exponential of 2 ulp, a sum of at most 16 + 6 levels, a quotient. An activation's slope is at most 1.13 and its own
evaluation within 16 e (1 + |z|). Each result is rounded once more, u times itself; f16 results below its normal range
are rounded to multiples of 2^-24. What is a whole number is equal.
"""
import ctypes as C
import math
import threading

import pytest
import torch

from burn_automata_amd import _abi, experts, layers
from burn_automata_amd._lib import lib
from burn_automata_amd.runtime import Context, ptr

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}
TYPES = (torch.float32, torch.bfloat16, torch.float16)
ACTS = {"identity": lambda v: v, "relu": torch.nn.functional.relu, "silu": torch.nn.functional.silu,
        "gelu": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}
INF = math.inf


def randn(*shape, seed, scale=1.0, dtype=torch.float32, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = shape[:-1] + (shape[-1] + pad,)
    t = (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)
    if not pad:
        return t
    t[..., shape[-1] - pad:] = math.nan  # what lies between the rows is not read
    return t[..., : shape[-1] - pad]


def check(got, want, bound, what):
    most = torch.finfo(got.dtype).max
    got, bound = got.double(), bound + U[got.dtype] * want.abs() + TINY[got.dtype]
    assert got.shape == want.shape, what
    over = (want.abs() + bound >= most) & (got == want.sign() * INF)  # past the type's largest value
    bad = ~(((got - want).abs() <= bound) | over)
    assert not bad.any(), (what, int(bad.sum()), float((got - want).abs()[bad].max()), float(bound[bad].max()))


# ------------------------------------------------------------------------------ references
def scores_of(logits, scores):
    """Scores in 64 bits and their bounds, relative."""
    l = logits.double()
    if scores == "sigmoid":
        return torch.sigmoid(l), torch.full_like(l, 32 * E)
    most = l.amax(1, keepdim=True)
    l = l - torch.where(most == -INF, 0.0, most)
    p = l.exp()
    return p / p.sum(1, keepdim=True).clamp_min(1e-300), (torch.where(l == -INF, 0.0, l.abs()) + 32) * E


def choose(logits, k, scores, bias, groups, top_groups):
    """The experts [rows, k], by a stable descending sort of exact keys."""
    l = logits.double()
    rows, count = l.shape
    p, _ = scores_of(logits, scores)
    b = torch.zeros(count, dtype=torch.float64, device="cuda") if bias is None else bias.double()
    shut = (l == -INF) | (b == -INF)
    key = l if bias is None else p + b
    if groups > 1:
        best, two = torch.where(shut, -INF, p + b).reshape(rows, groups, -1).sort(dim=2, descending=True, stable=True)
        two, none = two[:, :, :2], best[:, :, :2] == -INF
        # (s + s') + (b + b'), so that equal groups are equal in 64 bits, too
        value = sum(t.reshape(rows, groups, -1).gather(2, two).masked_fill(none, 0.0).sum(2) for t in (p, b.expand(rows, count)))
        value = torch.where(best[:, :, 0] == -INF, -INF, value)
        kept = value.sort(dim=1, descending=True, stable=True)[1][:, :top_groups]
        allowed = torch.zeros(rows, groups, dtype=torch.bool, device="cuda").scatter_(1, kept, True)
        shut = shut | ~allowed.repeat_interleave(count // groups, 1)
    best, at = torch.where(shut, -INF, key).sort(dim=1, descending=True, stable=True)
    return torch.where(best[:, :k] == -INF, -1, at[:, :k]).int()


def weights_of(logits, chosen, scores, renormalise, scale):
    p, rel = scores_of(logits, scores)
    at, live = chosen.long().clamp_min(0), chosen >= 0
    w = p.gather(1, at) * live
    err = w * rel.gather(1, at)
    if renormalise:
        z = w.sum(1, keepdim=True) + 1e-20
        err = err / z + w / z * (err.sum(1, keepdim=True) / z + 40 * E)
        w = w / z
    return w * scale, abs(scale) * (err + 4 * E * w) + 2.0 ** -126


def plan_of(chosen, count):
    key = torch.where((chosen < 0) | (chosen >= count), count, chosen).reshape(-1).long()
    order = key.sort(dim=0, stable=True)[1]
    slots = torch.empty_like(order)
    slots[order] = torch.arange(order.numel(), device="cuda")
    offsets = torch.bincount(key, minlength=count + 1).cumsum(0)[:count]
    return torch.cat([offsets.new_zeros(1), offsets]).int(), order.int(), slots.int().reshape(chosen.shape)


def check_plan(plan, chosen, count):
    offsets, order, slots = plan_of(chosen.reshape(-1, chosen.shape[-1]), count)
    assert torch.equal(plan.offsets, offsets) and torch.equal(plan.order, order) and torch.equal(plan.slots, slots)


def routed(rows, count, k, seed, none=0.0, skew=0.5):
    """A plan of random choices, and they."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    l = torch.randn(rows, count, generator=g, device="cuda") + skew * torch.randn(count, generator=g, device="cuda")
    chosen = l.sort(dim=1, descending=True)[1][:, :k].int()
    if none:
        chosen = torch.where(torch.rand(rows, k, generator=g, device="cuda") < none, -1, chosen)
    return experts.Plan(*plan_of(chosen, count)), chosen


# ------------------------------------------------------------------------------ routing
COUNTS = ((1, 1), (2, 1), (3, 3), (8, 2), (9, 4), (16, 16), (17, 5), (32, 32), (33, 6), (64, 8), (65, 7), (123, 5), (256, 8),
          (257, 32), (600, 9), (1024, 32))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("count,k", COUNTS)
def test_route(dtype, count, k):
    for n, (scores, bias, renormalise, rows) in enumerate((("softmax", False, True, 67), ("sigmoid", True, True, 300),
                                                          ("softmax", True, False, 131), ("sigmoid", False, False, 1))):
        logits = randn(rows, count, seed=count + n, scale=2.0, dtype=dtype, pad=(count + n) % 3)
        b = randn(count, seed=n, scale=0.1, dtype=torch.float32 if n % 2 else dtype) if bias else None
        r = experts.route(logits, k, scores, b, renormalise=renormalise, scale=1.0 + n)
        want = choose(logits, k, scores, b, 1, 1)
        assert torch.equal(r.experts, want), (scores, bias)
        check(r.weights, *weights_of(logits, want, scores, renormalise, 1.0 + n), "weights")
        check_plan(r.plan, want, count)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("count,groups,top_groups,k", ((4, 2, 1, 2), (8, 8, 3, 3), (32, 32, 5, 4), (30, 3, 2, 7), (60, 6, 2, 5),
                                                       (64, 64, 9, 9), (63, 7, 7, 8), (256, 8, 4, 8), (250, 10, 3, 6),
                                                       (512, 4, 1, 32), (1024, 64, 8, 16)))
def test_route_with_groups(dtype, count, groups, top_groups, k):
    for n, (scores, bias) in enumerate((("sigmoid", True), ("softmax", False))):
        logits = randn(211, count, seed=count + n, scale=1.5, dtype=dtype)
        b = randn(count, seed=n, scale=0.1) if bias else None
        r = experts.route(logits, k, scores, b, groups, top_groups)
        want = choose(logits, k, scores, b, groups, top_groups)
        assert torch.equal(r.experts, want), scores
        check(r.weights, *weights_of(logits, want, scores, True, 1.0), "weights")
        check_plan(r.plan, want, count)


@pytest.mark.parametrize("groups", (1, 4))
def test_equal_keys_go_to_the_lowest_index(groups):
    for count in (8, 24, 64, 256, 1024):
        for scores in ("softmax", "sigmoid"):
            g = torch.Generator(device="cuda").manual_seed(count)
            logits = torch.randint(-1, 2, (500, count), generator=g, device="cuda").float()
            logits[0] = 0.0
            logits[1] = -0.0
            logits[1, ::2] = 0.0
            logits[2] = torch.finfo(torch.float32).min
            bias = torch.randint(-1, 2, (count,), generator=g, device="cuda").float() * 0.25
            for b in (None, torch.zeros(count, device="cuda"), bias):
                r = experts.route(logits, 4, scores, b, groups, 2 if groups > 1 else 1)
                assert torch.equal(r.experts, choose(logits, 4, scores, b, groups, 2 if groups > 1 else 1)), (count, scores)


@pytest.mark.parametrize("groups", (1, 4))
@pytest.mark.parametrize("count", (8, 64, 256))
def test_keys_that_32_bits_do_not_tell_apart(count, groups):
    """Biases that bring every key to within 2^-25 of the same value: the order is that of 64 bits."""
    logits = randn(400, count, seed=count)
    logits[:] = logits[:1]
    logits[1:] += randn(399, count, seed=count + 1, scale=2.0 ** -22)
    bias = (1.5 - torch.sigmoid(logits[0].double())).float()
    got = experts.route(logits, 5, "sigmoid", bias, groups, 3 if groups > 1 else 1).experts
    want = choose(logits, 5, "sigmoid", bias, groups, 3 if groups > 1 else 1)
    assert torch.equal(got, want)
    near = (torch.sigmoid(logits) + bias)  # and f32 does not tell it
    assert not torch.equal(near.sort(dim=1, descending=True, stable=True)[1][:, :5].int(), choose(logits, 5, "sigmoid", bias, 1, 1))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("count,groups", ((5, 1), (24, 1), (24, 4), (256, 1), (256, 8)))
def test_closed_experts(dtype, count, groups):
    logits = randn(300, count, seed=count, dtype=dtype)
    g = torch.Generator(device="cuda").manual_seed(3)
    logits[torch.rand(300, count, generator=g, device="cuda") < 0.5] = -INF
    logits[::7] = -INF  # rows that nothing is left of
    logits[3] = -INF
    logits[3, count - 1] = 1.0
    bias = randn(count, seed=4, scale=0.1)
    bias[1] = -INF
    for scores in ("softmax", "sigmoid"):
        for b in (None, bias):
            k, top = min(4, count), min(2, groups)
            r = experts.route(logits, k, scores, b, groups, top)
            want = choose(logits, k, scores, b, groups, top)
            assert torch.equal(r.experts, want)
            assert (r.weights[want < 0] == 0).all() and torch.isfinite(r.weights).all()
            check(r.weights, *weights_of(logits, want, scores, True, 1.0), "weights")
            check_plan(r.plan, want, count)
            dw = randn(300, k, seed=5)
            dw[want < 0] = math.nan  # not read
            d = experts.route_adjoint(dw, logits, r.experts, scores)
            assert torch.isfinite(d).all() and (d[logits == -INF] == 0).all()


def test_nan_and_infinite_logits_stay_in_their_row():
    for count, groups in ((6, 1), (256, 1), (256, 8)):
        for b in (None, randn(count, seed=2, scale=0.1)):
            logits = randn(64, count, seed=1)
            clean = experts.route(logits, 3, "softmax", b, groups, max(1, groups // 2))
            logits[5, 2] = math.nan
            logits[6, 4] = INF
            r = experts.route(logits, 3, "softmax", b, groups, max(1, groups // 2))
            rest = [i for i in range(64) if i not in (5, 6)]
            assert torch.equal(r.experts[rest], clean.experts[rest]) and torch.equal(r.weights[rest], clean.weights[rest])
            assert ((r.experts >= 0) & (r.experts < count)).all() and r.weights[5].isnan().all()
    logits = randn(4, 16, seed=1)
    logits[1, 9] = math.nan
    logits[2, 3] = INF
    r = experts.route(logits, 2, "sigmoid", renormalise=False)
    assert r.experts[1, 0] == 9 and r.weights[1, 0].isnan() and r.experts[2, 0] == 3 and r.weights[2, 0] == 1.0


def route_adjoint_reference(dw, logits, chosen, scores, renormalise, scale):
    p, rel = scores_of(logits, scores)
    at, live = chosen.long().clamp_min(0), (chosen >= 0).double()
    g = torch.nan_to_num(dw.double()) * live
    s = p.gather(1, at) * live
    r = rel.amax(1, keepdim=True) + (chosen.shape[1] + 16) * E  # of a score, a sum of them and what they are times
    if renormalise:
        z = s.sum(1, keepdim=True) + 1e-20
        ds = scale * (g - (g * s).sum(1, keepdim=True) / z) / z * live
        size = abs(scale) * (g.abs() + (g.abs() * s).sum(1, keepdim=True) / z) / z * live
    else:
        ds = scale * g
        size = ds.abs()
    dense = torch.zeros_like(p).scatter_add_(1, at, ds)
    most = torch.zeros_like(p).scatter_add_(1, at, size)
    if scores == "sigmoid":
        return dense * p * (1 - p), 4 * r * most * p
    through, own = (ds * s).sum(1, keepdim=True), (size * s).sum(1, keepdim=True)
    if renormalise:
        # sum ds s = scale / z (sum g s - sum g s sum s / z) and sum s = z - 1e-20, so it is scale sum(g s) 1e-20 / z^2: as
        # the difference, even 64 bits leave 2^-53 of its terms, a million times as much
        through = scale * (g * s).sum(1, keepdim=True) / z * (1e-20 / z)
        own = abs(scale) * (g.abs() * s).sum(1, keepdim=True) / z * (1e-20 / z)
    return p * (dense - through), p * 4 * r * (most + own) + p * 2.0 ** -100


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("count,k", COUNTS)
def test_route_adjoint(dtype, count, k):
    for n, (scores, renormalise, rows) in enumerate((("softmax", True, 67), ("softmax", False, 301), ("sigmoid", True, 130),
                                                     ("sigmoid", False, 1))):
        logits = randn(rows, count, seed=count + n, scale=2.0, dtype=dtype, pad=(count + n) % 3)
        chosen = choose(logits, k, scores, None, 1, 1)
        chosen[torch.rand(rows, k, device="cuda") < 0.1] = -1
        dw = randn(rows, k, seed=n)
        got = experts.route_adjoint(dw, logits, chosen, scores, renormalise, 1.5)
        check(got, *route_adjoint_reference(dw, logits, chosen, scores, renormalise, 1.5), (scores, renormalise))


def test_route_adjoint_against_differences():
    """Central differences of the weights in 64 bits, h = 2^-17: the third derivative of a score is below 1, so they are within
    h^2 of the slope, and 2^-52 / h = 2^-35 of it by rounding."""
    for scores in ("softmax", "sigmoid"):
        for renormalise in (True, False):
            logits, dw = randn(20, 7, seed=1), randn(20, 3, seed=2)
            chosen = experts.route(logits, 3, scores, renormalise=renormalise).experts
            got = experts.route_adjoint(dw, logits, chosen, scores, renormalise).double()
            h = 2.0 ** -17
            for e in range(7):
                step = torch.zeros(7, dtype=torch.float64, device="cuda")
                step[e] = h
                up, down = (weights_of(logits.double() + s * step, chosen, scores, renormalise, 1.0)[0] for s in (1, -1))
                slope = ((up - down) * dw.double()).sum(1) / (2 * h)
                assert ((got[:, e] - slope).abs() <= 1e-5).all()  # 60 e of terms of size 3, and h^2 times theirs


@pytest.mark.parametrize("entries,count", ((0, 3), (1, 1), (1, 1024), (63, 5), (64, 5), (65, 5), (1000, 511), (1000, 512), (1025, 200),
                                           (4096, 9), (4097, 9), (8192, 300), (8193, 300), (8194, 1024), (16384, 8), (16385, 8), (16386, 1024),
                                           (32768, 65), (32769, 65), (50000, 1), (100003, 37), (300000, 256)))
def test_plan(entries, count):
    for k in (1, 2 if entries % 2 == 0 else 1):
        k = min(k, count)
        g = torch.Generator(device="cuda").manual_seed(entries)
        chosen = torch.randint(-2, count + 2, (entries // k, k), generator=g, device="cuda", dtype=torch.int32)
        chosen[chosen == -2] = -(1 << 31)
        check_plan(experts.plan(chosen, count), chosen, count)
        same = torch.full_like(chosen, count - 1)  # all with one expert
        check_plan(experts.plan(same, count), same, count)


def test_leading_dims_and_nothing_at_all():
    logits = randn(4, 5, 6, seed=1)
    r = experts.route(logits, 2)
    flat = experts.route(logits.reshape(20, 6), 2)
    assert r.experts.shape == r.weights.shape == (4, 5, 2) and torch.equal(r.experts.reshape(20, 2), flat.experts)
    assert torch.equal(r.plan.slots, flat.plan.slots) and r.plan.rows == 20 and r.plan.top_k == 2 and r.plan.experts == 6
    assert torch.equal(experts.plan(r.experts, 6).order, r.plan.order)
    d = experts.route_adjoint(r.weights, logits, r.experts)
    assert d.shape == logits.shape
    x, w = randn(4, 5, 8, seed=2), randn(6, 3, 8, seed=3)
    y = experts.linear(x, w, r.plan, gather=True).out
    assert y.shape == (40, 3) and experts.combine(y, r.plan, r.weights, randn(4, 5, 3, seed=4)).shape == (4, 5, 3)
    back = experts.linear_adjoint(y, x, w, r.plan, gather=True, bias=False)
    assert back.x.shape == x.shape and back.weight.shape == w.shape and back.bias is None
    none = experts.route(logits[:0].reshape(0, 6), 2)
    assert none.experts.shape == (0, 2) and (none.plan.offsets == 0).all() and none.plan.order.numel() == 0
    x = randn(0, 8, seed=2)
    assert experts.linear(x, w, none.plan, gather=True).out.shape == (0, 3)
    assert experts.combine(randn(0, 3, seed=1), none.plan, none.weights).shape == (0, 3)
    for act in ("identity", "gelu"):
        z = None if act == "identity" else randn(0, 3, seed=1)
        back = experts.linear_adjoint(randn(0, 3, seed=1), x, w, none.plan, z, act, gather=True)
        assert back.x.shape == (0, 8) and (back.weight == 0).all() and (back.bias == 0).all()
        added = torch.ones(6, 3, 8, device="cuda"), torch.ones(6, 3, device="cuda")
        experts.linear_adjoint(randn(0, 3, seed=1), x, w, none.plan, z, act, weight_adjoint=added[0], bias_adjoint=added[1])
        assert (added[0] == 1).all() and (added[1] == 1).all()


# ------------------------------------------------------------------------------ the experts' linear layers
def of_slots(plan):
    """Each slot's expert (the number of experts: none) and row."""
    slot = torch.arange(plan.order.numel(), device="cuda")
    expert = torch.searchsorted(plan.offsets[1:].long().contiguous(), slot, right=True)
    return expert, torch.div(plan.order.long(), plan.top_k, rounding_mode="floor")


def linear_reference(x, weight, bias, plan, act, gather):
    expert, row = of_slots(plan)
    rows = x.double()[row] if gather else x.double()
    n = weight.shape[1]
    z = torch.zeros(rows.shape[0], n, dtype=torch.float64, device="cuda")
    most = torch.zeros_like(z)
    for e in range(plan.experts):
        i = (expert == e).nonzero()[:, 0]
        if i.numel():
            z[i] = rows[i] @ weight[e].double().T
            most[i] = rows[i].abs() @ weight[e].double().abs().T
            if bias is not None:
                z[i] += bias[e].double()
                most[i] += bias[e].double().abs()
    err = (weight.shape[2] + 8) * E * most
    y = ACTS[act](z)
    return z, err, y, err * 1.13 + (0 if act == "identity" else 16 * E * (1 + z.abs()) * (1 + y.abs()))


# few slots an expert; small, narrow and large tiles; whole units or not; the direct tiles
LINEARS = ((1, 4, 2, 8, 8), (40, 16, 2, 1024, 1024), (1, 32, 4, 2048, 64), (3, 1024, 32, 33, 40), (17, 3, 2, 130, 66), (40, 256, 8, 72, 50), (200, 7, 3, 66, 128),
           (1000, 4, 2, 129, 18), (1000, 4, 1, 64, 33), (3000, 5, 2, 31, 200), (3000, 300, 4, 40, 24), (2000, 2, 1, 512, 512),
           (5000, 4, 2, 256, 512), (4096, 8, 4, 320, 264), (20000, 8, 2, 66, 128), (1100, 8, 2, 1024, 1024), (2100, 8, 2, 2048, 512))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,count,k,inputs,outputs", LINEARS)
def test_linear(dtype, rows, count, k, inputs, outputs):
    for n, act in enumerate(ACTS):
        gather, keep = n % 2 == 0, n > 1
        plan, _ = routed(rows, count, k, seed=rows + n, none=0.1 if n % 2 else 0.0)
        x = randn(rows if gather else rows * k, inputs, seed=n, dtype=dtype, pad=(0, 3, 8, 1)[n] if inputs % 8 else 0)
        w = randn(count, outputs, inputs, seed=5, scale=inputs ** -0.5, dtype=dtype)
        b = None if n == 0 else randn(count, outputs, seed=6, scale=0.2, dtype=torch.float32 if n == 1 else dtype)
        z, z_err, y, y_err = linear_reference(x, w, b, plan, act, gather)
        r = experts.linear(x, w, plan, b, act, gather, keep)
        live = int(plan.offsets[-1])
        check(r.out[:live], y[:live], y_err[:live], (act, "out"))
        assert (r.out[live:] == 0).all()
        if keep:
            check(r.preactivation[:live], z[:live], z_err[:live], (act, "z"))
            assert (r.preactivation[live:] == 0).all()
        else:
            assert r.preactivation is None


def adjoint_reference(dy, x, weight, z, plan, act, gather):
    """Gradients and their bounds; dz is rounded to the layer's type where there is an activation."""
    expert, row = of_slots(plan)
    rows = x.double()[row] if gather else x.double()
    dz = dy.double()
    dz_err = torch.zeros_like(dz)
    if act != "identity":
        leaf = z.double().requires_grad_()
        slope, = torch.autograd.grad(ACTS[act](leaf).sum(), leaf)
        dz_err = 32 * E * dz.abs() * (1 + z.double().abs())
        dz = dz * slope
    live = (expert < plan.experts)[:, None]
    dz, dz_err = torch.where(live, dz, 0.0), torch.where(live, dz_err, 0.0)
    rounded = dz_err + (0 if act == "identity" else U[dy.dtype] * dz.abs() + TINY[dy.dtype] * live)
    count, n, k = weight.shape
    dx = torch.zeros(rows.shape[0], k, dtype=torch.float64, device="cuda")
    dx_err, dw = torch.zeros_like(dx), torch.zeros(weight.shape, dtype=torch.float64, device="cuda")
    dw_err, db = torch.zeros_like(dw), torch.zeros(count, n, dtype=torch.float64, device="cuda")
    db_err = torch.zeros_like(db)
    for e in range(count):
        i = (expert == e).nonzero()[:, 0]
        if i.numel():
            w = weight[e].double()
            d, r = dz[i], rounded[i]
            dx[i] = d @ w
            dx_err[i] = r @ w.abs() + (n + 8) * E * ((d.abs() + r) @ w.abs())
            dw[e] = d.T @ rows[i]
            dw_err[e] = r.T @ rows[i].abs() + (i.numel() + 8) * E * ((d.abs() + r).T @ rows[i].abs())
            db[e] = d.sum(0)
            db_err[e] = dz_err[i].sum(0) + (i.numel() + 8) * E * d.abs().sum(0)
    if gather:
        dx = torch.zeros(x.reshape(-1, k).shape, dtype=torch.float64, device="cuda").index_add_(0, row, dx)
        most = torch.zeros_like(dx).index_add_(0, row, dx_err)
        dx_err = most + 40 * E * (dx.abs() + most)
    return (dx, dx_err), (dw, dw_err), (db, db_err)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,count,k,inputs,outputs", LINEARS)
def test_linear_adjoint(dtype, rows, count, k, inputs, outputs):
    for n, act in enumerate(ACTS):
        gather = n % 2 == 0
        plan, _ = routed(rows, count, k, seed=rows + n, none=0.1 if n % 2 else 0.0)
        slots, live = rows * k, int(plan.offsets[-1])
        x = randn(rows if gather else slots, inputs, seed=n, dtype=dtype, pad=(0, 3, 8, 1)[n] if inputs % 8 else 0)
        w = randn(count, outputs, inputs, seed=5, scale=inputs ** -0.5, dtype=dtype)
        dy = randn(slots, outputs, seed=6, scale=0.3, dtype=dtype, pad=n if outputs % 8 else 0)
        z = None if act == "identity" else randn(slots, outputs, seed=7, dtype=dtype)
        dy[live:] = math.nan  # slots without an expert are not read
        r = experts.linear_adjoint(dy, x, w, plan, z, act, gather)
        dx, dw, db = adjoint_reference(torch.nan_to_num(dy), x, w, z, plan, act, gather)
        check(r.x, *dx, (act, "x"))
        check(r.weight, *dw, (act, "weight"))
        check(r.bias, *db, (act, "bias"))
        if not gather:
            assert (r.x[live:] == 0).all()


# x's gradient in parts: a sum over many outputs, few slots
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gather", (True, False))
@pytest.mark.parametrize("rows,count,k,inputs,outputs", ((1, 9, 8, 30, 2779), (13, 3, 3, 61, 1041), (75, 13, 8, 44, 2240), (130, 4, 1, 8, 4097)))
def test_linear_adjoint_of_few_slots_and_many_outputs(dtype, gather, rows, count, k, inputs, outputs):
    for act, none in (("identity", 0.3), ("silu", 0.0)):
        plan, _ = routed(rows, count, k, seed=rows, none=none)
        slots, live = rows * k, int(plan.offsets[-1])
        x, w = randn(rows if gather else slots, inputs, seed=1, dtype=dtype), randn(count, outputs, inputs, seed=2, scale=0.2, dtype=dtype)
        dy = randn(slots, outputs, seed=3, scale=0.3, dtype=dtype)
        z = None if act == "identity" else randn(slots, outputs, seed=4, dtype=dtype)
        dy[live:] = math.nan
        (dx, dx_err), (dw, dw_err), (db, db_err) = adjoint_reference(torch.nan_to_num(dy), x, w, z, plan, act, gather)
        both, alone = experts.linear_adjoint(dy, x, w, plan, z, act, gather), experts.linear_adjoint(dy, x, w, plan, z, act, gather, parameters=False)
        for r in (both, alone):
            check(r.x, dx, dx_err, act)
            if not gather:
                assert (r.x[live:] == 0).all()
        check(both.weight, dw, dw_err, act)
        check(both.bias, db, db_err, act)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ("identity", "gelu"))
def test_gradients_that_are_added_to_and_left_out(dtype, act):
    for rows, inputs, outputs in ((300, 66, 40), (6000, 48, 64)):
        plan, _ = routed(rows, 6, 2, seed=1, none=0.1)
        x, w = randn(rows, inputs, seed=1, dtype=dtype), randn(6, outputs, inputs, seed=2, scale=0.1, dtype=dtype)
        dy = randn(rows * 2, outputs, seed=3, scale=0.3, dtype=dtype)
        z = None if act == "identity" else randn(rows * 2, outputs, seed=4, dtype=dtype)
        (dx, dx_err), (dw, dw_err), (db, db_err) = adjoint_reference(dy, x, w, z, plan, act, True)
        for kind in (torch.float32, dtype):
            gw, gb = randn(6, outputs, inputs, seed=5, dtype=kind), randn(6, outputs, seed=6, dtype=kind)
            w0, b0 = gw.double(), gb.double()
            r = experts.linear_adjoint(dy, x, w, plan, z, act, True, weight_adjoint=gw, bias_adjoint=gb)
            assert r.weight is gw and r.bias is gb
            check(gw, w0 + dw, dw_err + 2 * E * (w0.abs() + dw.abs()), "weight")
            check(gb, b0 + db, db_err + 2 * E * (b0.abs() + db.abs()), "bias")
        whole = experts.linear_adjoint(dy, x, w, plan, z, act, True)
        no_x = experts.linear_adjoint(dy, x, w, plan, z, act, True, inputs=False)
        only_x = experts.linear_adjoint(dy, x, w, plan, z, act, True, parameters=False)
        no_b = experts.linear_adjoint(dy, x, w, plan, z, act, True, bias=False)
        assert no_x.x is None and only_x.weight is None and only_x.bias is None and no_b.bias is None
        # the sums may be split otherwise, so each is held to its own bound
        for r in (whole, only_x, no_b):
            check(r.x, dx, dx_err, "x")
        for r in (whole, no_x, no_b):
            check(r.weight, dw, dw_err, "weight")
        for r in (whole, no_x):
            check(r.bias, db, db_err, "bias")


def test_bias_gradient_alone():
    plan, _ = routed(500, 5, 2, seed=1, none=0.2)
    ctx = Context(0)
    for act, code in (("identity", 0), ("silu", 3)):
        dy, z = randn(1000, 70, seed=2), randn(1000, 70, seed=3)
        db = torch.empty(5, 70, device="cuda")
        cfg = _abi.NpaExpertLinearCfg(500, 0, 0, 0, 0, 0, 0, 5, 2, 8, 70, 0, code, 0, 0, 0, 0)
        ctx.check(lib().npa_expert_linear_adjoint(ctx.handle, C.byref(cfg), None, None, ptr(z), ptr(plan.offsets), None, None,
                                                  ptr(dy), None, None, ptr(db)))
        ctx.synchronize()
        _, _, (want, err) = adjoint_reference(dy, randn(1000, 8, seed=4), randn(5, 70, 8, seed=5), z, plan, act, False)
        check(db, want, err, act)


@pytest.mark.parametrize("dtype", TYPES)
def test_all_rows_with_one_expert_and_experts_without_rows(dtype):
    for count, only in ((5, 0), (5, 4), (64, 17)):
        chosen = torch.full((700, 1), only, dtype=torch.int32, device="cuda")
        plan = experts.plan(chosen, count)
        x, w = randn(700, 96, seed=1, dtype=dtype), randn(count, 80, 96, seed=2, scale=0.1, dtype=dtype)
        z, z_err, y, y_err = linear_reference(x, w, None, plan, "identity", True)
        check(experts.linear(x, w, plan, gather=True).out, y, y_err, "out")
        dy = randn(700, 80, seed=3, dtype=dtype)
        r = experts.linear_adjoint(dy, x, w, plan, gather=True)
        dx, dw, db = adjoint_reference(dy, x, w, None, plan, "identity", True)
        check(r.x, *dx, "x")
        check(r.weight, *dw, "weight")
        check(r.bias, *db, "bias")
        others = [e for e in range(count) if e != only]
        assert (r.weight[others] == 0).all() and (r.bias[others] == 0).all()
    nobody = experts.plan(torch.full((300, 2), -1, dtype=torch.int32, device="cuda"), 3)
    x, w = randn(300, 96, seed=1, dtype=dtype), randn(3, 80, 96, seed=2, dtype=dtype)
    x[:] = math.nan
    assert (experts.linear(x, w, nobody, randn(3, 80, seed=1), "gelu", True).out == 0).all()
    r = experts.linear_adjoint(randn(600, 80, seed=3, dtype=dtype), x, w, nobody, gather=True)
    assert (r.x == 0).all() and (r.weight == 0).all() and (r.bias == 0).all()


@pytest.mark.parametrize("gather", (True, False))
def test_f32_infinities_and_small_numbers(gather):
    """f32 operands whose bf16 parts do not sum to them: the f32 result, and infinities and NaN in their rows only."""
    for rows, inputs, outputs in ((40, 70, 48), (900, 66, 128)):
        plan, _ = routed(rows, 3, 2, seed=1)
        n = rows if gather else rows * 2
        x, w = randn(n, inputs, seed=1), randn(3, outputs, inputs, seed=2)
        x[0, 0], x[1, 1], x[2, 2] = INF, math.nan, -INF
        clean = torch.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0)
        got = experts.linear(x, w, plan, gather=gather).out
        want = experts.linear(clean, w, plan, gather=gather).out
        _, row = of_slots(plan)
        odd = (row if gather else torch.arange(rows * 2, device="cuda")) < 3
        assert torch.equal(got[~odd], want[~odd]) and not torch.isfinite(got[odd]).any()
        small = randn(n, inputs, seed=3, scale=2.0 ** -124)
        z, err, _, _ = linear_reference(small, w, None, plan, "identity", gather)
        check(experts.linear(small, w, plan, gather=gather).out, z, err, "small")


# ------------------------------------------------------------------------------ combining
COMBINES = ((1, 4, 1, 1), (1, 32, 8, 5), (37, 3, 2, 7), (300, 8, 2, 18), (129, 9, 3, 66), (64, 40, 32, 130), (200, 4, 2, 513), (33, 5, 4, 4099),
            (7, 3, 2, 20003), (600, 5, 4, 1030))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,count,k,width", COMBINES)
def test_combine(dtype, rows, count, k, width):
    for n in range(4):
        plan, chosen = routed(rows, count, k, seed=rows + n, none=0.3 if n % 2 else 0.0)
        slots, live = rows * k, int(plan.offsets[-1])
        y = randn(slots, width, seed=n, dtype=dtype, pad=n)
        y[live:] = math.nan
        w = torch.rand(rows, k, device="cuda") if n else None
        res = randn(rows, width, seed=9, dtype=dtype, pad=n % 2) if n > 1 else None
        part = torch.nan_to_num(y.double())[plan.slots.long()]
        factor = (chosen >= 0).double() * (1 if w is None else w.double())
        terms = part * factor[:, :, None]
        want = terms.sum(1) + (0 if res is None else res.double())
        most = terms.abs().sum(1) + (0 if res is None else res.double().abs())
        if w is not None:
            w[chosen < 0] = math.nan  # not read
        check(experts.combine(y, plan, w, res), want, (k + 8) * E * most, "out")
        dout = randn(rows, width, seed=8, dtype=dtype, pad=n % 3)
        r = experts.combine_adjoint(dout, y, plan, w)
        expert, row = of_slots(plan)
        dy = dout.double()[row] * factor.reshape(-1)[plan.order.long()][:, None]
        check(r.y, dy, 2 * E * dy.abs(), "y")
        assert (r.y[live:] == 0).all()
        if w is None:
            assert r.weights is None
        else:
            prod = part * dout.double()[:, None] * (chosen >= 0)[:, :, None]
            check(r.weights, prod.sum(2), (width + 8) * E * prod.abs().sum(2), "weights")


def test_combine_over_its_residual():
    plan, _ = routed(200, 4, 2, seed=1)
    y, w, res = randn(400, 66, seed=2), torch.rand(200, 2, device="cuda"), randn(200, 66, seed=3)
    want = experts.combine(y, plan, w, res)
    ctx = Context(0)
    cfg = _abi.NpaCombineCfg(200, 0, 0, 0, 0, 0, 4, 2, 66, 0)
    ctx.check(lib().npa_expert_combine(ctx.handle, C.byref(cfg), ptr(y), ptr(plan.offsets), ptr(plan.slots), ptr(w), ptr(res), ptr(res)))
    ctx.synchronize()
    assert torch.equal(res, want)


# ------------------------------------------------------------------------------ together
def block(x, wr, w1, b1, w2, b2, count, k, dout):
    """A mixture of two-layer rules with a residual, forward and backward."""
    logits = layers.linear(x, wr).out
    r = experts.route(logits, k)
    h = experts.linear(x, w1, r.plan, b1, "gelu", True, True)
    y = experts.linear(h.out, w2, r.plan, b2)
    out = experts.combine(y.out, r.plan, r.weights, x)
    c = experts.combine_adjoint(dout, y.out, r.plan, r.weights)
    second = experts.linear_adjoint(c.y, h.out, w2, r.plan)
    first = experts.linear_adjoint(second.x, x, w1, r.plan, h.preactivation, "gelu", True)
    dl = experts.route_adjoint(c.weights, logits, r.experts)
    router = layers.linear_adjoint(dl, x, wr, bias=False)
    return [out, dout + first.x + router.x, router.weight, first.weight, first.bias, second.weight, second.bias, r.experts,
            r.plan.order, r.weights]


def block_inputs(rows, width, hidden, count, dtype=torch.float32, seed=0):
    return (randn(rows, width, seed=seed + 1, dtype=dtype), randn(count, width, seed=seed + 2, scale=width ** -0.5, dtype=dtype),
            randn(count, hidden, width, seed=seed + 3, scale=width ** -0.5, dtype=dtype), randn(count, hidden, seed=seed + 4, scale=0.1, dtype=dtype),
            randn(count, width, hidden, seed=seed + 5, scale=hidden ** -0.5, dtype=dtype), randn(count, width, seed=seed + 6, scale=0.1, dtype=dtype))


def test_a_block_against_reverse_differentiation():
    """The whole run in f32 against 64 bits for the experts it chose. Each gradient within 1e-5 of its largest element: sums
    of up to 500 f32 terms, 2^-24 * 500 = 3e-5 at the very worst of their absolute values and about 2^-24 * sqrt(500) of
    it for terms of either sign."""
    rows, width, hidden, count, k = 250, 34, 50, 5, 2
    args = block_inputs(rows, width, hidden, count)
    dout = randn(rows, width, seed=9)
    got = block(*args, count, k, dout)
    chosen = got[7].long()
    leaves = [t.double().requires_grad_() for t in args]
    x, wr, w1, b1, w2, b2 = leaves
    s = torch.softmax(x @ wr.T, 1).gather(1, chosen)
    s = s / (s.sum(1, keepdim=True) + 1e-20)
    out = x
    for j in range(k):
        e = chosen[:, j]
        h = ACTS["gelu"](torch.bmm(w1[e], x[:, :, None])[:, :, 0] + b1[e])
        out = out + s[:, j:j + 1] * (torch.bmm(w2[e], h[:, :, None])[:, :, 0] + b2[e])
    assert float((got[0].double() - out).abs().max()) < 1e-5 * float(out.abs().max())
    for g, want in zip(got[1:7], torch.autograd.grad((out * dout.double()).sum(), leaves)):
        assert float((g.double() - want).abs().max()) < 1e-5 * float(want.abs().max())


@pytest.mark.parametrize("dtype,rows,width,hidden,count", ((torch.float32, 600, 66, 128, 8), (torch.bfloat16, 3000, 256, 512, 4),
                                                           (torch.float16, 40, 50, 30, 300)))
def test_same_bits_each_time_eagerly_captured_and_on_other_streams(dtype, rows, width, hidden, count):
    args, dout = block_inputs(rows, width, hidden, count, dtype), randn(rows, width, seed=9, dtype=dtype)
    other = block_inputs(rows * 2, width, hidden, count, dtype, 50)
    other_dout = randn(rows * 2, width, seed=10, dtype=dtype)
    want = block(*args, count, 2, dout)
    want_other = block(*other, count, 2, other_dout)
    assert all(torch.equal(a, b) for a, b in zip(block(*args, count, 2, dout), want))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        assert all(torch.equal(a, b) for a, b in zip(block(*args, count, 2, dout), want))
        own = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=own):  # a context without a workspace
            got = block(*args, count, 2, dout)
        second = torch.cuda.CUDAGraph()
        with torch.cuda.graph(second, stream=own):  # and one with a workspace that is too small
            got_other = block(*other, count, 2, other_dout)
        for turn in range(3):
            for t in got + got_other:
                t.fill_(7)
            if turn % 2:
                second.replay()
                graph.replay()
            else:
                graph.replay()
                second.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(torch.equal(a, b) for a, b in zip(got_other, want_other))
            again = block(*other, count, 2, other_dout)
            torch.full((1 << 22,), math.nan, device="cuda")
            assert all(torch.equal(a, b) for a, b in zip(again, want_other))
        # the graph's inputs are read anew
        args[0].copy_(randn(rows, width, seed=77, dtype=dtype))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, block(*args, count, 2, dout)))


def test_two_threads_at_once():
    cases = [(block_inputs(500 + 100 * i, 66, 64, 6, seed=i), randn(500 + 100 * i, 66, seed=9)) for i in range(2)]
    want = [block(*a, 6, 2, d) for a, d in cases]
    torch.cuda.synchronize()
    right = [False, False]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            ok = True
            for _ in range(10):
                got = block(*cases[i][0], 6, 2, cases[i][1])
                torch.cuda.current_stream().synchronize()
                ok = ok and all(torch.equal(a, b) for a, b in zip(got, want[i]))
            right[i] = ok

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(right)


def test_a_plan_of_other_contents_is_no_access_outside():
    """Offsets, order and slots that are no plan's: results are of no use, and calls that follow are right."""
    rows, count, k = 500, 6, 2
    good, _ = routed(rows, count, k, seed=1)
    g = torch.Generator(device="cuda").manual_seed(2)
    anything = lambda *s: torch.randint(-(1 << 31), (1 << 31) - 1, s, generator=g, device="cuda", dtype=torch.int32)  # noqa: E731
    x, w1 = randn(rows, 66, seed=1), randn(count, 40, 66, seed=2)
    want = experts.linear(x, w1, good, gather=True).out
    for bad in (experts.Plan(anything(count + 1), anything(rows * k), anything(rows, k)),
                experts.Plan(good.offsets.flip(0).contiguous(), good.order, good.slots + 400)):
        y = experts.linear(x, w1, bad, gather=True).out
        experts.linear_adjoint(y, x, w1, bad, y, "gelu", True)
        experts.combine_adjoint(experts.combine(y, bad, torch.rand(rows, k, device="cuda")), y, bad, torch.rand(rows, k, device="cuda"))
        experts.route_adjoint(torch.rand(rows, k, device="cuda"), randn(rows, count, seed=3), anything(rows, k))
        torch.cuda.synchronize()
    assert torch.equal(experts.linear(x, w1, good, gather=True).out, want)


def test_weights_in_place():
    """A slice of the experts' inputs is taken where it lies, other views as copies."""
    plan, _ = routed(50, 4, 2, seed=1)
    wide, x = randn(4, 30, 64, seed=2), randn(50, 40, seed=3)
    assert experts._weight(wide[:, :, 8:48], plan, 40, x)[0].data_ptr() == wide.data_ptr() + 32
    want = experts.linear(x, wide[:, :, 8:48].contiguous(), plan, gather=True).out
    assert torch.equal(experts.linear(x, wide[:, :, 8:48], plan, gather=True).out, want)
    turned = wide[:, :, :30].transpose(1, 2)
    want = experts.linear(x[:, :30], turned.contiguous(), plan, gather=True).out
    assert torch.equal(experts.linear(x[:, :30], turned, plan, gather=True).out, want)


def test_host_arrays():
    """A context in host-I/O mode: the same results from host arrays."""
    rows, count, k, width = 70, 5, 2, 20
    x, l, w = randn(rows, width, seed=1), randn(rows, count, seed=2), randn(count, 12, width, seed=3)
    r = experts.route(l, k)
    lin = experts.linear(x, w, r.plan, gather=True)
    dy = randn(rows * k, 12, seed=4)
    back = experts.linear_adjoint(dy, x, w, r.plan, gather=True)
    out = experts.combine(lin.out, r.plan, r.weights)
    cadj = experts.combine_adjoint(out, lin.out, r.plan, r.weights)
    dl = experts.route_adjoint(cadj.weights, l, r.experts)
    torch.cuda.synchronize()
    ctx = Context(0, host_io=True)
    host = lambda t: t.cpu().contiguous()  # noqa: E731
    new = lambda *s, t=torch.float32: torch.full(s, 3, dtype=t)  # noqa: E731
    i32 = torch.int32
    hx, hl, hw, hdy = host(x), host(l), host(w), host(dy)
    ex, wt, of, od, sl = new(rows, k, t=i32), new(rows, k), new(count + 1, t=i32), new(rows * k, t=i32), new(rows, k, t=i32)
    cfg = _abi.NpaRouteCfg(rows, 0, 0, count, k, 1, 1, 0, 0, 0, 1, 1.0)
    ctx.check(lib().npa_expert_route(ctx.handle, C.byref(cfg), ptr(hl), None, ptr(ex), ptr(wt), ptr(of), ptr(od), ptr(sl)))
    for got, want in ((ex, r.experts), (wt, r.weights), (of, r.plan.offsets), (od, r.plan.order), (sl, r.plan.slots)):
        assert torch.equal(got, want.cpu())
    of2, od2, sl2 = new(count + 1, t=i32), new(rows * k, t=i32), new(rows, k, t=i32)
    ctx.check(lib().npa_expert_plan(ctx.handle, rows, k, count, ptr(ex), ptr(of2), ptr(od2), ptr(sl2)))
    assert torch.equal(of, of2) and torch.equal(od, od2) and torch.equal(sl, sl2)
    lc = _abi.NpaExpertLinearCfg(rows, 0, 0, 0, 0, 0, 0, count, k, width, 12, 0, 0, 0, 0, 0, 1)
    y = new(rows * k, 12)
    ctx.check(lib().npa_expert_linear(ctx.handle, C.byref(lc), ptr(hx), ptr(hw), None, ptr(of), ptr(od), ptr(y), None))
    assert torch.equal(y, lin.out.cpu())
    dx, dw, db = new(rows, width), new(count, 12, width), new(count, 12)
    ctx.check(lib().npa_expert_linear_adjoint(ctx.handle, C.byref(lc), ptr(hx), ptr(hw), None, ptr(of), ptr(od), ptr(sl), ptr(hdy),
                                              ptr(dx), ptr(dw), ptr(db)))
    for got, want in ((dx, back.x), (dw, back.weight), (db, back.bias)):
        assert torch.equal(got, want.cpu())
    cc = _abi.NpaCombineCfg(rows, 0, 0, 0, 0, 0, count, k, 12, 0)
    o, dyy, dwt = new(rows, 12), new(rows * k, 12), new(rows, k)
    ctx.check(lib().npa_expert_combine(ctx.handle, C.byref(cc), ptr(y), ptr(of), ptr(sl), ptr(wt), None, ptr(o)))
    ctx.check(lib().npa_expert_combine_adjoint(ctx.handle, C.byref(cc), ptr(y), ptr(of), ptr(sl), ptr(wt), ptr(o), ptr(dyy), ptr(dwt)))
    dlh = new(rows, count)
    ctx.check(lib().npa_expert_route_adjoint(ctx.handle, C.byref(cfg), ptr(hl), ptr(ex), ptr(dwt), ptr(dlh)))
    for got, want in ((o, out), (dyy, cadj.y), (dwt, cadj.weights), (dlh, dl)):
        assert torch.equal(got, want.cpu())


def test_refusals():
    plan, chosen = routed(50, 4, 2, seed=1)
    x, w, l = randn(50, 8, seed=1), randn(4, 6, 8, seed=2), randn(50, 4, seed=3)
    y = randn(100, 6, seed=4)
    bad = _abi.InvalidArgument
    for call, error in (
            (lambda: experts.route(l, 0), bad), (lambda: experts.route(l, 5), bad), (lambda: experts.route(l.double(), 2), bad),
            (lambda: experts.route(l, 2, "tanh"), bad), (lambda: experts.route(l, 2, bias=l[0, :3]), _abi.OutputShape),
            (lambda: experts.route(l, 2, bias=l[0].double()), bad), (lambda: experts.route(l, 2, groups=3), bad),
            (lambda: experts.route(l, 2, groups=0), bad), (lambda: experts.route(l, 2, groups=4, top_groups=1), bad),
            (lambda: experts.route(l, 2, groups=2, top_groups=3), bad), (lambda: experts.route(l, 2, groups=2, top_groups=0), bad),
            (lambda: experts.route(l, 2, scale=INF), bad), (lambda: experts.route(randn(2, 1025, seed=1), 2), bad),
            (lambda: experts.route(randn(2, 128, seed=1), 65, groups=128, top_groups=128), bad),
            (lambda: experts.route_adjoint(l[:, :2], l, chosen.long()), bad), (lambda: experts.route_adjoint(l, l, chosen), _abi.OutputShape),
            (lambda: experts.route_adjoint(l[:, :2].half(), l, chosen), bad),
            (lambda: experts.plan(chosen.long(), 4), bad), (lambda: experts.plan(chosen, 1), bad), (lambda: experts.plan(chosen, 1025), bad),
            (lambda: experts.Plan(plan.offsets.long(), plan.order, plan.slots), bad),
            (lambda: experts.Plan(plan.offsets, plan.order[:-1], plan.slots), _abi.OutputShape),
            (lambda: experts.Plan(plan.offsets, plan.order, plan.slots.t()), bad),
            (lambda: experts.linear(x, w, (plan.offsets, plan.order, plan.slots)), bad),
            (lambda: experts.linear(x, w, plan), _abi.OutputShape), (lambda: experts.linear(y, w, plan, gather=True), _abi.OutputShape),
            (lambda: experts.linear(x, w[:3], plan, gather=True), _abi.OutputShape), (lambda: experts.linear(x, w[0], plan, gather=True), _abi.OutputShape),
            (lambda: experts.linear(x, w.half(), plan, gather=True), bad), (lambda: experts.linear(x, w, plan, randn(6, seed=1), gather=True), _abi.OutputShape),
            (lambda: experts.linear(x, w, plan, None, "tanh", True), bad),
            (lambda: experts.linear_adjoint(y, x, w, plan, None, "gelu", True), bad),
            (lambda: experts.linear_adjoint(y[:99], x, w, plan, gather=True), _abi.OutputShape),
            (lambda: experts.linear_adjoint(y, x, w, plan, gather=True, weight_adjoint=w.clone()), bad),
            (lambda: experts.linear_adjoint(y, x, w, plan, gather=True, weight_adjoint=w[0].clone(), bias=False), _abi.OutputShape),
            (lambda: experts.combine(y[:99], plan), _abi.OutputShape), (lambda: experts.combine(y, plan, l), _abi.OutputShape),
            (lambda: experts.combine(y, plan, l[:, :2].half()), bad), (lambda: experts.combine(y, plan, None, x), _abi.OutputShape),
            (lambda: experts.combine(y, plan, None, y[:50].half()), bad),
            (lambda: experts.combine_adjoint(y, y, plan), _abi.OutputShape),
            (lambda: experts.combine(y, plan, ctx=Context(0, stream=torch.cuda.Stream().cuda_stream)), bad)):
        with pytest.raises(error):
            call()
    ctx = Context(0)
    L = lib()
    rc = _abi.NpaRouteCfg(50, 3, 0, 4, 2, 1, 1, 0, 0, 0, 1, 1.0)  # a stride below the row's length
    args = (ptr(l), None, ptr(chosen), ptr(torch.empty(50, 2, device="cuda")))
    assert L.npa_expert_route(ctx.handle, C.byref(rc), *args, None, None, None) == bad.code
    rc.logits_stride = 0
    assert L.npa_expert_route(ctx.handle, C.byref(rc), *args, None, ptr(plan.order), ptr(plan.slots)) == bad.code
    assert L.npa_expert_route(ctx.handle, C.byref(rc), None, None, args[2], args[3], None, None, None) == bad.code
    assert L.npa_expert_route(ctx.handle, None, *args, None, None, None) == bad.code
    rc.element_type = 3
    assert L.npa_expert_route(ctx.handle, C.byref(rc), *args, None, None, None) == bad.code
    lc = _abi.NpaExpertLinearCfg(50, 0, 0, 0, 0, 0, 0, 4, 2, 8, 6, 0, 0, 0, 0, 0, 1)
    out = torch.empty(100, 6, device="cuda")
    assert L.npa_expert_linear(ctx.handle, C.byref(lc), ptr(x), ptr(w), None, ptr(plan.offsets), None, ptr(out), None) == bad.code
    assert L.npa_expert_linear(ctx.handle, C.byref(lc), ptr(x), ptr(w), None, None, ptr(plan.order), ptr(out), None) == bad.code
    lc.out_dims = 1 << 29
    assert L.npa_expert_linear(ctx.handle, C.byref(lc), ptr(x), ptr(w), None, ptr(plan.offsets), ptr(plan.order), ptr(out), None) == bad.code
    cc = _abi.NpaCombineCfg(1 << 30, 0, 0, 0, 0, 0, 4, 2, 6, 0)
    assert L.npa_expert_combine(ctx.handle, C.byref(cc), ptr(y), ptr(plan.offsets), ptr(plan.slots), None, None, ptr(out)) == bad.code


def test_elements_past_32_bits():
    """2^32 and more elements of out, of its adjoint and of a combined y: the last rows, and gradients of all."""
    rows, count, k, inputs, outputs = 1_100_000, 4, 2, 64, 2048
    dtype, last = torch.bfloat16, 500
    plan, _ = routed(rows, count, k, seed=1)
    slots = rows * k
    assert slots * outputs > 1 << 32
    x, w = randn(rows, inputs, seed=2, dtype=dtype), randn(count, outputs, inputs, seed=3, scale=0.125, dtype=dtype)
    out = experts.linear(x, w, plan, gather=True).out
    tail = plan.order[-last:].long() // k  # of the last expert
    check(out[-last:], x[tail].double() @ w[-1].double().T, inputs * E * (x[tail].double().abs() @ w[-1].double().abs().T), "out")
    weights = torch.rand(rows, k, device="cuda")
    got = experts.combine(out, plan, weights)
    where = plan.slots[-last:].long()
    terms = weights[-last:].double()[..., None] * out[where].double()
    check(got[-last:], terms.sum(1), 4 * E * terms.abs().sum(1), "combine")
    del got
    # dx and dW through out as its own adjoint
    r = experts.linear_adjoint(out, x, w, plan, gather=True)
    mine = torch.bucketize(where, plan.offsets[1:-1].long(), right=True)  # the experts of the last rows' slots
    products = torch.stack([torch.stack([out[s].double() @ w[e].double() for s, e in zip(a, b)]) for a, b in zip(where[-20:].tolist(), mine[-20:].tolist())])
    sizes = torch.stack([torch.stack([out[s].double().abs() @ w[e].double().abs() for s, e in zip(a, b)]) for a, b in zip(where[-20:].tolist(), mine[-20:].tolist())])
    check(r.x[-20:], products.sum(1), (outputs + 4) * E * sizes.sum(1), "x")
    begin, end = plan.offsets[-2:].tolist()
    dw = torch.zeros(outputs, inputs, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(dw)
    for at in range(begin, end, 100_000):
        d, rows_of = out[at:min(at + 100_000, end)].double(), x[plan.order[at:min(at + 100_000, end)].long() // k].double()
        dw += d.T.contiguous() @ rows_of
        size += d.abs().T.contiguous() @ rows_of.abs()
    check(r.weight[-1], dw, (end - begin + 1000) * E * size, "weight")
    back = experts.combine_adjoint(x.new_ones(rows, outputs), out, plan, weights)
    entry = plan.order[-last:].long()
    want = weights.reshape(-1)[entry].double()[:, None].expand(-1, outputs)
    check(back.y[-last:], want, 0.0 * want, "y")
    sums, bound = out[where].double().sum(2), out[where].double().abs().sum(2)
    check(back.weights[-last:], sums, outputs * E * bound, "weights")
