"""The mixture's layers on layouts that the Python calls do not make themselves: rows of results apart, arrays that begin at
any element, padded rows and slices of weights for every form of the products, rows of a few elements, and f32 operands that
are not the sum of their bf16 parts, backward. References and bounds are those of test_gpu_experts."""
import ctypes as C
import math

import pytest
import torch

from burn_automata_amd import _abi, experts
from burn_automata_amd._lib import lib
from burn_automata_amd.runtime import Context, ptr
from tests.test_gpu_experts import (E, adjoint_reference, check, choose, linear_reference, of_slots, randn, route_adjoint_reference, routed,
                                    weights_of)

pytestmark = pytest.mark.gpu

CODES = {torch.float32: _abi.TYPE_F32, torch.bfloat16: _abi.TYPE_BF16, torch.float16: _abi.TYPE_F16}
TYPES = tuple(CODES)
FILL = 7.0


def apart(rows, cols, stride, offset, dtype, fill=FILL):
    """A matrix of `stride` elements a row that begins at element `offset` of an allocation filled with `fill`, and the latter."""
    whole = torch.full((offset + rows * stride + 8,), fill, device="cuda", dtype=dtype)
    return whole[offset:offset + rows * stride].reshape(rows, stride)[:, :cols], whole


def put(t, stride, offset):
    """A copy of t with such a layout, NaN between its rows."""
    m, _ = apart(t.shape[0], t.shape[1], stride, offset, t.dtype, math.nan)
    return m.copy_(t)


def untouched(m, whole):
    m.fill_(FILL)
    return bool((whole == FILL).all())


# few slots, small tiles, large ones, narrow ones, direct ones
SIZES = ((3, 4, 2, 40, 24), (300, 5, 3, 66, 50), (4000, 6, 2, 66, 128), (4000, 6, 2, 128, 18), (1100, 4, 2, 256, 512))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,count,k,inputs,outputs", SIZES)
@pytest.mark.parametrize("gap,offset", ((0, 1), (1, 0), (5, 3), (8, 8)))
def test_linear_layouts(dtype, rows, count, k, inputs, outputs, gap, offset):
    ctx = Context(0)
    for act, gather in (("gelu", True), ("identity", False)):
        plan, _ = routed(rows, count, k, seed=rows, none=0.1)
        slots, live, n_x = rows * k, int(plan.offsets[-1]), rows if gather else rows * k
        x0, w0 = randn(n_x, inputs, seed=1, dtype=dtype), randn(count, outputs, inputs, seed=2, scale=inputs ** -0.5, dtype=dtype)
        b, dy0, z0 = randn(count, outputs, seed=3, dtype=dtype), randn(slots, outputs, seed=4, dtype=dtype), randn(slots, outputs, seed=5, dtype=dtype)
        x, w = put(x0, inputs + gap, offset), put(w0.reshape(-1, inputs), inputs + gap, offset)
        dy, z_in = put(dy0, outputs + gap, offset), put(z0, outputs + gap, offset)
        dy[live:] = math.nan
        out, out_all = apart(slots, outputs, outputs + gap, offset, dtype)
        z, z_all = apart(slots, outputs, outputs + gap, offset, dtype)
        dx, dx_all = apart(n_x, inputs, inputs + gap, offset, dtype)
        cfg = _abi.NpaExpertLinearCfg(rows, inputs + gap, inputs + gap, outputs + gap, outputs + gap, outputs + gap, inputs + gap, count, k,
                                      inputs, outputs, CODES[dtype], _abi.ACT_IDENTITY if act == "identity" else _abi.ACT_GELU, CODES[dtype], CODES[dtype], 0, int(gather))
        torch.cuda.synchronize()
        ctx.check(lib().npa_expert_linear(ctx.handle, C.byref(cfg), ptr(x), ptr(w), ptr(b), ptr(plan.offsets), ptr(plan.order), ptr(out), ptr(z)))
        ctx.synchronize()
        z_want, z_err, y_want, y_err = linear_reference(x0, w0, b, plan, act, gather)
        check(out[:live], y_want[:live], y_err[:live], (act, "out"))
        check(z[:live], z_want[:live], z_err[:live], (act, "z"))
        assert (out[live:] == 0).all() and (z[live:] == 0).all() and untouched(out, out_all) and untouched(z, z_all)
        dw, dw_all = apart(count * outputs, inputs, inputs, offset, dtype)
        db, db_all = apart(1, count * outputs, count * outputs, offset, dtype)
        ctx.check(lib().npa_expert_linear_adjoint(ctx.handle, C.byref(cfg), ptr(x), ptr(w), None if act == "identity" else ptr(z_in), ptr(plan.offsets),
                                                  ptr(plan.order), ptr(plan.slots), ptr(dy), ptr(dx), ptr(dw), ptr(db)))
        ctx.synchronize()
        want = adjoint_reference(dy0, x0, w0, None if act == "identity" else z0, plan, act, gather)
        check(dx, *want[0], (act, "x"))
        check(dw.reshape(count, outputs, inputs), *want[1], (act, "weight"))
        check(db.reshape(count, outputs), *want[2], (act, "bias"))
        assert untouched(dx, dx_all) and untouched(dw, dw_all) and untouched(db, db_all)


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("rows,count,k,inputs,outputs", ((2100, 8, 2, 512, 2048), (9000, 4, 1, 320, 256), (1500, 3, 2, 1024, 1024)))
@pytest.mark.parametrize("gap", (8, 64))
def test_large_tiles_of_padded_rows(dtype, rows, count, k, inputs, outputs, gap):
    for act, gather in (("gelu", True), ("identity", False), ("silu", False), ("relu", True)):
        plan, _ = routed(rows, count, k, seed=rows, none=0.05)
        slots, live = rows * k, int(plan.offsets[-1])
        x = randn(rows if gather else slots, inputs, seed=1, dtype=dtype, pad=gap)
        w = randn(count, outputs, inputs, seed=2, scale=inputs ** -0.5, dtype=dtype, pad=gap)
        assert experts._weight(w, plan, inputs, x)[2] == inputs + gap  # taken in place
        dy = randn(slots, outputs, seed=3, scale=0.3, dtype=dtype, pad=gap)
        z = None if act == "identity" else randn(slots, outputs, seed=4, dtype=dtype, pad=gap)
        if not gather:
            x[live:] = math.nan
        dy[live:] = math.nan
        _, _, y, y_err = linear_reference(torch.nan_to_num(x), w, None, plan, act, gather)
        out = experts.linear(x, w, plan, None, act, gather).out
        check(out[:live], y[:live], y_err[:live], (act, "out"))
        assert (out[live:] == 0).all()
        r = experts.linear_adjoint(dy, x, w, plan, z, act, gather)
        want = adjoint_reference(torch.nan_to_num(dy), torch.nan_to_num(x), w, z, plan, act, gather)
        for got, (value, bound), what in zip((r.x, r.weight, r.bias), want, ("x", "weight", "bias")):
            check(got, value, bound, (act, what))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("inputs", (1, 2, 6, 7, 8, 9))
@pytest.mark.parametrize("outputs", (1, 3, 7, 9))
def test_layers_of_a_few_columns(dtype, inputs, outputs):
    for rows, count, k, gather in ((1, 1, 1, True), (5, 3, 2, False), (70, 4, 3, True), (2000, 7, 2, False), (9000, 2, 2, True)):
        plan, _ = routed(rows, count, k, seed=rows, none=0.2)
        slots, live = rows * k, int(plan.offsets[-1])
        for act in ("identity", "silu"):
            x, w = randn(rows if gather else slots, inputs, seed=1, dtype=dtype, pad=1), randn(count, outputs, inputs, seed=2, dtype=dtype)
            b = randn(count, outputs, seed=3)
            z_want, z_err, y, y_err = linear_reference(x, w, b, plan, act, gather)
            r = experts.linear(x, w, plan, b, act, gather, True)
            check(r.out[:live], y[:live], y_err[:live], "out")
            check(r.preactivation[:live], z_want[:live], z_err[:live], "z")
            assert (r.out[live:] == 0).all() and (r.preactivation[live:] == 0).all()
            dy = randn(slots, outputs, seed=4, dtype=dtype, pad=2)
            z = None if act == "identity" else randn(slots, outputs, seed=5, dtype=dtype)
            dy[live:] = math.nan
            r = experts.linear_adjoint(dy, x, w, plan, z, act, gather)
            want = adjoint_reference(torch.nan_to_num(dy), x, w, z, plan, act, gather)
            for got, (value, bound), what in zip((r.x, r.weight, r.bias), want, ("x", "weight", "bias")):
                check(got, value, bound, (act, what))


@pytest.mark.parametrize("gather", (True, False))
def test_f32_infinities_and_small_numbers_backward(gather):
    """What is not finite stays in its rows of x's gradient and in its expert's of the weights'; small operands keep f32's accuracy."""
    for rows, inputs, outputs in ((40, 70, 48), (900, 66, 128), (5000, 66, 18)):
        plan, _ = routed(rows, 4, 2, seed=1)
        n, slots = rows if gather else rows * 2, rows * 2
        expert, row = of_slots(plan)
        x, w, dy = randn(n, inputs, seed=1), randn(4, outputs, inputs, seed=2), randn(slots, outputs, seed=3)
        clean = experts.linear_adjoint(dy, x, w, plan, gather=gather)
        odd_slot = int(plan.offsets[1])  # the second expert's first
        dy[odd_slot, 3] = math.inf
        dy[odd_slot + 1, 5] = math.nan
        r = experts.linear_adjoint(dy, x, w, plan, gather=gather)
        odd = torch.zeros(n, dtype=torch.bool, device="cuda")
        odd[(row if gather else torch.arange(slots, device="cuda"))[odd_slot:odd_slot + 2]] = True
        assert torch.equal(r.x[~odd], clean.x[~odd]) and not torch.isfinite(r.x[odd]).any()
        for got, want in ((r.weight, clean.weight), (r.bias, clean.bias)):
            assert torch.equal(got[[0, 2, 3]], want[[0, 2, 3]])
            rest = [c for c in range(outputs) if c not in (3, 5)]
            assert torch.equal(got[1][rest], want[1][rest]) and not torch.isfinite(got[1][[3, 5]]).any()
        x = randn(n, inputs, seed=1)
        x[(row if gather else torch.arange(slots, device="cuda"))[odd_slot], 2] = -math.inf
        r = experts.linear_adjoint(randn(slots, outputs, seed=3), x, w, plan, gather=gather)
        assert torch.equal(r.x, clean.x) and torch.equal(r.bias, clean.bias) and not torch.isfinite(r.weight[1][:, 2]).any()
        rest = [c for c in range(inputs) if c != 2]
        assert torch.equal(r.weight[1][:, rest], clean.weight[1][:, rest])
        for x_scale, dy_scale in ((2.0 ** -124, 1.0), (1.0, 2.0 ** -124), (2.0 ** -60, 2.0 ** -60)):
            x, dy = randn(n, inputs, seed=4, scale=x_scale), randn(slots, outputs, seed=5, scale=dy_scale)
            r = experts.linear_adjoint(dy, x, w, plan, gather=gather)
            want = adjoint_reference(dy, x, w, None, plan, "identity", gather)
            for got, (value, bound), what in zip((r.x, r.weight, r.bias), want, ("x", "weight", "bias")):
                check(got, value, bound, (x_scale, dy_scale, what))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gap,offset", ((0, 1), (1, 0), (5, 3)))
def test_route_and_combine_layouts(dtype, gap, offset):
    ctx = Context(0)
    for rows, count, k, width in ((300, 5, 2, 3), (129, 64, 8, 18), (70, 250, 4, 66), (33, 700, 5, 1030)):
        l0 = randn(rows, count, seed=rows, dtype=dtype)
        logits = put(l0, count + gap, offset)
        want = choose(l0, k, "softmax", None, 1, 1)
        weights = torch.empty(rows, k, device="cuda")
        chosen = torch.empty(rows, k, dtype=torch.int32, device="cuda")
        rc = _abi.NpaRouteCfg(rows, count + gap, count + gap, count, k, 1, 1, CODES[dtype], CODES[dtype], _abi.SCORE_SOFTMAX, 1, 1.0)
        torch.cuda.synchronize()
        ctx.check(lib().npa_expert_route(ctx.handle, C.byref(rc), ptr(logits), None, ptr(chosen), ptr(weights), None, None, None))
        dl, dl_all = apart(rows, count, count + gap, offset, dtype)
        dw = randn(rows, k, seed=2)
        torch.cuda.synchronize()
        ctx.check(lib().npa_expert_route_adjoint(ctx.handle, C.byref(rc), ptr(logits), ptr(chosen), ptr(dw), ptr(dl)))
        ctx.synchronize()
        assert torch.equal(chosen, want)
        check(weights, *weights_of(l0, want, "softmax", True, 1.0), "weights")
        check(dl, *route_adjoint_reference(dw, l0, chosen, "softmax", True, 1.0), "logits")
        assert untouched(dl, dl_all)
        plan = experts.plan(want, count)
        y0, res0, dout0 = randn(rows * k, width, seed=3, dtype=dtype), randn(rows, width, seed=4, dtype=dtype), randn(rows, width, seed=5, dtype=dtype)
        y, res, dout = put(y0, width + gap, offset), put(res0, width + gap, offset), put(dout0, width + gap, offset)
        out, out_all = apart(rows, width, width + gap, offset, dtype)
        dy, dy_all = apart(rows * k, width, width + gap, offset, dtype)
        cc = _abi.NpaCombineCfg(rows, width + gap, width + gap, width + gap, width + gap, width + gap, count, k, width, CODES[dtype])
        torch.cuda.synchronize()
        ctx.check(lib().npa_expert_combine(ctx.handle, C.byref(cc), ptr(y), ptr(plan.offsets), ptr(plan.slots), ptr(weights), ptr(res), ptr(out)))
        dweights = torch.empty(rows, k, device="cuda")
        ctx.check(lib().npa_expert_combine_adjoint(ctx.handle, C.byref(cc), ptr(y), ptr(plan.offsets), ptr(plan.slots), ptr(weights), ptr(dout), ptr(dy), ptr(dweights)))
        ctx.synchronize()
        terms = y0.double()[plan.slots.long()] * weights.double()[:, :, None]
        check(out, terms.sum(1) + res0.double(), (k + 8) * E * (terms.abs().sum(1) + res0.double().abs()), "out")
        _, row = of_slots(plan)
        back = dout0.double()[row] * weights.reshape(-1).double()[plan.order.long()][:, None]
        check(dy, back, 2 * E * back.abs(), "y")
        prod = y0.double()[plan.slots.long()] * dout0.double()[:, None]
        check(dweights, prod.sum(2), (width + 8) * E * prod.abs().sum(2), "weights")
        assert untouched(out, out_all) and untouched(dy, dy_all)


@pytest.mark.parametrize("count,k", ((5, 4), (64, 8), (300, 32)))
def test_route_adjoint_of_an_expert_named_twice(count, k):
    logits, dw = randn(70, count, seed=count), randn(70, k, seed=1)
    g = torch.Generator(device="cuda").manual_seed(2)
    chosen = torch.randint(-1, count, (70, k), generator=g, device="cuda", dtype=torch.int32)
    chosen[:, 1] = chosen[:, 0]
    for scores in ("softmax", "sigmoid"):
        for renormalise in (True, False):
            got = experts.route_adjoint(dw, logits, chosen, scores, renormalise)
            check(got, *route_adjoint_reference(dw, logits, chosen, scores, renormalise, 1.0), (scores, renormalise))
