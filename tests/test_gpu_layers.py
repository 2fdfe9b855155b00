"""Layer norm and linear layer, forward and adjoint, against their definitions in 64 bits.

Tolerances, elementwise, from rounding alone. u is the unit roundoff of the array's type (f32 2^-24,
bf16 2^-8, f16 2^-11) and e = 2^-24 that of the f32 sums. A sum of K products in any order is within
(K + 8) e times the sum of their absolute values (the 8 covers the epilogue's few operations); the
norm's sums are trees of at most c = 64 + width / 1024 additions deep. An activation's slope is at most
1.13 and its own evaluation within 16 e (1 + |z|). Each result is rounded once more, u times itself;
f16 results below its normal range are rounded to multiples of 2^-24.
"""
import ctypes as C
import math

import pytest
import torch

from burn_automata_amd import _abi, layers
from burn_automata_amd._lib import lib
from burn_automata_amd.runtime import Context, ptr

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}
TYPES = (torch.float32, torch.bfloat16, torch.float16)
ACTS = ("identity", "relu", "gelu", "silu")


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
    over = (want.abs() + bound >= most) & (got == want.sign() * math.inf)  # past the type's largest value
    bad = ~(((got - want).abs() <= bound) | over)
    assert not bad.any(), (what, int(bad.sum()), float((got - want).abs()[bad].max()), float(bound[bad].max()))


# ------------------------------------------------------------------------------ layer norm
def norm_reference(x, gamma, beta, eps):
    x = x.double()
    var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
    rstd = 1.0 / torch.sqrt(var + eps)
    xh = (x - mean) * rstd
    c = (64 + x.shape[-1] / 1024) * E
    xh_err = c * (rstd * (x.abs() + 2 * x.abs().mean(-1, keepdim=True)) + 2 * xh.abs())
    g = torch.ones_like(x[:1]) if gamma is None else gamma.double()
    y = xh * g + (0 if beta is None else beta.double())
    err = xh_err * g.abs() + 4 * E * (y.abs() + (xh * g).abs())
    return y, err, mean, rstd, xh, xh_err, g, c


# widths on both sides of every change of lanes and vectors a lane, and past the widest row in registers
WIDTHS = (1, 2, 3, 7, 8, 31, 66, 126, 128, 129, 255, 257, 513, 1023, 1025, 2047, 2050, 4096, 4099, 8193, 16384,
          16385, 20003)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_norm_forward(dtype, width):
    rows = 37 if width < 4000 else 5
    x = randn(rows, width, seed=width, dtype=dtype, scale=1.5, pad=width % 3) + 0.7
    param = torch.float32 if width % 2 else dtype
    gamma, beta = (randn(width, seed=width + k, dtype=param) for k in (1, 2))
    r = layers.layer_norm(x, gamma, beta, 1e-5)
    y, err, mean, rstd, _, _, _, c = norm_reference(x, gamma, beta, 1e-5)
    check(r.out, y, err, "out")
    check(r.mean, mean[:, 0], 2 * c * x.double().abs().mean(1), "mean")
    check(r.rstd, rstd[:, 0], 4 * c * rstd[:, 0] * (1 + (x.double().abs().mean(1) * rstd[:, 0]) ** 2 * c), "rstd")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_norm_adjoint(dtype, width):
    rows = 301 if width < 4000 else 9
    x = randn(rows, width, seed=width, dtype=dtype, scale=1.5, pad=width % 3)
    dy = randn(rows, width, seed=width + 5, dtype=dtype, scale=0.3, pad=width % 2)
    param = dtype if width % 2 else torch.float32
    gamma = randn(width, seed=width + 1, dtype=param)
    f = layers.layer_norm(x, gamma, None, 1e-3)
    r = layers.layer_norm_adjoint(dy, x, f.mean, f.rstd, gamma)
    _, _, _, rstd, xh, xh_err, g, c = norm_reference(x, gamma, None, 1e-3)
    d = dy.double()
    t = d * g
    m1, m2 = t.mean(1, keepdim=True), (t * xh).mean(1, keepdim=True)
    dx = rstd * (t - m1 - xh * m2)
    mean_abs = (t * xh).abs().mean(1, keepdim=True)
    err = rstd * (4 * c * (t.abs() + t.abs().mean(1, keepdim=True) + xh.abs() * mean_abs)
                  + xh_err * mean_abs + xh.abs() * (t.abs() * xh_err).mean(1, keepdim=True))
    check(r.x, dx, err, "x")
    depth = (64 + rows) * E
    check(r.gamma, (d * xh).sum(0), depth * (d * xh).abs().sum(0) + (d.abs() * xh_err).sum(0), "gamma")
    check(r.beta, d.sum(0), depth * d.abs().sum(0), "beta")
    assert r.gamma.dtype == r.beta.dtype == param


def test_norm_without_parameters_and_in_place():
    x, dy = randn(65, 96, seed=1), randn(65, 96, seed=2)
    f = layers.layer_norm(x)
    y, err, *_ = norm_reference(x, None, None, 1e-5)
    check(f.out, y, err, "out")
    r = layers.layer_norm_adjoint(dy, x, f.mean, f.rstd)
    assert r.gamma is None and r.beta is None
    ctx = Context(0)
    cfg = _abi.NpaNormCfg(65, 0, 0, 0, 0, 96, 0, 0, 0, 1e-5)
    inplace, back = x.clone(), dy.clone()
    ctx.check(lib().npa_layer_norm_adjoint(ctx.handle, C.byref(cfg), ptr(x), None, ptr(f.mean), ptr(f.rstd), ptr(back),
                                           ptr(back), None, None))
    ctx.check(lib().npa_layer_norm(ctx.handle, C.byref(cfg), ptr(inplace), None, None, ptr(inplace), None, None))
    ctx.synchronize()
    assert torch.equal(inplace, f.out) and torch.equal(back, r.x)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", (1, 5, 18, 66, 200, 255, 256, 257, 600, 1023, 2050, 5000, 16384))
def test_norm_parameters_of_few_and_more_rows(dtype, width):
    """Rows on both sides of the sizes at which the last block joins the sums, and the calls after each other on
    the same workspace; dgamma and dbeta are sums of `rows` f32 products of three factors each."""
    for rows in (1, 2, 5, 24, 97, 1500, 9300):
        if rows * width > 1 << 23:
            break
        x, dy = randn(rows, width, seed=1, dtype=dtype), randn(rows, width, seed=2, dtype=dtype)
        gamma = randn(width, seed=3, dtype=dtype)
        mean, rstd = x.float().mean(1), torch.rand(rows, device="cuda") + 0.5
        r = layers.layer_norm_adjoint(dy, x, mean, rstd, gamma)
        m, s, d = mean.double()[:, None], rstd.double()[:, None], dy.double()
        most = (d.abs() * (x.double().abs() + m.abs()) * s).sum(0)
        check(r.gamma, (d * ((x.double() - m) * s)).sum(0), (rows + 8) * E * most, "gamma")
        check(r.beta, d.sum(0), (rows + 8) * E * d.abs().sum(0), "beta")
        again = layers.layer_norm_adjoint(dy, x, mean, rstd, gamma)
        assert all(torch.equal(getattr(r, k), getattr(again, k)) for k in ("x", "gamma", "beta"))


def test_norm_adjoint_replayed_in_a_graph():
    """Replays of a captured call, with eager calls of another size on the same workspace in between."""
    x, dy = randn(700, 66, seed=1), randn(700, 66, seed=2)
    gamma = randn(66, seed=3)
    mean, rstd = x.mean(1), torch.rand(700, device="cuda") + 0.5
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = layers.layer_norm_adjoint(dy, x, mean, rstd, gamma)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = layers.layer_norm_adjoint(dy, x, mean, rstd, gamma)
        for rows in (600, 7, 700):
            for t in (got.x, got.gamma, got.beta):
                t.fill_(math.nan)
            graph.replay()
            layers.layer_norm_adjoint(dy[:rows], x[:rows], mean[:rows], rstd[:rows], gamma)
            side.synchronize()
            assert all(torch.equal(getattr(got, k), getattr(want, k)) for k in ("x", "gamma", "beta"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", (66, 1023, 8200, 16390))
def test_norm_adjoint_over_its_input(dtype, width):
    rows = 70
    x, dy, gamma = randn(rows, width, seed=1, dtype=dtype), randn(rows, width, seed=2, dtype=dtype), randn(width, seed=3)
    f = layers.layer_norm(x, gamma)
    want = layers.layer_norm_adjoint(dy, x, f.mean, f.rstd, gamma)
    dg, db = torch.empty_like(gamma), torch.empty_like(gamma)
    ctx = Context(0)
    cfg = _abi.NpaNormCfg(rows, 0, 0, 0, 0, width, TYPES.index(dtype), 0, 0, 1e-5)
    torch.cuda.synchronize()
    ctx.check(lib().npa_layer_norm_adjoint(ctx.handle, C.byref(cfg), ptr(x), ptr(gamma), ptr(f.mean), ptr(f.rstd), ptr(dy),
                                           ptr(dy), ptr(dg), ptr(db)))
    ctx.synchronize()
    assert torch.equal(dy, want.x) and torch.equal(dg, want.gamma) and torch.equal(db, want.beta)


def test_norm_constant_rows_and_zero_eps():
    x = torch.full((3, 50), 2.5, device="cuda")
    f = layers.layer_norm(x, eps=1e-5)
    assert torch.equal(f.out, torch.zeros_like(x))
    f = layers.layer_norm(randn(4, 50, seed=3), eps=0.0)
    assert torch.isfinite(f.out).all()


def test_norm_rows_with_nan_and_infinity_stay_apart():
    x = randn(6, 70, seed=4)
    clean = layers.layer_norm(x).out
    x[1, 3], x[4, 0] = math.nan, math.inf
    out = layers.layer_norm(x).out
    for row in range(6):
        if row in (1, 4):
            assert torch.isnan(out[row]).any()
        else:
            assert torch.equal(out[row], clean[row])


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_gradients_are_added_to(dtype):
    x, dy = randn(130, 77, seed=5, dtype=dtype), randn(130, 77, seed=6, dtype=dtype)
    gamma = randn(77, seed=7)
    f = layers.layer_norm(x, gamma)
    once = layers.layer_norm_adjoint(dy, x, f.mean, f.rstd, gamma)
    dg, db = torch.ones(77, device="cuda"), torch.full((77,), 2.0, device="cuda")
    r = layers.layer_norm_adjoint(dy, x, f.mean, f.rstd, gamma, gamma_adjoint=dg, beta_adjoint=db)
    assert r.gamma is dg and r.beta is db
    assert torch.equal(dg, once.gamma + 1.0) and torch.equal(db, once.beta + 2.0)


def test_norm_of_no_rows():
    x = torch.empty(0, 33, device="cuda")
    f = layers.layer_norm(x)
    assert f.out.shape == (0, 33)
    gamma = torch.ones(33, device="cuda")
    r = layers.layer_norm_adjoint(x, x, f.mean, f.rstd, gamma)
    assert torch.equal(r.gamma, torch.zeros(33, device="cuda")) and torch.equal(r.beta, torch.zeros(33, device="cuda"))


def test_norm_difference_quotients():
    """The directional derivative of sum(dy * norm(x)) against its central difference in f64 of the same
    formula: the kernels' gradient of the definition's own slope. h = 2^-12 leaves a truncation error of
    about h^2 and the f32 gradient's e, both far below 1e-5 of the sum of absolute terms."""
    x, dy, v = (randn(20, 45, seed=k) for k in (11, 12, 13))
    gamma, beta = randn(45, seed=14), randn(45, seed=15)
    f = layers.layer_norm(x, gamma, beta)
    r = layers.layer_norm_adjoint(dy, x, f.mean, f.rstd, gamma)
    h = 2.0 ** -12
    at = lambda s: (norm_reference(x.double() + s * v.double(), gamma, beta, 1e-5)[0] * dy.double()).sum()  # noqa: E731
    slope = (at(h) - at(-h)) / (2 * h)
    terms = r.x.double() * v.double()
    assert abs(float(slope - terms.sum())) < 1e-5 * float(terms.abs().sum())


# ------------------------------------------------------------------------------ linear layer
def act64(z, name):
    return {"identity": lambda v: v, "relu": torch.relu, "silu": torch.nn.functional.silu,
            "gelu": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}[name](z)


def slope64(z, name):
    if name == "identity":
        return torch.ones_like(z)
    z = z.clone().requires_grad_()
    return torch.autograd.grad(act64(z, name).sum(), z)[0]


def forward_case(rows, k, n, dtype, act="identity", bias=True, residual=False, keep=False, pad=0, seed=0):
    x = randn(rows, k, seed=seed + 1, dtype=dtype, pad=pad)
    w = randn(n, k, seed=seed + 2, dtype=dtype, scale=1 / math.sqrt(k), pad=pad)
    b = randn(n, seed=seed + 3, dtype=torch.float32 if pad else dtype) if bias else None
    res = randn(rows, n, seed=seed + 4, dtype=dtype, pad=pad) if residual else None
    r = layers.linear(x, w, b, act, res, keep)
    z = x.double() @ w.double().T
    size = x.double().abs() @ w.double().abs().T
    if bias:
        z, size = z + b.double(), size + b.double().abs()
    y = act64(z, act)
    err = (k + 8) * E * size
    zerr = err
    err = 1.13 * err + (16 * E * (1 + z.abs()) if act in ("gelu", "silu") else 0)
    if residual:
        y = y + res.double()
        err = err + E * y.abs()
    check(r.out, y, err, ("out", rows, k, n, act))
    if keep:
        check(r.preactivation, z, zerr, "preactivation")
    else:
        assert r.preactivation is None


# sizes around the tiles and the short and long sums of every form of the product
SHAPES = ((1, 1, 1), (1, 8, 3), (1, 4096, 64), (2, 33, 1), (3, 64, 130), (5, 127, 17), (16, 256, 16), (17, 100, 33),
          (33, 66, 128), (64, 64, 64), (65, 65, 65), (100, 1000, 18), (128, 128, 128), (129, 31, 257), (200, 640, 200),
          (256, 512, 256), (257, 513, 300), (300, 2048, 72), (511, 70, 513), (1000, 123, 256), (2049, 66, 27))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_linear_forward(dtype, shape):
    pick = sum(shape)
    forward_case(*shape, dtype, ACTS[pick % 4], bias=pick % 3 != 0, residual=pick % 2 == 0, keep=pick % 5 < 2,
                 pad=(0, 0, 1, 8)[pick % 4], seed=pick)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
def test_linear_epilogue(dtype, act):
    for k, (bias, residual, keep) in enumerate(((0, 0, 0), (1, 0, 1), (0, 1, 1), (1, 1, 0))):
        forward_case(70, 96, 80, dtype, act, bool(bias), bool(residual), bool(keep), seed=100 + k)
        forward_case(3, 520, 40, dtype, act, bool(bias), bool(residual), bool(keep), pad=4, seed=200 + k)


def adjoint_case(rows, k, n, dtype, act="identity", bias=True, pad=0, seed=0):
    x = randn(rows, k, seed=seed + 1, dtype=dtype, pad=pad)
    w = randn(n, k, seed=seed + 2, dtype=dtype, scale=1 / math.sqrt(k), pad=pad)
    dy = randn(rows, n, seed=seed + 3, dtype=dtype, scale=0.25, pad=pad)
    z = randn(rows, n, seed=seed + 4, dtype=dtype, scale=1.5, pad=pad) if act != "identity" else None
    r = layers.linear_adjoint(dy, x, w, z, act, bias=bias)
    dz = dy.double() * (1 if z is None else slope64(z.double(), act))
    # the slope's own evaluation, and dz's rounding to the type where there is an activation
    derr = (0 if z is None else 16) * E * 1.13 * dy.double().abs() * (1 + (0 if z is None else z.double().abs()))
    bias_err = torch.as_tensor(derr, device="cuda").double().expand(rows, n) if z is not None else torch.zeros_like(dz)
    derr = bias_err + (0 if z is None else U[dtype]) * dz.abs() + (0 if z is None else TINY[dtype])
    xa, wa = x.double().abs(), w.double().abs()
    check(r.x, dz @ w.double(), derr @ wa + (n + 8) * E * (dz.abs() @ wa), ("x", rows, k, n, act))
    check(r.weight, dz.T @ x.double(), derr.T @ xa + (rows + 8) * E * (dz.abs().T @ xa), ("weight", rows, k, n, act))
    if bias:
        check(r.bias, dz.sum(0), bias_err.sum(0) + (rows + 8) * E * dz.abs().sum(0), ("bias", rows, k, n, act))
    else:
        assert r.bias is None


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES + ((4097, 66, 128), (9001, 20, 12)))
def test_linear_adjoint(dtype, shape):
    pick = sum(shape)
    adjoint_case(*shape, dtype, ACTS[pick % 4], bias=pick % 3 != 0, pad=(0, 0, 1, 8)[pick % 4], seed=pick)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
def test_linear_adjoint_activations(dtype, act):
    adjoint_case(150, 72, 88, dtype, act, True, seed=300)
    adjoint_case(7, 300, 45, dtype, act, True, pad=3, seed=400)


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_gradients_are_added_to(dtype):
    rows, k, n = 700, 70, 50
    x, w = randn(rows, k, seed=1, dtype=dtype), randn(n, k, seed=2, dtype=dtype)
    dy = randn(rows, n, seed=3, dtype=dtype, scale=0.1)
    dw, db = torch.zeros(n, k, device="cuda"), torch.zeros(n, device="cuda")
    for _ in range(2):  # twice the gradient: doubling is exact
        r = layers.linear_adjoint(dy, x, w, weight_adjoint=dw, bias_adjoint=db, inputs=False)
    assert r.x is None and r.weight is dw and r.bias is db
    want = dy.double().T @ x.double()
    check(dw, 2 * want, 2 * (rows + 9) * E * (dy.double().abs().T @ x.double().abs()), "weight")
    check(db, 2 * dy.double().sum(0), 2 * (rows + 9) * E * dy.double().abs().sum(0), "bias")


# Large aligned products of 16-bit types, loaded straight into LDS: partial tiles on both edges, sums of an odd
# number of steps, split sums (17,472 is 16 parts of 17 steps of 64 and one of a single step), padded rows.
@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("act,shape,pad", (("gelu", (4100, 320, 2056), 0), ("relu", (4096, 256, 2048), 8),
                                           ("silu", (600, 17472, 1032), 0), ("identity", (257, 17472, 1300), 8)))
def test_linear_forward_large(dtype, act, shape, pad):
    forward_case(*shape, dtype, act, residual=pad == 0, keep=pad == 8, pad=pad, seed=shape[0])


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("act,shape,pad", (("gelu", (4100, 2056, 320), 0), ("identity", (4097, 2048, 256), 8),
                                           ("silu", (17472, 1032, 600), 0), ("relu", (8192, 2056, 576), 8)))
def test_linear_adjoint_large(dtype, act, shape, pad):
    adjoint_case(*shape, dtype, act, pad=pad, seed=shape[0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", (1, 2, 15, 16, 17, 31, 32))
def test_linear_of_few_rows(dtype, rows):
    for k, n, pad in ((1, 17, 0), (7, 16, 1), (31, 15, 0), (32, 33, 8), (257, 1000, 3), (4104, 130, 0)):
        forward_case(rows, k, n, dtype, ACTS[(rows + k) % 4], residual=rows % 2 == 0, keep=k % 2 == 1, pad=pad, seed=rows + k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", ((3, 200, 40), (300, 70, 90), (4096, 256, 2048), (40, 2000, 24)))
def test_linear_onto_its_residual(dtype, shape):
    rows, k, n = shape
    x, w, res = (randn(*s, seed=7, dtype=dtype) for s in ((rows, k), (n, k), (rows, n)))
    want = layers.linear(x, w, None, "silu", res).out
    ctx = Context(0)
    kind = TYPES.index(dtype)
    cfg = _abi.NpaLinearCfg(rows, 0, 0, 0, 0, 0, 0, 0, k, n, kind, layers.Activation.silu, kind, kind, 0)
    torch.cuda.synchronize()
    ctx.check(lib().npa_linear(ctx.handle, C.byref(cfg), ptr(x), ptr(w), None, ptr(res), ptr(res), None))
    ctx.synchronize()
    assert torch.equal(res, want)


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_of_no_rows(dtype):
    x, w = torch.empty(0, 24, device="cuda", dtype=dtype), randn(40, 24, seed=1, dtype=dtype)
    assert layers.linear(x, w).out.shape == (0, 40)
    r = layers.linear_adjoint(torch.empty(0, 40, device="cuda", dtype=dtype), x, w)
    assert torch.equal(r.weight, torch.zeros_like(w)) and torch.equal(r.bias, torch.zeros_like(w[:, 0]))
    assert r.x.shape == (0, 24)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", ((5, 300, 20), (200, 300, 140), (600, 512, 512)))
def test_linear_nan_and_infinity_stay_in_their_row(dtype, shape):
    rows, k, n = shape
    x, w = randn(rows, k, seed=1, dtype=dtype), randn(n, k, seed=2, dtype=dtype)
    clean = layers.linear(x, w).out
    x[1, 7], x[3, 2] = math.nan, math.inf
    out = layers.linear(x, w).out
    assert torch.isnan(out[1]).all()
    assert torch.equal(out[3], torch.where(w[:, 2] > 0, math.inf, -math.inf).to(dtype))
    keep = [r for r in range(rows) if r not in (1, 3)]
    assert torch.equal(out[keep], clean[keep])


@pytest.mark.parametrize("shape", ((4, 64, 8), (200, 300, 140), (600, 512, 512)))
def test_linear_f32_keeps_the_whole_range(shape):
    """Values near f32's largest and far below 1 keep f32's relative accuracy."""
    rows, k, n = shape
    for scale_x, scale_w in ((1e37, 1e-37), (3e38, 1e-30), (1e-25, 1e-8), (1e-37, 1e20)):
        x = randn(rows, k, seed=1).clamp(-1, 1) * scale_x
        w = randn(n, k, seed=2).clamp(-1, 1) * scale_w
        got = layers.linear(x, w).out.double()
        want, size = x.double() @ w.double().T, x.double().abs() @ w.double().abs().T
        assert ((got - want).abs() <= (k + 8) * E * size + k * 2.0 ** -120 * max(scale_w, 1.0) * max(scale_x, 1.0)
                + 2.0 ** -126).all(), (scale_x, scale_w)


def test_relu_slope_at_zero_and_masked_infinities():
    z = torch.tensor([[0.0, -0.0, -1.0, 2.0, math.nan]], device="cuda")
    dy = torch.tensor([[1.0, math.inf, math.nan, 3.0, 1.0]], device="cuda")
    r = layers.linear_adjoint(dy, torch.ones(1, 1, device="cuda"), torch.zeros(5, 1, device="cuda"), z, "relu")
    assert torch.equal(r.bias, torch.tensor([0.0, 0.0, 0.0, 3.0, 0.0], device="cuda"))


@pytest.mark.parametrize("act", ("gelu", "silu"))
def test_slopes_far_out(act):
    z = torch.tensor([[-math.inf, -1e30, -60.0, 60.0, 1e30, math.inf]], device="cuda")
    r = layers.linear_adjoint(torch.ones_like(z), torch.ones(1, 1, device="cuda"), torch.zeros(6, 1, device="cuda"), z, act)
    assert torch.allclose(r.bias, torch.tensor([0.0, 0.0, 0.0, 1.0, 1.0, 1.0], device="cuda"), atol=1e-20)


def test_rows_past_32_bit_offsets():
    """Rows whose elements lie beyond 2^32 elements from the first."""
    far = (1 << 31) + 16
    base = torch.zeros(2 * far + 4096, dtype=torch.float16, device="cuda")
    x = base.as_strided((3, 1024), (far, 1))
    x.copy_(randn(3, 1024, seed=1))
    dense = x.contiguous()
    assert torch.equal(layers.layer_norm(x).out, layers.layer_norm(dense).out)
    w = randn(48, 1024, seed=2, dtype=torch.float16)
    assert torch.equal(layers.linear(x, w).out, layers.linear(dense, w).out)
    dy = randn(3, 48, seed=3, dtype=torch.float16)
    assert torch.equal(layers.linear_adjoint(dy, x, w).weight, layers.linear_adjoint(dy, dense, w).weight)


@pytest.mark.parametrize("dtype", TYPES)
def test_more_rows_than_one_launch_takes_at_once(dtype):
    rows = (1 << 20) + 77
    x, w = randn(rows, 24, seed=1, dtype=dtype), randn(16, 24, seed=2, dtype=dtype)
    y = layers.linear(x, w, activation="relu").out
    take = torch.tensor([0, 1, 4095, 65536, rows - 2, rows - 1], device="cuda")
    assert torch.equal(y[take][:2], layers.linear(x[:300].contiguous(), w, activation="relu").out[:2])
    want = torch.relu(x[take].double() @ w.double().T)
    check(y[take], want, 32 * E * (x[take].double().abs() @ w.double().abs().T), "out")
    adjoint = layers.linear_adjoint(y, x, w).weight
    terms = y.double().abs().T @ x.double().abs()
    check(adjoint, y.double().T @ x.double(), (rows + 8) * E * terms, "weight")


def test_more_columns_than_one_launch_takes_at_once():
    """Column sums and few rows whose launches of a thread, or a few, a column would be 2^32 threads."""
    width = (1 << 25) + 8
    x, dy = randn(1, width, seed=1, dtype=torch.float16), randn(1, width, seed=2, dtype=torch.float16)
    gamma = torch.ones(width, dtype=torch.float16, device="cuda")
    mean, rstd = torch.full((1,), 0.25, device="cuda"), torch.full((1,), 2.0, device="cuda")
    r = layers.layer_norm_adjoint(dy, x, mean, rstd, gamma)
    assert torch.equal(r.beta, dy[0])  # one row: no sum
    assert torch.equal(r.gamma, (dy[0].float() * ((x[0].float() - 0.25) * 2.0)).to(torch.float16))
    # one column in: each output and gradient is one product
    outputs = 1 << 28
    w = randn(outputs, 1, seed=3, dtype=torch.float16)
    two = torch.full((1, 1), 2.0, dtype=torch.float16, device="cuda")
    y = layers.linear(two, w).out
    assert torch.equal(y, w.T * 2)
    r = layers.linear_adjoint(y, two, w, inputs=False)
    assert torch.equal(r.bias, y[0]) and torch.equal(r.weight, y.T * 2)
    r = layers.linear_adjoint(y, two, w, y, "silu", inputs=False)  # the slope and bias in kernels of their own
    z = y.float()
    s = torch.sigmoid(z)
    bias = z * (s * (1.0 + z * (1.0 - s)))
    bound = U[torch.float16] * 2 * bias.abs() + 2 * 16 * E * (1 + z.abs()) * z.abs() + TINY[torch.float16]
    assert bool(((r.bias.float() - bias[0]).abs() <= bound[0]).all())  # both sides' slopes are f32


@pytest.mark.parametrize("dtype", TYPES)
def test_two_calls_give_the_same_bits(dtype):
    x, w, dy = (randn(*s, seed=k, dtype=dtype) for k, s in enumerate(((3000, 200), (90, 200), (3000, 90))))
    a, b = layers.linear_adjoint(dy, x, w), layers.linear_adjoint(dy, x, w)
    assert torch.equal(a.x, b.x) and torch.equal(a.weight, b.weight) and torch.equal(a.bias, b.bias)


def test_calls_follow_the_current_stream():
    """Without a context a call runs on torch's current stream, after the work queued there."""
    x, w = randn(4096, 512, seed=1), randn(512, 512, seed=2)
    want = layers.linear(x * 3.0, w).out
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = x
        for _ in range(20):
            y = y * 1.0
        y = layers.linear(y * 3.0, w).out
        total = layers.linear_adjoint(y, x, w).x
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, want) and torch.equal(total, layers.linear_adjoint(want, x, w).x)


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
def test_host_arrays(dtype):
    """Host-I/O mode: strided rows travel whole, and the elements between them come back unchanged."""
    x, w = randn(19, 40, seed=1, dtype=dtype), randn(30, 40, seed=2, dtype=dtype)
    want = layers.linear(x, w, activation="silu", keep_preactivation=True)
    back = layers.linear_adjoint(want.out, x, w, want.preactivation, "silu")
    ctx = Context(0, host_io=True)
    hx, hw = x.cpu(), w.cpu()
    out, z = torch.full((19, 33), 7.0, dtype=dtype), torch.empty(19, 30, dtype=dtype)
    kind = layers._TYPES[dtype]
    cfg = _abi.NpaLinearCfg(19, 0, 0, 0, 33, 0, 0, 0, 40, 30, kind, _abi.ACT_SILU, kind, kind, 0)
    ctx.check(lib().npa_linear(ctx.handle, C.byref(cfg), ptr(hx), ptr(hw), None, None, ptr(out), ptr(z)))
    assert torch.equal(out[:, :30], want.out.cpu()) and torch.equal(z, want.preactivation.cpu())
    assert (out[:18, 30:] == 7.0).all()
    cfg = _abi.NpaLinearCfg(19, 0, 0, 0, 0, 0, 33, 0, 40, 30, kind, _abi.ACT_SILU, kind, _abi.TYPE_F32, 1)
    dx, dw, db = torch.empty(19, 40, dtype=dtype), torch.ones(30, 40), torch.ones(30)
    ctx.check(lib().npa_linear_adjoint(ctx.handle, C.byref(cfg), ptr(hx), ptr(hw), ptr(z), ptr(out), ptr(dx), ptr(dw), ptr(db)))
    assert torch.equal(dx, back.x.cpu())
    assert torch.equal((dw - 1.0).to(dtype).sub(back.weight.cpu()).abs().max() <= 2 * U[dtype] * back.weight.abs().max().cpu()
                       + 2.0 ** -20, torch.tensor(True))
    nx = torch.empty(19, 40, dtype=dtype)
    ncfg = _abi.NpaNormCfg(19, 0, 0, 0, 0, 40, kind, kind, 0, 1e-5)
    ctx.check(lib().npa_layer_norm(ctx.handle, C.byref(ncfg), ptr(hx), None, None, ptr(nx), None, None))
    assert torch.equal(nx, layers.layer_norm(x).out.cpu())


def test_linear_difference_quotients():
    """As test_norm_difference_quotients, through gelu and in the weights' direction too."""
    x, w, dy = randn(30, 25, seed=1), randn(14, 25, seed=2, scale=0.2), randn(30, 14, seed=3)
    f = layers.linear(x, w, None, "gelu", keep_preactivation=True)
    r = layers.linear_adjoint(dy, x, w, f.preactivation, "gelu")
    vx, vw = randn(30, 25, seed=4).double(), randn(14, 25, seed=5).double()
    h = 2.0 ** -12
    at = lambda s: (act64((x.double() + s * vx) @ (w.double() + s * vw).T, "gelu") * dy.double()).sum()  # noqa: E731
    slope = (at(h) - at(-h)) / (2 * h)
    terms = torch.cat([(r.x.double() * vx).flatten(), (r.weight.double() * vw).flatten()])
    assert abs(float(slope - terms.sum())) < 1e-5 * float(terms.abs().sum())


# ------------------------------------------------------------------------------ refusals
def test_refusals():
    x, w = randn(4, 8, seed=1), randn(6, 8, seed=2)
    with pytest.raises(_abi.InvalidArgument, match="not a CUDA tensor"):
        layers.linear(x.cpu(), w)
    with pytest.raises(_abi.InvalidArgument, match="float64"):
        layers.layer_norm(x.double())
    with pytest.raises(_abi.InvalidArgument, match="expected torch.float32"):
        layers.linear(x, w.half())
    with pytest.raises(_abi.OutputShape, match="weight"):
        layers.linear(x, w[:, :7])
    with pytest.raises(_abi.OutputShape, match="bias"):
        layers.linear(x, w, torch.zeros(5, device="cuda"))
    with pytest.raises(_abi.OutputShape, match="residual"):
        layers.linear(x, w, residual=x)
    with pytest.raises(_abi.InvalidArgument, match="unknown activation"):
        layers.linear(x, w, activation="tan")
    with pytest.raises(_abi.InvalidArgument, match="unknown activation"):
        layers.linear(x, w, activation=9)
    with pytest.raises(_abi.OutputShape, match="gamma"):
        layers.layer_norm(x, torch.ones(9, device="cuda"))
    with pytest.raises(_abi.InvalidArgument, match="eps"):
        layers.layer_norm(x, eps=-1.0)
    with pytest.raises(_abi.InvalidArgument, match="eps"):
        layers.layer_norm(x, eps=math.nan)
    with pytest.raises(_abi.InvalidArgument, match="dims"):
        layers.layer_norm(torch.empty(4, 0, device="cuda"))
    with pytest.raises(_abi.InvalidArgument, match="preactivation"):
        layers.linear_adjoint(torch.zeros(4, 6, device="cuda"), x, w, None, "relu")
    with pytest.raises(_abi.OutputShape, match="out_adjoint"):
        layers.linear_adjoint(torch.zeros(4, 5, device="cuda"), x, w)
    with pytest.raises(_abi.InvalidArgument, match="together"):
        layers.linear_adjoint(torch.zeros(4, 6, device="cuda"), x, w, weight_adjoint=torch.zeros(6, 8, device="cuda"))
    f = layers.layer_norm(x)
    with pytest.raises(_abi.InvalidArgument, match="mean"):
        layers.layer_norm_adjoint(x, x, f.mean.half(), f.rstd)


def test_refusals_of_the_entry_points():
    x, w, y = randn(4, 8, seed=1), randn(6, 8, seed=2), torch.full((4, 6), 5.0, device="cuda")
    ctx = Context(0)

    def linear(cfg, a=x, b=w, out=y):
        return lib().npa_linear(ctx.handle, C.byref(cfg), ptr(a), ptr(b), None, None, ptr(out), None)

    def cfg(**kw):
        c = _abi.NpaLinearCfg(4, 0, 0, 0, 0, 0, 0, 0, 8, 6, 0, 0, 0, 0, 0)
        for k, v in kw.items():
            setattr(c, k, v)
        return c

    for bad, word in ((cfg(element_type=3), "element type"), (cfg(bias_type=1), "parameters"), (cfg(in_dims=0), "dims"),
                      (cfg(out_dims=1 << 31), "dims"), (cfg(rows=(1 << 30) + 1), "rows"), (cfg(x_stride=7), "stride"),
                      (cfg(out_stride=5), "stride"), (cfg(weight_stride=1 << 33), "stride"),
                      (cfg(activation=4), "activation")):
        assert linear(bad) == _abi.NPA_ERR_INVALID_ARGUMENT
        assert word in lib().npa_last_error(ctx.handle).decode(), word
    for a, b, out in ((None, w, y), (x, None, y), (x, w, None)):
        assert linear(cfg(), a, b, out) == _abi.NPA_ERR_INVALID_ARGUMENT
        assert "null" in lib().npa_last_error(ctx.handle).decode()
    odd = C.c_void_p(x.data_ptr() + 2)
    assert lib().npa_linear(ctx.handle, C.byref(cfg(rows=2)), odd, ptr(w), None, None, ptr(y), None) == _abi.NPA_ERR_INVALID_ARGUMENT
    assert "aligned" in lib().npa_last_error(ctx.handle).decode()
    assert lib().npa_linear(ctx.handle, None, ptr(x), ptr(w), None, None, ptr(y), None) == _abi.NPA_ERR_INVALID_ARGUMENT
    ctx.synchronize()
    assert (y == 5.0).all()
    n = _abi.NpaNormCfg(4, 0, 0, 0, 0, 8, 0, 0, 0, 1e-5)
    assert lib().npa_layer_norm(ctx.handle, C.byref(n), ptr(x), None, None, None, None, None) == _abi.NPA_ERR_INVALID_ARGUMENT
    assert lib().npa_layer_norm_adjoint(ctx.handle, C.byref(n), ptr(x), None, None, None, ptr(x), ptr(y), None, None) == \
        _abi.NPA_ERR_INVALID_ARGUMENT
