"""Layer norm at every change of lanes and vectors a lane, with rows that lie apart and NaN between them, and with
more rows than one launch has blocks. Tolerances and definitions are those of test_gpu_layers.py."""
import pytest
import torch

from burn_automata_amd import layers
from tests.test_gpu_layers import E, TYPES, check, norm_reference, randn

pytestmark = pytest.mark.gpu

# the widest rows of each shape: lanes a row times vectors a lane times elements a vector (4 of f32, 8 of 16 bits)
F32 = sorted({8 * 4, 16 * 4} | {lanes * n * 4 for lanes in (8, 16, 32, 64, 128, 256, 512, 1024) for n in (3, 4)})
HALF = sorted({8 * 8} | {lanes * 2 * 8 for lanes in (8, 16, 32, 64, 128, 256, 512, 1024)})
BOUNDS = [(torch.float32, b) for b in F32] + [(t, b) for t in TYPES[1:] for b in HALF]


def apart(rows, width, pad, seed, dtype, scale=1.0):
    """Rows of width + pad elements apart whose last pad are NaN: they do not affect the result."""
    t = randn(rows, width, seed=seed, dtype=dtype, scale=scale, pad=pad)
    assert t.stride() == (width + pad, 1) and (not pad or t.as_strided((rows - 1, pad), (width + pad, 1), width).isnan().all())
    return t


@pytest.mark.parametrize("dtype,bound", BOUNDS)
@pytest.mark.parametrize("pad", (0, 1, 3, 8))
def test_forward_and_adjoint_at_each_shape(dtype, bound, pad):
    # 3,071 and 3,073 stand for both sides of 3 x 256 x 4
    for width in (bound - 1, bound, bound + 1):
        if width == 3 * 1024:
            continue
        rows = 41 if width < 1000 else 6
        x = apart(rows, width, pad, width, dtype, 1.5)
        x += 0.7
        assert x.stride(0) == width + pad
        gamma, beta = randn(width, seed=1, dtype=dtype), randn(width, seed=2, dtype=dtype)
        f = layers.layer_norm(x, gamma, beta, 1e-5)
        y, err, mean, rstd, xh, xh_err, g, c = norm_reference(x, gamma, beta, 1e-5)
        size = x.double().abs().mean(1)
        check(f.out, y, err, ("out", width))
        check(f.mean, mean[:, 0], 2 * c * size, ("mean", width))
        check(f.rstd, rstd[:, 0], 4 * c * rstd[:, 0] * (1 + (size * rstd[:, 0]) ** 2 * c), ("rstd", width))
        dy = apart(rows, width, pad, width + 1, dtype, 0.3)
        r = layers.layer_norm_adjoint(dy, x, f.mean, f.rstd, gamma)
        d = dy.double()
        t = d * g
        dx = rstd * (t - t.mean(1, keepdim=True) - xh * (t * xh).mean(1, keepdim=True))
        most = (t * xh).abs().mean(1, keepdim=True)
        check(r.x, dx, rstd * (4 * c * (t.abs() + t.abs().mean(1, keepdim=True) + xh.abs() * most)
                               + xh_err * most + xh.abs() * (t.abs() * xh_err).mean(1, keepdim=True)), ("x", width))
        depth = (64 + rows) * E
        check(r.gamma, (d * xh).sum(0), depth * (d * xh).abs().sum(0) + (d.abs() * xh_err).sum(0), ("gamma", width))
        check(r.beta, d.sum(0), depth * d.abs().sum(0), ("beta", width))


@pytest.mark.parametrize("rows", (1, 2, 3))
@pytest.mark.parametrize("width", (1, 2, 3, 5, 7, 9, 15, 17))
def test_narrow_rows_apart(rows, width):
    for dtype in TYPES:
        x, dy = (apart(rows, width, 2, k, dtype) if rows > 1 else randn(1, width, seed=k, dtype=dtype) for k in (1, 2))
        f = layers.layer_norm(x, eps=1e-2)
        y, err, *_ = norm_reference(x, None, None, 1e-2)
        check(f.out, y, err, "out")
        dense = layers.layer_norm_adjoint(dy.contiguous(), x.contiguous(), f.mean, f.rstd)
        assert torch.equal(layers.layer_norm_adjoint(dy, x, f.mean, f.rstd).x, dense.x)


def test_wide_rows_past_the_blocks_of_a_launch():
    """Rows wider than registers hold, 77 more than the 2^20 blocks of a launch: the first blocks take a second row.
    Rows repeat every 4,096, so results do."""
    rows, width, period = (1 << 20) + 77, 16385, 4096
    base, back = randn(period, width, seed=1, dtype=torch.bfloat16), randn(period, width, seed=2, dtype=torch.bfloat16)
    f = layers.layer_norm(base)
    want = layers.layer_norm_adjoint(back, base, f.mean, f.rstd).x
    y, err, *_ = norm_reference(base[:64], None, None, 1e-5)
    check(f.out[:64], y, err, "out")

    def repeated(t):
        all_rows = torch.empty(rows, *t.shape[1:], dtype=t.dtype, device="cuda")
        for at in range(0, rows, period):
            all_rows[at:at + period] = t[: rows - at]
        return all_rows

    def same(got, t):
        return all(torch.equal(got[at:at + period], t[: rows - at]) for at in range(0, rows, period))

    x = repeated(base)
    r = layers.layer_norm(x)
    assert same(r.out, f.out) and same(r.mean, f.mean) and same(r.rstd, f.rstd)
    mean, rstd = r.mean, r.rstd
    del r
    dy = repeated(back)
    assert same(layers.layer_norm_adjoint(dy, x, mean, rstd).x, want)
    del x, dy
    torch.cuda.empty_cache()
