"""The dense layers' workspaces: calls that overlap against the rule, captured calls, threads that end."""
import ctypes as C

import pytest
import torch

from burn_automata_amd import _abi
from burn_automata_amd._lib import lib
from burn_automata_amd.runtime import Context, ptr

pytestmark = pytest.mark.gpu


def randn(*shape, seed, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def test_overlapping_calls_leave_the_context_usable():
    """Small calls of one context on two streams at once: what they return is not defined, and nothing is asked of
    it. Calls that follow alone are right again, of each number of blocks."""
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    ctx = Context(0, stream=first.cuda_stream)
    width = 66
    x, dy, gamma = randn(1500, width, seed=1), randn(1500, width, seed=2), randn(width, seed=3)
    mean, rstd = x.mean(1), torch.rand(1500, device="cuda") + 0.5
    dg, db, dx = torch.empty(width, device="cuda"), torch.empty(width, device="cuda"), torch.empty_like(x)

    def call(rows):
        cfg = _abi.NpaNormCfg(rows, 0, 0, 0, 0, width, 0, 0, 0, 0.0)
        ctx.check(lib().npa_layer_norm_adjoint(ctx.handle, C.byref(cfg), ptr(x), ptr(gamma), ptr(mean), ptr(rstd), ptr(dy),
                                               ptr(dx), ptr(dg), ptr(db)))

    sizes = (1500, 40, 700, 1, 300, 97, 1100)
    want = {}
    torch.cuda.synchronize()
    for rows in sizes:
        call(rows)
        ctx.synchronize()
        want[rows] = dg.clone(), db.clone()
        torch.cuda.synchronize()
        exact = dy[:rows].double().sum(0)
        assert ((want[rows][1].double() - exact).abs() <= (rows + 8) * 2.0 ** -24 * dy[:rows].double().abs().sum(0)).all()
    for k in range(200):
        ctx.set_stream((first, second)[k % 2].cuda_stream)
        call(sizes[k % 7])
    torch.cuda.synchronize()
    for rows in sizes:
        for _ in range(2):
            dg.fill_(float("nan"))
            db.fill_(float("nan"))
            torch.cuda.synchronize()
            call(rows)
            torch.cuda.synchronize()
            assert torch.equal(dg, want[rows][0]) and torch.equal(db, want[rows][1]), rows
