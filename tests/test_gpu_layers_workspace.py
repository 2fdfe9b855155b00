"""The dense layers' workspaces: calls that overlap against the rule, captured calls, threads that end."""
import ctypes as C
import math
import threading

import pytest
import torch

from burn_automata_amd import _abi, layers
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


def calls(rows, k, n, dtype=torch.bfloat16):
    """Calls of every operator that keep something in the workspace, by name."""
    x, w, dy = randn(rows, k, seed=1, dtype=dtype), randn(n, k, seed=2, dtype=dtype), randn(rows, n, seed=3, dtype=dtype)
    z, gamma = randn(rows, n, seed=4, dtype=dtype), randn(k, seed=5, dtype=dtype)
    mean, rstd = x.float().mean(1), torch.rand(rows, device="cuda") + 0.5
    narrow = randn(40, k, seed=6, dtype=dtype)

    def run():
        a, b = layers.linear_adjoint(dy, x, w, z, "gelu"), layers.linear_adjoint(dy, x, w)
        c, d = layers.layer_norm_adjoint(x, x, mean, rstd, gamma), layers.linear(narrow, w, None, "silu")
        e = layers.layer_norm(x, gamma)
        return [a.x, a.weight, a.bias, b.x, b.weight, b.bias, c.x, c.gamma, c.beta, d.out, e.out]

    return run


def library_bytes():
    """Device memory in use outside torch's allocator."""
    torch.cuda.synchronize()
    free, total = torch.cuda.mem_get_info()
    return total - free - torch.cuda.memory_reserved()


def check_replays(graph, got, want, between):
    for _ in range(3):
        for t in got:
            t.fill_(math.nan)
        graph.replay()
        torch.cuda.current_stream().synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        between()


@pytest.mark.parametrize("shape", ((300, 2048, 72), (700, 66, 128), (2048, 512, 2048)))
def test_a_captured_call_keeps_its_buffers(shape):
    """A larger call on the same context, after the capture, takes other buffers: the captured ones are still
    allocated, and replays are right whatever is written to memory that was allocated since."""
    side = torch.cuda.Stream()
    small, large = calls(*shape), calls(shape[0] * 4, shape[1], shape[2] * 2)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        want = small()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = small()
        spare = []

        def between():
            large()
            spare.append(torch.full((1 << 22,), math.nan, device="cuda"))

        check_replays(graph, got, want, between)


def test_outgrown_buffers_stay_allocated_only_where_a_graph_has_them():
    """dz of 8,192 x 4,096 bf16 (64 MiB) and of twice the rows: without a capture the larger takes the smaller's
    place, with one it comes beside it."""
    side = torch.cuda.Stream()
    rows, n = 8192, 4096
    dy, z = torch.ones(2 * rows, n, dtype=torch.bfloat16, device="cuda"), torch.ones(2 * rows, n, dtype=torch.bfloat16, device="cuda")
    x, w = torch.ones(2 * rows, 8, dtype=torch.bfloat16, device="cuda"), torch.ones(n, 8, dtype=torch.bfloat16, device="cuda")
    dx = torch.empty_like(x)
    mib = 1 << 20
    grown = []
    for capture in (False, True):
        ctx = Context(0, stream=side.cuda_stream)

        def call(r):
            cfg = _abi.NpaLinearCfg(r, 0, 0, 0, 0, 0, 0, 0, 8, n, _abi.TYPE_BF16, _abi.ACT_GELU, _abi.TYPE_BF16, _abi.TYPE_BF16, 0)
            ctx.check(lib().npa_linear_adjoint(ctx.handle, C.byref(cfg), None, ptr(w), ptr(z), ptr(dy), ptr(dx), None, None))

        with torch.cuda.stream(side):
            call(rows)
            torch.cuda.synchronize()
            if capture:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=side):
                    call(rows)
            before = library_bytes()
            call(2 * rows)
            grown.append(library_bytes() - before)
        ctx.close()
    assert 64 * mib - 8 * mib < grown[0] < 64 * mib + 8 * mib, grown
    assert 128 * mib - 8 * mib < grown[1] < 128 * mib + 8 * mib, grown


@pytest.mark.parametrize("shape", ((300, 2048, 72), (700, 66, 128), (2048, 512, 2048)))
def test_capture_on_a_stream_of_its_own(shape):
    """A call that has run on one stream is captured on another, whose context has no workspace yet; and again, at
    a larger size, when that context has one that is too small."""
    small, large = calls(*shape), calls(shape[0] * 4, shape[1], shape[2] * 2)
    side, own = torch.cuda.Stream(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want, want_large = small(), large()
    torch.cuda.synchronize()
    graphs = []
    for run in (small, large):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=own):
            graphs.append((graph, run()))
    for _ in range(2):
        check_replays(*graphs[0], want, large)
        check_replays(*graphs[1], want_large, small)


def test_capture_as_torch_does_it():
    """The default of torch.cuda.graph: a capture stream of torch's choice."""
    run = calls(900, 66, 128, torch.float32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            want = run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    check_replays(graph, got, want, run)


def test_a_capture_outlives_its_thread():
    """A thread warms up, captures and ends; the graph is replayed here, between calls of a further thread on the
    same stream."""
    own = torch.cuda.Stream()
    small, large = calls(700, 66, 128), calls(2000, 66, 256)
    torch.cuda.synchronize()
    made = []

    def capture():
        with torch.cuda.stream(own):
            want = small()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=own):
                got = small()
            own.synchronize()
        made.append((graph, got, want))

    def further():
        with torch.cuda.stream(own):
            made.append([t.clone() for t in large()])
            own.synchronize()

    def run(f):
        t = threading.Thread(target=f)
        t.start()
        t.join()

    run(capture)
    spare = []

    def between():
        run(further)
        spare.append(torch.full((1 << 22,), math.nan, device="cuda"))
        torch.cuda.synchronize()

    check_replays(*made[0], between)
    assert len(made) == 4 and all(torch.equal(a, b) for other in made[2:] for a, b in zip(made[1], other))


def test_a_context_on_another_stream_is_refused():
    x, w = randn(40, 24, seed=1), randn(16, 24, seed=2)
    f = layers.layer_norm(x)
    side = torch.cuda.Stream()
    ctx = Context(0, stream=side.cuda_stream)
    for call in (lambda: layers.linear(x, w, ctx=ctx), lambda: layers.linear_adjoint(randn(40, 16, seed=3), x, w, ctx=ctx),
                 lambda: layers.layer_norm(x, ctx=ctx),
                 lambda: layers.layer_norm_adjoint(x, x, f.mean, f.rstd, ctx=ctx)):
        with pytest.raises(_abi.InvalidArgument, match="current stream"):
            call()
    want = layers.linear(x, w).out
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        assert torch.equal(layers.linear(x, w, ctx=ctx).out, want)
    torch.cuda.synchronize()
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    assert torch.equal(layers.linear(x, w, ctx=ctx).out, want)
    assert torch.equal(layers.linear(x, w, ctx=Context(0)).out, want)
