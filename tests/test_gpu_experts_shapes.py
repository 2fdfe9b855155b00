"""Arrays of the right number of elements in another shape than the choices have are refused, not read in another order."""
import pytest
import torch

from burn_automata_amd import _abi, experts

pytestmark = pytest.mark.gpu


def test_turned_arrays_are_refused():
    rows, count, k, width, outputs = 6, 4, 3, 8, 5
    g = torch.Generator(device="cuda").manual_seed(1)
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    logits = randn(rows, count)
    r = experts.route(logits, k)
    y, w = randn(rows * k, width), randn(count, outputs, width)
    turned = r.weights.t()
    for call in (lambda: experts.combine(y, r.plan, turned), lambda: experts.combine(y, r.plan, turned.contiguous()),
                 lambda: experts.combine(y, r.plan, r.weights.reshape(2, -1)),
                 lambda: experts.combine_adjoint(randn(rows, width), y, r.plan, turned),
                 lambda: experts.route_adjoint(turned, logits, r.experts),
                 lambda: experts.linear(y, w, r.plan, randn(outputs, count))):
        with pytest.raises(_abi.OutputShape):
            call()


def test_leading_dims_and_flat_arrays_are_served():
    g = torch.Generator(device="cuda").manual_seed(1)
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    logits = randn(2, 3, 4)
    r = experts.route(logits, 3)
    y, w, b = randn(18, 8), randn(4, 5, 8), randn(4, 5)
    want = experts.combine(y, r.plan, r.weights)
    assert torch.equal(experts.combine(y, r.plan, r.weights.reshape(6, 3)), want)
    assert torch.equal(experts.combine(y, r.plan, r.weights.reshape(-1)), want)
    assert torch.equal(experts.linear(y, w, r.plan, b).out, experts.linear(y, w, r.plan, b.reshape(-1)).out)
    d = experts.route_adjoint(r.weights, logits, r.experts)
    assert torch.equal(experts.route_adjoint(r.weights.reshape(6, 3), logits, r.experts), d)
