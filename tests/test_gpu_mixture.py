"""A step of a mixture of update rules: its dense part against reverse differentiation in 64 bits, the particles' gradients
through the oracle's perception, difference quotients, and that a fit runs."""
import numpy as np
import pytest
import torch

from burn_automata_amd import synthetic as syn
from burn_automata_amd import training
from burn_automata_amd.training import MixtureRule, fit
from oracle import oracle as O
from tests.helpers import rel_err

pytestmark = pytest.mark.gpu


def _case(n=600, hidden=48, count=5, top_k=2, scores="softmax"):
    w = syn.workload("c1", particles=n)
    pos = torch.from_numpy(np.asarray(w["positions"], dtype=np.float32)).reshape(-1, 4).cuda()
    st = torch.from_numpy(np.asarray(w["states"], dtype=np.float32)).reshape(n, -1).cuda()
    g = torch.Generator(device="cuda").manual_seed(3)
    st = st + 0.3 * torch.randn(st.shape, generator=g, device="cuda")
    return MixtureRule(w["model"], w["grid"], hidden, count=count, top_k=top_k, scores=scores), pos, st, n


def _dense(rule, trace, pos, st, features):
    """The rows after a step in 64 bits, of the experts that the step chose, and its parameters."""
    p = {k: v.double().requires_grad_() for k, v in rule.parameters.items()}
    normed = torch.nn.functional.layer_norm(features, features.shape[1:], p["gamma"], p["beta"], 1e-5)
    logits = normed @ p["router"].T
    score = torch.softmax(logits, 1) if rule.scores == "softmax" else torch.sigmoid(logits)
    chosen = trace.mixed[1].experts.long()
    weight = score.gather(1, chosen)
    weight = weight / (weight.sum(1, keepdim=True) + 1e-20)
    rows = torch.cat([pos[:, :2], st], 1).double()
    for j in range(rule.top_k):
        e = chosen[:, j]
        h = torch.bmm(p["w1"][e], normed[:, :, None])[:, :, 0] + p["b1"][e]
        h = torch.nn.functional.gelu(h, approximate="tanh")
        rows = rows + weight[:, j:j + 1] * (torch.bmm(p["w2"][e], h[:, :, None])[:, :, 0] + p["b2"][e])
    return rows, p


@pytest.mark.parametrize("scores", ("softmax", "sigmoid"))
def test_dense_part_against_reverse_differentiation(scores):
    """Every gradient within 1e-5 of its largest element: sums of at most 600 f32 terms, 2^-24 * 600 = 4e-5 at the very
    worst of their absolute values and about 2^-24 * sqrt(600) of it for terms of either sign."""
    rule, pos, st, n = _case(scores=scores)
    nx, ns, trace = rule.forward(pos, st, 1, n)
    g = torch.Generator(device="cuda").manual_seed(5)
    dx = torch.zeros_like(pos)
    dx[:, :2] = torch.randn(n, 2, generator=g, device="cuda")
    ds = torch.randn(ns.shape, generator=g, device="cuda")
    rule.backward(trace, dx, ds)
    rows, p = _dense(rule, trace, pos, st, trace.features.double())
    got = torch.cat([nx[:, :2], ns], 1).double()
    assert float((got - rows).detach().abs().max()) < 1e-5 * float(rows.detach().abs().max())
    loss = (rows * torch.cat([dx[:, :2], ds], 1).double()).sum()
    for name, want in zip(p, torch.autograd.grad(loss, list(p.values()))):
        err = float((rule.gradients[name].double() - want).abs().max())
        assert err < 1e-5 * float(want.abs().max()), (name, err)


def test_particles_gradient_against_the_oracle():
    """The particles' gradients: the dense part's in 64 bits, through the oracle's perception adjoint. Its own bar
    against the device is 1e-4 of the largest element."""
    rule, pos, st, n = _case(hidden=32)
    _, ns, trace = rule.forward(pos, st, 1, n)
    g = torch.Generator(device="cuda").manual_seed(6)
    dx, ds = torch.zeros_like(pos), torch.randn(ns.shape, generator=g, device="cuda")
    dx[:, :2] = torch.randn(n, 2, generator=g, device="cuda")
    back_x, back_s = rule.backward(trace, dx, ds)
    f = trace.features.double().requires_grad_()
    rows, _ = _dense(rule, trace, pos, st, f)
    through, = torch.autograd.grad((rows * torch.cat([dx[:, :2], ds], 1).double()).sum(), f)
    want = O.perceive_adjoint_with_options(pos.cpu().numpy(), st.cpu().numpy(), 1, n, st.shape[1], rule.grid, rule.options,
                                           through.float().cpu().numpy())
    want_x = torch.from_numpy(np.asarray(want.position)).reshape(n, 4).cuda() + dx
    want_s = torch.from_numpy(np.asarray(want.state)).reshape(n, -1).cuda() + ds
    assert rel_err(back_x, want_x) < 1e-4 and rel_err(back_s, want_s) < 1e-4


def test_step_against_difference_quotients():
    """The derivative along a direction in the second layer's weights, in which the step is linear: central differences
    with h = 1 of a loss summed in 64 bits of f32 outputs of magnitude 1, whose rounding leaves 2^-24 sqrt(terms)."""
    rule, pos, st, n = _case()
    _, ns, trace = rule.forward(pos, st, 1, n)
    g = torch.Generator(device="cuda").manual_seed(7)
    ds = torch.randn(ns.shape, generator=g, device="cuda")
    rule.backward(trace, torch.zeros_like(pos), ds)
    w2 = rule.parameters["w2"].clone()
    v = torch.randn(w2.shape, generator=g, device="cuda") * 0.1

    def at(t):
        rule.parameters["w2"].copy_(w2 + t * v)
        return float((rule.forward(pos, st, 1, n)[1].double() * ds.double()).sum())

    slope = (at(1.0) - at(-1.0)) / 2
    terms = rule.gradients["w2"].double() * v.double()
    assert abs(slope - float(terms.sum())) < 1e-4 * float(terms.square().sum().sqrt())


def test_gradients_add_up_over_steps():
    rule, pos, st, n = _case(300)
    _, ns, trace = rule.forward(pos, st, 1, n)
    dx, ds = torch.zeros_like(pos), torch.ones_like(ns)
    rule.backward(trace, dx, ds)
    once = {k: v.clone() for k, v in rule.gradients.items()}
    rule.backward(trace, dx, ds)
    for k, v in rule.gradients.items():
        assert torch.allclose(v, 2 * once[k], rtol=1e-6, atol=1e-6 * float(once[k].abs().max())), k


def test_one_rule_of_one_is_the_rule_itself():
    """A mixture of one rule that every particle uses, of weight 1: the update rule of the same parameters. Both round
    sums of at most 66 f32 terms."""
    rule, pos, st, n = _case(count=1, top_k=1)
    plain = training.UpdateRule(rule.config, rule.grid, 48)
    for k in ("gamma", "beta"):
        plain.parameters[k].copy_(rule.parameters[k])
    for k in ("w1", "b1", "w2", "b2"):
        plain.parameters[k].copy_(rule.parameters[k][0])
    for a, b in zip(rule.forward(pos, st, 1, n)[:2], plain.forward(pos, st, 1, n)[:2]):
        assert float((a - b).abs().max()) < 66 * 2.0 ** -22 * float(b.abs().max())


def test_fit_and_the_command_run(capsys, monkeypatch):
    rule, pos, st, n = _case(300)
    target = torch.sin(pos[:, :1] + pos[:, 1:2] * torch.arange(1, st.shape[1] + 1, device="cuda"))
    losses = fit(rule, pos, st, target, 1, n, steps=2, iterations=4)
    assert len(losses) == 4 and all(np.isfinite(losses))
    assert all(float(g.abs().max()) > 0 for g in rule.gradients.values())
    monkeypatch.setattr("sys.argv", ["training", "--particles", "300", "--steps", "1", "--iterations", "2", "--experts", "3"])
    training.main()
    assert "300 particles, 1 steps: loss" in capsys.readouterr().out
