"""A step of a trained update rule, forward and backward, on the operators of ``kernels`` and ``layers``.

The rule is perception -> layer norm -> linear, gelu -> linear, added to the particles:

    rows  = [positions[:d] | states]                                  [T, d + S]
    next  = linear(gelu(linear(layer_norm(features))), residual=rows)

``UpdateRule.forward`` keeps what the way back reads, ``UpdateRule.backward`` adds the parameters' gradients to
``rule.gradients`` and returns the particles' own, so a rollout of several steps is a loop forward and a loop
backward. ``python -m burn_automata_amd.training`` fits a rule to a target on one GPU.
"""
from __future__ import annotations

import argparse
from dataclasses import dataclass

import torch

from . import kernels, layers
from .config import HashGridConfig, NpaConfig

ACTIVATION = layers.Activation.gelu


@dataclass
class StepTrace:
    """What UpdateRule.backward reads of one forward step."""

    positions: object
    states: object
    features: object
    norm: object
    hidden: object
    batch_size: int
    particle_count: int


class UpdateRule:
    """The parameters of a rule over ``config``'s perception (float32), and their gradients of the same shapes."""

    NAMES = ("gamma", "beta", "w1", "b1", "w2", "b2")

    def __init__(self, config: NpaConfig, grid: HashGridConfig, hidden: int | None = None, seed: int = 42,
                 device: int = 0):
        self.config, self.grid = config, grid
        self.options = config.perception_options()
        features, outputs = config.perception_dims(), config.update_dims()
        hidden = hidden or config.hidden_dims
        dev = f"cuda:{device}"
        g = torch.Generator(device=dev).manual_seed(seed)

        def normal(*shape, scale):
            return torch.randn(*shape, generator=g, device=dev) * scale

        self.parameters = {
            "gamma": torch.ones(features, device=dev), "beta": torch.zeros(features, device=dev),
            "w1": normal(hidden, features, scale=features ** -0.5), "b1": torch.zeros(hidden, device=dev),
            "w2": normal(outputs, hidden, scale=0.1 * hidden ** -0.5), "b2": torch.zeros(outputs, device=dev)}
        self.gradients = {k: torch.zeros_like(v) for k, v in self.parameters.items()}

    def zero_gradients(self):
        for g in self.gradients.values():
            g.zero_()

    def forward(self, positions, states, batch_size: int, particle_count: int, ctx=None):
        """(next positions [T, 4], next states [T, S], trace). Without ``ctx`` all of it runs on torch's current
        stream."""
        ctx = ctx or layers.current_context(positions.get_device())
        p, d, s = self.parameters, self.config.spatial_dims, self.config.state_dims
        states = states.reshape(-1, s)
        features = kernels.perceive_with_options(positions, states, batch_size, particle_count, s, self.grid,
                                                 self.options, ctx).features
        norm = layers.layer_norm(features, p["gamma"], p["beta"], ctx=ctx)
        hidden = layers.linear(norm.out, p["w1"], p["b1"], ACTIVATION, keep_preactivation=True, ctx=ctx)
        rows = torch.cat([positions[:, :d], states], dim=1)
        rows = layers.linear(hidden.out, p["w2"], p["b2"], residual=rows, ctx=ctx).out
        next_positions = positions.clone()
        next_positions[:, :d] = rows[:, :d]
        return next_positions, rows[:, d:].contiguous(), StepTrace(positions, states, features, norm, hidden,
                                                                   batch_size, particle_count)

    def backward(self, trace: StepTrace, position_adjoint, state_adjoint, ctx=None):
        """(position adjoint [T, 4], state adjoint [T, S]) of a step's inputs from those of its outputs; the
        parameters' gradients are added to ``gradients``."""
        ctx = ctx or layers.current_context(position_adjoint.get_device())
        p, g, d, s = self.parameters, self.gradients, self.config.spatial_dims, self.config.state_dims
        rows = torch.cat([position_adjoint[:, :d], state_adjoint.reshape(-1, s)], dim=1)
        back = layers.linear_adjoint(rows, trace.hidden.out, p["w2"], weight_adjoint=g["w2"], bias_adjoint=g["b2"],
                                     ctx=ctx)
        back = layers.linear_adjoint(back.x, trace.norm.out, p["w1"], trace.hidden.preactivation, ACTIVATION,
                                     weight_adjoint=g["w1"], bias_adjoint=g["b1"], ctx=ctx)
        back = layers.layer_norm_adjoint(back.x, trace.features, trace.norm.mean, trace.norm.rstd, p["gamma"],
                                         g["gamma"], g["beta"], ctx=ctx)
        through = kernels.perceive_adjoint_with_options(trace.positions, trace.states, trace.batch_size,
                                                        trace.particle_count, s, self.grid, self.options, back.x, ctx)
        # the residual's way past the rule; what lies past the spatial axes passes unchanged
        return position_adjoint + through.position, state_adjoint.reshape(-1, s) + through.state.reshape(-1, s)


def fit(rule: UpdateRule, positions, states, target, batch_size: int, particle_count: int, steps: int = 2,
        iterations: int = 50, rate: float = 0.01):
    """Adam on the mean squared distance of the states after ``steps`` steps to ``target`` [T, S]. Returns the
    loss before each iteration."""
    optimizer = torch.optim.Adam([rule.parameters[k] for k in rule.NAMES], lr=rate)
    for name in rule.NAMES:
        rule.parameters[name].grad = rule.gradients[name]
    losses = []
    for _ in range(iterations):
        x, s, traces = positions, states, []
        for _ in range(steps):
            x, s, trace = rule.forward(x, s, batch_size, particle_count)
            traces.append(trace)
        difference = s - target
        losses.append(float(difference.square().mean()))
        dx, ds = torch.zeros_like(x), difference * (2.0 / difference.numel())
        rule.zero_gradients()
        for trace in reversed(traces):
            dx, ds = rule.backward(trace, dx, ds)
        optimizer.step()
    return losses


def main():
    from . import synthetic

    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--particles", type=int, default=4096)
    ap.add_argument("--steps", type=int, default=2)
    ap.add_argument("--iterations", type=int, default=50)
    args = ap.parse_args()
    w = synthetic.workload("c1", particles=args.particles)
    positions = torch.from_numpy(w["positions"]).reshape(-1, 4).cuda()
    states = torch.from_numpy(w["states"]).reshape(args.particles, -1).cuda()
    rule = UpdateRule(w["model"], w["grid"])
    # each channel to a plane wave over the disk
    waves = torch.arange(1, states.shape[1] + 1, device="cuda") * 0.5
    target = torch.sin(positions[:, :1] * waves + positions[:, 1:2])
    losses = fit(rule, positions, states, target, 1, args.particles, args.steps, args.iterations)
    print(f"{args.particles} particles, {args.steps} steps: loss {losses[0]:.4f} -> {losses[-1]:.4f} in "
          f"{args.iterations} iterations")


if __name__ == "__main__":
    main()
