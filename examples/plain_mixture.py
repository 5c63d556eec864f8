"""Plain mixtures of adapters end to end: sessions with adapters of their own,
a gated mixture served in batches, and training of the adapters and the gate.

    python examples/plain_mixture.py [--hidden 1536] [--out 1536] [--rank 16] [--experts 8] [--tokens 4096] [--steps 20]

The projection is frozen and random, as are the teacher's adapters that the
training step learns to follow; all of it runs on one GPU through
provenloop_amd.mixture.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from provenloop_amd import mixture  # noqa: E402


class MixtureLinear(torch.nn.Module):
    """A frozen projection with n gated low-rank adapters, `choices` of them a token."""

    def __init__(self, weight, n, rank, choices, scale=2.0):
        super().__init__()
        d_out, d_in = weight.shape
        dev, dt = weight.device, weight.dtype
        self.register_buffer("weight", weight)
        self.register_buffer("scale", torch.full((n,), scale, device=dev))
        self.choices = choices
        self.gate = torch.nn.Parameter(torch.randn(n, d_in, device=dev) * d_in ** -0.5)
        self.lora_a = torch.nn.Parameter((torch.randn(n, rank, d_in, device=dev) * d_in ** -0.5).to(dt))
        self.lora_b = torch.nn.Parameter(torch.zeros(n, d_out, rank, device=dev, dtype=dt))

    def forward(self, x, allowed=None):
        routing = mixture.route(x.float() @ self.gate.t(), self.choices, mask=allowed)
        return mixture.lora_linear(x, self.weight, self.lora_a, self.lora_b, routing.experts, weights=routing.weights,
                                   scale=self.scale, groups=routing.groups)


@torch.no_grad()
def serve_sessions(weight, lora_a, lora_b, adapter_of_session):
    """One token of every session through the projection, each with its own adapter (or none: -1)."""
    x = torch.randn(len(adapter_of_session), weight.shape[1], device=weight.device).to(weight.dtype)
    ids = torch.tensor(adapter_of_session, dtype=torch.int32, device=weight.device)
    return x, mixture.lora_linear(x, weight, lora_a, lora_b, ids)


@torch.no_grad()
def experts_layer(x, gate, up, down, choices):
    """A mixture of full expert layers: route, products grouped by expert, weighted sum."""
    routing = mixture.route(x.float() @ gate.t(), choices)
    h = torch.nn.functional.silu(mixture.grouped_matmul(x, up, routing.groups))
    y = mixture.grouped_matmul(h, down, routing.groups)
    return (routing.weights[..., None] * y.float()).sum(1).to(x.dtype)


def train(model, teacher, tokens, steps, lr=1e-2):
    """The student's adapters and gate follow the teacher's outputs; returns the losses."""
    d_in = model.weight.shape[1]
    losses = []
    optimiser = torch.optim.Adam(model.parameters(), lr=lr)
    x = torch.randn(tokens, d_in, device=model.weight.device).to(model.weight.dtype)
    with torch.no_grad():
        want = teacher(x).float()
    for _ in range(steps):
        optimiser.zero_grad(set_to_none=True)
        loss = (model(x).float() - want).square().mean()
        loss.backward()
        optimiser.step()
        losses.append(loss.detach())
    return [float(v) for v in losses]


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, value in (("hidden", 1536), ("out", 1536), ("rank", 16), ("experts", 8), ("tokens", 4096), ("steps", 20)):
        p.add_argument("--" + name, type=int, default=value)
    a = p.parse_args(argv)
    torch.manual_seed(0)
    weight = (torch.randn(a.out, a.hidden, device="cuda") * a.hidden ** -0.5).bfloat16()
    teacher = MixtureLinear(weight, a.experts, a.rank, 2)
    with torch.no_grad():
        teacher.lora_b.normal_(std=0.3)
    student = MixtureLinear(weight, a.experts, a.rank, 2)
    student.gate.data.copy_(teacher.gate.data)

    _, y = serve_sessions(weight, teacher.lora_a, teacher.lora_b, [i % (a.experts + 1) - 1 for i in range(32)])
    print(f"32 sessions: {tuple(y.shape)}")
    up = (torch.randn(a.experts, 256, a.hidden, device="cuda") * a.hidden ** -0.5).bfloat16()
    down = (torch.randn(a.experts, a.hidden, 256, device="cuda") / 16).bfloat16()
    x = torch.randn(a.tokens, a.hidden, device="cuda").bfloat16()
    print(f"experts: {tuple(experts_layer(x, teacher.gate.data, up, down, 2).shape)}")
    losses = train(student, teacher, a.tokens, a.steps)
    print(f"training: loss {losses[0]:.4f} -> {losses[-1]:.4f} in {a.steps} steps")
    return losses


if __name__ == "__main__":
    main()
