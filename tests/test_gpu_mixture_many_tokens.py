"""More tokens than a launch with a workgroup for every few of them could have."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from provenloop_amd import mixture  # noqa: E402


def test_gate_gradient_of_more_than_2_to_the_26_tokens():
    t = (1 << 26) + 5
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    logits = torch.randn(t, 2, generator=g, device="cuda", dtype=torch.bfloat16).requires_grad_()
    dw = torch.randn(t, 1, generator=g, device="cuda")
    got, = torch.autograd.grad(mixture.route(logits, 1, normalize=False).weights, logits, dw)
    for at in (0, 1 << 22, (1 << 26) - 500, t - 1000):  # rows do not depend on each other
        part = logits[at:at + 1000].detach().requires_grad_()
        want, = torch.autograd.grad(mixture.route(part, 1, normalize=False).weights, part, dw[at:at + 1000])
        assert torch.equal(got[at:at + 1000], want)
        p = torch.softmax(part.detach().double(), 1)
        picked = torch.zeros_like(p).scatter_(1, part.detach().argmax(1, keepdim=True), 1.0)
        exact = p * (picked - (p * picked).sum(1, keepdim=True)) * dw[at:at + 1000]
        assert ((want.double() - exact).abs() <= exact.abs() * 2.0 ** -8 + 2.0 ** -18 * dw[at:at + 1000].abs()).all()
