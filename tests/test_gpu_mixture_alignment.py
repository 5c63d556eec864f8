"""Gradients that do not start on 16 bytes, as the backward of a concatenation hands them on, and wide outputs of operands that do not.

Widths are multiples of 8, so that nothing is copied for its width and the
kernels for unaligned operands run. Tolerances as in test_gpu_mixture.py.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

from provenloop_amd import mixture  # noqa: E402
from test_gpu_mixture import TYPES, choices, gen, grouped_oracle, lora_oracle, near, normal  # noqa: E402


# few rows and many, ranks of every padding, B^T dy in small and in large tiles (the last two)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("t,e,k,din,dout,rank", [(1, 3, 2, 64, 72, 8), (20, 4, 1, 264, 136, 16), (300, 5, 2, 72, 88, 12), (700, 7, 2, 129, 264, 30),
                                                 (2100, 5, 1, 72, 560, 40), (1000, 3, 6, 136, 1040, 100), (8000, 3, 2, 520, 88, 128),
                                                 (6000, 2, 4, 72, 200, 64)])
def test_lora_gradients(dtype, t, e, k, din, dout, rank):
    g, dt = gen(t + dout), TYPES[dtype]
    x, w = normal(g, t, din, dtype=dt).requires_grad_(), normal(g, dout, din, dtype=dt, std=din ** -0.5)
    a = normal(g, e, rank, din, dtype=dt, std=din ** -0.5).requires_grad_()
    b = normal(g, e, dout, rank, dtype=dt, std=0.3).requires_grad_()
    ids = choices(g, t, e, k)
    gate = torch.rand(t, k, generator=g, device="cuda").requires_grad_()
    scale = torch.rand(e, generator=g, device="cuda") * 2
    for dy in (normal(g, t, dout + 3, dtype=dt)[:, 1:1 + dout], normal(g, t * dout + 5, dtype=dt)[5:].view(t, dout)):
        assert dy.data_ptr() % 16 != 0
        y = mixture.lora_linear(x, w, a, b, ids, weights=gate, scale=scale)
        dx, da, db, dg = torch.autograd.grad(y, (x, a, b, gate), dy)
        ref, mag = lora_oracle(x.detach(), w, a.detach(), b.detach(), ids, gate.detach(), scale, None, dy)
        near(dx, ref["dx"], mag["dx"], dout + rank * k, mag["dxl"])
        near(da, ref["da"], mag["da"], dout + t * k, mag["da"])
        near(db, ref["db"], mag["db"], din + t * k, mag["db"])
        near(dg, ref["dg"], mag["dg"], din + dout + rank)
        # one gradient at a time
        for leaf, got in ((x, dx), (a, da), (b, db), (gate, dg)):
            y = mixture.lora_linear(x, w, a, b, ids, weights=gate, scale=scale)
            assert torch.equal(torch.autograd.grad(y, leaf, dy)[0], got)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("per_slot", [False, True])
@pytest.mark.parametrize("t,e,k,din,dout", [(1, 3, 2, 64, 72), (33, 4, 1, 264, 136), (150, 4, 2, 96, 80), (700, 2, 1, 520, 264), (2500, 4, 2, 77, 904),
                                            (3000, 40, 3, 200, 128)])
def test_grouped_gradients(dtype, per_slot, t, e, k, din, dout):
    g, dt = gen(t + dout), TYPES[dtype]
    ids = choices(g, t, e, k)
    x = normal(g, *((t, k, din) if per_slot else (t, din)), dtype=dt).requires_grad_()
    w = normal(g, e, dout, din, dtype=dt, std=0.5).requires_grad_()
    dy = normal(g, t * k * dout + 1, dtype=dt)[1:].view(t, k, dout)
    assert dy.data_ptr() % 16 != 0
    groups = mixture.group(ids, e)
    dx, dw = torch.autograd.grad(mixture.grouped_matmul(x, w, groups), (x, w), dy)
    (_, rdx, rdw), (_, mdx, mdw) = grouped_oracle(x.detach(), w.detach(), ids, k, dy)
    near(dx, rdx, mdx, dout * k)
    near(dw, rdw, mdw, t * k)
    for leaf, got in ((x, dx), (w, dw)):
        assert torch.equal(torch.autograd.grad(mixture.grouped_matmul(x, w, groups), leaf, dy)[0], got)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("t,k", [(16, 1), (9, 3), (32, 6)])
def test_few_tokens_of_very_wide_projections(dtype, t, k):
    """Large tiles without copies."""
    g, dt = gen(t), TYPES[dtype]
    din, dout, e, rank = 200, 33000, 7, 12
    x, w = normal(g, t, din + 3, dtype=dt)[:, 1:1 + din], normal(g, dout, din, dtype=dt, std=din ** -0.5)
    a, b = normal(g, e, rank, din, dtype=dt, std=din ** -0.5), normal(g, e, dout, rank, dtype=dt, std=0.3)
    ids, gate, bias = choices(g, t, e, k), torch.rand(t, k, generator=g, device="cuda"), normal(g, dout, dtype=dt)
    ref, mag = lora_oracle(x, w, a, b, ids, gate, None, bias)
    near(mixture.lora_linear(x, w, a, b, ids, weights=gate, bias=bias), ref["y"], mag["y"], din + rank * k, mag["low"])
