"""The mixture operators at sizes that reach each of their kernels, against the definitions in 64 bits.

Tolerances as in test_gpu_mixture.py: half a step of the output's type, 2^-23 a
rounding of a float sum, 2^-16 on the low-rank part.
"""
import importlib.util
import os

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

mixture = pytest.importorskip("provenloop_amd.mixture")

from test_gpu_mixture import TYPES, check_groups, choices, gen, grouped_oracle, lora_oracle, near, normal, route_oracle  # noqa: E402


# tiles of 256 x 128 and 256 x 256, y = x w^T and y = x w, with more choices than a tile keeps in LDS, many adapters a
# tile, ranks of every padding, widths that are copied to padded ones
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("t,e,k,din,dout,rank", [
    (2100, 5, 1, 72, 560, 16), (2100, 5, 2, 560, 72, 33), (2200, 9, 6, 136, 1040, 9), (8000, 6, 2, 72, 1100, 20),
    (8000, 3, 1, 1100, 88, 8), (1500, 40, 2, 200, 800, 128), (31, 4, 2, 203, 515, 12), (33, 4, 2, 203, 515, 12)])
def test_lora_linear_sizes(dtype, t, e, k, din, dout, rank):
    g = gen(t + dout)
    dt = TYPES[dtype]
    x, w = normal(g, t, din, dtype=dt).requires_grad_(), normal(g, dout, din, dtype=dt, std=din ** -0.5)
    a = normal(g, e, rank, din, dtype=dt, std=din ** -0.5).requires_grad_()
    b = normal(g, e, dout, rank, dtype=dt, std=0.3).requires_grad_()
    ids = choices(g, t, e, k)
    gate = torch.rand(t, k, generator=g, device="cuda").requires_grad_()
    scale = torch.rand(e, generator=g, device="cuda") * 2
    bias = normal(g, dout, dtype=dt)
    dy = normal(g, t, dout, dtype=dt)
    y = mixture.lora_linear(x, w, a, b, ids, weights=gate, scale=scale, bias=bias)
    dx, da, db, dg = torch.autograd.grad(y, (x, a, b, gate), dy)
    ref, mag = lora_oracle(x.detach(), w, a.detach(), b.detach(), ids, gate.detach(), scale, bias, dy)
    near(y.detach(), ref["y"], mag["y"], din + rank * k, mag["low"])
    near(dx, ref["dx"], mag["dx"], dout + rank * k, mag["dxl"])
    near(da, ref["da"], mag["da"], dout + t * k, mag["da"])
    near(db, ref["db"], mag["db"], din + t * k, mag["db"])
    near(dg, ref["dg"], mag["dg"], din + dout + rank)
    with torch.no_grad():
        near(mixture.lora_linear(x, w, a, b, ids, weights=gate, scale=scale, bias=bias), ref["y"], mag["y"], din + rank * k, mag["low"])


def test_lora_requests_of_ragged_lengths():
    """A prefill's requests, side by side, with an adapter each or none."""
    g = gen(21)
    t, e, din, dout, rank = 4000, 7, 264, 520, 24
    ends = torch.sort(torch.randint(0, t, (13,), generator=g, device="cuda")).values
    of = torch.searchsorted(ends, torch.arange(t, device="cuda"), right=True)
    ids = torch.randint(-1, e, (14,), generator=g, device="cuda", dtype=torch.int32)[of]
    x, w = normal(g, t, din, dtype=torch.bfloat16), normal(g, dout, din, dtype=torch.bfloat16, std=0.1)
    a, b = normal(g, e, rank, din, dtype=torch.bfloat16, std=0.1), normal(g, e, dout, rank, dtype=torch.bfloat16)
    ref, mag = lora_oracle(x, w, a, b, ids.view(t, 1), None, None, None)
    near(mixture.lora_linear(x, w, a, b, ids), ref["y"], mag["y"], din + rank, mag["low"])
    groups = mixture.group(ids, e)
    near(mixture.lora_linear(x, w, a, b, ids, groups=groups), ref["y"], mag["y"], din + rank, mag["low"])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("t,e,k,din,dout", [(9000, 3, 1, 96, 1100), (9000, 3, 1, 1104, 96), (3000, 300, 2, 64, 128), (700, 2, 1, 520, 264),
                                            (2500, 4, 2, 77, 900), (2100, 2, 3, 640, 31)])
def test_grouped_matmul_sizes(dtype, t, e, k, din, dout):
    g = gen(t + dout)
    ids = choices(g, t, e, k)
    x = normal(g, t, din, dtype=TYPES[dtype]).requires_grad_()
    w = normal(g, e, dout, din, dtype=TYPES[dtype], std=0.5).requires_grad_()
    dy = normal(g, t, k, dout, dtype=TYPES[dtype])
    y = mixture.grouped_matmul(x, w, mixture.group(ids, e))
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    (ry, rdx, rdw), (my, mdx, mdw) = grouped_oracle(x.detach(), w.detach(), ids, k, dy)
    near(y.detach(), ry, my, din)
    near(dx, rdx, mdx, dout * k)
    near(dw, rdw, mdw, t * k)
    assert (y[ids < 0] == 0).all()


def test_one_group_has_nearly_all():
    """Groups of very different sizes, some empty: the longest first, none left out."""
    g = gen(31)
    sizes = [0, 1, 3000, 0, 64, 65, 0, 129]
    ids = torch.cat([torch.full((n, 1), i, dtype=torch.int32) for i, n in enumerate(sizes)])[torch.randperm(sum(sizes), generator=torch.Generator().manual_seed(1))].cuda()
    t = len(ids)
    x = normal(g, t, 264, dtype=torch.bfloat16).requires_grad_()
    w = normal(g, 8, 136, 264, dtype=torch.bfloat16).requires_grad_()
    dy = normal(g, t, 1, 136, dtype=torch.bfloat16)
    y = mixture.grouped_matmul(x, w, mixture.group(ids, 8))
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    (ry, rdx, rdw), (my, mdx, mdw) = grouped_oracle(x.detach(), w.detach(), ids, 1, dy)
    near(y.detach(), ry, my, 264)
    near(dx, rdx, mdx, 136)
    near(dw, rdw, mdw, t)
    assert (dw[[0, 3, 6]] == 0).all()


@pytest.mark.parametrize("dtype,t,e,k", [("f16", 64, 512, 32), ("f32", 70, 200, 32), ("bf16", 300, 40, 30), ("f16", 500, 16, 16),
                                         ("f32", 9, 8, 8), ("f32", 2200000, 3, 2), ("bf16", 70000, 24, 5)])
@pytest.mark.parametrize("normalize", [True, False])
def test_route_sizes(dtype, t, e, k, normalize):
    g = gen(t + e)
    logits = normal(g, t, e, dtype=TYPES[dtype], std=2.0)
    mask = torch.rand(t, e, generator=g, device="cuda") < 0.8
    mask[::7] = False
    r = mixture.route(logits, k, mask=mask, normalize=normalize)
    w, ids, _, _ = route_oracle(logits, mask, k, normalize)
    assert np.array_equal(r.experts.cpu().numpy(), ids)
    steps = 2 * logits.float().abs().max().item() + (k if normalize else e) + 8  # as in test_gpu_mixture.test_route
    np.testing.assert_allclose(r.weights.cpu().numpy(), w, rtol=steps * 2.0 ** -23, atol=2.0 ** -126)
    check_groups(r.groups, e)


@pytest.mark.parametrize("t", [1, 20, 3000])
def test_serving_in_a_graph(t):
    """The path without gradients, captured: every replay equals the eager result on the inputs of the time."""
    g = gen(t)
    x = normal(g, t, 200, dtype=torch.float16)
    w, we = normal(g, 333, 200, dtype=torch.float16), normal(g, 6, 72, 200, dtype=torch.float16)
    a, b = normal(g, 6, 8, 200, dtype=torch.float16), normal(g, 6, 333, 8, dtype=torch.float16)
    logits = normal(g, t, 6)

    @torch.no_grad()
    def step():
        r = mixture.route(logits, 2)
        return [mixture.lora_linear(x, w, a, b, r.experts, weights=r.weights), mixture.grouped_matmul(x, we, r.groups),
                mixture.lora_linear(x, w, a, b, r.experts[:, :1].contiguous())]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(4):
        x.copy_(normal(gen(50 + i), t, 200, dtype=torch.float16))
        logits.copy_(normal(gen(70 + i), t, 6))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(outs, step())), i


def test_the_gradients_are_not_differentiable_again():
    x = torch.randn(40, 8, device="cuda").requires_grad_()
    r = mixture.route(x, 2)
    dx, = torch.autograd.grad(r.weights.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="second time"):
        dx.sum().backward()


def test_the_example_learns():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "plain_mixture.py")
    spec = importlib.util.spec_from_file_location("plain_mixture", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses = example.main(["--hidden", "256", "--out", "192", "--rank", "8", "--experts", "4", "--tokens", "512", "--steps", "12"])
    assert np.isfinite(losses).all() and losses[-1] < 0.7 * losses[0]
