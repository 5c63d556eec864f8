"""The gate with sigmoid scores, a bias for balance and nodes of experts, against its definition in 64 bits.

Choices are whole numbers and have to be equal: the definition decides in 64
bits, whose own rounding (2^-53) no random input here comes near, and equal
numbers go to the lowest index. Weights are float: a score has the errors of
expf's argument, expf (two steps), a sum and a quotient, a weight those of the
sum of the chosen, a quotient and the scale.
"""
import itertools

import numpy as np
import pytest
import torch

from test_gpu_mixture import TYPES, check_groups, gen, normal

pytestmark = pytest.mark.gpu

mixture = pytest.importorskip("provenloop_amd.mixture")


def oracle(logits, k, mask=None, normalize=True, score="softmax", bias=None, scale=1.0, nodes=1, top_nodes=1, node_best=1):
    """(weights, experts, scores, ranks) in 64 bits."""
    l = logits.detach().double().cpu().numpy()
    t, e = l.shape
    ok = ~(l == -np.inf)
    if mask is not None:
        ok &= np.broadcast_to(mask.cpu().numpy(), l.shape)
    with np.errstate(all="ignore"):
        if score == "softmax":
            p = np.where(ok, np.exp(l - np.where(ok, l, -np.inf).max(1, keepdims=True, initial=-np.inf)), 0)
            s = p / np.where(p.sum(1, keepdims=True) == 0, 1, p.sum(1, keepdims=True))
        else:
            s = np.where(ok, 1 / (1 + np.exp(-l)), 0)
        c = s if bias is None else s + bias.double().cpu().numpy()
        ok = ok & ~(c == -np.inf) if bias is not None else ok
        by = np.where(ok, c if bias is not None else l, -np.inf)
        if top_nodes < nodes:
            per = e // nodes
            up = -np.sort(-np.where(ok, c if bias is not None or node_best == 2 else l, -np.inf).reshape(t, nodes, per), axis=2)
            value = up[:, :, 0].copy()
            if node_best == 2 and per > 1:
                value += np.where(up[:, :, 1] == -np.inf, 0, up[:, :, 1])
            best = np.argsort(-value, axis=1, kind="stable")[:, :top_nodes]
            kept = np.zeros((t, nodes), bool)
            np.put_along_axis(kept, best, True, 1)
            by = np.where(np.repeat(kept, per, 1), by, -np.inf)
        rank = np.argsort(-by, axis=1, kind="stable")[:, :k]
        has = np.take_along_axis(by, rank, 1) > -np.inf
        sel = np.where(has, np.take_along_axis(s, rank, 1), 0)
        z = sel.sum(1, keepdims=True) if normalize else np.ones((t, 1))
        w = scale * sel / np.where(z == 0, 1, z)
    return w, np.where(has, rank, -1), s, rank


FORMS = [dict(score="sigmoid"), dict(score="sigmoid", bias=True), dict(score="softmax", bias=True, scale=2.5),
         dict(score="softmax", scale=0.5)]
NODES = [(1, 1, 1, 1, 1, 1), (1, 3, 2, 1, 1, 1), (7, 8, 4, 4, 2, 1), (65, 9, 2, 3, 1, 2), (300, 60, 5, 5, 2, 1), (1025, 64, 8, 8, 4, 2),
         (700, 65, 5, 13, 3, 2), (129, 200, 32, 4, 2, 2), (33, 512, 4, 512, 100, 1), (40, 512, 8, 256, 9, 2), (64, 512, 8, 2, 1, 2),
         (5000, 16, 3, 8, 2, 2), (40000, 6, 2, 3, 2, 1), (2100, 256, 8, 8, 4, 2), (90, 256, 6, 32, 3, 1), (20, 1, 1, 1, 1, 2)]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("form", range(len(FORMS)))
@pytest.mark.parametrize("t,e,k,nodes,top,best", NODES)
def test_gate(dtype, form, t, e, k, nodes, top, best):
    g = gen(t + e + k)
    logits = normal(g, t, e, dtype=TYPES[dtype], std=2.0)
    opts = dict(FORMS[form], nodes=nodes, top_nodes=top, node_best=best)
    if opts.get("bias"):
        opts["bias"] = normal(g, e, std=0.05)
    for normalize, masked in itertools.product((True, False), (True, False)):
        mask = None
        if masked:
            mask = torch.rand(t, e, generator=g, device="cuda") < 0.6
            mask[::5] = False  # rows with no expert
        r = mixture.route(logits, k, mask=mask, normalize=normalize, **opts)
        w, ids, _, _ = oracle(logits, k, mask, normalize, **opts)
        assert np.array_equal(r.experts.cpu().numpy(), ids)
        steps = 2 * logits.float().abs().max().item() + e + 12
        np.testing.assert_allclose(r.weights.cpu().numpy(), w, rtol=steps * 2.0 ** -23, atol=2.0 ** -126)
        check_groups(r.groups, e)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("e,nodes,top,best", [(8, 1, 1, 1), (64, 8, 2, 2), (48, 4, 2, 1), (256, 8, 4, 2), (500, 5, 2, 2)])
def test_near_ties(score, e, nodes, top, best):
    """Few different logits and biases, and sums that only 64 bits tell apart."""
    g = gen(e)
    t, k = 700, min(8, e // nodes * top)
    logits = torch.randint(-3, 4, (t, e), generator=g, device="cuda").float() / 2
    step = torch.randint(0, 3, (e,), generator=g, device="cuda").float()
    for bias in (step * 0.001, step * 2.0 ** -24, step * 2.0 ** -30, torch.zeros(e, device="cuda"), 1000 + step * 2.0 ** -14):
        opts = dict(score=score, bias=bias, nodes=nodes, top_nodes=top, node_best=best)
        assert np.array_equal(mixture.route(logits, k, **opts).experts.cpu().numpy(), oracle(logits, k, **opts)[1])
    # scores a float step apart, biases that take the difference back or nearly
    l = normal(g, t, 1).expand(t, e).contiguous()
    l += torch.arange(e, device="cuda") * 2.0 ** -22
    s = torch.sigmoid(l[0].double()) if score == "sigmoid" else torch.softmax(l[0].double(), 0)
    bias = (s.mean() - s).float()
    opts = dict(score=score, bias=bias, nodes=nodes, top_nodes=top, node_best=best)
    w, ids, sc, _ = oracle(l, k, **opts)
    got = mixture.route(l, k, **opts).experts.cpu().numpy()
    c = np.sort(sc + bias.double().cpu().numpy(), axis=1)
    clear = (np.diff(c, axis=1) > 2.0 ** -48).all(1)  # 64 bits of another exp may differ by a few steps of 2^-53
    if nodes == 1 and score == "sigmoid":  # a softmax does not change with a row's shift: there all rows are one
        assert clear.sum() > t // 4
    if nodes == 1 or best == 1:
        assert np.array_equal(got[clear], ids[clear])


@pytest.mark.parametrize("per", [2, 8, 12, 16, 64])
def test_nodes_that_only_64_bits_tell_apart(per):
    """Two nodes whose sums are equal in float, of experts that differ clearly: one is kept, the larger."""
    logits = torch.full((9, 4 * per), -6.0, device="cuda")
    logits[:, 0::per], logits[:, 1::per] = 2.0, 1.0
    for first, second in ((1, 2), (2, 1), (3, 0)):
        for more in (2.0 ** -25, -2.0 ** -26, 0.0):  # float's neighbours of 1/4
            bias = torch.full((4 * per,), -0.5, device="cuda")
            bias[first * per], bias[first * per + 1] = 0.25, 0.0
            bias[second * per], bias[second * per + 1] = 0.0, 0.25 + more
            for score, top in (("sigmoid", 1), ("softmax", 1)):
                opts = dict(score=score, bias=bias, nodes=4, top_nodes=top, node_best=2)
                got = mixture.route(logits, 2, **opts).experts.cpu().numpy()
                if more:
                    assert np.array_equal(got, oracle(logits, 2, **opts)[1])
                else:  # (s + 1/4) + t and s + (t + 1/4): one number, and 64 bits round each to either side of it
                    assert (got == [first * per, first * per + 1]).all() or (got == [second * per + 1, second * per]).all()


def test_many_tokens_whose_nodes_come_near():
    """A prefill's tokens, a few of which have nodes nearer than float tells apart."""
    for seed, (e, nodes, top) in enumerate([(256, 8, 4), (256, 8, 4), (96, 8, 3), (512, 16, 4)] * 6):
        g = gen(200 + seed)
        logits = normal(g, 65536, e, dtype=torch.bfloat16, std=1.5)
        bias = (torch.randn(e, generator=g, device="cuda") * 20).round() * 0.001
        opts = dict(score="sigmoid", bias=bias, nodes=nodes, top_nodes=top, node_best=2)
        r = mixture.route(logits, 8, **opts)
        # the definition in 64 bits, on the GPU: the host's takes long
        c = 1 / (1 + torch.exp(-logits.double())) + bias.double()
        value = torch.sort(c.view(-1, nodes, e // nodes), dim=2, descending=True).values[:, :, :2].sum(2)
        kept = torch.zeros_like(value, dtype=torch.bool).scatter_(1, torch.sort(value, dim=1, descending=True, stable=True).indices[:, :top], True)
        c = c.masked_fill(~kept.repeat_interleave(e // nodes, 1), -float("inf"))
        assert torch.equal(r.experts, torch.sort(c, dim=1, descending=True, stable=True).indices[:, :8].to(torch.int32))


def test_extremes_and_bad_values():
    inf, nan = float("inf"), float("nan")
    z = torch.zeros(4, device="cuda")

    def chosen(rows, k, **o):
        r = mixture.route(torch.tensor(rows, device="cuda"), k, **o)
        return r.experts.tolist(), r.weights.cpu()

    # scores that are all 0 or all 1 in float
    ids, w = chosen([[-200.0, -201.0, -202.0, -300.0], [50.0, 60.0, 70.0, 80.0]], 2, score="sigmoid")
    assert ids == [[0, 1], [3, 2]]
    torch.testing.assert_close(w, torch.tensor([[0.73105858, 0.26894142], [0.5, 0.5]]), rtol=2.0 ** -20, atol=0)
    ids, w = chosen([[-200.0, -201.0, -202.0, -300.0]], 2, score="softmax", bias=torch.tensor([0.0, 0.0, 9.0, 8.0], device="cuda"))
    # the softmax of the two that were chosen: exp(-98) = 2.75e-43, a subnormal float
    assert ids == [[2, 3]] and w[0, 0] == 1 and abs(float(w[0, 1]) - np.exp(-98.0)) <= 2.0 ** -148
    # not chosen: a bias of -inf, even where nothing else is left; a bias of +inf comes first
    ids, w = chosen([[1.0, 2.0, 3.0, 4.0]], 3, score="sigmoid", bias=torch.tensor([0.0, inf, -inf, -inf], device="cuda"))
    assert ids == [[1, 0, -1]] and w[0, 2] == 0
    # rows whose mask leaves nothing, or nothing on the best node
    mask = torch.tensor([[False] * 4, [True, False, False, True]], device="cuda")
    ids, w = chosen([[1.0, 2.0, 3.0, 4.0]] * 2, 2, mask=mask, score="sigmoid", bias=z, nodes=2, top_nodes=1, node_best=2)
    assert ids == [[-1, -1], [3, -1]] and w[0].tolist() == [0, 0] and w[1].tolist() == [1, 0]
    # lowest values of the type are allowed, -inf is not
    low = torch.finfo(torch.float32).min
    ids, w = chosen([[low, low, -inf, low], [-inf] * 4], 4, score="sigmoid", bias=z)
    assert ids == [[0, 1, 3, -1], [-1] * 4]
    torch.testing.assert_close(w[0], torch.tensor([1 / 3, 1 / 3, 1 / 3, 0]), rtol=2.0 ** -20, atol=0)
    # NaN and infinities where the mask hides them change nothing; an allowed NaN is chosen first and shows
    bad = [[nan, 1.0, inf, 0.5]] * 2
    mask = torch.tensor([[False, True, False, True], [True, True, False, True]], device="cuda")
    for o in (dict(), dict(bias=z), dict(bias=z, nodes=2, top_nodes=2), dict(nodes=2, top_nodes=2, node_best=2)):
        x = torch.tensor(bad, device="cuda", requires_grad=True)
        r = mixture.route(x, 2, mask=mask, score="sigmoid", **o)
        assert r.experts.tolist() == [[1, 3], [0, 1]], o
        s = torch.sigmoid(torch.tensor([1.0, 0.5], dtype=torch.float64))
        torch.testing.assert_close(r.weights[0].detach().cpu().double(), s / s.sum(), rtol=2.0 ** -20, atol=0)
        assert torch.isnan(r.weights[1, 0])
        grad, = torch.autograd.grad(r.weights[0, 0], x)
        assert torch.isfinite(grad[0]).all() and grad[0, 0] == 0 and grad[0, 2] == 0
    # a NaN bias is the largest
    ids, _ = chosen([[1.0, 2.0, 3.0, 4.0]], 2, score="sigmoid", bias=torch.tensor([0.0, nan, 0.0, 0.0], device="cuda"))
    assert ids == [[1, 3]]
    ids, w = chosen([[inf, 0.0, 0.0, -1.0]], 2, score="sigmoid", bias=z)
    assert ids == [[0, 1]]
    torch.testing.assert_close(w, torch.tensor([[2 / 3, 1 / 3]]), rtol=2.0 ** -20, atol=0)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("e,k,nodes,top,best", [(4, 2, 1, 1, 1), (13, 5, 1, 1, 1), (64, 8, 8, 2, 1), (200, 12, 1, 1, 1), (512, 8, 4, 2, 2)])
def test_zeros_of_both_signs(dtype, e, k, nodes, top, best):
    """-0 and 0 are equal, and go to the lowest index."""
    g = gen(e)
    logits = torch.randint(-1, 2, (300, e), generator=g, device="cuda").float()
    logits = torch.where(torch.rand(300, e, generator=g, device="cuda") < 0.5, logits, -logits).to(TYPES[dtype])
    assert bool((torch.signbit(logits) & (logits == 0)).any())
    bias = torch.where(torch.rand(e, generator=g, device="cuda") < 0.5, 0.0, -0.0)
    for opts in (dict(score="sigmoid"), dict(scale=2.0), dict(score="sigmoid", bias=bias)):
        opts = dict(opts, nodes=nodes, top_nodes=top, node_best=best)
        r = mixture.route(logits, k, **opts)
        w, ids, _, _ = oracle(logits, k, **opts)
        assert np.array_equal(r.experts.cpu().numpy(), ids)
        np.testing.assert_allclose(r.weights.cpu().numpy(), w, rtol=2.0 ** -18, atol=0)
        check_groups(r.groups, e)


@pytest.mark.parametrize("e", [16, 40, 64, 130, 256, 300, 512])
def test_every_number_of_choices(e):
    """1 to 32, each with weights that are its own sum's."""
    g = gen(e)
    logits = normal(g, 40, e)
    bias = normal(g, e, std=0.1)
    for k in range(1, min(e, 32) + 1):
        for opts in (dict(score="sigmoid"), dict(bias=bias)):
            r = mixture.route(logits, k, **opts)
            w, ids, _, _ = oracle(logits, k, **opts)
            assert np.array_equal(r.experts.cpu().numpy(), ids), k
            np.testing.assert_allclose(r.weights.cpu().numpy(), w, rtol=2.0 ** -18, atol=2.0 ** -126)


def test_strides_and_masks():
    g = gen(3)
    wide = normal(g, 50, 40, dtype=torch.bfloat16)
    mask = torch.rand(24, generator=g, device="cuda") < 0.7
    bias = normal(g, 48, std=0.1)[::2]
    opts = dict(score="sigmoid", bias=bias, nodes=4, top_nodes=2, node_best=2)
    for logits in (wide[:, 5:29], wide.t()[:24].t(), wide[:1, :24].expand(50, 24)):
        for m in (mask, mask.expand(50, 24), None):
            r = mixture.route(logits, 4, mask=m, **opts)
            w, ids, _, _ = oracle(logits, 4, mask=m, **opts)
            assert np.array_equal(r.experts.cpu().numpy(), ids)
            np.testing.assert_allclose(r.weights.cpu().numpy(), w, rtol=2.0 ** -18, atol=2.0 ** -126)


def test_plain_keywords_are_the_plain_gate():
    g = gen(4)
    logits = normal(g, 300, 24)
    want = mixture.route(logits, 3)
    for opts in (dict(score="softmax", scale=1.0, nodes=1), dict(nodes=6, top_nodes=6, node_best=2)):
        r = mixture.route(logits, 3, **opts)
        assert torch.equal(r.weights, want.weights) and torch.equal(r.experts, want.experts)
    r = mixture.route(logits, 3, scale=2.0)
    assert torch.equal(r.weights, 2 * want.weights) and torch.equal(r.experts, want.experts)


@pytest.mark.parametrize("dtype,t,e,k", [("f32", 1, 3, 2), ("f32", 257, 13, 3), ("bf16", 100, 64, 8), ("f16", 70, 130, 4), ("f32", 9, 300, 8)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("normalize", [True, False])
def test_gradient(dtype, t, e, k, score, normalize):
    g = gen(e)
    logits = normal(g, t, e, dtype=TYPES[dtype], std=1.5).requires_grad_()
    mask = torch.rand(t, e, generator=g, device="cuda") < 0.7
    mask[::6] = False
    opts = dict(mask=mask, normalize=normalize, score=score, bias=normal(g, e, std=0.1), scale=2.5)
    dw = normal(g, t, k)
    got, = torch.autograd.grad(mixture.route(logits, k, **opts).weights, logits, dw)
    w, ids, s, rank = oracle(logits, k, **opts)
    # through the scores: weights' gradient in the chosen scores, then the scores' in the logits
    d = dw.double().cpu().numpy() * 2.5 * (ids >= 0)
    sel = np.take_along_axis(s, rank, 1) * (ids >= 0)
    z = sel.sum(1, keepdims=True)
    z[z == 0] = 1
    ds = np.zeros((t, e))
    np.put_along_axis(ds, rank, (d - (sel / z * d).sum(1, keepdims=True)) / z * (ids >= 0) if normalize else d, 1)
    want = s * (ds - (s * ds).sum(1, keepdims=True)) if score == "softmax" else ds * s * (1 - s)
    size = np.abs(d).max() * (k + 1)
    tol = torch.finfo(TYPES[dtype]).eps / 2 * np.abs(want) + (e + k + 24) * 2.0 ** -23 * size
    assert (np.abs(got.double().cpu().numpy() - want) <= tol).all()
    # and against differences of the definition, where no choice changes
    t0 = int(np.argmax(ids[:, k - 1] >= 0))
    l = logits.detach().double()
    one = dict(opts, mask=mask[t0:t0 + 1])
    for i in range(min(e, 6)):
        h = 1e-6
        up, down = l[t0:t0 + 1].clone(), l[t0:t0 + 1].clone()
        up[0, i] += h
        down[0, i] -= h
        (wu, iu, _, _), (wd, idn, _, _) = oracle(up, k, **one), oracle(down, k, **one)
        if np.array_equal(iu, idn):
            slope = ((wu - wd) * dw[t0].double().cpu().numpy()).sum() / (2 * h)
            assert abs(slope - float(got[t0, i])) <= 1e-6 + torch.finfo(TYPES[dtype]).eps * abs(slope) + tol[t0, i]


@pytest.mark.parametrize("t", [0, 1, 2048, 2049, 100000])
def test_lengths(t):
    g = gen(t)
    logits = normal(g, t, 16, std=1.0)
    opts = dict(score="sigmoid", bias=normal(g, 16, std=0.1), nodes=4, top_nodes=2, node_best=2)
    r = mixture.route(logits, 1, **opts)
    w, ids, _, _ = oracle(logits, 1, **opts) if t else (np.zeros((0, 1)), np.zeros((0, 1), int), None, None)
    assert np.array_equal(r.experts.cpu().numpy(), ids)
    check_groups(r.groups, 16)


def test_streams_graphs_and_runs():
    """With 4-bit experts after it: on another stream, again, and captured, bit for bit the same."""
    g = gen(13)
    logits, x = normal(g, 900, 32, dtype=torch.bfloat16), normal(g, 900, 128, dtype=torch.bfloat16)
    bias = torch.randint(-9, 9, (32,), generator=g, device="cuda").float() * 0.001
    e4 = mixture.quantize4(normal(g, 32, 64, 128, dtype=torch.bfloat16), 64)
    dy = normal(g, 900, 64)

    def step(logits, x):
        r = mixture.route(logits, 4, score="sigmoid", bias=bias, scale=2.5, nodes=8, top_nodes=3, node_best=2)
        y = (r.weights[..., None] * mixture.grouped_matmul(x, e4, r.groups).float()).sum(1)
        return [y.detach(), r.experts, *torch.autograd.grad(y, (logits, x), dy)]

    def leaves():
        return [logits.clone().requires_grad_(), x.clone().requires_grad_()]

    want = step(*leaves())
    assert all(torch.equal(p, q) for p, q in zip(want, step(*leaves())))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(*leaves())
        static = leaves()
        step(*static)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*static)
    for i in range(4):
        with torch.no_grad():
            static[0].copy_(normal(gen(50 + i), 900, 32, dtype=torch.bfloat16))
        bias.copy_(torch.randint(-9, 9, (32,), generator=gen(60 + i), device="cuda").float() * 0.001)
        graph.replay()
        torch.cuda.synchronize()
        eager = step(*[v.detach().clone().requires_grad_() for v in static])
        assert all(torch.equal(p, q) for p, q in zip(outs, eager)), i
