"""Infinities and NaN in one adapter, token or coefficient: where the definition has them, and nowhere else.

The oracle takes every adapter's own rows alone, in 64 bits on the CPU, so that
nothing is multiplied that the definition does not multiply. Tolerances of the
finite outputs as in test_gpu_mixture.py.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

from provenloop_amd import mixture  # noqa: E402
from test_gpu_mixture import TYPES, choices, gen, near, normal  # noqa: E402

INF, NAN = float("inf"), float("nan")

# t, adapters, choices, d_in, d_out, rank: large tiles of both shapes each way, more choices than a tile lists, small tiles
SIZES = [(2100, 5, 1, 72, 560, 16), (2100, 5, 2, 560, 72, 33), (2200, 9, 6, 136, 1040, 9), (8000, 6, 2, 72, 1100, 20),
         (8000, 3, 1, 1100, 88, 8), (300, 4, 2, 72, 88, 12), (40, 4, 2, 264, 136, 16)]


def low_rank(x, a, b, ids, gate, scale):
    """sum_j gate_tj scale_e b_e (a_e x_t) over each token's own adapters, and its magnitude."""
    x, a, b, ids = x.detach().cpu().double(), a.detach().cpu().double(), b.detach().cpu().double(), ids.cpu()
    y, size = torch.zeros(len(x), b.shape[1], dtype=torch.float64), torch.zeros(len(x), b.shape[1], dtype=torch.float64)
    for e in range(a.shape[0]):
        for j in range(ids.shape[1]):
            rows = torch.nonzero(ids[:, j] == e)[:, 0]
            if len(rows):
                c = (gate[rows, j].detach().cpu().double() if gate is not None else torch.ones(len(rows), dtype=torch.float64))[:, None]
                c = c * float(scale[e]) if scale is not None else c
                y[rows] += c * ((x[rows] @ a[e].t()) @ b[e].t())
                size[rows] += c.abs() * ((x[rows].abs() @ a[e].abs().t()) @ b[e].abs().t())
    return y.cuda(), size.cuda()


def agrees(got, want, magnitude, n, low):
    """The same infinities and NaN, and the finite values within their tolerance."""
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[torch.isinf(want)].double(), want[torch.isinf(want)])
    near(got[fine], want[fine], magnitude[fine], n, low[fine])


def case(t, e, k, din, dout, rank, dtype):
    g, dt = gen(t + dout), TYPES[dtype]
    c = dict(x=normal(g, t, din, dtype=dt), w=normal(g, dout, din, dtype=dt, std=din ** -0.5),
             a=normal(g, e, rank, din, dtype=dt, std=din ** -0.5), b=normal(g, e, dout, rank, dtype=dt, std=0.3),
             ids=choices(g, t, e, k), gate=torch.rand(t, k, generator=g, device="cuda"),
             scale=torch.rand(e, generator=g, device="cuda") + 0.5, dy=normal(g, t, dout, dtype=dt))
    return c


def passes(c):
    """(y, y without a graph, dx)"""
    x = c["x"].clone().requires_grad_()
    y = mixture.lora_linear(x, c["w"], c["a"], c["b"], c["ids"], weights=c["gate"], scale=c["scale"])
    dx, = torch.autograd.grad(y, x, c["dy"])
    with torch.no_grad():
        return y.detach(), mixture.lora_linear(c["x"], c["w"], c["a"], c["b"], c["ids"], weights=c["gate"], scale=c["scale"]), dx


def check_forward(c, got):
    x, w = c["x"].double().cpu(), c["w"].double().cpu()
    low, size = low_rank(c["x"], c["a"], c["b"], c["ids"], c["gate"], c["scale"])
    main, whole = (x @ w.t()).cuda(), (x.abs() @ w.abs().t()).cuda()
    agrees(got, main + low, whole + size, c["x"].shape[1] + c["a"].shape[1] * c["ids"].shape[1], size)


def check_dx(c, got):
    dy, w = c["dy"].double().cpu(), c["w"].double().cpu()
    low, size = low_rank(c["dy"], c["b"].transpose(1, 2), c["a"].transpose(1, 2), c["ids"], c["gate"], c["scale"])
    main, whole = (dy @ w).cuda(), (dy.abs() @ w.abs()).cuda()
    agrees(got, main + low, whole + size, c["dy"].shape[1] + c["a"].shape[1] * c["ids"].shape[1], size)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("sizes", SIZES)
def test_a_bad_adapter_stays_with_its_tokens(sizes, dtype):
    """Infinities and NaN in the B (and, for dx, the A) of an adapter in use: other tokens' rows are bit for bit what
    they are without them."""
    c = case(*sizes, dtype)
    clean = passes(c)
    e = 1
    mine = (c["ids"] == e).any(1)
    assert mine.any() and not mine.all()
    bad = dict(c, b=c["b"].clone())
    bad["b"][e, 3, 0], bad["b"][e, 10, -1], bad["b"][e, 11, 1], bad["b"][e, -1, 2] = INF, NAN, -INF, INF
    y, served, _ = passes(bad)
    for got, was in ((y, clean[0]), (served, clean[1])):
        assert torch.equal(got[~mine], was[~mine])
        check_forward(bad, got)
    bad = dict(c, a=c["a"].clone())
    bad["a"][e, 0, 5], bad["a"][e, -1, 8], bad["a"][e, 1, -1] = INF, NAN, -INF
    dx = passes(bad)[2]
    assert torch.equal(dx[~mine], clean[2][~mine])
    check_dx(bad, dx)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("sizes", SIZES)
def test_infinite_coefficients(sizes, dtype):
    """An infinite, or no, number in a token, in its weights or in what A makes of it: infinities where the definition has them."""
    c = case(*sizes, dtype)
    clean = passes(c)
    t = len(c["x"])
    touched = torch.zeros(t, dtype=torch.bool, device="cuda")
    bad = dict(c, gate=c["gate"].clone(), x=c["x"].clone(), dy=c["dy"].clone())
    for i, (what, value) in enumerate((("gate", INF), ("gate", -INF), ("gate", NAN), ("x", INF), ("x", NAN), ("dy", -INF), ("dy", NAN))):
        bad[what][3 * i + 1, 0] = value
        touched[3 * i + 1] = True
    for got, was, check in zip(passes(bad), clean, (check_forward, check_forward, check_dx)):
        assert torch.equal(got[~touched], was[~touched])
        check(bad, got)
    bad = dict(c, a=c["a"].clone())  # every token of one adapter has an infinite rank
    bad["a"][1, 0, 5] = INF
    for got in passes(bad)[:2]:
        check_forward(bad, got)
    bad = dict(c, b=c["b"].clone())
    bad["b"][1, 3, 0] = -INF
    check_dx(bad, passes(bad)[2])


@pytest.mark.parametrize("sizes", SIZES)
def test_coefficients_near_the_largest_float(sizes):
    """Products of weight and coefficient at and beyond float's range, brought back by a small factor."""
    c = case(*sizes, "bf16")
    c["a"], c["b"] = c["a"] * 0.125, c["b"] * 0.125
    c["gate"][::7] = 3e38
    c["gate"][1::7] = -1.5e38
    c["scale"][:] = 1
    y, served, dx = passes(c)
    check_forward(c, y)
    check_forward(c, served)
    check_dx(c, dx)


def adapter_gradients(c):
    """(da, db) in 64 bits, and their magnitudes, from each adapter's own tokens."""
    x, dy, gate = c["x"].cpu().double(), c["dy"].cpu().double(), c["gate"].cpu().double()
    a, b, ids = c["a"].cpu().double(), c["b"].cpu().double(), c["ids"].cpu()
    out = [torch.zeros_like(a), torch.zeros_like(b), torch.zeros_like(a), torch.zeros_like(b)]
    for e in range(a.shape[0]):
        for j in range(ids.shape[1]):
            rows = torch.nonzero(ids[:, j] == e)[:, 0]
            if len(rows):
                cf = gate[rows, j][:, None] * float(c["scale"][e])
                cv, cu = cf * (dy[rows] @ b[e]), cf * (x[rows] @ a[e].t())
                out[0][e] += cv.t() @ x[rows]
                out[1][e] += dy[rows].t() @ cu
                out[2][e] += (cf.abs() * (dy[rows].abs() @ b[e].abs())).t() @ x[rows].abs()
                out[3][e] += dy[rows].abs().t() @ (cf.abs() * (x[rows].abs() @ a[e].abs().t()))
    return [v.cuda() for v in out]


def gradients(c):
    a, b = c["a"].clone().requires_grad_(), c["b"].clone().requires_grad_()
    y = mixture.lora_linear(c["x"], c["w"], a, b, c["ids"], weights=c["gate"], scale=c["scale"])
    return torch.autograd.grad(y, (a, b), c["dy"])


def check_gradients(c, da, db):
    ra, rb, sa, sb = adapter_gradients(c)
    t, k = c["ids"].shape
    agrees(da, ra, sa, c["dy"].shape[1] + t * k, sa)
    agrees(db, rb, sb, c["x"].shape[1] + t * k, sb)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("sizes", SIZES + [(900, 3, 1, 72, 264, 100)])
def test_gradients_of_bad_tokens_and_adapters(sizes, dtype):
    """Infinities in a token, its gradient, its weight or an adapter show in the gradients of the adapters concerned, as
    infinities where the definition has them; the others' are bit for bit what they are without them."""
    c = case(*sizes, dtype)
    clean = gradients(c)
    for what, at, value in (("x", (5, 3), INF), ("dy", (6, 2), -INF), ("x", (9, 0), NAN), ("gate", (11, 0), INF), ("a", (1, 0, 4), INF),
                            ("b", (1, 7, 0), -INF), ("dy", (13, 1), NAN)):
        bad = dict(c, **{what: c[what].clone()})
        bad[what][at] = value
        if what == "gate":
            c["ids"][11, 0] = bad["ids"][11, 0] = 1
            clean = gradients(c)
        touched = {at[0]} if what in ("a", "b") else set(c["ids"][at[0]].tolist())
        da, db = gradients(bad)
        for e in range(len(c["a"])):
            if e not in touched:
                assert torch.equal(da[e], clean[0][e]) and torch.equal(db[e], clean[1][e])
        check_gradients(bad, da, db)


def test_gradients_of_coefficients_near_the_largest_float():
    """A scaled coefficient between bf16's largest value and float's makes a finite gradient."""
    c = case(600, 2, 1, 72, 88, 16, "bf16")
    c["ids"][:] = 0
    c["ids"][::3] = 1
    c["x"][:], c["dy"][:], c["gate"][:], c["scale"][0] = 0, 2.0 ** -10, 1, 1.999
    c["a"][0, 3, :], c["b"][0] = 0, 0
    c["x"][1, 7], c["a"][0, 3, 7] = 1, 2.0 ** 127
    da, db = gradients(c)
    assert float(db[0, :, 3].abs().min()) > 1e35
    check_gradients(c, da, db)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_bad_values_in_unaligned_operands(dtype):
    """The same in the kernels for operands and gradients that do not start on 16 bytes."""
    c = case(32, 5, 3, 200, 33000, 12, dtype)
    shift = lambda v: torch.cat([v.new_zeros(1), v.flatten()])[1:].view(v.shape)  # noqa: E731
    c["x"] = shift(c["x"])
    c["b"][1, 3, 0], c["b"][1, -1, 2], c["gate"][4, 0], c["x"][9, 0] = INF, NAN, -INF, INF
    with torch.no_grad():
        check_forward(c, mixture.lora_linear(c["x"], c["w"], c["a"], c["b"], c["ids"], weights=c["gate"], scale=c["scale"]))
    c = case(700, 5, 2, 136, 264, 20, dtype)
    c["dy"] = shift(c["dy"])
    c["a"][1, 0, 5], c["a"][1, -1, 8], c["gate"][4, 0], c["dy"][9, 0] = INF, NAN, -INF, INF
    assert c["dy"].data_ptr() % 16 != 0
    check_dx(c, passes(c)[2])
    c["a"] = c["a"].nan_to_num(0.5, 0.5, 0.5)
    check_gradients(c, *gradients(c))


@pytest.mark.parametrize("t", [40, 2100])
def test_bad_values_of_slots_without_an_expert(t):
    """Weights, gradients and rows of slots that have no expert are never read into anything."""
    c = case(t, 5, 2, 72, 560, 16, "bf16")
    none = c["ids"] < 0
    assert none.any()
    clean = [*passes(c), *gradients(c)]
    bad = dict(c, gate=torch.where(none, torch.full_like(c["gate"], NAN), c["gate"]))
    assert all(torch.equal(p, q) for p, q in zip([*passes(bad), *gradients(bad)], clean))
    w = normal(gen(1), 5, 136, 72, dtype=torch.bfloat16).requires_grad_()
    x = c["x"].clone()
    x[none.all(1)] = NAN
    groups = mixture.group(c["ids"], 5)
    dy = normal(gen(2), t, 2, 136, dtype=torch.bfloat16)
    results = []
    for xs, d in ((c["x"], dy), (x, torch.where(none[..., None], torch.full_like(dy, INF), dy))):
        xs = xs.clone().requires_grad_()
        y = mixture.grouped_matmul(xs, w, groups)
        results.append([y.detach(), *torch.autograd.grad(y, (xs, w), d)])
    assert all(torch.equal(p, q) for p, q in zip(*results))
    logits = normal(gen(3), t, 5).requires_grad_()
    mask = torch.rand(t, 5, generator=gen(4), device="cuda") < 0.4
    for normalize in (True, False):
        r = mixture.route(logits, 3, mask=mask, normalize=normalize)
        dw = normal(gen(5), t, 3)
        want, = torch.autograd.grad(r.weights, logits, dw, retain_graph=True)
        got, = torch.autograd.grad(r.weights, logits, torch.where(r.experts < 0, torch.full_like(dw, NAN), dw))
        assert torch.equal(got, want) and (r.experts < 0).any()
