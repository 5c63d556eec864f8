"""4-bit weights and the products with them, against their definitions in 64 bits.

A 4-bit weight is defined to the bit: scale * (code - zero), rounded to the
scales' type; quantizing too, since no value lies so near a tie that float's
rounding of the quotient could move it. The products' tolerances are those of
test_gpu_mixture.py, on the values that dequantize4 gives.
"""
import numpy as np
import pytest
import torch

from test_gpu_mixture import TYPES, choices, gen, grouped_oracle, lora_oracle, near, normal

pytestmark = pytest.mark.gpu

mixture = pytest.importorskip("provenloop_amd.mixture")


def checkpoint(g, shape, size, dtype, zeros, std=0.1):
    groups = -(-shape[-1] // size)
    codes = torch.randint(0, 16, shape, generator=g, device="cuda", dtype=torch.uint8)
    scales = normal(g, *shape[:-1], groups, dtype=dtype, std=std)  # of both signs
    z = torch.randint(0, 16, scales.shape, generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    return codes, scales, z


def values(codes, scales, zeros, size):
    """On the host in 64 bits, rounded once (torch rounds to nearest even)."""
    at = np.arange(codes.shape[-1]) // size
    c, s = codes.cpu().double(), scales.cpu().double()[..., at]
    z = 8.0 if zeros is None else zeros.cpu().double()[..., at]
    return (s * (c - z)).to(scales.dtype)


def same(got, want):
    """Equal bit for bit, signs of zeros aside, with NaN where want has them."""
    got, want = got.cpu(), want.cpu()
    assert got.shape == want.shape and got.dtype == want.dtype
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    assert torch.equal(got.masked_fill(nan, 0).float(), want.masked_fill(nan, 0).float())


SHAPES = [((1, 1), 32), ((16, 64), 32), ((17, 65), 64), ((3, 200), 128), ((256, 1536), 64), ((129, 31), 32), ((40, 96), 1 << 30),
          ((2, 48, 160), 32), ((3, 15, 127), 64), ((5, 33, 513), 128), ((1, 512, 3584), 256), ((4, 16, 4096), 4096)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("shape,size", SHAPES)
def test_pack_and_values(dtype, zeros, shape, size):
    g = gen(shape[-1])
    codes, scales, z = checkpoint(g, shape, size, TYPES[dtype], zeros)
    w = mixture.pack4(codes, scales, size, zeros=z)
    assert w.shape == shape and w.dtype == TYPES[dtype] and w.group_size == size and w.zeros == zeros
    same(mixture.dequantize4(w), values(codes, scales, z, size))
    # the high bits of codes and zeros are not read
    same(mixture.dequantize4(mixture.pack4(codes | 0xf0, scales, size, zeros=None if z is None else z | 0xa0)),
         values(codes, scales, z, size))


def test_pack_strides():
    g = gen(2)
    big = torch.randint(0, 16, (3, 50, 300), generator=g, device="cuda", dtype=torch.uint8)
    _, scales, _ = checkpoint(g, (3, 50, 130), 64, torch.bfloat16, False)
    for codes in (big[:, :, :130], big[:, :, 3:133], big[:, :, 1:].transpose(1, 2)[:, :130].transpose(1, 2), big[:1, :, :130].expand(3, 50, 130)):
        same(mixture.dequantize4(mixture.pack4(codes, scales, 64)), values(codes, scales, None, 64))
    turned = scales.transpose(0, 1).contiguous().transpose(0, 1)
    same(mixture.dequantize4(mixture.pack4(big[:, :, :130], turned, 64)), values(big[:, :, :130], scales, None, 64))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_scales_at_the_ends_of_the_range(dtype):
    """Subnormal, largest and bad scales: what the products cannot use makes its own group NaN and no other."""
    dt = TYPES[dtype]
    top = 2.0 ** 120 if dtype == "bf16" else 65504.0
    tiny = float(torch.finfo(dt).smallest_normal) / 4
    bad = [float("inf"), -float("inf"), float("nan")] + ([3e38, -2.0 ** 121] if dtype == "bf16" else [])
    fine = [top, -top, tiny, -tiny, 0.0, float(torch.finfo(dt).smallest_normal)]
    scales = torch.tensor([fine + bad], dtype=dt, device="cuda")
    n = scales.shape[1]
    codes = torch.arange(16, dtype=torch.uint8, device="cuda").repeat(1, 2 * n)
    for zeros in (None, torch.full((1, n), 15, dtype=torch.uint8, device="cuda")):
        want = values(codes, scales, zeros, 32)
        want[:, 32 * len(fine):] = float("nan")
        same(mixture.dequantize4(mixture.pack4(codes, scales, 32, zeros=zeros)), want)


def quantized(w, size, zeros):
    """The definition on the host, scale and codes in 64 bits."""
    w = w.cpu()
    v = torch.nn.functional.pad(w.double(), (0, -w.shape[-1] % size)).unflatten(-1, (-1, size))
    low, high = v.amin(-1, keepdim=True).clamp(max=0), v.amax(-1, keepdim=True).clamp(min=0)
    s = ((high - low) / 15 if zeros else torch.maximum(high, -low) / 7).to(w.dtype).double()
    by = torch.where(s > 0, s, torch.ones_like(s))
    if zeros:
        z = torch.round(-low / by).clamp(0, 15)
        q = torch.round(v / by) + z
        q = q.clamp(0, 15) - z
    else:
        q = torch.round(v / by).clamp(-7, 7)
    out = (s * q).to(w.dtype)
    bad = ~torch.isfinite(v).all(-1, keepdim=True) | ~torch.isfinite(s)
    out = torch.where(bad, torch.full_like(out, float("nan")), out)
    return out.flatten(-2)[..., :w.shape[-1]]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("shape,size", SHAPES)
def test_quantize(dtype, zeros, shape, size):
    g = gen(shape[-1] + 1)
    size = min(size, 8192)
    w = normal(g, *shape, dtype=TYPES[dtype], std=0.02)
    same(mixture.dequantize4(mixture.quantize4(w, size, zeros=zeros)), quantized(w, size, zeros))
    # few different values: many of them are on a tie
    w = (torch.randint(-7, 8, shape, generator=g, device="cuda") / 2).to(TYPES[dtype])
    same(mixture.dequantize4(mixture.quantize4(w, size, zeros=zeros)), quantized(w, size, zeros))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("zeros", [False, True])
def test_quantize_extremes(dtype, zeros):
    dt = TYPES[dtype]
    info = torch.finfo(dt)
    w = torch.zeros(12, 96, dtype=dt)
    w[0] = 0.5
    w[1] = -3.0
    w[2, ::2], w[2, 1::2] = 1.0, -1.0
    w[3, 40] = float("nan")
    w[4, 70] = float("inf")
    w[5, 3] = -float("inf")
    w[6] = info.tiny
    w[7, :32] = info.smallest_normal / 8
    w[8, 64:] = -float(info.max) if dtype == "f16" else -2.0 ** 120
    w[9, 5] = -0.0
    w[10, 0], w[10, 31] = 15.0, -1e-4
    w[11, :] = torch.linspace(-1, 7, 96).to(dt)
    same(mixture.dequantize4(mixture.quantize4(w.cuda(), 32, zeros=zeros)), quantized(w, 32, zeros))


def test_quantize_strides():
    g = gen(4)
    big = normal(g, 3, 40, 300, dtype=torch.bfloat16)
    for w in (big[:, :, :130], big[:, :, 1:131], big.transpose(1, 2)[:, :200], big[:1].expand(3, 40, 300), big[1, 3:20, 7:9]):
        for size in (32, 128, 256):
            same(mixture.dequantize4(mixture.quantize4(w, size)), quantized(w, size, False))


# ---------------------------------------------------------------- grouped products
GROUPED4 = [(1, 1, 1, 8, 8, 32), (1, 5, 2, 64, 16, 64), (3, 4, 1, 72, 200, 32), (17, 3, 2, 1536, 256, 128), (64, 8, 1, 128, 129, 64),
            (130, 6, 3, 100, 70, 64), (129, 2, 2, 33, 65, 32), (500, 16, 2, 264, 136, 128), (1000, 3, 1, 513, 40, 64),
            (300, 40, 4, 64, 1, 1024), (40, 2, 1, 1, 24, 32), (2000, 7, 2, 320, 384, 32), (16, 4, 2, 3584, 512, 128),
            (5000, 2, 1, 192, 272, 64), (40, 3, 1, 1290, 1030, 256), (700, 2, 2, 1536, 300, 64)]


@pytest.mark.parametrize("dtype,zeros", [("bf16", False), ("bf16", True), ("f16", False), ("f16", True)])
@pytest.mark.parametrize("per_slot", [False, True])
@pytest.mark.parametrize("t,e,k,din,dout,size", GROUPED4)
def test_grouped_matmul(dtype, zeros, per_slot, t, e, k, din, dout, size):
    g = gen(din + dout)
    ids = choices(g, t, e, k)
    w4 = mixture.pack4(*checkpoint(g, (e, dout, din), size, TYPES[dtype], zeros)[:2], size) if not zeros else None
    if zeros:
        codes, scales, z = checkpoint(g, (e, dout, din), size, TYPES[dtype], True)
        w4 = mixture.pack4(codes, scales, size, zeros=z)
    w = mixture.dequantize4(w4)
    x = normal(g, *((t, k, din) if per_slot else (t, din)), dtype=TYPES[dtype]).requires_grad_()
    dy = normal(g, t, k, dout, dtype=TYPES[dtype])
    groups = mixture.group(ids, e)
    y = mixture.grouped_matmul(x, w4, groups)
    dx, = torch.autograd.grad(y, x, dy)
    (ry, rdx, _), (my, mdx, _) = grouped_oracle(x.detach(), w, ids, k, dy)
    near(y.detach(), ry, my, din)
    near(dx, rdx, mdx, dout * k)
    assert (y[ids < 0] == 0).all()
    with torch.no_grad():
        near(mixture.grouped_matmul(x, w4, groups), ry, my, din)


@pytest.mark.parametrize("t", [20, 1500])
def test_grouped_strides_and_alignment(t):
    g = gen(11)
    e, k, din, dout = 4, 2, 96, 80
    ids = choices(g, t, e, k)
    w4 = mixture.pack4(*checkpoint(g, (e, dout, din), 32, torch.bfloat16, False)[:2], 32)
    w = mixture.dequantize4(w4)
    big = normal(g, t, 200, dtype=torch.bfloat16)
    dbig = normal(g, t, k, 200, dtype=torch.bfloat16)
    for x in (big[:, :din], big[:, 3:3 + din], big.t()[:din].t(), big[:1, :din].expand(t, din)):
        for dy in (dbig[:, :, :dout], dbig[:, :, 5:5 + dout], dbig[:1, :1, :1].expand(t, k, dout)):
            xr = x.detach().requires_grad_()
            y = mixture.grouped_matmul(xr, w4, mixture.group(ids, e))
            (ry, rdx, _), (my, mdx, _) = grouped_oracle(x, w, ids, k, dy)
            near(y.detach(), ry, my, din)
            near(torch.autograd.grad(y, xr, dy)[0], rdx, mdx, dout * k)


@pytest.mark.parametrize("cols,size", [(33, 32), (40, 32), (40, 64), (130, 128)])
@pytest.mark.parametrize("t", [1, 40])
def test_columns_behind_the_last_have_no_value(t, cols, size):
    """Scales at which a code that stands in their place would be an infinity, which times x's zeros is NaN."""
    g = gen(cols + t)
    codes = torch.randint(0, 6, (2, 24, cols), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.full((2, 24, -(-cols // size)), 12288.0, dtype=torch.float16, device="cuda")
    z = torch.zeros(scales.shape, dtype=torch.uint8, device="cuda")
    x = normal(g, t, cols, dtype=torch.float16, std=2.0 ** -10)
    v = values(codes, scales, z, size).double()
    w = mixture.pack4(codes, scales, size, zeros=z)
    groups = mixture.group(torch.zeros(t, 1, dtype=torch.int32, device="cuda"), 2)
    w1 = mixture.pack4(codes[0], scales[0], size, zeros=z[0])
    none = torch.full((t,), -1, dtype=torch.int32, device="cuda")
    a, b = normal(g, 1, 8, cols, dtype=torch.float16), normal(g, 1, 24, 8, dtype=torch.float16)
    want = x.cpu().double() @ v[0].T
    # products of two f16 are exact in float; cols - 1 additions of them and one rounding to f16
    bound = want.abs() * 2.0 ** -11 + (cols * 2.0 ** -23) * (x.cpu().double().abs() @ v[0].abs().T)
    for y in (mixture.grouped_matmul(x, w, groups)[:, 0], mixture.lora_linear(x, w1, a, b, none)):
        assert bool(((y.cpu().double() - want).abs() <= bound).all())


@pytest.mark.parametrize("t", [20, 2500])
def test_bad_values_stay_where_they_are(t):
    """A NaN scale shows in its row of its expert alone; a token's infinity in its own outputs, with the sign of its weight."""
    g = gen(6)
    codes, scales, _ = checkpoint(g, (4, 64, 128), 32, torch.bfloat16, False)
    codes[0, 5, 3], codes[0, 6, 3] = 15, 1
    scales = scales.abs()
    scales[3] = float("nan")
    scales[1, 9, 2] = float("inf")
    w4 = mixture.pack4(codes, scales, 32)
    x = normal(g, t, 128, dtype=torch.bfloat16)
    ids = torch.randint(0, 3, (t, 1), generator=g, device="cuda", dtype=torch.int32)
    ids[7], ids[11] = 0, 0
    x[7], x[11, 3] = float("nan"), float("inf")
    y = mixture.grouped_matmul(x, w4, mixture.group(ids, 4))[:, 0]
    fine = torch.ones(t, dtype=torch.bool, device="cuda")
    fine[7] = fine[11] = False
    ok = torch.isfinite(y) | ((ids == 1) & (torch.arange(64, device="cuda") == 9))
    assert ok[fine].all() and torch.isnan(y[7]).all()
    assert torch.isnan(y[fine & (ids[:, 0] == 1), 9]).all()
    assert y[11, 5] == float("inf") and y[11, 6] == -float("inf")
    want = torch.sign(codes[0, :, 3].double() - 8) * float("inf")
    assert torch.equal(y[11].double().nan_to_num(nan=7), want.nan_to_num(nan=7))


# ---------------------------------------------------------------- shared projection with adapters
LORA4 = [(1, 1, 1, 64, 64, 1, 32), (1, 4, 1, 1536, 256, 16, 64), (2, 3, 2, 72, 100, 8, 32), (7, 16, 1, 128, 72, 32, 64),
         (33, 5, 3, 65, 33, 5, 32), (64, 64, 1, 256, 128, 64, 128), (65, 3, 2, 96, 264, 128, 32), (130, 2, 1, 48, 40, 17, 64),
         (300, 100, 1, 128, 192, 16, 128), (700, 8, 2, 264, 136, 16, 64), (1030, 3, 2, 200, 129, 20, 32),
         (2500, 6, 4, 136, 72, 40, 1024), (600, 300, 2, 64, 72, 4, 64), (1200, 4, 2, 1100, 1290, 16, 128)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("t,e,k,din,dout,rank,size", LORA4)
def test_lora_linear(dtype, t, e, k, din, dout, rank, size):
    g = gen(t + din)
    dt = TYPES[dtype]
    codes, scales, z = checkpoint(g, (dout, din), size, dt, t % 2 == 0, std=din ** -0.5 / 5)
    w4 = mixture.pack4(codes, scales, size, zeros=z)
    w = mixture.dequantize4(w4)
    x = normal(g, t, din, dtype=dt).requires_grad_()
    a = normal(g, e, rank, din, dtype=dt, std=din ** -0.5).requires_grad_()
    b = normal(g, e, dout, rank, dtype=dt, std=0.3).requires_grad_()
    ids = choices(g, t, e, k)
    gate = torch.rand(t, k, generator=g, device="cuda").requires_grad_()
    scale = torch.rand(e, generator=g, device="cuda") * 2
    bias = normal(g, dout, dtype=dt)
    dy = normal(g, t, dout, dtype=dt)
    y = mixture.lora_linear(x, w4, a, b, ids, weights=gate, scale=scale, bias=bias)
    dx, da, db, dg = torch.autograd.grad(y, (x, a, b, gate), dy)
    ref, mag = lora_oracle(x.detach(), w, a.detach(), b.detach(), ids, gate.detach(), scale, bias, dy)
    n = din + rank * k
    near(y.detach(), ref["y"], mag["y"], n, mag["low"])
    near(dx, ref["dx"], mag["dx"], dout + rank * k, mag["dxl"])
    near(da, ref["da"], mag["da"], dout + t * k, mag["da"])
    near(db, ref["db"], mag["db"], din + t * k, mag["db"])
    near(dg, ref["dg"], mag["dg"], din + dout + rank)
    with torch.no_grad():
        near(mixture.lora_linear(x, w4, a, b, ids, weights=gate, scale=scale, bias=bias), ref["y"], mag["y"], n, mag["low"])
        plain, pmag = lora_oracle(x, w, a, b, ids, None, None, None)
        near(mixture.lora_linear(x, w4, a, b, ids if k > 1 else ids[:, 0]), plain["y"], pmag["y"], n, pmag["low"])


@pytest.mark.parametrize("t", [9, 300, 1500])
def test_lora_strides(t):
    g = gen(9)
    big = normal(g, t, 300, dtype=torch.float16)
    codes, scales, z = checkpoint(g, (88, 96), 64, torch.float16, True)
    w4 = mixture.pack4(codes, scales, 64, zeros=z)
    w = mixture.dequantize4(w4)
    a = normal(g, 4, 16, 160, dtype=torch.float16, std=0.1)[:, :, 1:97]
    b = normal(g, 4, 88, 40, dtype=torch.float16, std=0.3)[:, :, 3:19]
    ids = torch.randint(-1, 4, (t, 1), generator=g, device="cuda", dtype=torch.int32)
    for x in (big[:, :96], big[:, 5:101], big[:1, :96].expand(t, 96), big.t()[:96].t()):
        ref, mag = lora_oracle(x, w, a, b, ids, None, None, None)
        near(mixture.lora_linear(x, w4, a, b, ids), ref["y"], mag["y"], 96 + 16, mag["low"])


def test_gradients_against_differences():
    """dx of a scalar function against its differences, each evaluated in 64 bits on the values of the weights."""
    g = gen(21)
    codes, scales, z = checkpoint(g, (24, 40), 32, torch.float16, True)
    w4 = mixture.pack4(codes, scales, 32, zeros=z)
    w = mixture.dequantize4(w4).double()
    a, b = normal(g, 2, 4, 40, dtype=torch.float16, std=0.2), normal(g, 2, 24, 4, dtype=torch.float16, std=0.2)
    ids = torch.tensor([[0], [1], [-1]], dtype=torch.int32, device="cuda")
    x = normal(g, 3, 40, dtype=torch.float16).requires_grad_()
    dy = normal(g, 3, 24, dtype=torch.float16)
    dx, = torch.autograd.grad(mixture.lora_linear(x, w4, a, b, ids), x, dy)

    def f(v):
        low = torch.stack([(v[i] @ a[e].double().t()) @ b[e].double().t() if e >= 0 else torch.zeros(24, device="cuda", dtype=torch.float64)
                           for i, e in enumerate(ids[:, 0].tolist())])
        return ((v @ w.t() + low) * dy.double()).sum()

    for i, j in ((0, 0), (1, 17), (2, 39), (0, 31)):
        up, down = x.detach().double().clone(), x.detach().double().clone()
        up[i, j] += 2.0 ** -10
        down[i, j] -= 2.0 ** -10
        slope = (f(up) - f(down)) / 2.0 ** -9
        assert abs(float(slope) - float(dx[i, j])) <= 2.0 ** -11 * abs(float(slope)) + 2.0 ** -12


def test_streams_graphs_and_runs():
    """On another stream, again, and captured with a router and 4-bit experts: bit for bit the eager results."""
    g = gen(13)
    x = normal(g, 600, 128, dtype=torch.bfloat16)
    w4 = mixture.quantize4(normal(g, 96, 128, dtype=torch.bfloat16), 32)
    e4 = mixture.quantize4(normal(g, 5, 96, 128, dtype=torch.bfloat16), 64, zeros=True)
    a, b = normal(g, 5, 16, 128, dtype=torch.bfloat16), normal(g, 5, 96, 16, dtype=torch.bfloat16)
    logits = normal(g, 600, 5)
    dy = normal(g, 600, 96, dtype=torch.bfloat16)

    def step(x, a, b, logits):
        r = mixture.route(logits, 2)
        y = mixture.lora_linear(x, w4, a, b, r.experts, weights=r.weights)
        z = mixture.grouped_matmul(x, e4, r.groups)
        few = mixture.grouped_matmul(x[:4], e4, mixture.group(r.experts[:4], 5))
        both = (r.weights[..., None] * z.float()).sum(1)
        return [y.detach(), z.detach(), few.detach(), *torch.autograd.grad([y, both], (x, a, b, logits), [dy, dy.float()])]

    def leaves():
        return [v.clone().requires_grad_() for v in (x, a, b, logits)]

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
        g2 = gen(100 + i)
        with torch.no_grad():
            static[0].copy_(normal(g2, 600, 128, dtype=torch.bfloat16))
            static[3].copy_(normal(g2, 600, 5))
        graph.replay()
        torch.cuda.synchronize()
        eager = step(*[v.detach().clone().requires_grad_() for v in static])
        assert all(torch.equal(p, q) for p, q in zip(outs, eager)), i


def test_no_tokens_and_empty_groups():
    w4 = mixture.quantize4(torch.ones(3, 8, 16, dtype=torch.bfloat16, device="cuda"), 32)
    none = torch.empty(0, 2, dtype=torch.int32, device="cuda")
    x = torch.empty(0, 16, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    y = mixture.grouped_matmul(x, w4, mixture.group(none, 3))
    assert y.shape == (0, 2, 8) and torch.autograd.grad(y, x, torch.empty_like(y))[0].shape == x.shape
    a, b = torch.zeros(3, 4, 16, dtype=torch.bfloat16, device="cuda"), torch.zeros(3, 8, 4, dtype=torch.bfloat16, device="cuda")
    one = w4._replace(data=mixture.quantize4(torch.ones(8, 16, dtype=torch.bfloat16, device="cuda"), 32).data, shape=(8, 16))
    assert mixture.lora_linear(x, one, a, b, none).shape == (0, 8)
    for t in (3, 2000):
        ids = torch.full((t, 1), -1, dtype=torch.int32, device="cuda")
        x = torch.full((t, 16), float("nan"), dtype=torch.bfloat16, device="cuda", requires_grad=True)
        y = mixture.grouped_matmul(x, w4, mixture.group(ids, 3))
        assert (y == 0).all() and (torch.autograd.grad(y, x, torch.ones_like(y))[0] == 0).all()


def test_codes_beyond_32_bits():
    """Experts whose codes lie more than 2^32 bytes into the data."""
    g = gen(14)
    e, dout, din = 4200, 1024, 2048  # 4.4 GB of codes
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of GPU memory")
    one = checkpoint(g, (1, dout, din), 128, torch.bfloat16, False)[:2]
    with pytest.raises(ValueError, match="experts"):
        w4 = mixture.pack4(one[0].expand(e, dout, din), one[1].expand(e, dout, din // 128), 128)
        mixture.grouped_matmul(torch.zeros(1, din, dtype=torch.bfloat16, device="cuda"), w4, mixture.Groups(
            torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"),
            torch.zeros(e + 1, dtype=torch.int32, device="cuda"), e))
    del w4
    e, dout, din = 1024, 4096, 2176
    codes, scales, _ = checkpoint(g, (1, dout, din), 128, torch.bfloat16, False)
    w4 = mixture.pack4(codes.expand(e, dout, din), scales.expand(e, dout, din // 128), 128)
    assert w4.data.numel() > 1 << 32
    x = normal(g, 3, din, dtype=torch.bfloat16)
    ids = torch.tensor([[1023], [0], [1000]], dtype=torch.int32, device="cuda")
    w = values(codes, scales, None, 128)[0].cuda()
    y = mixture.grouped_matmul(x, w4, mixture.group(ids, e))[:, 0]
    near(y, x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t(), din)
