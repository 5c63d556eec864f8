"""Gates with balanced choices and 4-bit weights, beside the operators of
perf/operators.py, as measurable cases.

Every case is a dict of plain values; `kind` names the operator:

  gate      a gate of T tokens over E experts whose scores are a softmax or
            sigmoids, the choice made by score + bias within the best nodes of
            experts; weights, choices and the slots grouped by expert;
  quantize  frozen weights to 4 bits with a scale (and a zero) per group of
            columns, and the values that these stand for;
  grouped4  matrix products grouped by expert with 4-bit experts;
  lora4     a shared 4-bit projection with the low-rank adapters of many
            requests (or a gated mixture of them) added in the same pass.

A 4-bit weight is the value scale * (code - zero) rounded to the type of the
scales, which is x's. `train` cases return the gradients beside the outputs (the
4-bit weights are frozen and have none). Widths are those of bench.py and tests/
(hidden 1536 with q and v of 1536 and 256 outputs and rank 16; hidden 3584 with
512 outputs and rank 32; 32 sessions), or generic ones.

Where `own` is false, `run` computes the operators from elementary torch
operations in 32 bits (the scores that decide a choice in 64), rounded once at
the end; where it is true, through provenloop_amd.mixture.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# what the largest listed cases cost: lora4_prefill's operations, quantize_experts' bytes
FLOPS_MAX = 2 * 8192 * 3584 * 3584 + 2 * 8192 * 32 * (3584 + 3584)
WEIGHTS_MAX = 8 * 1536 * 3584


def listed():
    return [
        # One decoded token through a gate of sigmoid scores with a bias for
        # balance: pure latency.
        dict(name="gate_token", kind="gate", dtype="f32", t=1, e=64, k=6, score="sigmoid", bias=True, nodes=1,
             top_nodes=1, node_best=1, masked=False, normalize=True, scale=1.0, train=False),
        # A large prefill batch over 256 experts on 8 nodes, of which a token
        # may use the 4 whose two best experts are the best.
        dict(name="gate_prefill", kind="gate", dtype="bf16", t=65536, e=256, k=8, score="sigmoid", bias=True, nodes=8,
             top_nodes=4, node_best=2, masked=False, normalize=True, scale=2.5, train=False),
        # A training step's gate: odd sizes, softmax scores, experts withheld
        # from some tokens, and the logits' gradient.
        dict(name="gate_train", kind="gate", dtype="f32", t=4099, e=60, k=5, score="softmax", bias=True, nodes=5,
             top_nodes=2, node_best=1, masked=True, normalize=False, scale=1.0, train=True),
        # The v projection of a small model to 4 bits, with zeros.
        dict(name="quantize_v", kind="quantize", dtype="bf16", e=1, din=1536, dout=256, size=64, zeros=True),
        # 8 experts to 4 bits when a model is loaded.
        dict(name="quantize_experts", kind="quantize", dtype="f16", e=8, din=1536, dout=3584, size=128, zeros=False),
        # Experts' products while 16 sessions decode: few rows per expert, the
        # weights are what has to be read.
        dict(name="grouped4_decode", kind="grouped4", dtype="f16", t=16, e=8, k=2, din=3584, dout=512, size=128,
             zeros=True, train=False),
        # The same for a prefill batch: large matrix products of ragged sizes.
        dict(name="grouped4_prefill", kind="grouped4", dtype="bf16", t=8192, e=8, k=2, din=1536, dout=3584, size=128,
             zeros=False, train=False),
        # A training step through 16 frozen experts: output and gradient of the
        # tokens.
        dict(name="grouped4_train", kind="grouped4", dtype="bf16", t=4093, e=16, k=2, din=1536, dout=1536, size=64,
             zeros=False, train=True),
        # One token of one session through its q projection and adapter.
        dict(name="lora4_token", kind="lora4", dtype="bf16", t=1, e=4, k=1, din=1536, dout=1536, rank=16, requests=1,
             gated=False, size=64, zeros=False, train=False),
        # 32 sessions decode together, each with an adapter of its own.
        dict(name="lora4_sessions", kind="lora4", dtype="bf16", t=32, e=32, k=1, din=3584, dout=3584, rank=32,
             requests=32, gated=False, size=128, zeros=False, train=False),
        # Prefill of 20 requests of ragged lengths, an adapter each or none:
        # the largest case.
        dict(name="lora4_prefill", kind="lora4", dtype="bf16", t=8192, e=8, k=1, din=3584, dout=3584, rank=32,
             requests=20, gated=False, size=128, zeros=True, train=False),
        # A training step of the adapters and their gate beside the frozen q
        # projection: gradients of the tokens, A, B and the gate weights.
        dict(name="lora4_train", kind="lora4", dtype="bf16", t=4096, e=8, k=2, din=1536, dout=1536, rank=16,
             requests=0, gated=True, size=64, zeros=False, train=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)) - 1e-9)))))


def _width(rng, lo, hi):
    """A feature width: mostly a multiple of 8, as models have them, any number otherwise."""
    n = _log_int(rng, lo, hi)
    return n if rng.random() < 0.25 else max(8, n // 8 * 8)


def draw(rng):
    kind = rng.choice(["gate", "gate", "quantize", "grouped4", "grouped4", "lora4", "lora4"])
    train = rng.random() < 0.35
    if kind == "gate":
        per = _log_int(rng, 1, 64)
        nodes = rng.randint(1, min(8, 256 // per))
        if per * nodes < 2:
            nodes = 2
        top_nodes = rng.randint(1, nodes)
        return dict(kind=kind, dtype=rng.choice(["bf16", "f16", "f32"]), t=_log_int(rng, 1, 65536), e=per * nodes,
                    k=rng.randint(1, min(8, per * top_nodes)), score=rng.choice(["softmax", "sigmoid"]),
                    bias=rng.random() < 0.7, nodes=nodes, top_nodes=top_nodes, node_best=rng.randint(1, 2),
                    masked=rng.random() < 0.4, normalize=rng.random() < 0.6, scale=rng.choice([1.0, 2.5]), train=train)
    case = dict(kind=kind, dtype=rng.choice(["bf16", "f16"]), e=_log_int(rng, 1, 64), din=_width(rng, 64, 4096),
                dout=_width(rng, 64, 4096), size=rng.choice([32, 64, 128]), zeros=rng.random() < 0.5)
    if kind != "lora4":
        while case["e"] > 1 and case["e"] * case["din"] * case["dout"] > WEIGHTS_MAX:
            case["e"] = case["e"] * 3 // 4
    if kind == "quantize":
        return case
    case.update(t=_log_int(rng, 1, 8192), k=rng.randint(1, min(4, case["e"])), train=train)
    if kind == "lora4":
        gated = rng.random() < 0.5
        case.update(rank=_log_int(rng, 1, 64), gated=gated, requests=0)
        if not gated:
            case.update(k=1, requests=_log_int(rng, 1, case["t"]))
    while case["t"] > 1 and _cost(case) > FLOPS_MAX:
        case["t"] = case["t"] * 3 // 4
    return case


def _cost(case):
    """Operations of a pass; the plain form of `lora4` takes every adapter's columns."""
    f = work(case)["flops"]
    if case["kind"] == "lora4":
        f += 2 * case["t"] * case["e"] * case["rank"] * (case["din"] + case["dout"])
    return f


# ---------------------------------------------------------------- inputs
def _normal(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * std


def _choices(g, t, e, k):
    """k distinct experts a token, some experts favoured (ragged groups, possibly empty ones)."""
    score = _normal(g, t, e) + _normal(g, 1, e, std=1.0)
    return torch.sort(score, dim=1, descending=True, stable=True).indices[:, :k].to(torch.int32).contiguous()


def _four_bits(g, st, case, dt, shape):
    """Codes, scales and zeros of a weight as a checkpoint holds them: about normal values of 1 / sqrt(d_in)."""
    groups = -(-case["din"] // case["size"])
    st["codes"] = (_normal(g, *shape, std=2.6) + 8).round_().clamp_(0, 15).to(torch.uint8)
    spread = torch.rand(*shape[:-1], groups, generator=g, device="cuda") + 0.5
    st["scales"] = (spread * (case["din"] ** -0.5 / 2.6)).to(dt)
    st["zeros"] = None
    if case["zeros"]:
        st["zeros"] = torch.randint(6, 11, (*shape[:-1], groups), generator=g, device="cuda").to(torch.uint8)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    e = case["e"]
    st = dict(case=case)
    if case["kind"] == "quantize":
        shape = (case["dout"], case["din"]) if e == 1 else (e, case["dout"], case["din"])
        st["w"] = _normal(g, *shape, std=case["din"] ** -0.5).to(dt)
        return st
    t, k = case["t"], case["k"]
    if case["kind"] == "gate":
        st["logits"] = _normal(g, t, e, std=1.5).to(dt)
        # as balancing leaves it: a few steps of 0.001 up or down
        st["bias"] = (_normal(g, e, std=20).round_() * 0.001) if case["bias"] else None
        st["mask"] = None
        if case["masked"]:
            # sessions without some of the experts; one token in 50 without any
            allowed = torch.rand(t, e, generator=g, device="cuda") < 0.8
            st["mask"] = allowed & (torch.rand(t, 1, generator=g, device="cuda") >= 0.02)
        if case["train"]:
            st["dweights"] = _normal(g, t, k)
        leaves = ["logits"]
    elif case["kind"] == "grouped4":
        din, dout = case["din"], case["dout"]
        st["x"] = _normal(g, t, din).to(dt)
        _four_bits(g, st, case, dt, (e, dout, din))
        st["experts"] = _choices(g, t, e, k)
        if case["train"]:
            st["dy"] = _normal(g, t, k, dout).to(dt)
        leaves = ["x"]
    else:
        din, dout, r = case["din"], case["dout"], case["rank"]
        st["x"] = _normal(g, t, din).to(dt)
        _four_bits(g, st, case, dt, (dout, din))
        st["a"] = _normal(g, e, r, din, std=din ** -0.5).to(dt)
        st["b"] = _normal(g, e, dout, r, std=0.1).to(dt)
        st["scale"] = torch.full((e,), 2.0, device="cuda")
        if case["gated"]:
            st["experts"] = _choices(g, t, e, k)
            st["weights"] = torch.softmax(_normal(g, t, k, std=1.5), dim=1)
        else:
            # contiguous requests of ragged lengths, an adapter each; one in eight has none
            n = case["requests"]
            ends = torch.sort(torch.rand(n, generator=g, device="cuda")).values * t if n < t else \
                torch.arange(1, n + 1, device="cuda", dtype=torch.float32)
            of = torch.searchsorted(ends.contiguous(), torch.arange(t, device="cuda", dtype=torch.float32), right=True)
            ids = torch.randint(0, e, (n + 1,), generator=g, device="cuda")
            ids[torch.rand(n + 1, generator=g, device="cuda") < 0.125] = -1
            st["experts"] = ids[of].to(torch.int32).view(t, 1).contiguous()
            st["weights"] = None
        if case["train"]:
            st["dy"] = _normal(g, t, dout).to(dt)
        leaves = ["x", "a", "b"] + (["weights"] if case["gated"] else [])
    if case["train"]:
        for name in leaves:
            st[name].requires_grad_()
        st["leaves"] = leaves
    if own:
        from provenloop_amd import mixture

        if case["kind"] != "gate":  # the weights as a server lays them out once, when it loads them
            st["w4"] = mixture.pack4(st["codes"], st["scales"], case["size"], zeros=st["zeros"])
    return st


# ---------------------------------------------------------------- the framework's operators
def _run_own(st):
    from provenloop_amd import mixture

    case = st["case"]
    if case["kind"] == "gate":
        r = mixture.route(st["logits"], case["k"], mask=st["mask"], normalize=case["normalize"], score=case["score"],
                          bias=st["bias"], scale=case["scale"], nodes=case["nodes"], top_nodes=case["top_nodes"],
                          node_best=case["node_best"])
        out = [r.weights.detach(), r.experts, r.groups.order, r.groups.offsets]
        y, dy = r.weights, st.get("dweights")
    elif case["kind"] == "quantize":
        return [mixture.dequantize4(mixture.quantize4(st["w"], case["size"], zeros=case["zeros"]))]
    elif case["kind"] == "grouped4":
        groups = mixture.group(st["experts"], case["e"])
        y, dy = mixture.grouped_matmul(st["x"], st["w4"], groups), st.get("dy")
        out = [y.detach()]
    else:
        y = mixture.lora_linear(st["x"], st["w4"], st["a"], st["b"], st["experts"], weights=st["weights"],
                                scale=st["scale"])
        out, dy = [y.detach()], st.get("dy")
    if case["train"]:
        out += torch.autograd.grad(y, [st[n] for n in st["leaves"]], dy)
    return out


# ---------------------------------------------------------------- plain forms
def _plain_gate(st):
    case, l = st["case"], st["logits"].detach().double()
    t, e = l.shape
    k, nodes = case["k"], case["nodes"]
    allowed = l > -math.inf
    if st["mask"] is not None:
        allowed = allowed & st["mask"]
    masked = torch.where(allowed, l, torch.full_like(l, -math.inf))
    if case["score"] == "softmax":
        big = masked.amax(1, keepdim=True)
        p = torch.exp(masked - torch.where(big > -math.inf, big, torch.zeros_like(big)))
        total = p.sum(1, keepdim=True)
        score = p / torch.where(total > 0, total, torch.ones_like(total))
    else:
        score = torch.where(allowed, 1 / (1 + torch.exp(-l)), torch.zeros_like(l))
    rank = masked
    if st["bias"] is not None:
        rank = torch.where(allowed, score + st["bias"].double(), masked)
    elif nodes > 1 and case["node_best"] == 2:
        rank = torch.where(allowed, score, masked)
    if nodes > 1:
        best = torch.sort(rank.view(t, nodes, -1), dim=2, descending=True).values[:, :, :case["node_best"]]
        value = torch.where(best > -math.inf, best, torch.zeros_like(best)).sum(2)
        value = torch.where(best[:, :, 0] > -math.inf, value, torch.full_like(value, -math.inf))
        kept = torch.sort(value, dim=1, descending=True, stable=True).indices[:, :case["top_nodes"]]
        keep = torch.zeros(t, nodes, dtype=torch.bool, device=l.device).scatter_(1, kept, True)
        rank = torch.where(keep.repeat_interleave(e // nodes, dim=1), rank, torch.full_like(rank, -math.inf))
    top, index = torch.sort(rank, dim=1, descending=True, stable=True)
    top, index = top[:, :k], index[:, :k]
    chosen = top > -math.inf
    experts = torch.where(chosen, index, torch.full_like(index, -1)).to(torch.int32)
    s = torch.where(chosen, torch.gather(score, 1, index), torch.zeros_like(top))
    total = s.sum(1, keepdim=True) if case["normalize"] else torch.ones_like(s[:, :1])
    share = s / torch.where(total > 0, total, torch.ones_like(total))
    slots = experts.reshape(-1)
    key = torch.where(slots < 0, torch.full_like(slots, e), slots)
    order = torch.sort(key, stable=True).indices.to(torch.int32)
    counts = torch.zeros(e + 1, dtype=torch.int64, device=l.device).scatter_add_(
        0, key.long(), torch.ones_like(key, dtype=torch.int64))[:e]
    offsets = torch.cat([counts.new_zeros(1), torch.cumsum(counts, 0)]).to(torch.int32)
    out = [(share * case["scale"]).float(), experts, order, offsets]
    if case["train"]:
        dw = st["dweights"].double() * case["scale"]
        inner = (share * dw).sum(1, keepdim=True)
        # the share's gradient in the chosen logits; all logits move an unnormalized softmax
        if case["normalize"]:
            own_part = share * (dw - inner) * (1 if case["score"] == "softmax" else 1 - s)
        else:
            own_part = share * dw * (1 if case["score"] == "softmax" else 1 - s)
        grad = torch.zeros_like(l).scatter_add_(1, index, own_part)
        if case["score"] == "softmax" and not case["normalize"]:
            grad = grad - score * inner
        out.append(grad.to(st["logits"].dtype))
    return out


def _plain_quantize(st):
    """The largest value of a group of columns gives its scale; codes by rounding to even."""
    case, w = st["case"], st["w"]
    size, din = case["size"], case["din"]
    groups = -(-din // size)
    v = torch.zeros(*w.shape[:-1], groups * size, device=w.device)
    v[..., :din] = w.float()
    v = v.view(*w.shape[:-1], groups, size)
    if case["zeros"]:
        low, high = v.amin(-1, keepdim=True).clamp(max=0), v.amax(-1, keepdim=True).clamp(min=0)
        scale = ((high - low) / 15).to(w.dtype).float()
    else:
        scale = (v.abs().amax(-1, keepdim=True) / 7).to(w.dtype).float()
    by = torch.where(scale > 0, scale, torch.ones_like(scale))
    zero = torch.round(-low / by).clamp(0, 15) if case["zeros"] else torch.full_like(scale, 8)
    codes = (torch.round(v / by) + zero).clamp(0 if case["zeros"] else 1, 15)
    back = (scale * (codes - zero)).view(*w.shape[:-1], -1)[..., :din]
    return [back.to(w.dtype)]


def _plain_weights(st):
    """The values of 4-bit weights, in float but rounded to x's type as they are defined."""
    size, codes = st["case"]["size"], st["codes"]
    din = codes.shape[-1]
    scale = st["scales"].float().repeat_interleave(size, dim=-1)[..., :din]
    zero = 8.0 if st["zeros"] is None else st["zeros"].float().repeat_interleave(size, dim=-1)[..., :din]
    return (scale * (codes.float() - zero)).to(st["scales"].dtype).float()


def _plain_grouped(st):
    """The slots sorted by expert, one product per expert that has any."""
    case, dt = st["case"], st["x"].dtype
    t, e, k = case["t"], case["e"], case["k"]
    slots, order = torch.sort(st["experts"].reshape(-1), stable=True)
    bounds = torch.searchsorted(slots, torch.arange(e + 1, device="cuda", dtype=torch.int32)).tolist()
    w = _plain_weights(st)
    xs = st["x"].detach().float()[order // k]
    ys = torch.zeros(t * k, case["dout"], device="cuda")
    if case["train"]:
        ds = st["dy"].float().view(t * k, -1)[order]
        dxs = torch.zeros_like(xs)
    for i in range(e):
        s = slice(bounds[i], bounds[i + 1])
        if s.start == s.stop:
            continue
        torch.mm(xs[s], w[i].t(), out=ys[s])
        if case["train"]:
            torch.mm(ds[s], w[i], out=dxs[s])
    y = torch.empty_like(ys)
    y[order] = ys
    out = [y.view(t, k, -1).to(dt)]
    if case["train"]:
        dx = torch.empty_like(dxs)
        dx[order] = dxs
        out.append(dx.view(t, k, -1).sum(1).to(dt))
    return out


def _plain_lora(st):
    """Every adapter's columns for every token, the tokens' own kept."""
    case, dt = st["case"], st["x"].dtype
    t, e, r = case["t"], case["e"], case["rank"]
    x, w = st["x"].detach().float(), _plain_weights(st)
    a, b = st["a"].detach().float(), st["b"].detach().float()
    ids = st["experts"].long()
    g = st["weights"].detach() if case["gated"] else torch.ones(ids.shape, device="cuda")
    c = torch.where(ids >= 0, g * st["scale"][ids.clamp(min=0)], torch.zeros_like(g))
    gate = torch.zeros(t, e, device="cuda").scatter_add_(1, ids.clamp(min=0), c)[:, :, None]
    a2, b2 = a.reshape(e * r, -1), b.permute(1, 0, 2).reshape(-1, e * r)
    u = (x @ a2.t()).view(t, e, r)
    gu = (gate * u).view(t, e * r)
    out = [(x @ w.t() + gu @ b2.t()).to(dt)]
    if case["train"]:
        dy = st["dy"].float()
        v = (dy @ b2).view(t, e, r)
        gv = (gate * v).view(t, e * r)
        dx = dy @ w + gv @ a2
        da = (gv.t() @ x).view(a.shape)
        db = (dy.t() @ gu).view(-1, e, r).permute(1, 0, 2)
        out += [dx.to(dt), da.to(dt), db.contiguous().to(dt)]
        if case["gated"]:
            dg = (u * v).sum(2) * st["scale"]
            picked = torch.gather(dg, 1, ids.clamp(min=0))
            out.append(torch.where(ids >= 0, picked, torch.zeros_like(picked)))
    return out


def run(state):
    if own:
        return _run_own(state)
    return {"gate": _plain_gate, "quantize": _plain_quantize, "grouped4": _plain_grouped,
            "lora4": _plain_lora}[state["case"]["kind"]](state)


# ---------------------------------------------------------------- what a pass cannot do without
def _weight_bytes(case):
    """Codes, scales of 2 bytes and zeros of 4 bits of one matrix."""
    groups = -(-case["din"] // case["size"])
    return case["dout"] * (case["din"] + groups * (5 if case["zeros"] else 4)) // 2


def work(case):
    if case["kind"] == "quantize":
        n = case["e"] * case["dout"] * case["din"]
        return {"bytes": 4 * n + case["e"] * _weight_bytes(case), "flops": 6 * n}
    size = 4 if case["dtype"] == "f32" else 2
    t, e, k = case["t"], case["e"], case["k"]
    slots = t * k
    if case["kind"] == "gate":
        nbytes = t * e * (size + (1 if case["masked"] else 0)) + slots * 12 + (e + 1) * 4 + e * 4 * case["bias"]
        flops = 6 * t * e
        if case["train"]:
            nbytes += slots * 4 + t * e * size
            flops += 3 * t * e
        return {"bytes": nbytes, "flops": flops}
    din, dout = case["din"], case["dout"]
    used = min(e, slots)
    if case["kind"] == "grouped4":
        nbytes = size * (t * din + slots * dout) + used * _weight_bytes(case) + slots * 4
        flops = 2 * slots * din * dout
        if case["train"]:
            nbytes += size * (slots * dout + t * din)
            flops *= 2
        return {"bytes": nbytes, "flops": flops}
    r = case["rank"]
    nbytes = size * (t * (din + dout) + used * r * (din + dout)) + _weight_bytes(case) + slots * 8
    flops = 2 * t * din * dout + 2 * slots * r * (din + dout)
    if case["train"]:
        nbytes += size * (t * (din + dout) + e * r * (din + dout)) + slots * 4
        flops = 4 * t * din * dout + 6 * slots * r * (din + dout)
    return {"bytes": nbytes, "flops": flops}


# ---------------------------------------------------------------- the definitions in 64 bits
def _exact_gate(st):
    """On the host's numpy, row by row where nodes decide."""
    case = st["case"]
    t, e, k = case["t"], case["e"], case["k"]
    l = st["logits"].detach().double().cpu().numpy()
    ok = np.isfinite(l) if st["mask"] is None else np.isfinite(l) & st["mask"].cpu().numpy()
    if case["score"] == "softmax":
        top = np.max(np.where(ok, l, -np.inf), axis=1, keepdims=True)
        p = np.where(ok, np.exp(l - np.where(np.isfinite(top), top, 0.0)), 0.0)
        z = p.sum(1, keepdims=True)
        s = p / np.where(z == 0, 1.0, z)
    else:
        s = np.where(ok, np.exp(-np.logaddexp(0.0, -l)), 0.0)
    two = case["nodes"] > 1 and case["node_best"] == 2
    c = s + st["bias"].double().cpu().numpy() if case["bias"] else s if two else l
    c = np.where(ok, c, -np.inf)
    per = e // case["nodes"]
    if case["nodes"] > 1:
        up = -np.sort(-c.reshape(t, case["nodes"], per), axis=2)
        value = up[:, :, 0].copy()
        if case["node_best"] == 2 and per > 1:
            value += np.where(np.isfinite(up[:, :, 1]), up[:, :, 1], 0.0)
        first = np.argsort(-value, axis=1, kind="stable")[:, :case["top_nodes"]]
        kept = np.zeros((t, case["nodes"]), bool)
        np.put_along_axis(kept, first, True, 1)
        c = np.where(np.repeat(kept, per, axis=1), c, -np.inf)
    rank = np.argsort(-c, axis=1, kind="stable")[:, :k]
    has = np.isfinite(np.take_along_axis(c, rank, 1))
    sel = np.take_along_axis(s, rank, 1) * has
    z = sel.sum(1, keepdims=True) if case["normalize"] else np.ones((t, 1))
    z[z == 0] = 1.0
    share = sel / z
    experts = np.where(has, rank, -1).astype(np.int32)
    flat = experts.ravel()
    order = np.argsort(np.where(flat < 0, e, flat), kind="stable").astype(np.int32)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[flat >= 0], minlength=e))]).astype(np.int32)
    out = [share * case["scale"], experts, order, offsets]
    if case["train"]:
        dw = st["dweights"].double().cpu().numpy() * case["scale"]
        mean = (share * dw).sum(1, keepdims=True)
        # d share_i / d s_j, then d s_j / d l
        ds = ((dw - mean) / z if case["normalize"] else dw) * has
        full = np.zeros((t, e))
        np.put_along_axis(full, rank, ds, 1)
        if case["score"] == "softmax":
            grad = s * (full - (s * full).sum(1, keepdims=True))
        else:
            grad = full * s * (1 - s)
        out.append(grad)
    return [torch.from_numpy(np.ascontiguousarray(o)).cuda() for o in out]


def _exact_quantize(st):
    """Group by group of columns; the scale is a value of the weights' type."""
    case, dt = st["case"], st["w"].dtype
    w = st["w"].double()
    out = torch.empty_like(w)
    for at in range(0, case["din"], case["size"]):
        v = w[..., at:at + case["size"]]
        if case["zeros"]:
            low = torch.minimum(v.min(-1, keepdim=True).values, torch.zeros((), device="cuda", dtype=torch.float64))
            high = torch.maximum(v.max(-1, keepdim=True).values, torch.zeros((), device="cuda", dtype=torch.float64))
            s = ((high - low) / 15).to(dt).double()
            z = torch.clamp(torch.round(-low / s), 0, 15)
            q = torch.clamp(torch.round(v / s) + z, 0, 15) - z
        else:
            s = (v.abs().max(-1, keepdim=True).values / 7).to(dt).double()
            q = torch.clamp(torch.round(v / s), -7, 7)
        out[..., at:at + case["size"]] = torch.where(s > 0, (s * q).to(dt).double(), torch.zeros_like(v))
    return [out]


def _exact_weight(codes, scales, zeros, size):
    w = torch.empty(codes.shape, dtype=torch.float64, device="cuda")
    for j in range(scales.shape[-1]):
        z = 8.0 if zeros is None else zeros[:, j:j + 1].double()
        s = scales[:, j:j + 1]
        w[:, j * size:(j + 1) * size] = (s.double() * (codes[:, j * size:(j + 1) * size].double() - z)).to(s.dtype)
    return w


def _exact_grouped(st):
    case = st["case"]
    t, k = case["t"], case["k"]
    ids = st["experts"].cpu().numpy()
    x = st["x"].detach().double()
    y = torch.zeros(t, k, case["dout"], dtype=torch.float64, device="cuda")
    dx = torch.zeros(t, case["din"], dtype=torch.float64, device="cuda")
    for e in range(case["e"]):
        if not (ids == e).any():
            continue
        we = _exact_weight(st["codes"][e], st["scales"][e], None if st["zeros"] is None else st["zeros"][e],
                           case["size"])
        wt = we.t().contiguous()
        for j in range(k):
            rows = torch.from_numpy(np.flatnonzero(ids[:, j] == e)).cuda()
            if len(rows) == 0:
                continue
            y[rows, j] = torch.mm(x[rows], wt)
            if case["train"]:
                dx.index_add_(0, rows, torch.mm(st["dy"][rows, j].double(), we))
    return [y, dx] if case["train"] else [y]


def _exact_lora(st):
    """Adapter by adapter, on the tokens that have it."""
    case = st["case"]
    t, k = case["t"], case["k"]
    ids = st["experts"].cpu().numpy()
    x = st["x"].detach().double()
    w = _exact_weight(st["codes"], st["scales"], st["zeros"], case["size"])
    y = torch.mm(x, w.t().contiguous())
    if case["train"]:
        dy = st["dy"].double()
        dx = torch.mm(dy, w)
        da = torch.zeros(st["a"].shape, dtype=torch.float64, device="cuda")
        db = torch.zeros(st["b"].shape, dtype=torch.float64, device="cuda")
        dg = torch.zeros(t, k, dtype=torch.float64, device="cuda")
    for e in range(case["e"]):
        a, b = st["a"][e].detach().double(), st["b"][e].detach().double()
        s = float(st["scale"][e])
        for j in range(k):
            rows = torch.from_numpy(np.flatnonzero(ids[:, j] == e)).cuda()
            if len(rows) == 0:
                continue
            g = st["weights"][rows, j].detach().double()[:, None] if case["gated"] else 1.0
            u = torch.mm(x[rows], a.t().contiguous())
            y.index_add_(0, rows, torch.mm(s * g * u, b.t().contiguous()))
            if case["train"]:
                v = torch.mm(dy[rows], b)
                dx.index_add_(0, rows, torch.mm(s * g * v, a))
                da[e] += torch.mm((s * g * v).t().contiguous(), x[rows])
                db[e] += torch.mm(dy[rows].t().contiguous(), s * g * u)
                dg[rows, j] = s * (u * v).sum(1)
    if not case["train"]:
        return [y]
    return [y, dx, da, db] + ([dg] if case["gated"] else [])


def exact(case, seed):
    st = prepare(case, seed)
    return {"gate": _exact_gate, "quantize": _exact_quantize, "grouped4": _exact_grouped,
            "lora4": _exact_lora}[case["kind"]](st)
