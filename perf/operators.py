"""The plain (unencrypted) mixture-of-adapters operators as measurable cases.

Every case is a dict of plain values; `kind` names the operator:

  route    softmax gate of T tokens over E experts: the k chosen experts, their
           weights, and the (token, choice) slots grouped by expert;
  grouped  matrix products grouped by expert, with ragged group sizes;
  lora     a shared projection with the low-rank adapters of many requests
           (or a gated mixture of them) added in the same pass.

`train` cases return the gradients beside the outputs. Widths are those of
bench.py and tests/ (hidden 1536 with q and v of 1536 and 256 outputs and rank
16; hidden 3584 with 512 outputs and rank 32; 3 experts a projection; 32
sessions), or generic ones.

Where `own` is false, `run` computes the operators from elementary torch
operations in 32 bits, rounded once at the end; where it is true, through
provenloop_amd.mixture.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# what the largest listed cases cost: lora_prefill's operations, grouped_train's bytes
FLOPS_MAX = 2 * 8192 * 3584 * 3584 + 2 * 8192 * 32 * (3584 + 3584)
BYTES_MAX = 2 * (2 * 4093 * 1536 + 2 * 8186 * 1536 + 2 * 16 * 1536 * 1536)


def listed():
    return [
        # One token through CryptoMOE's gate of 3 experts: pure latency.
        dict(name="route_token", kind="route", dtype="f32", t=1, e=3, k=2, masked=False, normalize=True, train=False),
        # A large prefill batch through a wide gate, some experts withheld
        # from some sessions.
        dict(name="route_prefill", kind="route", dtype="bf16", t=65536, e=64, k=8, masked=True, normalize=True,
             train=False),
        # A training step's gate: odd sizes, full softmax weights, rows with
        # no expert allowed, and the logits' gradient.
        dict(name="route_train", kind="route", dtype="f32", t=4099, e=13, k=3, masked=True, normalize=False,
             train=True),
        # Experts' products while 16 sessions decode: few rows per expert, the
        # weights are what has to be read.
        dict(name="grouped_decode", kind="grouped", dtype="f16", t=16, e=8, k=2, din=3584, dout=512, train=False),
        # The same for a prefill batch: large matrix products of ragged sizes.
        dict(name="grouped_prefill", kind="grouped", dtype="bf16", t=8192, e=8, k=2, din=1536, dout=3584,
             train=False),
        # A training step of 16 experts: output, gradient of the tokens and of
        # every expert's weight.
        dict(name="grouped_train", kind="grouped", dtype="bf16", t=4093, e=16, k=2, din=1536, dout=1536, train=True),
        # One token of one session through its q projection and adapter.
        dict(name="lora_token", kind="lora", dtype="bf16", t=1, e=4, k=1, din=1536, dout=1536, rank=16,
             requests=1, gated=False, train=False),
        # 32 sessions decode together, each with an adapter of its own.
        dict(name="lora_sessions", kind="lora", dtype="bf16", t=32, e=32, k=1, din=3584, dout=3584, rank=32,
             requests=32, gated=False, train=False),
        # A batch of 250 such sessions, of a few adapters' requests and others.
        dict(name="lora_many", kind="lora", dtype="f16", t=250, e=100, k=1, din=1536, dout=1536, rank=16,
             requests=250, gated=False, train=False),
        # Prefill of 20 requests of ragged lengths, an adapter each or none:
        # the largest case.
        dict(name="lora_prefill", kind="lora", dtype="bf16", t=8192, e=8, k=1, din=3584, dout=3584, rank=32,
             requests=20, gated=False, train=False),
        # CryptoMOE's experts in the clear: a gated mixture of 2 of 3 adapters
        # beside the v projection, an odd number of tokens.
        dict(name="lora_mixture", kind="lora", dtype="f16", t=1021, e=3, k=2, din=1536, dout=256, rank=16,
             requests=0, gated=True, train=False),
        # A training step of the adapters and their gate beside the frozen q
        # projection: gradients of the tokens, A, B and the gate weights.
        dict(name="lora_train", kind="lora", dtype="bf16", t=4096, e=8, k=2, din=1536, dout=1536, rank=16,
             requests=0, gated=True, train=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)) - 1e-9)))))


def _width(rng, lo, hi):
    """A feature width: mostly a multiple of 8, as models have them, any number otherwise."""
    n = _log_int(rng, lo, hi)
    return n if rng.random() < 0.25 else max(8, n // 8 * 8)


def draw(rng):
    kind = rng.choice(["route", "grouped", "lora", "lora"])
    train = rng.random() < 0.35
    if kind == "route":
        e = _log_int(rng, 2, 128)
        return dict(kind=kind, dtype=rng.choice(["bf16", "f16", "f32"]), t=_log_int(rng, 1, 65536), e=e,
                    k=rng.randint(1, min(8, e)), masked=rng.random() < 0.5, normalize=rng.random() < 0.6, train=train)
    case = dict(kind=kind, dtype=rng.choice(["bf16", "f16"]), t=_log_int(rng, 1, 8192), e=_log_int(rng, 1, 64), k=1,
                din=_width(rng, 64, 4096), dout=_width(rng, 64, 4096), train=train)
    case["k"] = rng.randint(1, min(4, case["e"]))
    if kind == "lora":
        gated = rng.random() < 0.5
        case.update(rank=_log_int(rng, 1, 64), gated=gated, requests=0)
        if not gated:
            case.update(k=1, requests=_log_int(rng, 1, case["t"]))
    while case["t"] > 1 and _cost(case) > FLOPS_MAX:
        case["t"] = case["t"] * 3 // 4
    while case["e"] > 1 and work(case)["bytes"] > BYTES_MAX:
        case["e"] = case["e"] * 3 // 4
        case["k"] = min(case["k"], case["e"])
    return case


def _cost(case):
    """Operations of a pass; the plain form of `lora` takes every adapter's columns."""
    f = work(case)["flops"]
    if case["kind"] == "lora":
        f += 2 * case["t"] * case["e"] * case["rank"] * (case["din"] + case["dout"])
    return f


# ---------------------------------------------------------------- inputs
def _normal(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * std


def _choices(g, t, e, k):
    """k distinct experts a token, some experts favoured (ragged groups, possibly empty ones)."""
    score = _normal(g, t, e) + _normal(g, 1, e, std=1.0)
    return torch.sort(score, dim=1, descending=True, stable=True).indices[:, :k].to(torch.int32).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    t, e, k = case["t"], case["e"], case["k"]
    st = dict(case=case)
    if case["kind"] == "route":
        st["logits"] = _normal(g, t, e, std=1.5).to(dt)
        st["mask"] = None
        if case["masked"]:
            # sessions without some of the experts; one token in 50 without any
            allowed = torch.rand(t, e, generator=g, device="cuda") < 0.8
            st["mask"] = allowed & (torch.rand(t, 1, generator=g, device="cuda") >= 0.02)
        if case["train"]:
            st["dweights"] = _normal(g, t, k)
        leaves = ["logits"]
    elif case["kind"] == "grouped":
        din, dout = case["din"], case["dout"]
        st["x"] = _normal(g, t, din).to(dt)
        st["w"] = _normal(g, e, dout, din, std=din ** -0.5).to(dt)
        st["experts"] = _choices(g, t, e, k)
        if case["train"]:
            st["dy"] = _normal(g, t, k, dout).to(dt)
        leaves = ["x", "w"]
    else:
        din, dout, r = case["din"], case["dout"], case["rank"]
        st["x"] = _normal(g, t, din).to(dt)
        st["weight"] = _normal(g, dout, din, std=din ** -0.5).to(dt)
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
    return st


# ---------------------------------------------------------------- the framework's operators
def _run_own(st):
    from provenloop_amd import mixture

    case = st["case"]
    if case["kind"] == "route":
        r = mixture.route(st["logits"], case["k"], mask=st["mask"], normalize=case["normalize"])
        out = [r.weights.detach(), r.experts, r.groups.order, r.groups.offsets]
        y, dy = r.weights, st.get("dweights")
    elif case["kind"] == "grouped":
        groups = mixture.group(st["experts"], case["e"])
        y, dy = mixture.grouped_matmul(st["x"], st["w"], groups), st.get("dy")
        out = [y.detach()]
    else:
        y = mixture.lora_linear(st["x"], st["weight"], st["a"], st["b"], st["experts"], weights=st["weights"],
                                scale=st["scale"])
        out, dy = [y.detach()], st.get("dy")
    if case["train"]:
        out += torch.autograd.grad(y, [st[n] for n in st["leaves"]], dy)
    return out


# ---------------------------------------------------------------- plain forms
def _plain_route(st):
    case, logits = st["case"], st["logits"].detach().float()
    e, k = case["e"], case["k"]
    allowed = logits > -math.inf
    if st["mask"] is not None:
        allowed = allowed & st["mask"]
    masked = torch.where(allowed, logits, torch.full_like(logits, -math.inf))
    top, index = torch.sort(masked, dim=1, descending=True, stable=True)
    top, index = top[:, :k], index[:, :k]
    chosen = top > -math.inf
    experts = torch.where(chosen, index, torch.full_like(index, -1)).to(torch.int32)
    big = top[:, :1]
    big = torch.where(big > -math.inf, big, torch.zeros_like(big))
    num = torch.where(chosen, torch.exp(top - big), torch.zeros_like(top))
    full = torch.where(allowed, torch.exp(masked - big), torch.zeros_like(masked))
    total = (num if case["normalize"] else full).sum(1, keepdim=True)
    total = torch.where(total > 0, total, torch.ones_like(total))
    weights = num / total
    slots = experts.reshape(-1)
    key = torch.where(slots < 0, torch.full_like(slots, e), slots)
    order = torch.sort(key, stable=True).indices.to(torch.int32)
    counts = (key[:, None] == torch.arange(e, device=key.device, dtype=key.dtype)[None, :]).sum(0)
    offsets = torch.cat([counts.new_zeros(1), torch.cumsum(counts, 0)]).to(torch.int32)
    out = [weights, experts, order, offsets]
    if case["train"]:
        dw = st["dweights"]
        inner = (weights * dw).sum(1, keepdim=True)
        picked = index.long()
        if case["normalize"]:
            grad = torch.zeros_like(logits).scatter_(1, picked, weights * (dw - inner))
        else:
            grad = (-full / total * inner).scatter_add_(1, picked, weights * dw)
        out.append(grad.to(st["logits"].dtype))
    return out


def _plain_grouped(st):
    """The slots sorted by expert, one product per expert that has any."""
    case, dt = st["case"], st["x"].dtype
    t, e, k = case["t"], case["e"], case["k"]
    slots, order = torch.sort(st["experts"].reshape(-1), stable=True)
    bounds = torch.searchsorted(slots, torch.arange(e + 1, device="cuda", dtype=torch.int32)).tolist()
    w = st["w"].detach().float()
    xs = st["x"].detach().float()[order // k]
    ys = torch.zeros(t * k, case["dout"], device="cuda")
    if case["train"]:
        ds = st["dy"].float().view(t * k, -1)[order]
        dxs, dw = torch.zeros_like(xs), torch.zeros_like(w)
    for i in range(e):
        s = slice(bounds[i], bounds[i + 1])
        if s.start == s.stop:
            continue
        torch.mm(xs[s], w[i].t(), out=ys[s])
        if case["train"]:
            torch.mm(ds[s], w[i], out=dxs[s])
            torch.mm(ds[s].t(), xs[s], out=dw[i])
    y = torch.empty_like(ys)
    y[order] = ys
    out = [y.view(t, k, -1).to(dt)]
    if case["train"]:
        dx = torch.empty_like(dxs)
        dx[order] = dxs
        out += [dx.view(t, k, -1).sum(1).to(dt), dw.to(dt)]
    return out


def _plain_lora(st):
    """Every adapter's columns for every token, the tokens' own kept."""
    case, dt = st["case"], st["x"].dtype
    t, e, r = case["t"], case["e"], case["rank"]
    x, w = st["x"].detach().float(), st["weight"].float()
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
    return {"route": _plain_route, "grouped": _plain_grouped, "lora": _plain_lora}[state["case"]["kind"]](state)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    t, e, k = case["t"], case["e"], case["k"]
    slots = t * k
    if case["kind"] == "route":
        nbytes = t * e * (size + (1 if case["masked"] else 0)) + slots * 12 + (e + 1) * 4
        flops = 4 * t * e
        if case["train"]:
            nbytes += slots * 4 + t * e * size
            flops += 3 * t * e
        return {"bytes": nbytes, "flops": flops}
    din, dout = case["din"], case["dout"]
    used = min(e, slots)
    if case["kind"] == "grouped":
        nbytes = size * (t * din + used * din * dout + slots * dout) + slots * 4
        flops = 2 * slots * din * dout
        if case["train"]:
            nbytes += size * (slots * dout + t * din + e * din * dout)
            flops *= 3
        return {"bytes": nbytes, "flops": flops}
    r = case["rank"]
    nbytes = size * (t * (din + dout) + din * dout + used * r * (din + dout)) + slots * 8
    flops = 2 * t * din * dout + 2 * slots * r * (din + dout)
    if case["train"]:
        nbytes += size * (t * (din + dout) + e * r * (din + dout)) + slots * 4
        flops = 4 * t * din * dout + 6 * slots * r * (din + dout)
    return {"bytes": nbytes, "flops": flops}


# ---------------------------------------------------------------- the definitions in 64 bits
def _exact_route(st):
    """Row by row on the host's numpy: p = exp(l - max) / sum over what the mask leaves."""
    case = st["case"]
    t, e, k = case["t"], case["e"], case["k"]
    l = st["logits"].detach().double().cpu().numpy()
    ok = np.isfinite(l) if st["mask"] is None else np.isfinite(l) & st["mask"].cpu().numpy()
    rank = np.argsort(np.where(ok, -l, np.inf), axis=1, kind="stable")[:, :k]
    has = np.take_along_axis(ok, rank, 1)
    top = np.max(np.where(ok, l, -np.inf), axis=1, keepdims=True)
    p = np.where(ok, np.exp(l - np.where(np.isfinite(top), top, 0.0)), 0.0)
    sel = np.take_along_axis(p, rank, 1) * has
    z = (sel if case["normalize"] else p).sum(1, keepdims=True)
    z[z == 0] = 1.0
    wts = sel / z
    experts = np.where(has, rank, -1).astype(np.int32)
    flat = experts.ravel()
    order = np.concatenate([np.flatnonzero(flat == x) for x in list(range(e)) + [-1]]).astype(np.int32)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[flat >= 0], minlength=e))]).astype(np.int32)
    out = [wts, experts, order, offsets]
    if case["train"]:
        dw = st["dweights"].double().cpu().numpy()
        mean = (wts * dw).sum(1, keepdims=True)
        grad = np.zeros((t, e)) if case["normalize"] else -(p / z) * mean
        rows = np.repeat(np.arange(t), k)
        add = wts * (dw - mean) if case["normalize"] else wts * dw
        np.add.at(grad, (rows, rank.ravel()), add.ravel())
        out.append(grad)
    return [torch.from_numpy(np.ascontiguousarray(o)).cuda() for o in out]


def _exact_grouped(st):
    case = st["case"]
    t, k = case["t"], case["k"]
    ids = st["experts"].cpu().numpy()
    x, w = st["x"].detach().double(), st["w"].detach()
    y = torch.zeros(t, k, case["dout"], dtype=torch.float64, device="cuda")
    dx = torch.zeros(t, case["din"], dtype=torch.float64, device="cuda")
    dw = torch.zeros(w.shape, dtype=torch.float64, device="cuda") if case["train"] else None
    for e in range(case["e"]):
        we = w[e].double()
        for j in range(k):
            rows = torch.from_numpy(np.flatnonzero(ids[:, j] == e)).cuda()
            if len(rows) == 0:
                continue
            y[rows, j] = torch.mm(x[rows], we.t().contiguous())
            if case["train"]:
                d = st["dy"][rows, j].double()
                dx.index_add_(0, rows, torch.mm(d, we))
                dw[e] += torch.mm(d.t().contiguous(), x[rows])
    return [y, dx, dw] if case["train"] else [y]


def _exact_lora(st):
    """Adapter by adapter, on the tokens that have it."""
    case = st["case"]
    t, k = case["t"], case["k"]
    ids = st["experts"].cpu().numpy()
    x, w = st["x"].detach().double(), st["weight"].double()
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
    return {"route": _exact_route, "grouped": _exact_grouped, "lora": _exact_lora}[case["kind"]](st)
