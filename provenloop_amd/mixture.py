"""Plain (unencrypted) mixtures of low-rank adapters on torch tensors.

The adapters that `zero_moai` serves under encryption, in the clear: for
sessions that did not ask for encryption, for prefills and batches, and for
training the adapters and their gate. Three operators that fit together:

  route          softmax gate with top-k per token (`zero_moai.softmax_gate`
                 for a whole batch, on the GPU), slots grouped by expert
  grouped_matmul matrix products grouped by expert, with ragged group sizes
  lora_linear    a frozen shared projection with the adapters of many requests,
                 or a gated mixture of them, in one pass

A slot is a (token, choice) pair, numbered token * k + choice; expert -1 means
none. Work is queued on torch's current stream of the tensors' device, and
nothing waits for it. All three are differentiable (see each for what in) and
can be captured into a graph. Values are bf16 or f16 with sums in float; the
gate's logits may be f32 too. The C entry points are in
include/tensafe_he.h (th_route, th_group, th_grouped_matmul, th_lora_linear).

The reference applies a single adapter to a single hidden state in the clear
(demonstrator/server/inference_engine.py:1234-1242); batches, gates and
gradients have no counterpart there.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import _lib

__all__ = ["Groups", "Routing", "group", "route", "grouped_matmul", "lora_linear"]

_TYPES = {torch.bfloat16: _lib.TH_BF16, torch.float16: _lib.TH_F16}
_GATE_TYPES = {**_TYPES, torch.float32: _lib.TH_F32}
_RANK_PAD = 4  # u rows: the rank rounded up to this


class Groups(NamedTuple):
    """The (token, choice) slots grouped by expert (`group`, `route`)."""

    experts: torch.Tensor  # [T, k] int32, -1: none
    order: torch.Tensor    # [T * k] int32: slots sorted by expert, stable, those without one last
    offsets: torch.Tensor  # [n_groups + 1] int32: where each expert's slots begin in order
    n_groups: int


class Routing(NamedTuple):
    weights: torch.Tensor  # [T, k] float32
    experts: torch.Tensor  # [T, k] int32
    groups: Groups


def _queue(device):
    """Makes `device` current for the calls of this thread; its current stream."""
    if device.index != torch.cuda.current_device():
        return torch.cuda.device(device), torch._C._cuda_getCurrentRawStream(device.index)
    return None, torch._C._cuda_getCurrentRawStream(device.index)


def _call(device, fn, *args):
    guard, stream = _queue(device)
    if guard is None:
        rc = fn(*args, stream)
    else:
        with guard:
            rc = fn(*args, stream)
    if rc:
        _lib.check(rc)


def _need(ok, message):
    if not ok:
        raise ValueError(message)


def _on_gpu(name, *tensors):
    dev = tensors[0].device
    if dev.type != "cuda":
        raise ValueError(f"{name}: tensors must be on the GPU (there is no CPU path)")
    for t in tensors[1:]:
        if t is not None and t.device != dev:
            raise ValueError(f"{name}: all tensors must be on one device")
    return dev


def _rows(t):
    """t with unit column stride and rows that do not overlap (a copy only if it has none)."""
    if t.dim() and t.shape[-1] > 1 and t.stride(-1) != 1:
        return t.contiguous()
    if any(s < t.shape[-1] and n > 1 for s, n in zip(t.stride()[:-1], t.shape[:-1])):
        return t.contiguous()
    return t


def _ld(t, dim=-2):
    """Row stride; of a single row its length, which every row check takes."""
    return t.stride(dim) if t.shape[dim] > 1 else t.shape[-1]


def _work(device, fn, *args):
    n = C.c_size_t()
    rc = fn(*args, C.byref(n))
    if rc:
        _lib.check(rc)
    if n.value == 0:
        return None, 0
    t = torch.empty(n.value, dtype=torch.uint8, device=device)
    return t, n.value


def _ptr(t):
    return None if t is None else t.data_ptr()


def _experts(name, experts, device):
    _need(isinstance(experts, torch.Tensor) and experts.dtype == torch.int32, f"{name}: experts must be an int32 tensor")
    if experts.dim() == 1:
        experts = experts.unsqueeze(1)
    _need(experts.dim() == 2, f"{name}: experts must be [T] or [T, k]")
    return experts.contiguous()


# ---------------------------------------------------------------- grouping and gate
def group(experts, n_groups: int) -> Groups:
    """Groups the slots of experts [T, k] (or [T]; int32, anything outside
    [0, n_groups) is none) by expert: a stable sort on the GPU."""
    lib = _lib.load()
    experts = _experts("group", experts, None)
    dev = _on_gpu("group", experts)
    t, k = experts.shape
    order = torch.empty(t * k, dtype=torch.int32, device=dev)
    offsets = torch.empty(max(0, n_groups) + 1, dtype=torch.int32, device=dev)
    work, size = _work(dev, lib.th_group_workspace, t, n_groups, k)
    _call(dev, lib.th_group, experts.data_ptr(), t, n_groups, k, order.data_ptr(), offsets.data_ptr(), _ptr(work),
          size)
    return Groups(experts, order, offsets, n_groups)


def _route(logits, mask, k, normalize):
    lib = _lib.load()
    dev = logits.device
    t, e = logits.shape
    weights = torch.empty(t, k, dtype=torch.float32, device=dev)
    experts = torch.empty(t, k, dtype=torch.int32, device=dev)
    order = torch.empty(t * k, dtype=torch.int32, device=dev)
    offsets = torch.empty(e + 1, dtype=torch.int32, device=dev)
    work, size = _work(dev, lib.th_group_workspace, t, e, k)
    _call(dev, lib.th_route, _GATE_TYPES[logits.dtype], logits.data_ptr(), _ld(logits), t, e, _ptr(mask),
          _mask_ld(mask), k, int(normalize), weights.data_ptr(), experts.data_ptr(), order.data_ptr(),
          offsets.data_ptr(), _ptr(work), size)
    return weights, experts, order, offsets


def _mask_ld(mask):
    if mask is None or mask.dim() == 1 or mask.stride(0) == 0:
        return 0
    return _ld(mask)


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, mask, k, normalize):
        weights, experts, order, offsets = _route(logits, mask, k, normalize)
        ctx.save_for_backward(logits, weights, experts)
        ctx.mask, ctx.k, ctx.normalize = mask, k, normalize
        ctx.mark_non_differentiable(experts, order, offsets)
        return weights, experts, order, offsets

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dweights, *_):
        logits, weights, experts = ctx.saved_tensors
        dweights = dweights.contiguous()
        t, e = logits.shape
        dlogits = torch.empty(t, e, dtype=logits.dtype, device=logits.device)
        _call(logits.device, _lib.load().th_route_backward, _GATE_TYPES[logits.dtype], logits.data_ptr(), _ld(logits),
              t, e, _ptr(ctx.mask), _mask_ld(ctx.mask), ctx.k, int(ctx.normalize), weights.data_ptr(),
              experts.data_ptr(), dweights.data_ptr(), dlogits.data_ptr())
        return dlogits, None, None, None


def route(logits, k: int, mask=None, normalize: bool = True) -> Routing:
    """Softmax gate with top-k.

    logits [T, E] (bf16, f16 or f32; E <= 512); mask [T, E] or [E] bool, False
    where a token must not use an expert (a logit of -inf says the same). The k
    largest logits of each token are chosen, ties to the lowest index; weights
    are exp(l - max) over their sum (normalize=True) or over the sum of all
    allowed experts. Tokens with fewer than k allowed experts have -1 and
    weight 0 there. Differentiable in the logits.
    """
    _need(isinstance(logits, torch.Tensor) and logits.dtype in _GATE_TYPES, "route: logits must be bf16, f16 or f32")
    _need(logits.dim() == 2, "route: logits must be [T, E]")
    dev = _on_gpu("route", logits, mask)
    if mask is not None:
        _need(mask.dtype == torch.bool, "route: mask must be bool")
        _need(tuple(mask.shape) in (tuple(logits.shape), (logits.shape[1],)), "route: mask must be [T, E] or [E]")
        if mask.shape[-1] > 1 and mask.stride(-1) != 1:
            mask = mask.contiguous()
        if mask.dim() == 2 and mask.shape[0] > 1 and 0 < mask.stride(0) < mask.shape[1]:
            mask = mask.contiguous()
    logits = _rows(logits)
    if logits.requires_grad and torch.is_grad_enabled():
        weights, experts, order, offsets = _Route.apply(logits, mask, k, normalize)
    else:
        weights, experts, order, offsets = _route(logits, mask, k, normalize)
    return Routing(weights, experts, Groups(experts, order, offsets, logits.shape[1]))


# ---------------------------------------------------------------- grouped products
def _grouped_args(x, w, groups):
    t, k = groups.experts.shape
    e, n, d = w.shape
    return _lib.Grouped(_TYPES[x.dtype], int(x.dim() == 3), t, k, e, d, n, x.data_ptr(), w.data_ptr(), _ld(x),
                        _ld(w), w.stride(0), groups.order.data_ptr(), groups.offsets.data_ptr())


def _grouped(x, w, groups):
    t, k = groups.experts.shape
    y = torch.empty(t, k, w.shape[1], dtype=x.dtype, device=x.device)
    _call(x.device, _lib.load().th_grouped_matmul, C.byref(_grouped_args(x, w, groups)), y.data_ptr(), w.shape[1])
    return y


class _GroupedMatmul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, groups):
        ctx.save_for_backward(x, w)
        ctx.groups = groups
        return _grouped(x, w, groups)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        lib = _lib.load()
        dy = dy.contiguous()
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if ctx.needs_input_grad[0] else None
        dw = torch.empty(w.shape, dtype=w.dtype, device=w.device) if ctx.needs_input_grad[1] else None
        args = _grouped_args(x, w, ctx.groups)
        work, size = _work(x.device, lib.th_grouped_matmul_backward_workspace, C.byref(args))
        _call(x.device, lib.th_grouped_matmul_backward, C.byref(args), dy.data_ptr(), w.shape[1], _ptr(dx), _ptr(dw),
              _ptr(work), size)
        return dx, dw, None


def grouped_matmul(x, w, groups: Groups):
    """y[t, j] = w[expert of (t, j)] @ x[t]: matrix products grouped by expert.

    x [T, d_in], or [T, k, d_in] with a row per slot; w [E, d_out, d_in];
    groups from `route` or `group` with E groups. Returns [T, k, d_out], zero
    for slots without an expert. Differentiable in x and w.
    """
    _need(isinstance(x, torch.Tensor) and x.dtype in _TYPES, "grouped_matmul: x must be bf16 or f16")
    _need(w.dtype == x.dtype, "grouped_matmul: x and w must have one type")
    t, k = groups.experts.shape
    _need(w.dim() == 3 and w.shape[0] == groups.n_groups, "grouped_matmul: w must be [n_groups, d_out, d_in]")
    _need(tuple(x.shape) in ((t, w.shape[2]), (t, k, w.shape[2])),
          "grouped_matmul: x must be [T, d_in] or [T, k, d_in]")
    _on_gpu("grouped_matmul", x, w, groups.order)
    if x.dim() == 3:
        x = x.contiguous()
    x, w = _rows(x), _rows(w)
    if (x.requires_grad or w.requires_grad) and torch.is_grad_enabled():
        return _GroupedMatmul.apply(x, w, groups)
    return _grouped(x, w, groups)


# ---------------------------------------------------------------- shared projection with adapters
def _lora_args(x, weight, bias, a, b, experts, gate, scale, order, offsets):
    t, k = experts.shape
    return _lib.LoraLinear(_TYPES[x.dtype], k, t, x.shape[1], weight.shape[0], a.shape[1], a.shape[0], x.data_ptr(),
                           weight.data_ptr(), _ptr(bias), a.data_ptr(), b.data_ptr(), _ld(x), _ld(weight), _ld(a),
                           a.stride(0), _ld(b), b.stride(0), experts.data_ptr(), _ptr(gate), _ptr(scale),
                           _ptr(order), _ptr(offsets))


def _lora(args, x, d_out, u):
    lib = _lib.load()
    y = torch.empty(x.shape[0], d_out, dtype=x.dtype, device=x.device)
    ref = C.byref(args)
    work, size = _work(x.device, lib.th_lora_linear_workspace, ref, int(u is not None))
    _call(x.device, lib.th_lora_linear, ref, y.data_ptr(), d_out, _ptr(u), _ptr(work), size)
    return y


class _LoraLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, a, b, gate, weight, bias, experts, scale, groups):
        t, k = experts.shape
        if groups is None:  # the backward pass needs them again
            groups = group(experts, a.shape[0])
        u = torch.empty(t * k, -(-a.shape[1] // _RANK_PAD) * _RANK_PAD, dtype=torch.float32, device=x.device)
        ctx.save_for_backward(x, a, b, gate, weight, bias, experts, scale, groups.order, groups.offsets, u)
        args = _lora_args(x, weight, bias, a, b, experts, gate, scale, groups.order, groups.offsets)
        return _lora(args, x, weight.shape[0], u)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, a, b, gate, weight, bias, experts, scale, order, offsets, u = ctx.saved_tensors
        lib = _lib.load()
        dy = _rows(dy)

        def like(i, t):
            return torch.empty(t.shape, dtype=t.dtype, device=t.device) if ctx.needs_input_grad[i] else None

        dx, da, db, dgate = like(0, x), like(1, a), like(2, b), like(3, gate)
        args = _lora_args(x, weight, bias, a, b, experts, gate, scale, order, offsets)
        ref = C.byref(args)
        work, size = _work(x.device, lib.th_lora_linear_backward_workspace, ref)
        _call(x.device, lib.th_lora_linear_backward, ref, u.data_ptr(), dy.data_ptr(), _ld(dy), _ptr(dx), _ptr(da),
              _ptr(db), _ptr(dgate), _ptr(work), size)
        return dx, da, db, dgate, None, None, None, None, None


def lora_linear(x, weight, lora_a, lora_b, experts, weights=None, scale=None, bias=None,
                groups: Optional[Groups] = None):
    """y[t] = weight @ x[t] + bias + sum_j weights[t, j] scale[e] B[e] @ (A[e] @ x[t]), e = experts[t, j].

    x [T, d_in]; weight [d_out, d_in] and bias [d_out] frozen; lora_a
    [n, rank, d_in] and lora_b [n, d_out, rank] (PEFT's layout; rank <= 128,
    shorter adapters padded with zeros); experts [T] or [T, k] int32, outside
    [0, n) none: each request's adapter, or `route`'s choice; weights [T, k]
    float32 or None (ones): `route`'s; scale [n] float32 or None (ones). The
    low-rank products stay in float. groups: of `experts`, if the caller has
    them. Differentiable in x, lora_a, lora_b and weights.
    """
    _need(isinstance(x, torch.Tensor) and x.dtype in _TYPES, "lora_linear: x must be bf16 or f16")
    for name, t in (("weight", weight), ("lora_a", lora_a), ("lora_b", lora_b), ("bias", bias)):
        _need(t is None or t.dtype == x.dtype, f"lora_linear: {name} must have x's type")
    _need(x.dim() == 2 and weight.dim() == 2 and weight.shape[1] == x.shape[1],
          "lora_linear: x must be [T, d_in] and weight [d_out, d_in]")
    n, r = lora_a.shape[0], lora_a.shape[1] if lora_a.dim() == 3 else 0
    _need(tuple(lora_a.shape) == (n, r, x.shape[1]), "lora_linear: lora_a must be [n, rank, d_in]")
    _need(tuple(lora_b.shape) == (n, weight.shape[0], r), "lora_linear: lora_b must be [n, d_out, rank]")
    experts = _experts("lora_linear", experts, x.device)
    _need(experts.shape[0] == x.shape[0], "lora_linear: experts must have a row per token")
    _need(bias is None or (tuple(bias.shape) == (weight.shape[0],)), "lora_linear: bias must be [d_out]")
    if weights is not None:
        if weights.dim() == 1:
            weights = weights.unsqueeze(1)
        _need(weights.dtype == torch.float32 and weights.shape == experts.shape,
              "lora_linear: weights must be float32 and shaped as experts")
        weights = weights.contiguous()
    if scale is not None:
        _need(scale.dtype == torch.float32 and tuple(scale.shape) == (n,), "lora_linear: scale must be float32 [n]")
        scale = scale.contiguous()
    _on_gpu("lora_linear", x, weight, lora_a, lora_b, experts, weights, scale, bias)
    x, weight, lora_a, lora_b = _rows(x), _rows(weight), _rows(lora_a), _rows(lora_b)
    if bias is not None:
        bias = bias.contiguous()
    if groups is not None:
        _need(groups.n_groups == n and groups.experts.shape == experts.shape, "lora_linear: groups of other experts")
    if torch.is_grad_enabled():
        _need(not any(t is not None and t.requires_grad for t in (weight, bias, scale)),
              "lora_linear: weight, bias and scale are frozen and have no gradient")
        if any(t is not None and t.requires_grad for t in (x, lora_a, lora_b, weights)):
            return _LoraLinear.apply(x, lora_a, lora_b, weights, weight, bias, experts, scale, groups)
    args = _lora_args(x, weight, bias, lora_a, lora_b, experts, weights, scale,
                      *((None, None) if groups is None else (groups.order, groups.offsets)))
    return _lora(args, x, weight.shape[0], None)
