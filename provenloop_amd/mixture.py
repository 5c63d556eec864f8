"""Plain (unencrypted) mixtures of low-rank adapters on torch tensors.

The adapters that `zero_moai` serves under encryption, in the clear: for
sessions that did not ask for encryption, for prefills and batches, and for
training the adapters and their gate. Three operators that fit together:

  route          gate with top-k per token (`zero_moai.softmax_gate` for a whole
                 batch, on the GPU; also with sigmoid scores, a bias for balance
                 and experts on nodes), slots grouped by expert
  grouped_matmul matrix products grouped by expert, with ragged group sizes
  lora_linear    a frozen shared projection with the adapters of many requests,
                 or a gated mixture of them, in one pass

The experts of grouped_matmul and the projection of lora_linear may have 4 bits
a weight (`Weight4`): `quantize4` makes them of bf16 or f16 ones, `pack4` lays out
a checkpoint's codes and scales, `dequantize4` gives the values that they stand
for. They are frozen: the products have gradients of everything else.

A slot is a (token, choice) pair, numbered token * k + choice; expert -1 means
none. Work is queued on torch's current stream of the tensors' device, and
nothing waits for it. All three are differentiable (see each for what in; in
reverse mode, once) and can be captured into a graph; forward-mode derivatives
and tracing are refused. Values are bf16 or f16 with sums in float; the
gate's logits may be f32 too. At most 1024 experts or adapters (512 for a gate),
32 choices a token and rank 128. The C entry points are in
include/tensafe_he.h (th_route, th_group, th_grouped_matmul, th_lora_linear).

The reference applies a single adapter to a single hidden state in the clear
(demonstrator/server/inference_engine.py:1234-1242); batches, gates and
gradients have no counterpart there.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib

_lib.load()  # the library that the binding calls

try:
    from . import _mixture_torch as _ext  # noqa: E402
except ImportError as e:
    raise ImportError(f"the binding of the mixture operators cannot be loaded ({e}): build it against this torch with "
                      "`make -C provenloop_amd/csrc mixture`") from e

__all__ = ["Groups", "Routing", "Weight4", "group", "route", "quantize4", "pack4", "dequantize4", "grouped_matmul",
           "lora_linear"]


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


class Weight4(NamedTuple):
    """Frozen weights of 4 bits: the values scale * (code - zero), rounded to dtype,
    with a scale (and a zero) for each row's group_size neighbouring columns. At
    most 2^30 columns, below 2^28 rows in all.

    Made by `quantize4` and `pack4`; used in place of a weight by `grouped_matmul`
    and `lora_linear`. data is the layout that the kernels read, half a byte a
    weight and 2 (with zeros 3) bytes a group, and is all that a copy to another
    device or a checkpoint has to take along: w._replace(data=w.data.to(device)).
    """

    data: torch.Tensor   # uint8
    shape: tuple         # (d_out, d_in) or (E, d_out, d_in)
    dtype: torch.dtype   # bf16 or f16, of the scales and values and of the products' other operands
    group_size: int
    zeros: bool


# ---------------------------------------------------------------- 4-bit weights
_TYPES = {torch.bfloat16: 1, torch.float16: 2}  # TH_BF16, TH_F16


def quantize4(weight, group_size: int = 128, zeros: bool = False) -> Weight4:
    """weight [d_out, d_in] or [E, d_out, d_in] (bf16 or f16) to 4 bits.

    group_size: columns of a scale, a power of two from 32 on (one that reaches
    d_in: a scale a row). Without zeros, scale = max |w| / 7 of the group and the
    codes stand for -7 .. 7 scales; with zeros, scale = (max - min) / 15 over the
    group's values and 0, and zero = -min / scale. Scales are rounded to the
    weight's type first, codes to the nearest value (ties to even). A group with
    an infinity or NaN becomes NaN, in bf16 also one whose scale is above 2^120.
    Has no gradient.
    """
    return Weight4(_ext.quantize4(weight, group_size, zeros), tuple(weight.shape), weight.dtype, group_size, bool(zeros))


def pack4(codes, scales, group_size: int, zeros=None) -> Weight4:
    """A checkpoint's 4-bit weights for the products here.

    codes [d_out, d_in] or [E, d_out, d_in] uint8, a code (the low 4 bits) a byte;
    scales [..., d_out, ceil(d_in / group_size)] bf16 or f16, which gives the
    values' type; zeros like scales in uint8 (0 .. 15), or None: 8 everywhere.
    Scales of infinity or NaN, for bf16 also above 2^120, make their group NaN.
    """
    return Weight4(_ext.pack4(codes, scales, group_size, zeros), tuple(codes.shape), scales.dtype, group_size,
                   zeros is not None)


def dequantize4(weight: Weight4):
    """The values of 4-bit weights: exactly those that the products multiply with."""
    return _ext.dequantize4(*_four(weight))


def _four(w):
    if w.dtype not in _TYPES:
        raise ValueError("a 4-bit weight's dtype must be bf16 or f16")
    return w.data, _TYPES[w.dtype], w.shape, w.group_size, w.zeros


# ---------------------------------------------------------------- grouping and gate
def group(experts, n_groups: int) -> Groups:
    """Groups the slots of experts [T, k] (or [T]; int32, anything outside
    [0, n_groups) is none) by expert: a stable sort on the GPU."""
    return Groups(*_ext.group(experts, n_groups), n_groups)


def route(logits, k: int, mask=None, normalize: bool = True, *, score: str = "softmax", bias=None, scale: float = 1.0,
          nodes: int = 1, top_nodes: int = 1, node_best: int = 1) -> Routing:
    """Gate with top-k, by softmax or sigmoid scores, balanced by a bias and by nodes.

    logits [T, E] (bf16, f16 or f32; E <= 512); mask [T, E] or [E] bool, False
    where a token must not use an expert (a logit of -inf says the same). The k
    largest logits of each token are chosen, ties to the lowest index; weights
    are exp(l - max) over their sum (normalize=True) or over the sum of all
    allowed experts. Tokens with fewer than k allowed experts have -1 and
    weight 0 there. Differentiable in the logits.

    score: "softmax" as above, or "sigmoid", s = 1 / (1 + exp(-l)) and weights s,
    or s over the sum of the chosen ones (normalize=True). scale: a positive
    number that multiplies the weights. bias [E] float32, which takes part in the
    choice alone: the k largest s + bias are chosen in place of the k largest
    logits (an expert whose bias is -inf never is; one of a large finite bias is
    a last choice, and costs a prefill time). Balancing raises it for experts
    with few slots and lowers it for those with many, as groups.offsets counts
    them. nodes: the experts lie in order on that many nodes, E / nodes each, and
    a token uses those of top_nodes nodes alone: of the nodes whose largest s +
    bias (without a bias, largest logit), or sum of the two largest s + bias
    (node_best=2; without a bias, of the two largest s), is largest. What scores
    decide is decided in 64 bits.
    """
    weights, experts, order, offsets = _ext.route(logits, k, mask, normalize, score, bias, scale, nodes, top_nodes, node_best)
    return Routing(weights, experts, Groups(experts, order, offsets, logits.shape[1]))


# ---------------------------------------------------------------- grouped products
def grouped_matmul(x, w, groups: Groups):
    """y[t, j] = w[expert of (t, j)] @ x[t]: matrix products grouped by expert.

    x [T, d_in], or [T, k, d_in] with a row per slot; w [E, d_out, d_in];
    groups from `route` or `group` with E groups. Returns [T, k, d_out], zero
    for slots without an expert. Differentiable in x and w. w may be a `Weight4`
    of shape (E, d_out, d_in), which has no gradient.
    """
    if isinstance(w, Weight4):
        return _ext.grouped_matmul4(x, *_four(w), *groups)
    return _ext.grouped_matmul(x, w, *groups)


# ---------------------------------------------------------------- shared projection with adapters
def lora_linear(x, weight, lora_a, lora_b, experts, weights=None, scale=None, bias=None,
                groups: Optional[Groups] = None):
    """y[t] = weight @ x[t] + bias + sum_j weights[t, j] scale[e] B[e] @ (A[e] @ x[t]), e = experts[t, j].

    x [T, d_in]; weight [d_out, d_in] (or a `Weight4` of that shape) and bias
    [d_out] frozen; lora_a [n, rank, d_in] and lora_b [n, d_out, rank] (PEFT's layout; rank <= 128,
    shorter adapters padded with zeros); experts [T] or [T, k] int32, outside
    [0, n) none: each request's adapter, or `route`'s choice; weights [T, k]
    float32 or None (ones): `route`'s; scale [n] float32 or None (ones). The
    low-rank products stay in float. groups: of `experts`, if the caller has
    them. Differentiable in x, lora_a, lora_b and weights.
    """
    order, offsets = (None, None) if groups is None else groups[1:3]
    if isinstance(weight, Weight4):
        return _ext.lora_linear4(x, *_four(weight), lora_a, lora_b, experts, weights, scale, bias, order, offsets)
    return _ext.lora_linear(x, weight, lora_a, lora_b, experts, weights, scale, bias, order, offsets)
