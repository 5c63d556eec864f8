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

__all__ = ["Groups", "Routing", "group", "route", "grouped_matmul", "lora_linear"]


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


# ---------------------------------------------------------------- grouping and gate
def group(experts, n_groups: int) -> Groups:
    """Groups the slots of experts [T, k] (or [T]; int32, anything outside
    [0, n_groups) is none) by expert: a stable sort on the GPU."""
    return Groups(*_ext.group(experts, n_groups), n_groups)


def route(logits, k: int, mask=None, normalize: bool = True) -> Routing:
    """Softmax gate with top-k.

    logits [T, E] (bf16, f16 or f32; E <= 512); mask [T, E] or [E] bool, False
    where a token must not use an expert (a logit of -inf says the same). The k
    largest logits of each token are chosen, ties to the lowest index; weights
    are exp(l - max) over their sum (normalize=True) or over the sum of all
    allowed experts. Tokens with fewer than k allowed experts have -1 and
    weight 0 there. Differentiable in the logits.
    """
    weights, experts, order, offsets = _ext.route(logits, k, mask, normalize)
    return Routing(weights, experts, Groups(experts, order, offsets, logits.shape[1]))


# ---------------------------------------------------------------- grouped products
def grouped_matmul(x, w, groups: Groups):
    """y[t, j] = w[expert of (t, j)] @ x[t]: matrix products grouped by expert.

    x [T, d_in], or [T, k, d_in] with a row per slot; w [E, d_out, d_in];
    groups from `route` or `group` with E groups. Returns [T, k, d_out], zero
    for slots without an expert. Differentiable in x and w.
    """
    return _ext.grouped_matmul(x, w, *groups)


# ---------------------------------------------------------------- shared projection with adapters
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
    order, offsets = (None, None) if groups is None else groups[1:3]
    return _ext.lora_linear(x, weight, lora_a, lora_b, experts, weights, scale, bias, order, offsets)
