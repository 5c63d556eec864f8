"""Uses of torch that the mixture operators do not support are refused: without a word, they would be left out of the results.

The refusals come before anything is asked of a GPU; the calls that do reach one are marked.
"""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from provenloop_amd import mixture

T, E, K, D_IN, D_OUT, RANK = 6, 4, 2, 16, 8, 4


def tensors(device):
    g = torch.Generator().manual_seed(1)

    def normal(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, generator=g).to(dtype).to(device)

    ids = torch.randint(0, E, (T, K), generator=g).to(torch.int32).to(device)
    groups = mixture.Groups(ids, torch.arange(T * K, dtype=torch.int32, device=device), torch.zeros(E + 1, dtype=torch.int32, device=device), E)
    return dict(logits=normal(T, E, dtype=torch.float32), x=normal(T, D_IN), w=normal(E, D_OUT, D_IN), weight=normal(D_OUT, D_IN),
                a=normal(E, RANK, D_IN), b=normal(E, D_OUT, RANK), gate=normal(T, K, dtype=torch.float32),
                scale=normal(E, dtype=torch.float32), bias=normal(D_OUT), ids=ids, groups=groups)


CALLS = {
    "route": (lambda c: mixture.route(c["logits"], K).weights, ["logits"]),
    "grouped_matmul": (lambda c: mixture.grouped_matmul(c["x"], c["w"], c["groups"]), ["x", "w"]),
    "lora_linear": (lambda c: mixture.lora_linear(c["x"], c["weight"], c["a"], c["b"], c["ids"], weights=c["gate"], scale=c["scale"],
                                                  bias=c["bias"]), ["x", "weight", "a", "b", "gate", "scale", "bias"]),
}
DUALS = [(name, arg) for name, (_, args) in CALLS.items() for arg in args]


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("name,arg", DUALS)
def test_forward_mode_derivatives(name, arg, device):
    c = tensors(device)
    for grad in (True, False):
        with forward_ad.dual_level(), torch.set_grad_enabled(grad):
            c2 = dict(c, **{arg: forward_ad.make_dual(c[arg], torch.ones_like(c[arg]))})
            with pytest.raises(NotImplementedError, match="forward-mode"):
                CALLS[name][0](c2)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("name", [*CALLS, "group"])
def test_tracing(name, device):
    c = tensors(device)
    call, args = CALLS.get(name, (lambda c: mixture.group(c["ids"], E).order, ["ids"]))
    arg = args[0]
    with pytest.raises(NotImplementedError, match="trace"):
        torch.jit.trace(lambda v: call(dict(c, **{arg: v})), (c[arg],))
    from torch.fx.experimental.proxy_tensor import make_fx

    with pytest.raises(NotImplementedError, match="trace"):
        make_fx(lambda v: call(dict(c, **{arg: v})))(c[arg])


@pytest.mark.gpu
@pytest.mark.parametrize("name", CALLS)
def test_forward_mode_derivatives_of_gradients(name):
    """A gradient's own tangent (a Hessian's product, forward over reverse) is refused too."""
    c = tensors("cuda")
    c["groups"] = mixture.group(c["ids"], E)
    call, args = CALLS[name]
    leaf = c[args[0]].requires_grad_()
    y = call(c)
    with forward_ad.dual_level():
        dy = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, leaf, dy)


@pytest.mark.gpu
@pytest.mark.parametrize("name", CALLS)
def test_function_transforms(name):
    """torch.func's vmap, grad and jvp raise."""
    c = tensors("cuda")
    c["groups"] = mixture.group(c["ids"], E)
    call, args = CALLS[name]
    arg = args[0]

    def f(v):
        return call(dict(c, **{arg: v}))

    with pytest.raises(RuntimeError):
        torch.func.vmap(f)(torch.stack([c[arg], c[arg]]))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda v: f(v).float().sum())(c[arg])
    with pytest.raises(RuntimeError):
        torch.func.jvp(f, (c[arg],), (torch.ones_like(c[arg]),))
