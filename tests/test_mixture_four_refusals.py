"""What the 4-bit weights and the balanced gate refuse, before anything reaches a GPU."""
import ctypes as C

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from provenloop_amd import _lib, mixture

from test_mixture_refusals import P, grouped, lora, refused

BF16 = torch.bfloat16


def weight(**kw):
    d = dict(dtype=1, matrices=3, d_out=8, d_in=16, group=32, zeros=0, data=P)
    d.update(kw)
    return C.byref(_lib.Weight4(**d))


BAD_WEIGHTS = [(dict(dtype=3), "dtype"), (dict(dtype=0), "dtype"), (dict(matrices=0), "positive"), (dict(d_out=0), "positive"),
               (dict(d_in=0), "positive"), (dict(d_in=(1 << 30) + 1), "2^30"), (dict(group=16), "power of two"),
               (dict(group=96), "power of two"), (dict(group=1 << 31), "power of two")]

BAD_WEIGHTS += [(dict(d_out=1 << 28), "2^28"), (dict(matrices=1 << 24), "2^28"), (dict(matrices=0xffffffff, d_out=1 << 30, d_in=1 << 30), "2^28")]

@pytest.mark.parametrize("change,text", BAD_WEIGHTS + [(dict(data=None), "null data"), (dict(data=P + 8), "multiple of 16")])
def test_weights(change, text):
    L = _lib.load()
    w = weight(**change)
    size = C.c_size_t()
    if (change, text) in BAD_WEIGHTS:
        refused(L.th_weight4_bytes(w, C.byref(size)), text)
    refused(L.th_pack4(w, P, 16, 128, P, None, None), text)
    refused(L.th_quantize4(w, P, 16, 128, None), text)
    refused(L.th_dequantize4(w, P, 16, 128, None), text)
    refused(L.th_grouped_matmul4(grouped(), w, P, 8, P, 1 << 40, None), text)
    refused(L.th_grouped_matmul4_backward(grouped(), w, P, 8, P, P, 1 << 40, None), text)
    refused(L.th_grouped_matmul4_workspace(grouped(), w, C.byref(size)), text)
    refused(L.th_grouped_matmul4_backward_workspace(grouped(), w, C.byref(size)), text)
    refused(L.th_lora_linear4(lora(), w, P, 8, None, P, 1 << 40, None), text)
    refused(L.th_lora_linear4_backward(lora(), w, P, P, 8, P, P, P, P, P, 1 << 40, None), text)
    refused(L.th_lora_linear4_workspace(lora(), w, 0, C.byref(size)), text)
    refused(L.th_lora_linear4_backward_workspace(lora(), w, C.byref(size)), text)


def test_bytes():
    """Half a byte a weight and two or three a scale, rows and columns rounded up."""
    L = _lib.load()
    size = C.c_size_t()

    def of(matrices, d_out, d_in, group, zeros):
        assert L.th_weight4_bytes(weight(matrices=matrices, d_out=d_out, d_in=d_in, group=group, zeros=zeros, data=None), C.byref(size)) == 0
        return size.value

    assert of(1, 16, 64, 32, 0) == 512 + 2 * 16 * 2
    assert of(1, 16, 64, 64, 1) == 512 + 16 * 3
    assert of(3, 17, 65, 128, 0) == 3 * (2 * 2 * 512 + 32 * 2)
    assert of(1, 16, 4096, 1 << 30, 0) == 64 * 512 + 16 * 2
    assert of(1024, 4096, 2176, 128, 0) > 1 << 32


def test_rows_and_null_arguments():
    L = _lib.load()
    w, wz = weight(), weight(zeros=1)
    refused(L.th_pack4(w, None, 16, 128, P, None, None), "null codes")
    refused(L.th_pack4(w, P, 15, 128, P, None, None), "codes: the row stride")
    refused(L.th_pack4(w, P, 16, 128, None, None, None), "null scales")
    refused(L.th_pack4(w, P, 16, 128, P, P, None), "zeros")
    refused(L.th_pack4(wz, P, 16, 128, P, None, None), "zeros")
    refused(L.th_quantize4(w, None, 16, 128, None), "null values")
    refused(L.th_quantize4(w, P, 15, 128, None), "values: the row stride")
    refused(L.th_dequantize4(w, P, 15, 128, None), "values: the row stride")
    refused(L.th_weight4_bytes(w, None), "null output")
    refused(L.th_weight4_bytes(None, C.byref(C.c_size_t())), "null weight")


@pytest.mark.parametrize("change", [dict(dtype=2), dict(matrices=2), dict(matrices=4), dict(d_out=9), dict(d_in=17)])
def test_other_operands(change):
    L = _lib.load()
    text = "dtype" if "dtype" in change else "other sizes"
    refused(L.th_grouped_matmul4(grouped(), weight(**change), P, 8, P, 1 << 40, None), text)
    refused(L.th_grouped_matmul4_backward(grouped(), weight(**change), P, 8, P, P, 1 << 40, None), text)
    one = dict(dict(matrices=1), **change)
    refused(L.th_lora_linear4(lora(), weight(**one), P, 8, None, P, 1 << 40, None), text)
    refused(L.th_lora_linear4_backward(lora(), weight(**one), P, P, 8, P, P, P, P, P, 1 << 40, None), text)


def test_products():
    L = _lib.load()
    w, one, size = weight(), weight(matrices=1), C.c_size_t()
    # the 16-bit weights of the descriptors are not looked at
    assert L.th_grouped_matmul4_workspace(grouped(w=None, ldw=0), w, C.byref(size)) == 0
    assert L.th_lora_linear4_workspace(lora(weight=None, ldw=0), one, 0, C.byref(size)) == 0
    refused(L.th_grouped_matmul4(None, w, P, 8, P, 1 << 40, None), "null descriptor")
    refused(L.th_grouped_matmul4(grouped(), None, P, 8, P, 1 << 40, None), "null weight")
    refused(L.th_lora_linear4(lora(), None, P, 8, None, P, 1 << 40, None), "null weight")
    refused(L.th_grouped_matmul4(grouped(), w, P, 7, P, 1 << 40, None), "y: the row stride")
    refused(L.th_grouped_matmul4(grouped(), w, None, 8, P, 1 << 40, None), "null y")
    refused(L.th_grouped_matmul4_backward(grouped(), w, P, 8, None, P, 1 << 40, None), "null dx")
    refused(L.th_grouped_matmul4_backward(grouped(), w, None, 8, P, P, 1 << 40, None), "null dy")
    assert L.th_grouped_matmul4_backward_workspace(grouped(), w, C.byref(size)) == 0 and size.value > 0
    refused(L.th_grouped_matmul4_backward(grouped(), w, P, 8, P, P, size.value - 1, None), "bytes")
    assert L.th_lora_linear4_backward_workspace(lora(), one, C.byref(size)) == 0
    refused(L.th_lora_linear4_backward(lora(), one, P, P, 8, P, P, P, P, P, size.value - 1, None), "bytes")


def gate(**kw):
    d = dict(dtype=3, score=1, normalize=1, n_experts=8, choices=2, nodes=4, top_nodes=2, node_best=2, tokens=4, ld=8, mask_ld=0,
             logits=P, mask=None, bias=None, scale=1.0)
    d.update(kw)
    return C.byref(_lib.Gate(**d))


@pytest.mark.parametrize("change,text", [
    (dict(dtype=4), "dtype"), (dict(score=2), "score"), (dict(n_experts=513, ld=513, nodes=1, top_nodes=1), "512"), (dict(choices=0), "choices"),
    (dict(choices=9), "choices"), (dict(choices=5), "top_nodes nodes"), (dict(nodes=3), "equally"), (dict(nodes=0), "equally"),
    (dict(top_nodes=0), "top_nodes"), (dict(top_nodes=5), "top_nodes"), (dict(node_best=0), "node_best"), (dict(node_best=3), "node_best"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(ld=7), "row stride"), (dict(mask=P, mask_ld=7), "mask"), (dict(logits=None), "null logits"), (dict(tokens=-1), "negative")])
def test_gates(change, text):
    L = _lib.load()
    refused(L.th_gate(gate(**change), P, P, P, P, None, 0, None), text)
    refused(L.th_gate_backward(gate(**change), P, P, P, P, None), text)
    refused(L.th_gate_workspace(gate(**change), C.byref(C.c_size_t())), text)


def test_gate_outputs():
    L = _lib.load()
    refused(L.th_gate(None, P, P, P, P, None, 0, None), "null descriptor")
    refused(L.th_gate(gate(), None, P, P, P, None, 0, None), "null output")
    refused(L.th_gate_backward(gate(), P, P, None, P, None), "null argument")
    refused(L.th_gate(gate(tokens=1 << 20), P, P, P, P, None, 0, None), "workspace")
    size, plain = C.c_size_t(), C.c_size_t()
    assert L.th_gate_workspace(gate(tokens=5000), C.byref(size)) == 0 and size.value > 0
    refused(L.th_gate(gate(tokens=5000), P, P, P, P, P, size.value - 1, None), "bytes")
    # without a bias, nodes or sigmoids it is the plain gate, with its workspace
    assert L.th_gate_workspace(gate(tokens=5000, score=0, nodes=1, top_nodes=1), C.byref(size)) == 0
    assert L.th_group_workspace(5000, 8, 2, C.byref(plain)) == 0 and size.value == plain.value


def test_python_gate():
    l = torch.zeros(4, 8)
    for kw, text in ((dict(score="relu"), "score"), (dict(bias=torch.zeros(7)), "bias"), (dict(bias=torch.zeros(8, dtype=BF16)), "bias"),
                     (dict(bias=torch.zeros(8, requires_grad=True)), "no gradient"), (dict(nodes=0), "nodes"), (dict(nodes=9), "nodes"),
                     (dict(nodes=4, top_nodes=5), "top_nodes"), (dict(bias=torch.zeros(8)), "on the GPU")):
        with pytest.raises(ValueError, match=text):
            mixture.route(l, 2, **kw)


def four(*shape, dtype=BF16, group_size=32, zeros=False):
    """A weight with data of the right size on the CPU, which every call refuses in the end."""
    n, at = C.c_size_t(), len(shape) - 2
    w = _lib.Weight4(1, shape[0] if at else 1, shape[at], shape[at + 1], group_size, zeros, None)
    assert _lib.load().th_weight4_bytes(C.byref(w), C.byref(n)) == 0
    return mixture.Weight4(torch.zeros(n.value, dtype=torch.uint8), shape, dtype, group_size, zeros)


def test_python_weights():
    w = torch.zeros(8, 16, dtype=BF16)
    codes, scales = torch.zeros(8, 16, dtype=torch.uint8), torch.ones(8, 1, dtype=BF16)
    for call, text in (
            (lambda: mixture.quantize4(w, 48), "power of two"), (lambda: mixture.quantize4(w, 0), "group_size"),
            (lambda: mixture.quantize4(w.float(), 32), "bf16 or f16"), (lambda: mixture.quantize4(w[0], 32), "d_out, d_in"),
            (lambda: mixture.quantize4(w[:0], 32), "sizes"), (lambda: mixture.quantize4(w, 32), "on the GPU"),
            (lambda: mixture.pack4(codes.int(), scales, 32), "uint8"), (lambda: mixture.pack4(codes, scales.float(), 32), "bf16 or f16"),
            (lambda: mixture.pack4(codes, scales[:7], 32), "scales"), (lambda: mixture.pack4(codes, scales, 32, zeros=scales), "uint8"),
            (lambda: mixture.pack4(codes, scales, 32, zeros=codes), "zeros"), (lambda: mixture.pack4(codes, scales, 32), "on the GPU"),
            (lambda: mixture.dequantize4(four(8, 16)), "on the GPU"),
            (lambda: mixture.dequantize4(four(8, 16)._replace(dtype=torch.float32)), "dtype"),
            (lambda: mixture.dequantize4(four(8, 16)._replace(shape=(8, 200))), "pack4 or quantize4"),
            (lambda: mixture.dequantize4(four(8, 16)._replace(data=torch.zeros(4096, dtype=torch.int8))), "pack4 or quantize4"),
            (lambda: mixture.dequantize4(four(8, 16)._replace(shape=(8, 0))), "sizes")):
        with pytest.raises(ValueError, match=text):
            call()


def test_python_products():
    x = torch.zeros(4, 16, dtype=BF16)
    ids = torch.zeros(4, 1, dtype=torch.int32)
    groups = mixture.Groups(ids, ids.view(-1), torch.zeros(4, dtype=torch.int32), 3)
    a, b = torch.zeros(3, 4, 16, dtype=BF16), torch.zeros(3, 8, 4, dtype=BF16)
    for w, text in ((four(3, 8, 16), "on the GPU"), (four(2, 8, 16), "n_groups"), (four(8, 16), "n_groups"),
                    (four(3, 8, 16, dtype=torch.float16), "one type"), (four(3, 8, 24), "x must be")):
        with pytest.raises(ValueError, match=text):
            mixture.grouped_matmul(x, w, groups)
    for w, text in ((four(8, 16), "on the GPU"), (four(1, 8, 16), "weight"), (four(8, 16, dtype=torch.float16), "x's type"),
                    (four(8, 24), "d_in"), (four(9, 16), "lora_b")):
        with pytest.raises(ValueError, match=text):
            mixture.lora_linear(x, w, a, b, ids)


def test_modes():
    """Forward-mode derivatives and tracing are refused, as for the other operators."""
    w, s = torch.zeros(8, 16, dtype=BF16), torch.ones(8, 1, dtype=BF16)
    codes = torch.zeros(8, 16, dtype=torch.uint8)
    x, ids = torch.zeros(4, 16, dtype=BF16), torch.zeros(4, 1, dtype=torch.int32)
    groups = mixture.Groups(ids, ids.view(-1), torch.zeros(4, dtype=torch.int32), 3)
    a, b = torch.zeros(3, 4, 16, dtype=BF16), torch.zeros(3, 8, 4, dtype=BF16)
    calls = {"quantize4": (lambda v: mixture.quantize4(v, 32).data, w), "pack4": (lambda v: mixture.pack4(codes, v, 32).data, s),
             "grouped": (lambda v: mixture.grouped_matmul(v, four(3, 8, 16), groups), x),
             "lora": (lambda v: mixture.lora_linear(v, four(8, 16), a, b, ids), x),
             "route": (lambda v: mixture.route(v, 2, score="sigmoid").weights, torch.zeros(4, 8)),
             "bias": (lambda v: mixture.route(torch.zeros(4, 8), 2, bias=v).weights, torch.zeros(8))}
    for call, v in calls.values():
        with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            call(forward_ad.make_dual(v, torch.ones_like(v)))
        with pytest.raises(NotImplementedError, match="trace"):
            torch.jit.trace(call, (v,))
    with pytest.raises(NotImplementedError, match="trace"):
        torch.jit.trace(lambda v: mixture.dequantize4(four(8, 16)._replace(data=v)), (four(8, 16).data,))
