"""What the plain mixture-of-adapters operators refuse, before anything reaches a GPU."""
import ctypes as C

import pytest
import torch

from provenloop_amd import _lib

mixture = pytest.importorskip("provenloop_amd.mixture")

P = 0x1000  # a pointer that a check looks at and nothing reads


def refused(rc, text):
    assert rc == _lib.TH_EINVAL and text in _lib.last_error(), (rc, _lib.last_error())


def test_group_and_route():
    L = _lib.load()
    size = C.c_size_t()
    refused(L.th_group_workspace(-1, 3, 1, C.byref(size)), "negative")
    refused(L.th_group_workspace(5, 0, 1, C.byref(size)), "number of experts")
    refused(L.th_group_workspace(5, 1025, 1, C.byref(size)), "number of experts")
    refused(L.th_group_workspace(5, 3, 33, C.byref(size)), "choices")
    refused(L.th_group_workspace(1 << 30, 3, 2, C.byref(size)), "below 2^31")
    refused(L.th_group(None, 5, 3, 1, P, P, None, 0, None), "null argument")
    assert L.th_group_workspace(1 << 20, 3, 2, C.byref(size)) == 0 and size.value > 0
    refused(L.th_group(P, 1 << 20, 3, 2, P, P, None, 0, None), "workspace")
    refused(L.th_group(P, 1 << 20, 3, 2, P, P, 0x1000, size.value - 1, None), "bytes")
    refused(L.th_group(P, 1 << 20, 3, 2, P, P, 0x1010, size.value, None), "256")

    def route(dtype=1, ld=8, t=4, e=8, mask_ld=0, k=2):
        return L.th_route(dtype, P, ld, t, e, P, mask_ld, k, 1, P, P, P, P, None, 0, None)

    refused(route(dtype=4), "dtype")
    refused(route(ld=7), "row stride")
    refused(route(k=9), "choices")
    refused(route(k=0), "choices")
    refused(route(e=513, ld=513), "512")
    refused(route(mask_ld=7), "mask")


def grouped(**kw):
    d = dict(dtype=1, x_per_slot=0, tokens=4, choices=2, experts=3, d_in=16, d_out=8, x=P, w=P, ldx=16, ldw=16, ldwe=128,
             order=P, offsets=P)
    d.update(kw)
    return C.byref(_lib.Grouped(**d))


@pytest.mark.parametrize("change,text", [
    (dict(dtype=3), "dtype"), (dict(tokens=-1), "negative"), (dict(choices=0), "choices"), (dict(experts=0), "experts"),
    (dict(d_in=0), "positive"), (dict(d_out=0), "positive"), (dict(x=None), "null x"), (dict(w=None), "null w"),
    (dict(ldx=15), "x: the row stride"), (dict(ldw=15), "w: the row stride"), (dict(order=None), "null groups"),
    (dict(tokens=1 << 30), "below 2^31")])
def test_grouped(change, text):
    L = _lib.load()
    refused(L.th_grouped_matmul(grouped(**change), P, 8, None), text)
    refused(L.th_grouped_matmul_backward(grouped(**change), P, 8, P, P, P, 1 << 40, None), text)


def test_grouped_outputs():
    L = _lib.load()
    refused(L.th_grouped_matmul(None, P, 8, None), "null descriptor")
    refused(L.th_grouped_matmul(grouped(), None, 8, None), "null y")
    refused(L.th_grouped_matmul(grouped(), P, 7, None), "y: the row stride")
    refused(L.th_grouped_matmul_backward(grouped(), P, 8, P, P, None, 0, None), "workspace")


def lora(**kw):
    d = dict(dtype=1, choices=2, tokens=4, d_in=16, d_out=8, rank=4, adapters=3, x=P, weight=P, bias=None, a=P, b=P, ldx=16,
             ldw=16, lda=16, lda_adapter=64, ldb=4, ldb_adapter=32, experts=P, gate=None, scale=None, order=None, offsets=None)
    d.update(kw)
    return C.byref(_lib.LoraLinear(**d))


@pytest.mark.parametrize("change,text", [
    (dict(dtype=3), "dtype"), (dict(rank=0), "rank"), (dict(rank=129), "rank"), (dict(adapters=1025), "experts"),
    (dict(x=None), "null x"), (dict(weight=None), "null weight"), (dict(a=None), "null weight"), (dict(experts=None), "experts"),
    (dict(lda=15), "a: the row stride"), (dict(ldb=3), "b: the row stride"), (dict(ldw=15), "weight: the row stride"),
    (dict(order=P), "go together"), (dict(d_out=0), "positive")])
def test_lora(change, text):
    L = _lib.load()
    refused(L.th_lora_linear(lora(**change), P, 8, None, 0x1000, 1 << 40, None), text)
    refused(L.th_lora_linear_backward(lora(**change), P, P, 8, P, P, P, P, 0x1000, 1 << 40, None), text)


def test_lora_workspaces():
    L = _lib.load()
    size = C.c_size_t()
    assert L.th_lora_linear_backward_workspace(lora(), C.byref(size)) == 0
    refused(L.th_lora_linear_backward(lora(), P, P, 8, P, P, P, P, 0x1000, size.value - 1, None), "bytes")
    refused(L.th_lora_linear_backward(lora(), None, P, 8, None, None, P, None, 0x1000, size.value, None), "null u")
    refused(L.th_lora_linear(lora(), P, 7, None, 0x1000, 1 << 40, None), "y: the row stride")


def test_python_arguments():
    x = torch.zeros(4, 16, dtype=torch.bfloat16)
    ids = torch.zeros(4, 1, dtype=torch.int32)
    with pytest.raises(ValueError, match="on the GPU"):
        mixture.route(torch.zeros(4, 8), 2)
    with pytest.raises(ValueError, match="bf16, f16 or f32"):
        mixture.route(torch.zeros(4, 8, dtype=torch.float64), 2)
    with pytest.raises(ValueError, match="on the GPU"):
        mixture.group(ids, 3)
    with pytest.raises(ValueError, match="int32"):
        mixture.group(ids.long(), 3)
    with pytest.raises(ValueError, match="int32"):
        mixture.lora_linear(x, torch.zeros(8, 16, dtype=torch.bfloat16), torch.zeros(3, 4, 16, dtype=torch.bfloat16),
                            torch.zeros(3, 8, 4, dtype=torch.bfloat16), ids.long())
    with pytest.raises(ValueError, match="weight must have x's type"):
        mixture.lora_linear(x, torch.zeros(8, 16), torch.zeros(3, 4, 16, dtype=torch.bfloat16),
                            torch.zeros(3, 8, 4, dtype=torch.bfloat16), ids)
    with pytest.raises(ValueError, match="lora_b must be"):
        mixture.lora_linear(x, torch.zeros(8, 16, dtype=torch.bfloat16), torch.zeros(3, 4, 16, dtype=torch.bfloat16),
                            torch.zeros(3, 8, 5, dtype=torch.bfloat16), ids)
    groups = mixture.Groups(ids, ids.view(-1), torch.zeros(4, dtype=torch.int32), 3)
    with pytest.raises(ValueError, match="w must be"):
        mixture.grouped_matmul(x, torch.zeros(2, 8, 16, dtype=torch.bfloat16), groups)
    with pytest.raises(ValueError, match="x must be"):
        mixture.grouped_matmul(x[:3], torch.zeros(3, 8, 16, dtype=torch.bfloat16), groups)
    with pytest.raises(ValueError, match="one type"):
        mixture.grouped_matmul(x, torch.zeros(3, 8, 16), groups)
