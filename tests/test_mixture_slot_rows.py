"""Row strides of what has a row per slot are checked by the number of slots, also for a single token. Nothing here reaches a GPU."""
import ctypes as C

from provenloop_amd import _lib
from test_mixture_refusals import P, grouped, refused


def test_rows_of_a_single_tokens_slots():
    L = _lib.load()
    refused(L.th_grouped_matmul(grouped(tokens=1), P, 7, None), "y: the row stride")
    refused(L.th_grouped_matmul(grouped(tokens=1), P, 0, None), "y: the row stride")
    refused(L.th_grouped_matmul(grouped(tokens=1, x_per_slot=1, ldx=15), P, 8, None), "x: the row stride")
    refused(L.th_grouped_matmul_backward(grouped(tokens=1), P, 7, P, P, P, 1 << 40, None), "dy: the row stride")
    refused(L.th_grouped_matmul_backward(grouped(tokens=1, x_per_slot=1, ldx=15), P, 8, P, P, P, 1 << 40, None), "x: the row stride")
    size = C.c_size_t()
    refused(L.th_grouped_matmul_backward_workspace(grouped(tokens=1, x_per_slot=1, ldx=15), C.byref(size)), "x: the row stride")
    # a single row has no stride
    assert L.th_grouped_matmul_backward_workspace(grouped(tokens=1, ldx=0), C.byref(size)) == 0
    assert L.th_grouped_matmul_backward_workspace(grouped(tokens=1, choices=1, x_per_slot=1, ldx=0), C.byref(size)) == 0
