"""A bias of -inf withholds its expert from every token of a balanced gate, also where the expert's score is NaN."""
import pytest
import torch

from test_gpu_mixture import TYPES, check_groups

pytestmark = pytest.mark.gpu

mixture = pytest.importorskip("provenloop_amd.mixture")

INF, NAN = float("inf"), float("nan")


def chosen(rows, bias, k, dtype="f32", **o):
    r = mixture.route(torch.tensor(rows, device="cuda", dtype=TYPES[dtype]), k, bias=torch.tensor(bias, device="cuda"), **o)
    check_groups(r.groups, len(bias))
    return r.experts.tolist(), r.weights.cpu()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_sigmoids(dtype):
    ids, w = chosen([[NAN, 1.0, 2.0, 3.0], [0.0, NAN, 2.0, 3.0]], [-INF, 0.0, 0.0, 0.0], 2, dtype, score="sigmoid")
    assert ids == [[3, 2], [1, 3]]  # a NaN that is not withheld is still the first choice
    s = torch.sigmoid(torch.tensor([3.0, 2.0], dtype=torch.float64))
    # a score: expf and its argument, a sum, a quotient; then a sum, a quotient and the scale: 10 steps at most
    torch.testing.assert_close(w[0].double(), s / s.sum(), rtol=10 * 2.0 ** -23, atol=0)
    # nothing is left
    ids, w = chosen([[NAN, NAN, INF, 3.0]], [-INF, -INF, -INF, 0.5], 3, dtype, score="sigmoid")
    assert ids == [[3, -1, -1]] and w[0].tolist() == [1, 0, 0]
    ids, w = chosen([[NAN, NAN]], [-INF, -INF], 2, dtype, score="sigmoid")
    assert ids == [[-1, -1]] and w[0].tolist() == [0, 0]


def test_softmax():
    """One infinite or NaN logit makes every share NaN; the withheld expert is no choice for that."""
    for bad in (INF, NAN):
        ids, _ = chosen([[bad, 1.0, 2.0, 3.0]], [-INF, 0.0, 0.0, 0.0], 3)
        assert ids == [[1, 2, 3]]


@pytest.mark.parametrize("per", [2, 8, 40])
def test_nodes(per):
    """Nor does its node count as NaN: node 1 has the larger scores and is kept."""
    rows, bias = [[NAN] + [0.0] * (per - 1) + [5.0, 4.0] + [-9.0] * (per - 2)], [-INF] + [0.0] * (2 * per - 1)
    for best in (1, 2):
        ids, _ = chosen(rows, bias, 2, score="sigmoid", nodes=2, top_nodes=1, node_best=best)
        assert ids == [[per, per + 1]]
