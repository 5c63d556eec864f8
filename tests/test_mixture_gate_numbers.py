"""Numbers that 32 bits do not hold are refused by the gate, not taken for what their low bits say."""
import pytest
import torch

from provenloop_amd import mixture


@pytest.mark.parametrize("node_best", [-1, 0, 3, (1 << 32) + 1, (1 << 32) + 2, -(1 << 32) + 1])
def test_node_best(node_best):
    with pytest.raises(ValueError, match="node_best"):
        mixture.route(torch.zeros(4, 8), 2, nodes=4, top_nodes=2, node_best=node_best)


@pytest.mark.parametrize("name,value", [("nodes", (1 << 32) + 4), ("top_nodes", (1 << 32) + 2), ("top_nodes", -(1 << 32) + 2)])
def test_nodes(name, value):
    with pytest.raises(ValueError, match="nodes"):
        mixture.route(torch.zeros(4, 8), 2, **dict(dict(nodes=4, top_nodes=2), **{name: value}))
