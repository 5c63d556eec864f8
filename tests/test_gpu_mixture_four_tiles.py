"""Products with 4-bit weights through every tile that a rule picks, with and without adapters (see test_mixture_four_tiles.py).

The comparisons and their tolerances are those of test_gpu_mixture_four.py, at sizes in the middle of each tile's range: ragged
last tiles in rows and columns, contractions that end inside a line, groups of unequal size and empty ones.
"""
import pytest

import test_gpu_mixture_four as four

pytestmark = pytest.mark.gpu

# tokens, experts, choices, d_in, d_out, columns of a scale
GROUPED = [(9, 2, 2, 1539, 500, 32), (13, 6, 2, 1290, 1500, 64), (100, 4, 1, 1539, 1100, 128), (400, 2, 1, 1539, 1000, 64),
           (768, 64, 2, 520, 1500, 64), (512, 8, 1, 1539, 1570, 128), (511, 8, 1, 1600, 1600, 32)]
# tokens, adapters, choices, d_in, d_out, rank, columns of a scale; zeros where the tokens are even
LORA = [(9, 3, 2, 1539, 500, 12, 64), (20, 4, 1, 1290, 3570, 16, 256), (51, 3, 1, 1290, 3570, 8, 128), (200, 4, 1, 1536, 1500, 16, 64),
        (201, 2, 2, 1539, 1500, 33, 128), (380, 3, 2, 1536, 3570, 16, 64), (379, 5, 1, 1290, 3570, 5, 32), (230, 5, 1, 1539, 3570, 20, 128),
        (255, 32, 1, 1536, 3584, 32, 128)]


@pytest.mark.parametrize("dtype,zeros", [("bf16", False), ("bf16", True), ("f16", False), ("f16", True)])
@pytest.mark.parametrize("t,e,k,din,dout,size", GROUPED)
def test_grouped_matmul(dtype, zeros, t, e, k, din, dout, size):
    four.test_grouped_matmul(dtype, zeros, t % 2 == 0, t, e, k, din, dout, size)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("t,e,k,din,dout,rank,size", LORA)
def test_lora_linear(dtype, t, e, k, din, dout, rank, size):
    four.test_lora_linear(dtype, t, e, k, din, dout, rank, size)
