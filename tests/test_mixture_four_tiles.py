"""The sizes of test_gpu_mixture_four_tiles.py reach every tile of the products with 4-bit weights, with and without adapters."""
import test_gpu_mixture_four_tiles as cases
from test_mixture_rules import evaluate  # noqa: F401  (a fixture)

TILES = ["16x16", "16x32", "32x32_ONCE", "64x32_ONCE", "32x32", "64x32"]


def test_every_tile_has_a_product(evaluate):
    # rows, columns, contraction and groups as the product sees them: slots of E experts, or tokens of one weight
    for sizes in ([(t * k, dout, din, e) for t, e, k, din, dout, _ in cases.GROUPED],
                  [(t, dout, din, 1) for t, _, _, din, dout, _, _ in cases.LORA]):
        assert evaluate([f"four_narrow({r}, {n}, {k}, {g})" for r, n, k, g in sizes]) == [1] * len(sizes)
        assert set(evaluate([f"four_tile({r}, {n}, {g})" for r, n, k, g in sizes])) == set(evaluate([f"FOUR_{t}" for t in TILES]))
