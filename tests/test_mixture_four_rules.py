"""Rules on sizes for 4-bit weights and for gates with balanced choices (mixture_rules.h), evaluated by a host program."""
from test_mixture_rules import evaluate  # noqa: F401  (a fixture)


def test_bytes(evaluate):
    """Blocks of 16 rows x 64 columns of codes; a scale, and with zeros a byte, for each row of them and each group."""
    cases = [(r, c, g, z) for r in (1, 15, 16, 17, 256, 1536) for c in (2, 62, 64, 66, 1536, 3584) for g in (32, 64, 128, 1 << 12, 1 << 30)
             for z in (0, 1)]
    got = evaluate([f"four_bytes(four_layout({r}, {c}, {g}), 3, {z})" for r, c, g, z in cases])
    for (rows, cols, group, zeros), size in zip(cases, got):
        strips, blocks = -(-rows // 16), -(-cols // 64)
        groups = -(-blocks * 64 // group)
        assert size == 3 * (strips * blocks * 512 + groups * strips * 16 * (2 + zeros))


def test_large_matrices_pass_32_bits(evaluate):
    got, = evaluate(["four_bytes(four_layout(1 << 20, 1 << 16, 128), 8, 1)"])
    assert got == 8 * ((1 << 35) + (1 << 29) * 3)


def test_which_products_keep_the_codes(evaluate):
    """Each side as measured: decodes and small batches, and many small groups, keep them; large products take values."""
    cases = {(1, 1536, 1536, 1): 1, (256, 3584, 3584, 1): 1, (512, 3584, 3584, 1): 1, (768, 3584, 3584, 1): 0, (1024, 1536, 1536, 1): 1,
             (4096, 1536, 1536, 1): 0, (8192, 3584, 3584, 1): 0, (32, 512, 3584, 8): 1, (800, 1536, 3584, 8): 1, (2048, 1536, 1536, 8): 0,
             (1536, 1536, 1536, 64): 1, (4096, 512, 1536, 16): 0, (16384, 3584, 1536, 8): 0}
    assert evaluate([f"four_narrow({r}, {n}, {k}, {g})" for r, n, k, g in cases]) == list(cases.values())


def test_which_tile(evaluate):
    cases = {(1, 1536, 1): "16x16", (16, 3584, 1): "16x16", (200, 256, 1): "16x16", (32, 512, 8): "16x16",
             (16, 8192, 1): "16x32", (32, 3584, 8): "16x32", (32, 3584, 1): "16x32", (64, 3584, 1): "32x32_ONCE",
             (128, 3584, 1): "64x32_ONCE", (1021, 512, 1): "64x32_ONCE", (384, 3584, 1): "32x32", (512, 1536, 8): "32x32",
             (1536, 1536, 64): "32x32", (256, 3584, 1): "64x32", (512, 3584, 1): "64x32"}
    assert evaluate([f"four_tile({r}, {n}, {g}) == FOUR_{t}" for (r, n, g), t in cases.items()]) == [1] * len(cases)


def test_every_tile_is_reached(evaluate):
    """No variant of the kernel is without a product that keeps its codes and takes it."""
    sizes = [(r, n, 1536, 1) for r in (1, 32, 64, 128, 256, 384) for n in (256, 1536, 3584)]
    got = evaluate([f"four_narrow({r}, {n}, {k}, {g}) ? four_tile({r}, {n}, {g}) : -1" for r, n, k, g in sizes])
    assert set(got) - {-1} == set(range(6))


def test_gate_chunks_cover_the_tokens_and_stay_few(evaluate):
    cases = [(t, k) for t in (1, 2, 63, 64, 1023, 2049, 4099, 8192, 8193, 65536, 1 << 20, 1 << 26, (1 << 31) // 32 - 1) for k in (1, 6, 8, 32)
             if t * k < 1 << 31]
    tokens = evaluate([f"gate_chunk_tokens({t}, {k})" for t, k in cases])
    chunks = evaluate([f"gate_chunks({t}, {k})" for t, k in cases])
    for (t, k), per, n in zip(cases, tokens, chunks):
        assert per >= 1 and n * per >= t > (n - 1) * per
        assert n <= 1100  # every workgroup adds up the others' counts
