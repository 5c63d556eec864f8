"""The mixture operators' rules on sizes (mixture_rules.h), evaluated by a host program."""
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "provenloop_amd", "csrc")


@pytest.fixture(scope="module")
def evaluate(tmp_path_factory):
    def run(exprs):
        d = tmp_path_factory.mktemp("rules")
        src, exe = d / "rules.cpp", d / "rules"
        body = "".join(f'  printf("%lld\\n", (long long)({e}));\n' for e in exprs)
        src.write_text('#include "mixture_rules.h"\n#include <stdio.h>\nusing namespace th;\nint main() {\n' + body + "}\n")
        subprocess.run(["g++", "-std=c++20", "-Wall", "-Werror", "-I", CSRC, str(src), "-o", str(exe)], check=True)
        return [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]

    return run


def test_chunks_cover_the_tokens_and_stay_few(evaluate):
    cases = [(t, k) for t in (1, 2, 63, 64, 1023, 1024, 2048, 2049, 65536, 1 << 20, 1 << 26, (1 << 31) // 32 - 1) for k in (1, 2, 8, 32)
             if t * k < 1 << 31]
    tokens = evaluate([f"group_chunk_tokens({t}, {k})" for t, k in cases])
    chunks = evaluate([f"group_chunks({t}, {k})" for t, k in cases])
    for (t, k), per, n in zip(cases, tokens, chunks):
        assert per >= 1 and n * per >= t > (n - 1) * per
        assert n <= 1100  # every workgroup adds up the others' counts
        if t * k <= 2048:
            assert n == 1 or per * k > 2048 - k


def test_partial_sums_have_places(evaluate):
    """Spans of any split of the slots among the adapters fit the number the workspace is laid out for."""
    for slots, adapters, cols in ((1, 1, 64), (1000, 7, 1536), (16384, 64, 3584), (32768, 1, 4096), (3, 300, 8)):
        span, = evaluate([f"lowrank_span({slots}, {cols})"])
        assert 256 <= span <= 2048
        most, = evaluate([f"lowrank_spans({slots}, {adapters}, {span})"])
        for split in ([slots], [1] * min(adapters, slots) + [slots - min(adapters, slots)],
                      [slots // adapters + (i < slots % adapters) for i in range(adapters)]):
            if len([s for s in split if s]) > adapters:
                split = [split[-1] + split[0]] + split[1:-1]
            assert sum(split) == slots and sum(-(-s // span) for s in split) <= most


def test_which_tiles(evaluate):
    """A decode's and a prefill's products take the kernels measured to be faster there."""
    narrow = {(1, 1536, 1536, 1): 1, (32, 3584, 3584, 1): 1, (250, 1536, 1536, 1): 1, (1021, 256, 1536, 1): 1, (256, 3584, 3584, 1): 1,
              (512, 3584, 3584, 1): 0, (1024, 1536, 1536, 1): 0, (8192, 3584, 3584, 1): 0, (8192, 32, 3584, 8): 1, (32, 512, 3584, 8): 1,
              (64, 4096, 512, 8): 0, (64, 3584, 3584, 8): 1}
    assert evaluate([f"narrow_product({r}, {n}, {k}, {g})" for r, n, k, g in narrow]) == list(narrow.values())
    tile = {(1, 1536, 1): 0, (32, 512, 8): 0, (8192, 16, 8): 3, (4096, 16, 8): 0, (32, 3584, 1): 1, (250, 1536, 1): 2, (1021, 256, 1): 2}
    assert evaluate([f"narrow_tile({r}, {n}, {g})" for r, n, g in tile]) == list(tile.values())
    square = {(8192, 3584, 1): 1, (4096, 1536, 1): 0, (16384, 3584, 8): 1, (8186, 1536, 16): 1, (8192, 8192, 1): 1}
    assert evaluate([f"wide_square({r}, {n}, {g})" for r, n, g in square]) == list(square.values())


def test_which_operands_are_copied(evaluate):
    assert evaluate([f"pad_operands({r}, {k})" for r, k in ((1, 203), (32, 1016), (33, 8), (1, 1024))]) == [0, 0, 1, 1]
