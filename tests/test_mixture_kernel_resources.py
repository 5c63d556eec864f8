"""Registers, scratch and LDS of the mixture operators' kernels, read from the built library's kernel descriptors.

Their tile rules count on a number of wavefronts per SIMD and workgroups per CU.
"""
import os
import re
import struct

import pytest

from test_kernel_resources import LIB, _kernels

BF16, F16 = "DF16b", "DF16_"
CU_LDS = 160 << 10


@pytest.fixture(scope="module")
def kernels():
    """{mangled name: (wavefronts per SIMD its registers allow, scratch bytes per lane, LDS bytes beside what a launch asks for)}"""
    if not os.path.exists(LIB):
        pytest.skip("the HIP library is not built")
    lib = open(LIB, "rb").read()
    out = {}
    for m in re.finditer(b"__CLANG_OFFLOAD_BUNDLE__", lib):
        count, = struct.unpack_from("<Q", lib, m.start() + 24)
        if count > 16:
            continue  # the magic as a string, not a bundle
        pos = m.start() + 32
        for _ in range(count):
            off, size, idlen = struct.unpack_from("<QQQ", lib, pos)
            target = lib[pos + 24:pos + 24 + idlen]
            pos += 24 + idlen
            if b"gfx950" not in target:
                continue
            for name, kd in _kernels(lib[m.start() + off:m.start() + off + size]):
                lds, scratch = struct.unpack_from("<II", kd)
                rsrc1, = struct.unpack_from("<I", kd, 48)
                out[name] = (min(8, 512 // (8 * ((rsrc1 & 63) + 1))), scratch, lds)
    assert out
    return out


def find(kernels, pattern):
    found = {n: v for n, v in kernels.items() if re.search(pattern, n)}
    assert found, pattern
    return found


def test_scratch(kernels):
    """Only the 256 x 256 products of y = x w have any: a few addresses outside their main loop."""
    for name, (_, scratch, _) in find(kernels, "narrow_kernel|wide_kernel|unaligned_kernel|outer_kernel|low_sum|route|place_kernel|count_kernel").items():
        square = re.search("wide_kernelI.*Li256ELi256ELi2ELi4ELi2ELb1E", name)
        assert scratch <= (24 if square else 0), name


@pytest.mark.parametrize("pattern,waves", [
    ("wide_kernelI", 2),                                    # 8 wavefronts, one workgroup a CU
    ("12outer_kernelI", 4),                                 # 8 wavefronts, two workgroups
    ("narrow_kernelI.*Li1ELi1ELi8ELi2E", 4),                # 8 wavefronts, two workgroups
    ("narrow_kernelI.*Li1ELi1ELi4ELi2ELb.ELb1ELb.E", 5),    # 4 wavefronts, five workgroups
    ("narrow_kernelI.*Li2ELi2ELi4ELi2E", 2),
    ("low_outer_kernelI.*Li1E", 2),                         # 4 wavefronts, two workgroups
    ("low_outer_kernelI.*Li[248]E", 1),                     # one
    ("unaligned_(outer_)?kernelI", 2)])                     # 4 wavefronts, two workgroups
def test_wavefronts(kernels, pattern, waves):
    for name, (w, _, _) in find(kernels, pattern).items():
        assert w >= waves, name


def test_two_low_rank_gradients_share_a_cu(kernels):
    """Up to rank 16 a workgroup asks for half a CU's LDS: any more beside it would leave the CU to one."""
    for name, (_, _, lds) in find(kernels, "low_outer_kernelI.*Li1E").items():
        assert 2 * (256 * (128 * 2 + 2 * 16 * 2) + lds) <= CU_LDS, name
