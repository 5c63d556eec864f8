"""Registers, scratch and LDS of the balanced gate and of 4-bit weights' own kernels, read from the built library's kernel descriptors."""
import pytest

from test_mixture_kernel_resources import CU_LDS, find, kernels  # noqa: F401  (a fixture)


@pytest.mark.parametrize("name", ["16quantize4_kernel", "12pack4_kernel", "18dequantize4_kernel", "24balanced_backward_kernel"])
def test_no_scratch(kernels, name):
    for kernel, (_, scratch, _) in find(kernels, name).items():
        assert scratch == 0, kernel


# lanes of a token, chunks of 8 experts a lane, passes of 8 choices: bytes of scratch a lane at most. A workgroup of 16
# wavefronts has 128 registers a lane; above 128 experts, or above 64 with more than 8 choices, a few values do not fit.
SCRATCH = {(1, 1, 1): 0, (2, 1, 1): 0, (4, 1, 1): 0, (8, 1, 1): 0, (8, 2, 1): 0, (8, 4, 1): 28, (16, 4, 1): 56,
           (1, 1, 4): 0, (2, 1, 4): 0, (4, 1, 4): 0, (8, 1, 4): 0, (8, 2, 4): 44, (8, 4, 4): 260, (16, 4, 4): 260}


def test_scratch_of_the_balanced_gate(kernels):
    seen = 0
    for (lanes, chunks, passes), most in SCRATCH.items():
        for kernel, (_, scratch, _) in find(kernels, f"15balanced_kernelI.*Li{lanes}ELi{chunks}ELi{passes}EE").items():
            assert scratch <= most, kernel
            seen += 1
    assert seen == len(find(kernels, "15balanced_kernelI")) == 3 * len(SCRATCH)


def test_a_workgroup_of_the_balanced_gate_fits_a_cu(kernels):
    """16 wavefronts, 4 a SIMD; LDS: numbers of the lanes or doubles of the wavefronts, biases, and 17 words an expert and one more."""
    for lanes, chunks, _ in SCRATCH:
        numbers, exact = 1024 * 3 * chunks * 4, 16 * 64 * max(1, lanes * chunks // 8) * 8
        lds = max(numbers, exact) + 8 * lanes * chunks * 4 + 17 * (8 * lanes * chunks + 1) * 4
        for kernel, (per_simd, _, more) in find(kernels, f"15balanced_kernelI.*Li{lanes}ELi{chunks}ELi").items():
            assert per_simd >= 4 and lds + more <= CU_LDS, kernel
