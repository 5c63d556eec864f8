"""Registers and LDS of the products with 4-bit weights; registers are read from the built library's kernel descriptors."""
import pytest

from test_mixture_kernel_resources import CU_LDS, find, kernels  # noqa: F401  (a fixture)


@pytest.mark.parametrize("mt,nt,wavefronts,workgroups", [(1, 1, 8, 1), (1, 2, 8, 1), (2, 2, 8, 1), (4, 2, 8, 1), (2, 2, 4, 3), (4, 2, 4, 2)])
def test_workgroups_of_a_cu(kernels, mt, nt, wavefronts, workgroups):
    """As many as the tiles' rule counts on, with adapters too: lora_linear's products always have them."""
    # two lines a wavefront: its rows' values, 1 KiB of codes, 256 bytes for scales and zeros
    lds = wavefronts * 2 * (16 * mt * (128 // nt) * 2 + 1024 + 256)
    found = find(kernels, f"narrow_kernelI.*Li{mt}ELi{nt}ELi{wavefronts}ELi2ELb0ELb1ELb[01]ELb1EE")
    assert len(found) == 4  # two types, with and without adapters
    for name, (per_simd, _, more) in found.items():
        assert min(4 * per_simd // wavefronts, CU_LDS // (lds + more)) >= workgroups, name
