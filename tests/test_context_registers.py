"""Registers of the kernel for few rows of attention over a context in two parts: its plan counts on so many workgroups of four wavefronts per CU, one
wavefront of each on a SIMD (host only)."""
import pytest

from test_kernel_registers import kernels  # noqa: F401


@pytest.mark.parametrize("dims, workgroups", [(64, 3), (96, 2), (128, 2), (192, 2), (256, 2)])  # (f32 above 128: one)
def test_workgroups_per_cu(kernels, dims, workgroups):  # noqa: F811
    found = [(k, v) for k, v in kernels.items() if "context_rows_kernel" in k and f"Li{dims}ELi" in k]
    assert len(found) == (5 if dims <= 128 else 3)  # f32 in 16 columns, 16-bit types in 16 and in 32
    for k, v in found:
        at_once = 1 if dims > 128 and "context_rows_kernelIfL" in k else workgroups
        assert (v["vgpr_count"] + 7) // 8 * 8 * at_once <= 512, k
        assert v["group_segment_fixed_size"] * at_once <= 160 * 1024, k
        assert v["vgpr_spill_count"] == 0, k
