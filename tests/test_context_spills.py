"""Registers that the tiled kernels of attention over a context in two parts spill (host only): to memory at most 16 in f32 and two above head_dim 128 in 16 bits, none below."""
from test_kernel_registers import kernels  # noqa: F401


def test_vector_registers(kernels):  # noqa: F811
    tiled = {k: v["vgpr_spill_count"] for k, v in kernels.items() if "rows_kernel" not in k and ("ContextParams" in k or "ContextBoth" in k)}
    assert len(tiled) > 40
    for name, spilled in tiled.items():
        most = 16 if "prefill_f32_terms_kernel" in name else 2 if "wide_rows32" in name else 0
        assert spilled <= most, (name, spilled)
