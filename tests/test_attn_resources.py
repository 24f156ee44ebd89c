"""The built gfx950 code objects: the kernels around the attention layers use no scratch (the attention's
loads stay on their way in up to 256 registers; a spilled one would be waited for behind all of them)."""
import pytest

from test_kernel_resources import kernels  # noqa: F401  (the fixture)

GUARDED = ("rms_fwd_kernel", "rms_bwd_kernel", "rotary_kernel", "paged_write_kernel", "paged_read_kernel",
           "paged_attn_kernel", "paged_attn_join_kernel")


@pytest.mark.parametrize("name", GUARDED)
def test_no_scratch(kernels, name):  # noqa: F811
    found = {k: v for k, v in kernels.items() if name in k}
    assert found
    for k, v in found.items():
        assert v.get("private_segment_fixed_size", 0) == 0 and v.get("vgpr_spill_count", 0) == 0, k
