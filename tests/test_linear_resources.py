"""The built gfx950 code objects: linear attention's and layer norm's kernels use no scratch.

The gradient walk keeps its operands in up to 256 registers and its next tiles' loads in flight: a
spilled one is waited for behind every load before it, which cost a tenth of the kernel where it
happened.  Reads the AMDGPU metadata of avelang_amd/libgdn.so as the chains' test does; CPU only.
"""
import pytest

from test_kernel_resources import kernels  # noqa: F401  (the fixture)

GUARDED = ("lin_grad_kernel", "lin_walk_kernel", "lin_segment_kernel", "lin_join_kernel",
           "lin_recurrent_kernel", "norm_fwd_kernel", "norm_bwd_kernel")


@pytest.mark.parametrize("name", GUARDED)
def test_no_scratch(kernels, name):  # noqa: F811
    found = {k: v for k, v in kernels.items() if name in k}
    assert found
    for k, v in found.items():
        assert v.get("private_segment_fixed_size", 0) == 0 and v.get("vgpr_spill_count", 0) == 0, k
