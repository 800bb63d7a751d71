"""The attention kernels keep everything in registers: o, Q, the scores and the loads in flight together come near the
limit of a wave, and one value in scratch would be moved in every tile."""
import pytest

from test_kernel_resources_cpu import kernels, matching      # noqa: F401 (a fixture)


@pytest.mark.parametrize("pattern,vgprs", [
    (r"void k_attn_rows<\w+, (64|128), ", 256),         # two waves per SIMD
    (r"void k_attn_rows<\w+, 256, ", 512),              # one
    (r"void k_attn_keys<\w+, (64|128), ", 256),
    (r"void k_attn_keys<\w+, 256, ", 512),
    (r"void k_attn_join<", 96),
])
def test_no_scratch(kernels, pattern, vgprs):            # noqa: F811
    over = {n: (k[".vgpr_count"], k[".vgpr_spill_count"], k[".private_segment_fixed_size"])
            for n, k in matching(kernels, pattern).items()
            if k[".vgpr_count"] > vgprs or k[".vgpr_spill_count"] or k[".private_segment_fixed_size"]}
    assert not over, over
