"""The kernels that walk many queries' rows use all registers that there are: the compiled code keeps none of them in memory.  Runs without a GPU, as
test_inflight_registers.py."""

import re
import shutil

import pytest

from ajllm_amd import asm_check

SOURCE = """
#include "tree_attention.h"
namespace ajq {
template __global__ void shared_attention_walk_kernel<128, uint16_t, 2>(SharedAttention);
template __global__ void shared_attention_walk_kernel<128, float, 1>(SharedAttention);
template __global__ void shared_attention_many_kernel<128, float, 2>(SharedAttention);
template __global__ void tree_attention_walk_kernel<128, uint16_t, 2, 4>(TreeAttention);
template __global__ void tree_attention_walk_kernel<128, uint16_t, 2, 8>(TreeAttention);
template __global__ void tree_attention_laid_kernel<128, float, 2, false>(TreeAttention);
}
"""


@pytest.mark.skipif(shutil.which("hipcc") is None, reason="needs hipcc")
def test_kernels_of_many_queries_spill_no_register():
    listing = asm_check.compile_device_asm(SOURCE)
    for what in ("private_segment_fixed_size", "vgpr_spill_count", "sgpr_spill_count"):
        found = dict(zip(re.findall(r"^    \.name: +(\S+)", listing, flags=re.M), re.findall(rf"^    \.{what}: +(\d+)", listing, flags=re.M)))
        assert len([name for name in found if "_walk_" in name or "_many_" in name or "_laid_" in name]) == 6, sorted(found)
        assert set(found.values()) == {"0"}, (what, found)
    assert "scratch_" not in listing
