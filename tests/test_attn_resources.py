"""Registers and scratch of the built attention kernels, read from the library's code objects."""
from __future__ import annotations

import pytest
from test_kernel_resources import _find


@pytest.mark.parametrize("kernel", ["decode_kernelI", "prompt_kernelI", "prompt_join_kernelI", "rope_kernelI"])
def test_attention_kernels_keep_their_values_in_registers(kernel):
    """No vector register of theirs is spilled and none of their arrays lies in scratch."""
    found = [k for part in ("NS_4Bf16E", "NS_3F16E") for k in _find("113" + kernel if kernel[0] == "d" else kernel)
             if part in k[".name"]]
    assert len(found) >= 12
    for k in found:
        assert k[".vgpr_spill_count"] == 0 and k[".private_segment_fixed_size"] == 0, k[".name"]


@pytest.mark.parametrize("hd,most", [(64, 128), (128, 168), (256, 256)])
def test_attention_workgroups_share_a_cu(hd, most):
    """Workgroups of four waves that a CU has registers for: four of 64 values, three of 128, two
    of 256 (prompts that are not halved, decode steps)."""
    for k in _find(f"Li{hd}E"):
        name = k[".name"]
        if "prompt_kernelI" in name and "Li2EEEv" not in name or "113decode_kernelI" in name:
            assert k[".vgpr_count"] <= most, (name, k[".vgpr_count"])
