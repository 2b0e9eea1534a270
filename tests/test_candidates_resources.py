"""Registers and scratch of the built kernels of a step of several candidates, read from the library's code objects."""
from __future__ import annotations

import pytest
from test_kernel_resources import _find


@pytest.mark.parametrize("kernel,forms", [("13shared_kernelI", 30), ("18shared_join_kernelI", 16), ("13logits_kernelI", 45),
                                          ("13sample_kernelI", 9)])
def test_values_stay_in_registers(kernel, forms):
    """No vector register is spilled and no array lies in scratch."""
    found = _find(kernel)
    assert len(found) >= forms
    for k in found:
        assert k[".vgpr_spill_count"] == 0 and k[".private_segment_fixed_size"] == 0, k[".name"]


@pytest.mark.parametrize("hd,nt,most", [(64, 0, 168), (64, 1, 168), (64, 2, 168), (128, 0, 168), (128, 1, 168), (128, 2, 256),
                                        (256, 0, 256), (256, 1, 256), (256, 2, 512)])
def test_workgroups_share_a_cu(hd, nt, most):
    """Workgroups of four waves that a CU has registers for: three of 64 and 128 values, two of 256, one less with two
    tiles of rows where sums are larger."""
    found = [k for k in _find("13shared_kernelI") if f"Li{hd}E" in k[".name"] and f"Li{nt}EEEv" in k[".name"]]
    assert len(found) == (2 if nt == 2 else 4)
    for k in found:
        assert k[".vgpr_count"] <= most, (k[".name"], k[".vgpr_count"])
