"""Registers of the paged attention and sampling kernels, from the metadata that the compiler leaves in the library: 20
registers in scratch memory cost a token of 32 sequences of up to 131072 rows 416 us against 297."""

from __future__ import annotations

import re

import pytest

from sva_amd import _lib

from .test_kernel_resources import kernels


def test_tiles_and_weights_stay_in_registers():
    if not _lib.LIB_PATH.exists():
        pytest.skip("the library is not built")
    attention, sample = 0, 0
    for name, k in kernels(_lib.LIB_PATH).items():
        if re.search(r"paged_attention_kernelILi\d+ELi\d+ELb\dE", name):
            attention += 1
        elif "sample_kernel" in name:
            sample += 1
        else:
            continue
        assert k[".private_segment_fixed_size"] == 0 and k[".vgpr_spill_count"] == 0, name
    assert attention == 18 and sample == 3  # three types of three widths, whole and padded; three types
