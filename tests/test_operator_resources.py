"""Registers of the prompt and 4-bit attention kernels, from the metadata that the compiler leaves in the library: a tile
that went through scratch memory cost 231 us for 8192 tokens against 143."""

from __future__ import annotations

import pytest

from sva_amd import _lib

from .test_kernel_resources import kernels


def test_tiles_stay_in_registers():
    if not _lib.LIB_PATH.exists():
        pytest.skip("the library is not built")
    found = kernels(_lib.LIB_PATH)
    prompt = {k: v for k, v in found.items() if "prompt_kernelILi1ELi64ELi0E" in k or "prompt_kernelILi2ELi64ELi0E" in k}
    cache4 = {k: v for k, v in found.items() if "cache4_attention_kernel" in k and "ELb0E" in k}
    assert len(prompt) == 2 and len(cache4) == 12  # two 16-bit types; four widths of three query types
    for name, k in {**prompt, **cache4}.items():
        assert k[".private_segment_fixed_size"] == 0 and k[".vgpr_spill_count"] == 0, name
    wide = {k: v for k, v in found.items() if "prompt_kernelILi1ELi128ELi0E" in k or "prompt_kernelILi2ELi128ELi0E" in k}
    assert len(wide) == 2 and all(k[".private_segment_fixed_size"] <= 64 for k in wide.values())
