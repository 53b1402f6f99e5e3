"""Scratch memory of the prompt and 4-bit attention kernels that do not fit their registers: no more than they were
measured with (bytes a lane)."""

from __future__ import annotations

import re

import pytest

from sva_amd import _lib

from .test_kernel_resources import kernels


def test_scratch_of_wide_and_padded_rows_stays_bounded():
    if not _lib.LIB_PATH.exists():
        pytest.skip("the library is not built")
    prompt, cache4 = {}, {}
    for name, k in kernels(_lib.LIB_PATH).items():
        m = re.search(r"prompt_kernelILi(\d+)ELi(\d+)ELi(\d+)E", name)
        if m:
            prompt[tuple(map(int, m.groups()))] = k[".private_segment_fixed_size"]
        m = re.search(r"cache4_attention_kernelILi(\d+)ELb(\d)ELi(\d+)E", name)
        if m:
            cache4[tuple(map(int, m.groups()))] = k[".private_segment_fixed_size"]
    # type (fp32, bf16, fp16) x head_dim x form, and the few-row forms of the 16-bit types
    assert len(prompt) == 27 + 18 and len(cache4) == 18
    for (dtype, dim, form), size in prompt.items():
        most = 0 if dim == 64 or (dim == 128 and (dtype == 0 or form >= 4)) else 96 if dim == 128 else 480
        assert size <= most, (dtype, dim, form, size)
    for (blocks, padded, terms), size in cache4.items():
        assert size <= (0 if not padded or blocks == 8 or terms == 1 else 48 if terms == 2 else 240), (blocks, terms)
