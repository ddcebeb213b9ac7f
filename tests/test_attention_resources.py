"""Registers of the rotary, cache and attention kernels, from the code objects' own metadata."""
from pathlib import Path

import pytest

from tests.test_kernel_resources import _gpu_images, _kernels
from trifuse_amd import _lib


@pytest.mark.parametrize("name,least", [("rotary_kernel", 2), ("cache_append_kernel", 20), ("cache_read_kernel", 6),
                                        ("attention_few_kernel", 8), ("attention_tile_kernel", 12), ("attention_join_kernel", 8)])
def test_no_spills(name, least):
    data = Path(_lib.LIB_PATH).read_bytes()
    found = {k[".name"]: k for image in _gpu_images(data) for k in _kernels(image) if name in k[".name"]}
    assert len(found) >= least, len(found)
    bad = {n: (k[".vgpr_spill_count"], k[".private_segment_fixed_size"]) for n, k in found.items()
           if k[".vgpr_spill_count"] or k[".private_segment_fixed_size"]}
    assert not bad
