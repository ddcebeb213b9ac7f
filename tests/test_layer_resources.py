"""Register spills of the kernels around the block, from the code objects' own metadata."""
from pathlib import Path

import pytest

from tests.test_kernel_resources import _gpu_images, _kernels
from trifuse_amd import _lib


@pytest.mark.parametrize("name,least", [("igemm_tile_kernel", 11), ("igemm_few_kernel", 12), ("token_logprobs_kernel", 6),
                                        ("norm_residual_kernel", 28), ("quantize_kernel", 28)])
def test_kernels_keep_their_registers(name, least):
    data = Path(_lib.LIB_PATH).read_bytes()
    found = {k[".name"]: k for image in _gpu_images(data) for k in _kernels(image) if name in k[".name"]}
    assert len(found) >= least
    bad = {n: (k[".vgpr_spill_count"], k[".private_segment_fixed_size"]) for n, k in found.items()
           if k[".vgpr_spill_count"] or k[".private_segment_fixed_size"]}
    assert not bad
