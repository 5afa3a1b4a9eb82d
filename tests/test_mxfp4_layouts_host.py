"""CPU: which strides of an MXFP4 cache are taken."""

import pytest
import torch

from my_vllm_amd import ops

B = ops.MXFP4_PAGE_BYTES


def _cache(pages, heads, page_stride, head_stride):
    memory = torch.zeros(B + page_stride * (pages - 1) + head_stride * (heads - 1), dtype=torch.uint8)
    return memory.as_strided((pages, heads, B), (page_stride, head_stride, 1))


@pytest.mark.parametrize("layout", [(4, 2, 2 * B, B), (4, 2, B, 4 * B), (4, 2, 2 * B + 16, B), (4, 2, B + 16, 4 * B + 48),
                                    (1, 3, 16, B), (3, 1, B, 16), (1, 1, 0, 0), (2, 3, 3 * B, B)])
def test_blocks_apart_are_taken(layout):
    cache = _cache(*layout)
    ops._check_mxfp4_caches(cache, cache.clone(memory_format=torch.preserve_format) if cache.is_contiguous() else cache,
                            cache.device)
    seen = torch.zeros(cache.untyped_storage().nbytes(), dtype=torch.int32)
    pages, heads, page_stride, head_stride = layout
    for p in range(pages):
        for h in range(heads):
            first = p * page_stride + h * head_stride
            seen[first:first + B] += 1
    assert seen.max() == 1  # what the check is for


@pytest.mark.parametrize("layout", [(4, 2, B, B), (4, 2, 2 * B - 16, B), (4, 2, B, 4 * B - 16), (2, 2, B + 16, B),
                                    (3, 3, 2 * B, B), (2, 1, B - 16, B), (1, 2, B, B - 16), (2, 2, 0, B)])
def test_overlapping_blocks_are_refused(layout):
    cache = _cache(*layout)
    with pytest.raises(ValueError, match="apart"):
        ops._check_mxfp4_caches(cache, cache, cache.device)
