"""MXFP4 caches of other strides on the GPU: taken and written block by block, or refused."""

import pytest
import torch

from my_vllm_amd import ops
from oracle import mxfp4

pytestmark = pytest.mark.gpu
B = ops.MXFP4_PAGE_BYTES


def _strided(gpu, page_stride, head_stride, pages=4, heads=2):
    size = B + page_stride * (pages - 1) + head_stride * (heads - 1)
    memory = torch.full((2, size), 0x33, dtype=torch.uint8, device=gpu)
    return memory, [m.as_strided((pages, heads, B), (page_stride, head_stride, 1), m.storage_offset()) for m in memory]


@pytest.mark.parametrize("page_stride,head_stride", [(2 * B, B), (B, 4 * B), (2 * B + 16, B), (B + 16, 4 * B + 48)])
def test_strided_caches(gpu, page_stride, head_stride):
    memory, (kc, vc) = _strided(gpu, page_stride, head_stride)
    gen = torch.Generator().manual_seed(1)
    k, v = (torch.randn(20, 2, 128, generator=gen).to(torch.bfloat16) for _ in range(2))
    slots = torch.randperm(64, generator=gen)[:20]
    ops.store_kvcache_mxfp4(k.to(gpu), v.to(gpu), kc, vc, slots.to(gpu))
    inside = torch.zeros(memory.size(1), dtype=torch.bool)
    for p in range(4):
        for h in range(2):
            inside[p * page_stride + h * head_stride:][:B] = True
    for rows, cache, raw in ((k, kc, memory[0]), (v, vc, memory[1])):
        want = torch.full((4, 2, B), 0x33, dtype=torch.uint8)
        mxfp4.store(rows, want, slots.tolist())
        assert torch.equal(cache.cpu(), want)
        assert (raw.cpu()[~inside] == 0x33).all()
    for got, cache in zip(ops.load_kvcache_mxfp4(kc, vc, slots.to(gpu)), (kc, vc)):
        held = mxfp4.values(cache.cpu().contiguous()).reshape(-1, 2, 128)[slots]
        assert torch.equal(got.cpu().double(), held)


@pytest.mark.parametrize("page_stride,head_stride", [(B, B), (2 * B - 16, B), (B, 4 * B - 16)])
def test_overlapping_blocks_are_refused(gpu, page_stride, head_stride):
    # Two workgroups would write one byte.
    memory, (kc, vc) = _strided(gpu, page_stride, head_stride)
    k = torch.zeros(3, 2, 128, dtype=torch.bfloat16, device=gpu)
    slots = torch.arange(3, device=gpu)
    with pytest.raises(ValueError, match="apart"):
        ops.store_kvcache_mxfp4(k, k, kc, vc, slots)
    with pytest.raises(ValueError, match="apart"):
        ops.load_kvcache_mxfp4(kc, vc, slots)
    assert (memory == 0x33).all()
