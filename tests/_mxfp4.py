"""Shared pieces of the MXFP4 tests."""

from __future__ import annotations

import torch

from oracle import mxfp4


def attention_bound(expected, spread, largest, keys: int, dtype: torch.dtype, p_dtype: torch.dtype):
    """How far an attention output may be off, element by element.

    With A the average of |V| under the exact probabilities (``spread``):
    P is rounded once to ``p_dtype`` (half a step each, so that of A);
    a score is a sum of 128 products in fp32, off by at most 136 * 2^-24 of the
    sum of its |q||k| (``largest``), which moves P and the row sum by as much
    each, and its scaling, subtraction and exp2 by 8 * 2^-24 of its size; the
    sums over ``keys`` terms and the split's merge add 2 (keys + 64) * 2^-24.
    The result is rounded once to ``dtype``."""
    step = torch.finfo(p_dtype).eps / 2
    fp32 = 2.0 ** -24
    scores = 2 * (136 + 8) * fp32 * largest
    relative = step + scores + 2 * (keys + 64) * fp32
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps  # a subnormal step
    return relative * (1 + step) * spread + torch.finfo(dtype).eps / 2 * (1 + relative) * expected.abs() + tiny


def assert_within(actual: torch.Tensor, expected: torch.Tensor, bound: torch.Tensor) -> None:
    actual = actual.double().cpu()
    assert actual.shape == expected.shape
    assert torch.isfinite(actual).all(), "non-finite attention output"
    over = (actual - expected).abs() / bound
    assert float(over.max()) <= 1.0, f"off by {float(over.max()):.3g} times the bound"


def cache_pool(batch, device, layers: int = 2):
    """The batch's caches in MXFP4 as layer 1 of a pool ``[2, layers, P, H, 1088]``,
    on the device and (contiguous) on the CPU."""
    k, v = mxfp4.cache_of(batch.k_cache), mxfp4.cache_of(batch.v_cache)
    pool = torch.full((2, layers, *k.shape), 0xff, dtype=torch.uint8, device=device)
    pool[0, 1], pool[1, 1] = k.to(device), v.to(device)
    return pool[0, 1], pool[1, 1], k, v


def poison_stale(cache: torch.Tensor, block_tables, kv_lengths, seed: int) -> None:
    """Everything past the sequences' ends: arbitrary codes under NaN scales (CPU, in place)."""
    gen = torch.Generator().manual_seed(seed)
    keep = torch.zeros(cache.shape[0], 16, dtype=torch.bool)
    for row, kv in zip(block_tables.cpu(), kv_lengths):
        for token in range(kv):
            keep[row[token // 16], token % 16] = True
    codes = torch.randint(0, 256, cache[..., :1024].shape, generator=gen, dtype=torch.uint8)
    stale = ~keep[:, None, :, None]
    cache[..., :1024] = torch.where(stale, codes.unflatten(-1, (16, 64)),
                                    cache[..., :1024].unflatten(-1, (16, 64))).flatten(-2)
    cache[..., 1024:] = torch.where(stale, torch.tensor(255, dtype=torch.uint8),
                                    cache[..., 1024:].unflatten(-1, (16, 4))).flatten(-2)


def random_cache(pages: int, heads: int, seed: int) -> torch.Tensor:
    """A cache of arbitrary codes under scales of 2^-5 .. 1 (CPU)."""
    gen = torch.Generator().manual_seed(seed)
    cache = torch.randint(0, 256, (pages, heads, mxfp4.BLOCK), generator=gen, dtype=torch.uint8)
    cache[..., 1024:] = torch.randint(122, 128, (pages, heads, 64), generator=gen, dtype=torch.uint8)
    return cache


def subnormal_bound(keys: int, value: float, p_dtype: torch.dtype) -> float:
    """What :func:`attention_bound` leaves out: a probability below the type's normal
    range, relative to a reference that the largest of its row reaches, is rounded by
    up to half a subnormal step, so the average of ``keys`` values of at most
    ``value`` by that often as much."""
    info = torch.finfo(p_dtype)
    return keys * value * info.tiny * info.eps / 2
