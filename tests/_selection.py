"""Shared pieces of the page selection tests."""

from __future__ import annotations

import numpy as np
import torch

PAGE, DIM = 16, 128


def tables_for(counts, num_pages: int, seed: int, width: int | None = None) -> torch.Tensor:
    """Block tables of distinct pages in a random order; behind a row's last page
    a page id that no cache holds."""
    order = np.random.default_rng(seed).permutation(num_pages)
    width = max(max(counts), 1) if width is None else width
    table = np.full((len(counts), width), 0x7ffffff0, np.int32)
    first = 0
    for s, n in enumerate(counts):
        table[s, :n] = order[first:first + n]
        first += n
    return torch.from_numpy(table)


def keys(num_pages: int, heads: int, dtype: torch.dtype, seed: int) -> torch.Tensor:
    """Pages of keys whose rows share a centre and whose channels are of unlike size."""
    gen = torch.Generator().manual_seed(seed)
    channels = torch.exp(0.5 * torch.randn(heads, DIM, generator=gen))
    centre = 0.5 * torch.randn(num_pages, 1, heads, DIM, generator=gen)
    return ((torch.randn(num_pages, PAGE, heads, DIM, generator=gen) + centre) * channels).to(dtype)


def bounds_of(k_cache: torch.Tensor) -> torch.Tensor:
    wide = k_cache.double()
    return torch.stack((wide.amin(1), wide.amax(1)), 2).to(k_cache.dtype)


def queries(rows: int, heads: int, dtype: torch.dtype, seed: int) -> torch.Tensor:
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(rows, heads, DIM, generator=gen).to(dtype)


def page_counts(lens) -> list[int]:
    return [(max(n, 0) + PAGE - 1) // PAGE for n in lens]


def same(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Equal values, NaN where the other has one."""
    a, b = a.double().cpu(), b.double().cpu()
    return a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())
