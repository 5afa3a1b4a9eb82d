"""The MXFP4 KV cache and attention over it, in 64 bits on the CPU.

Written from the format's definition (OCP microscaling FP4: e2m1 elements, one
E8M0 scale for 32) and this package's choice of scale, apart from the kernels:
values are picked from the grid by distance, scales by exact exponents.
"""

from __future__ import annotations

import math

import numpy as np
import torch

PAGE = 16
DIM = 128
GROUP = 32
BLOCK = PAGE * (DIM // 2 + DIM // GROUP)
GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
# Largest exponent of a scale: every value read back is finite in the type.
MAX_EXPONENT = {torch.bfloat16: 125, torch.float16: 13}


def quantise(rows: torch.Tensor) -> tuple[np.ndarray, np.ndarray]:
    """(codes ``[..., 128]``, scale bytes ``[..., 4]``), uint8, of bf16/fp16 rows."""
    x = rows.double().cpu().numpy().reshape(*rows.shape[:-1], DIM // GROUP, GROUP)
    finite = np.isfinite(x).all(-1)
    size = np.where(finite[..., None], np.abs(x), 0.0)
    amax = size.max(-1)
    # The smallest e with amax <= 7 * 2^e; amax = m * 2^p, 0.5 <= m < 1, 7 = 0.875 * 2^3.
    m, p = np.frexp(amax)
    e = np.where(m <= 0.875, p - 3, p - 2)
    e = np.clip(np.where(amax == 0, -127, e), -127, MAX_EXPONENT[rows.dtype])
    scaled = np.ldexp(size, -e[..., None])
    # The nearest grid value; of two as near, the one of even code.
    away = np.abs(scaled[..., None] - GRID)
    best = away.min(-1, keepdims=True)
    code = np.where(away == best, np.arange(8) + np.where(np.arange(8) % 2 == 0, 0, 100), 1000).min(-1) % 100
    code = code + np.where(np.signbit(x) & finite[..., None], 8, 0)
    byte = np.where(finite, e + 127, 255)
    return code.reshape(rows.shape).astype(np.uint8), byte.astype(np.uint8)


def block_of(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """Blocks ``uint8 [..., 1088]`` of pages of codes ``[..., 16, 128]`` and scales ``[..., 16, 4]``."""
    pairs = codes[..., 0::2] | (codes[..., 1::2] << 4)
    lead = codes.shape[:-2]
    return np.concatenate([pairs.reshape(*lead, -1), scales.reshape(*lead, -1)], -1)


def cache_of(cache: torch.Tensor) -> torch.Tensor:
    """The MXFP4 cache ``uint8 [P, H, 1088]`` of a bf16/fp16 one ``[P, 16, H, 128]``."""
    codes, scales = quantise(cache.transpose(1, 2).contiguous())
    return torch.from_numpy(block_of(codes, scales))


def store(rows: torch.Tensor, cache: torch.Tensor, slots: list[int]) -> None:
    """Writes rows ``[N, H, 128]`` into a cache (CPU, in place) slot by slot."""
    codes, scales = quantise(rows)
    pairs = codes[..., 0::2] | (codes[..., 1::2] << 4)
    blocks = cache.numpy()
    for t, slot in enumerate(slots):
        if 0 <= slot < blocks.shape[0] * PAGE:
            page, token = divmod(slot, PAGE)
            blocks[page, :, 64 * token:64 * token + 64] = pairs[t]
            blocks[page, :, 1024 + 4 * token:1024 + 4 * token + 4] = scales[t]


def values(cache: torch.Tensor) -> torch.Tensor:
    """The float64 values ``[P, 16, H, 128]`` of a cache."""
    blocks = cache.cpu().numpy()
    lead = blocks.shape[:-1]
    pairs = blocks[..., :1024].reshape(*lead, PAGE, DIM // 2)
    codes = np.stack([pairs & 15, pairs >> 4], -1).reshape(*lead, PAGE, DIM)
    size = GRID[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    byte = blocks[..., 1024:].reshape(*lead, PAGE, DIM // GROUP).astype(np.int64)
    scale = np.where(byte == 255, np.nan, np.ldexp(1.0, byte - 127))
    return torch.from_numpy(size * scale.repeat(GROUP, -1)).transpose(1, 2)


def attention(q, k_cache, v_cache, block_tables, query_lengths, kv_lengths, scale: float | None = None):
    """(outputs, bound sums) in float64, ``[T, Hq, 128]`` each: causal attention
    over the values of the two caches, and the same average of |V|.  Also
    returns the largest sum of |q||k| * scale of a score, for error bounds."""
    k_all, v_all = values(k_cache), values(v_cache)
    hq, hkv = q.shape[1], k_cache.shape[1]
    scale = 1 / math.sqrt(DIM) if scale is None else scale
    out = torch.empty(q.shape, dtype=torch.float64)
    spread = torch.empty(q.shape, dtype=torch.float64)
    largest, first = 0.0, 0
    for s, (n, kv) in enumerate(zip(query_lengths, kv_lengths)):
        pages = block_tables[s, :(kv + PAGE - 1) // PAGE].long().cpu()
        k = k_all[pages].reshape(-1, hkv, DIM)[:kv]
        v = v_all[pages].reshape(-1, hkv, DIM)[:kv]
        for h in range(hq):
            g = h // (hq // hkv)
            rows = q[first:first + n, h].double().cpu()
            scores = rows @ k[:, g].T * scale
            hidden = torch.arange(kv)[None] > torch.arange(kv - n, kv)[:, None]
            prob = torch.softmax(scores.masked_fill(hidden, -math.inf), -1)
            # A masked key has no weight, whatever its value.
            out[first:first + n, h] = torch.where(hidden[..., None], 0.0, prob[..., None] * v[None, :, g]).sum(1) \
                if torch.isnan(v).any() else prob @ v[:, g]
            spread[first:first + n, h] = prob @ v[:, g].abs()
            largest = max(largest, float((rows.abs() @ k[:, g].abs().T).nan_to_num(0).max()) * scale)
        first += n
    return out, spread, largest
