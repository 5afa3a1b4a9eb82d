"""Page bounds, page selection and attention over selected pages, in 64 bits on
the CPU, one page, head and row at a time — test infrastructure only.

Pinned in ``tests/test_page_selection_host.py``: bounds against a sort of every
column, the selection against hand-made scores with ties, and the attention
against ``oracle.reference.paged_attention`` where a list holds every page.
"""

from __future__ import annotations

import math

import numpy as np
import torch

PAGE = 16


def page_bounds(k_cache, bounds, block_tables, seq_lens, new_tokens) -> torch.Tensor:
    """``bounds`` after a step that appended ``new_tokens[s]`` tokens to sequence s."""
    out = bounds.clone()
    for row, n, new in zip(block_tables.tolist(), seq_lens, new_tokens):
        for pos in range(max(0, n - new), n):
            if pos % PAGE == PAGE - 1 and pos // PAGE < len(row) and 0 <= row[pos // PAGE] < len(k_cache):
                page = row[pos // PAGE]
                keys = k_cache[page].double()
                out[page, :, 0] = keys.amin(0).to(out.dtype)
                out[page, :, 1] = keys.amax(0).to(out.dtype)
    return out


def page_scores(q, bounds) -> np.ndarray:
    """Scores of pages ``bounds [n, 2, 128]`` for the queries ``q [G, 128]`` of a KV
    head: the sum over queries and channels of the larger of q min and q max (that of
    max for a positive q, of min for a negative one); NaN if either product is."""
    queries = q.double().numpy()
    up = np.where(queries < 0, 0.0, queries).sum(0)
    down = np.where(queries > 0, 0.0, queries).sum(0)
    box = bounds.double().numpy()
    finite = np.isfinite(box).all((1, 2)) & np.isfinite(queries).all()
    scores = np.zeros(len(box))
    for j, ok in enumerate(finite):
        if ok:  # the same sum, queries of one sign taken together
            scores[j] = math.fsum(np.concatenate((box[j, 1] * up, box[j, 0] * down)))
        else:
            with np.errstate(invalid="ignore"):
                low, high = queries * box[j, 0], queries * box[j, 1]
                larger = np.where(queries < 0, low, high)
                scores[j] = np.where(np.isnan(low) | np.isnan(high), math.nan, larger).sum()
    return scores


def chosen(scores, want: int) -> list[int]:
    """Places of the ``want`` highest scores: NaN above all, ties to the lowest place."""
    order = sorted(range(len(scores)), key=lambda j: (not math.isnan(scores[j]), -scores[j] if
                                                      not math.isnan(scores[j]) else 0.0, j))
    return sorted(order[:want])


def select_pages(q, bounds, block_tables, seq_lens, num_selected: int, sink: int, recent: int):
    """(tables ``[S, H, num_selected]``, lens ``[S]``)."""
    heads = bounds.shape[1]
    group = q.shape[1] // heads
    tables = torch.full((len(q), heads, num_selected), -1, dtype=torch.int32)
    lens = torch.zeros(len(q), dtype=torch.int32)
    for s, (row, length) in enumerate(zip(block_tables, seq_lens)):
        n = (max(length, 0) + PAGE - 1) // PAGE
        taken = min(n, num_selected)
        lens[s] = max(length, 0) - PAGE * (n - taken)
        for h in range(heads):
            if n <= num_selected:
                places = list(range(n))
            else:
                middle = row[sink:n - recent].long()
                scores = page_scores(q[s, h * group:(h + 1) * group], bounds[middle, h])
                best = chosen(scores, num_selected - sink - recent)
                places = [*range(sink), *(sink + j for j in best), *range(n - recent, n)]
            tables[s, h, :taken] = row[places]
    return tables, lens


def attention(q, k_cache, v_cache, tables, lens, scale: float):
    """(output, average of |V| under the probabilities, largest sum of |q||k| times
    the scale) in float64 of each row over its lists."""
    rows, hq, dim = q.shape
    heads = k_cache.shape[2]
    group = hq // heads
    out = torch.zeros(rows, hq, dim, dtype=torch.float64)
    spread, largest = torch.zeros_like(out), torch.zeros(rows, hq, 1, dtype=torch.float64)
    for s in range(rows):
        n = int(lens[s])
        if n <= 0:
            continue
        for h in range(heads):
            pages = tables[s, h, : (n + PAGE - 1) // PAGE].long()
            k, v = (c[pages, :, h].reshape(-1, dim)[:n].double() for c in (k_cache, v_cache))
            mine = slice(h * group, (h + 1) * group)
            queries = q[s, mine].double()
            p = torch.softmax(queries @ k.t() * scale, -1)
            out[s, mine], spread[s, mine] = p @ v, p @ v.abs()
            largest[s, mine] = (queries.abs() @ k.abs().t()).amax(-1, keepdim=True) * scale
    return out, spread, largest
