"""CPU: the attention tests' bounds tell a coarser type of the probabilities, and the planner cuts whole tiles."""

import math

import numpy as np
import pytest
import torch

from my_vllm_amd.attention_backend import plan_decode_shared
from oracle import mxfp4
from tests._mxfp4 import attention_bound, subnormal_bound
from workloads import make_paged_batch

FEW_KEYS = [2, 3, 4, 5, 7, 15, 16, 17, 31, 33, 64, 65]  # those of test_gpu_mxfp4_forms.py
BF16, FP16 = torch.bfloat16, torch.float16


def _decode_with_rounded_probabilities(batch, k, v, p_dtype, dtype):
    """Decode in 64 bits but for P, rounded once to ``p_dtype`` against the row's largest score, and the result."""
    hq, hkv = batch.q.shape[1], k.shape[1]
    k_all, v_all = mxfp4.values(k), mxfp4.values(v)
    out = torch.empty(batch.q.shape, dtype=torch.float64)
    for s, kv in enumerate(batch.kv_lengths):
        pages = batch.common.block_tables[s, :(kv + 15) // 16].long()
        rows_k, rows_v = (c[pages].reshape(-1, hkv, 128)[:kv] for c in (k_all, v_all))
        for h in range(hq):
            g = h // (hq // hkv)
            scores = batch.q[s, h].double() @ rows_k[:, g].T / math.sqrt(128)
            p = torch.exp(scores - scores.max())
            out[s, h] = (p.to(p_dtype).double() @ rows_v[:, g]) / p.sum()
    return out.to(dtype).double()


@pytest.mark.parametrize("hq,hkv", [(16, 8), (40, 8), (12, 4), (16, 1)])
def test_the_fp16_bound_holds_fp16_probabilities_and_refuses_bf16_ones(hq, hkv):
    batch = make_paged_batch(hq, [1] * len(FEW_KEYS), FEW_KEYS, 0, hq, hkv, dtype=FP16)
    k, v = mxfp4.cache_of(batch.k_cache), mxfp4.cache_of(batch.v_cache)
    expected, spread, largest = mxfp4.attention(batch.q, k, v, batch.common.block_tables, batch.query_lengths,
                                                batch.kv_lengths)
    bound = (attention_bound(expected, spread, largest, max(FEW_KEYS), FP16, FP16)
             + subnormal_bound(max(FEW_KEYS), float(mxfp4.values(v).abs().max()), FP16))
    for p_dtype, within in ((FP16, True), (BF16, False)):
        off = (_decode_with_rounded_probabilities(batch, k, v, p_dtype, FP16) - expected).abs() / bound
        assert (float(off.max()) <= 1) is within


@pytest.mark.parametrize("counts,hkv,cus", [([5, 1, 40, 8, 1, 129], 5, 256), ([1875], 8, 256), ([75], 8, 256),
                                            ([2000, 1, 2, 3], 8, 256), ([17] * 300, 8, 256), ([9, 8, 7], 2, 1),
                                            ([300] * 37, 4, 304)])
def test_shared_plans_cut_between_tiles(counts, hkv, cus):
    # A tile is two pages: pieces and their quarters begin at even pages and end at
    # even ones or with the sequence.
    items = plan_decode_shared(counts, 3, 7, hkv, cus, always=True)[0]
    pages = np.array(counts)[items[:, 0] - 3]
    assert (items[:, 1] % 2 == 0).all()
    assert ((items[:, 2] % 2 == 0) | (items[:, 2] == pages)).all()
