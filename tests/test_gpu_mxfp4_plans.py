"""Decode graph states and plans of MXFP4 and of 16-bit caches on the GPU: neither fits the other's."""

import pytest
import torch

from my_vllm_amd.attention_backend import MI355XAttentionBackend, MI355XMXFP4AttentionBackend
from tests.test_gpu_mxfp4 import _on
from workloads import make_paged_batch

pytestmark = pytest.mark.gpu


def test_states_take_their_own_kinds_plans(gpu):
    wide, fp4 = (cls(16, 4, 128, 16, torch.bfloat16) for cls in (MI355XAttentionBackend, MI355XMXFP4AttentionBackend))
    common = _on(make_paged_batch(1, [1] * 3, [40, 900, 17], 0, 16, 4).common, gpu)
    states = {b: b.create_full_decode_graph_state(3, 3 * common.block_tables.size(1), gpu) for b in (wide, fp4)}
    plans = {b: b.build_plan(common) for b in (wide, fp4)}
    for own, other in ((wide, fp4), (fp4, wide)):
        assert own.full_decode_graph_metadata_fits(states[own], plans[own])
        assert not own.full_decode_graph_metadata_fits(states[other], plans[own])
        assert not own.full_decode_graph_metadata_fits(states[other], plans[other])
    assert not wide.full_decode_graph_metadata_fits(states[wide], plans[fp4])
    with pytest.raises(ValueError, match="does not fit"):
        wide.plan_full_decode_graph(states[wide], plans[fp4])
