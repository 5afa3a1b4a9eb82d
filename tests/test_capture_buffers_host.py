"""CPU: which buffers a step inside a graph capture takes (the capture is played)."""

import pytest
import torch

from my_vllm_amd import ops
from my_vllm_amd.attention_backend import MI355XAttentionBackend, MI355XMXFP4AttentionBackend


@pytest.mark.parametrize("cls", [MI355XAttentionBackend, MI355XMXFP4AttentionBackend])
def test_a_capture_takes_no_buffer_of_eager_steps(monkeypatch, cls):
    backend = cls(16, 8, 128, 16, torch.bfloat16)
    cpu, playing = torch.device("cpu"), [None]
    monkeypatch.setattr(cls, "_capture_of", lambda self, device: playing[0])
    counters = ops.decode_workspace_bytes(0, 1, 1)
    small, large = (ops.decode_workspace_bytes(slots, 8, 2) for slots in (3, 4000))
    q = torch.zeros(5, 16, 128, dtype=torch.bfloat16)
    # As in a forward: the output first, then the workspace.
    eager_out, eager = backend._get_reusable_attention_output(q), backend._get_workspace(small, cpu)
    captured, outs = [], []
    for playing[0] in ((7, 1), (7, 2), (8, 1)):  # two streams of one capture, then another capture
        outs += [backend._get_reusable_attention_output(q) for _ in range(2)]
        first = backend._get_workspace(small, cpu)
        assert (first[:counters] == 0).all()
        first[:4] = 1  # a launch leaves its counters clear: nothing clears them again for the next layer
        assert backend._get_workspace(small, cpu) is first and first[0] == 1
        grown = backend._get_workspace(large, cpu)
        assert grown.numel() >= large and (grown[:counters] == 0).all()
        assert backend._get_workspace(small, cpu) is grown
        captured += [first, grown]
    starts = [t.data_ptr() for t in (eager, *captured)]
    assert len(set(starts)) == len(starts)
    assert len({t.data_ptr() for t in (eager_out, *outs)}) == 1 + len(outs)
    # Eager steps go on with theirs, and grow them as before.
    playing[0] = None
    assert backend._get_reusable_attention_output(q).data_ptr() == eager_out.data_ptr()
    assert backend._get_workspace(small, cpu) is eager
    assert backend._get_workspace(large, cpu).numel() >= large and backend._workspace is not eager
    # The zeros of an unplaced capture are not an eager workspace's.
    fresh = cls(16, 8, 128, 16, torch.bfloat16)
    playing[0] = (9, 1)
    fresh._get_reusable_attention_output(q)
    fresh._get_workspace(small, cpu)
    assert fresh._workspace is None and fresh._output_buffer is None
