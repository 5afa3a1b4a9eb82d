"""Captured steps keep memory of their own: eager steps that grow the backend's
buffers, other captures and other tensors neither change a replay nor are
changed by one."""

import pytest
import torch

from my_vllm_amd.attention_backend import MI355XAttentionBackend, MI355XMXFP4AttentionBackend
from oracle import mxfp4
from tests.test_gpu_mxfp4 import _on
from tests._util import set_decode_planning
from workloads import make_paged_batch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _step(cls, seed, q_lens, ctx, prefills, gpu):
    batch = make_paged_batch(seed, q_lens, ctx, prefills, 32, 8)
    caches = (batch.k_cache, batch.v_cache)
    if cls is MI355XMXFP4AttentionBackend:
        caches = tuple(mxfp4.cache_of(c) for c in caches)
    return batch.q.to(gpu), *(c.to(gpu) for c in caches), _on(batch.common, gpu)


def _forward(backend, step, plan=None):
    q, k, v, common = step
    return backend.forward(q, None, None, k, v, plan or backend.build_plan(common))


STEPS = {
    "decode": ([1] * 5, [5000, 17, 90, 1000, 33], 0),
    "mixed": ([40, 1, 1], [300, 3000, 2000], 1),
}


@pytest.mark.parametrize("eager_first", [True, False])
@pytest.mark.parametrize("kind,schedule", [("decode", "listed"), ("decode", "claims"), ("mixed", None)])
@pytest.mark.parametrize("cls", [MI355XAttentionBackend, MI355XMXFP4AttentionBackend])
def test_replays_beside_eager_steps_that_grow_the_buffers(gpu, monkeypatch, cls, kind, schedule, eager_first):
    if schedule == "claims" and cls is MI355XMXFP4AttentionBackend:
        schedule = "shared"
    set_decode_planning(monkeypatch, schedule=schedule)
    step = _step(cls, 1, *STEPS[kind], gpu)
    want = _forward(cls(32, 8, 128, 16, BF16), step).clone()
    backend = cls(32, 8, 128, 16, BF16)
    plan = backend.build_plan(step[3])
    assert plan.metadata.num_decode_part_slots > 0
    if eager_first:
        assert torch.equal(_forward(backend, step, plan), want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _forward(backend, step, plan).clone()
    # More partial slots and more rows: both eager buffers are replaced (or made).
    large = _step(cls, 2, [1] * 40, [2000 + 7 * i for i in range(40)], 0, gpu)
    large_want = _forward(cls(32, 8, 128, 16, BF16), large).clone()
    assert torch.equal(_forward(backend, large), large_want)
    torch.cuda.synchronize()
    # Whatever was given back is taken by these.
    fresh = [torch.full((n << 20,), 0xa5, dtype=torch.uint8, device=gpu) for n in (1, 1, 2, 4, 8)]
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert all((t == 0xa5).all() for t in fresh)
        assert torch.equal(_forward(backend, large), large_want)
        assert torch.equal(_forward(backend, step), want)


@pytest.mark.parametrize("cls", [MI355XAttentionBackend, MI355XMXFP4AttentionBackend])
def test_two_graphs_of_one_backend_replay_at_once(gpu, monkeypatch, cls):
    # Split steps of two layers, captured from one backend, on two streams: each as alone.
    set_decode_planning(monkeypatch, schedule="listed")
    backend = cls(32, 8, 128, 16, BF16)
    graphs = []
    for seed, ctx in ((3, [4000, 900, 2500]), (4, [3000] * 6)):
        step = _step(cls, seed, [1] * len(ctx), ctx, 0, gpu)
        plan = backend.build_plan(step[3])
        assert plan.metadata.num_decode_part_slots > 0
        swapped = (step[0], step[2], step[1], step[3])
        want = [_forward(backend, s, plan).clone() for s in (step, swapped)]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = [_forward(backend, s, plan).clone() for s in (step, swapped)]
        graphs.append((graph, outs, want, torch.cuda.Stream(), (step, plan)))
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, outs, _, stream, _ in graphs:
            with torch.cuda.stream(stream):
                for _ in range(4):
                    graph.replay()
        torch.cuda.synchronize()
        for _, outs, want, _, _ in graphs:
            assert all(torch.equal(a, b) for a, b in zip(outs, want))
