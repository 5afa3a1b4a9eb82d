"""Captured steps keep memory of their own: eager steps that grow the backend's
buffers, other captures and other tensors neither change a replay nor are
changed by one."""

import pytest
import torch

from my_vllm_amd.attention_backend import MI355XAttentionBackend, MI355XMXFP4AttentionBackend
from tests._mxfp4 import random_cache
from tests.test_gpu_mxfp4 import _on
from tests._util import set_decode_planning
from workloads import make_paged_batch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _step(cls, seed, q_lens, ctx, prefills, gpu):
    batch = make_paged_batch(seed, q_lens, ctx, prefills, 32, 8, device=gpu, rng_device="cuda")
    caches = (batch.k_cache, batch.v_cache)
    if cls is MI355XMXFP4AttentionBackend:
        caches = tuple(random_cache(batch.k_cache.shape[0], 8, 2 * seed + i).to(gpu) for i in (0, 1))
    return batch.q, *caches, batch.common


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


@pytest.mark.parametrize("kind,schedule", [("decode", "claims"), ("mixed", None)])
def test_the_layers_of_a_capture_share_counters(gpu, monkeypatch, kind, schedule):
    # Launches that count in the workspace (claims, arrivals), layer after layer of one graph.
    set_decode_planning(monkeypatch, schedule=schedule)
    backend = MI355XAttentionBackend(32, 8, 128, 16, BF16)
    step = _step(MI355XAttentionBackend, 5, *STEPS[kind], gpu)
    q, k, v, common = step
    plan = backend.build_plan(common)
    layers = [step, (q, v, k, common), (q, k, k, common)]
    want = [_forward(backend, s, plan).clone() for s in layers]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [_forward(backend, s, plan).clone() for s in layers]
    for _ in range(3):
        for out in outs:
            out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
        assert torch.equal(_forward(backend, step, plan), want[0])


def test_captured_folded_stores(gpu):
    # The step's rows written inside the captured decode launches of two layers.
    backend, eager = (MI355XAttentionBackend(32, 8, 128, 16, BF16) for _ in range(2))
    batch = make_paged_batch(6, [1] * 4, [5000, 17, 64, 1200], 0, 32, 8)
    common, q = _on(batch.common, gpu), batch.q.to(gpu)
    plan = backend.build_plan(common)
    assert plan.metadata.num_decode_part_slots > 0
    k, v = batch.k_new.to(gpu), batch.v_new.to(gpu)
    caches = [(batch.k_cache.to(gpu), batch.v_cache.to(gpu)) for _ in range(2)]
    backend.forward_with_kv_store(q, k, v, *caches[0], common.slot_mapping, plan)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [backend.forward_with_kv_store(q, k, v, *c, common.slot_mapping, plan).clone() for c in caches]
    for seed in range(3):
        k.copy_(torch.randn(k.shape, generator=torch.Generator().manual_seed(seed)))
        v.copy_(torch.randn(v.shape, generator=torch.Generator().manual_seed(10 + seed)))
        for kc, vc in caches:
            kc.copy_(batch.k_cache)
            vc.copy_(batch.v_cache)
        graph.replay()
        torch.cuda.synchronize()
        kc, vc = batch.k_cache.to(gpu), batch.v_cache.to(gpu)
        want = eager.forward_with_kv_store(q, k, v, kc, vc, common.slot_mapping, eager.build_plan(common))
        assert not eager.fused_store_error() and not backend.fused_store_error()
        for out, cache in zip(outs, caches):
            assert torch.equal(out, want) and torch.equal(cache[0], kc) and torch.equal(cache[1], vc)
