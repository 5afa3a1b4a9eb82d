"""GPU: the backend whose decode rows attend to selected pages, as a model runner
drives it: prefill chunks, decode steps and MIXED steps over one cache whose
pages and bounds grow with the sequences, eager and from a captured graph.
Every step is checked against the 64-bit oracle."""

import math

import pytest
import torch

from my_vllm_amd import ops
from my_vllm_amd.attention_backend import MI355XAttentionBackend, MI355XSparseAttentionBackend
from my_vllm_amd.contract import AttentionRoute, CommonAttentionMetadata
from oracle import selection
from oracle.reference import paged_attention
from tests._mxfp4 import assert_within, attention_bound
from tests._selection import PAGE, bounds_of, queries, same
from tests._util import assert_attention_close
from workloads import make_paged_batch

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
SCALE = 1 / math.sqrt(128)


class Runner:
    """A cache of ``pages`` pages whose free pages are dealt out in a shuffled order."""

    def __init__(self, gpu, hq, hkv, dtype, pages, seed, **numbers):
        self.gpu, self.hq, self.hkv, self.dtype = gpu, hq, hkv, dtype
        self.numbers = {"selected_pages": 6, "sink_pages": 1, "recent_pages": 2, **numbers}
        self.backend = MI355XSparseAttentionBackend(hq, hkv, 128, PAGE, dtype, **self.numbers)
        self.gen = torch.Generator().manual_seed(seed)
        self.k, self.v = (torch.full((pages, PAGE, hkv, 128), math.nan, dtype=dtype) for _ in range(2))
        self.bounds = torch.full((pages, hkv, 2, 128), math.nan, dtype=dtype)
        self.k_gpu, self.v_gpu, self.bounds_gpu = self.k.to(gpu), self.v.to(gpu), self.bounds.to(gpu)
        self.free = torch.randperm(pages, generator=self.gen).tolist()
        self.rows, self.lens = [], []

    def batch(self, new, prefills):
        """(common, slots) of a step that appends ``new[s]`` tokens to sequence s."""
        for s, count in enumerate(new):
            if s == len(self.rows):
                self.rows.append([])
                self.lens.append(0)
            self.lens[s] += count
            while len(self.rows[s]) * PAGE < self.lens[s]:
                self.rows[s].append(self.free.pop())
        counts = [len(row) for row in self.rows]
        table = torch.full((len(new), max(counts)), -1, dtype=torch.int32)
        for s, row in enumerate(self.rows):
            table[s, :len(row)] = torch.tensor(row)
        slots = [self.rows[s][p // PAGE] * PAGE + p % PAGE for s, count in enumerate(new)
                 for p in range(self.lens[s] - count, self.lens[s])]
        starts = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32)
        self.table = table
        decodes = len(new) - prefills
        return CommonAttentionMetadata(
            num_prefill_seqs=prefills, num_decode_seqs=decodes, num_prefill_tokens=sum(new) - decodes,
            num_decode_tokens=decodes, query_start_loc=starts.to(self.gpu),
            seq_lens=torch.tensor(self.lens, dtype=torch.int32, device=self.gpu),
            slot_mapping=torch.tensor(slots, dtype=torch.int32, device=self.gpu), block_tables=table.to(self.gpu),
            max_q_len=max(new), max_kv_len=max(self.lens), block_counts=tuple(counts), num_kv_blocks=sum(counts),
            num_prefill_kv_blocks=sum(counts[:prefills]), trusted=True), slots

    def rows_of(self, tokens):
        centre = 0.7 * torch.randn(1, self.hkv, 128, generator=self.gen)
        return [(torch.randn(tokens, self.hkv, 128, generator=self.gen) + centre).to(self.dtype) for _ in range(2)]

    def host_store(self, k, v, slots, new):
        for cache, values in ((self.k, k), (self.v, v)):
            cache.view(-1, self.hkv, 128)[slots] = values
        self.bounds = selection.page_bounds(self.k, self.bounds, self.table, self.lens, new)

    def check(self, out, q, new, prefills):
        first = sum(new[:prefills])
        if prefills:
            want = paged_attention(q[:first], self.k, self.v, self.table, new[:prefills], self.lens[:prefills])
            assert_attention_close(out[:first], want)
        if prefills < len(new):
            lens = self.lens[prefills:]
            tables, kept = selection.select_pages(q[first:], self.bounds, self.table[prefills:], lens,
                                                  *self.numbers.values())
            expected, spread, largest = selection.attention(q[first:], self.k, self.v, tables, kept, SCALE)
            assert_within(out[first:], expected, attention_bound(expected, spread, largest, max(lens), self.dtype,
                                                                 self.dtype))
        assert same(self.bounds_gpu, self.bounds)

    def step(self, new, prefills, separate=False):
        common, slots = self.batch(new, prefills)
        plan = self.backend.build_plan(common)
        k, v = self.rows_of(sum(new))
        q = queries(sum(new), self.hq, self.dtype, sum(self.lens))
        self.host_store(k, v, slots, new)
        k, v, caches = k.to(self.gpu), v.to(self.gpu), (self.k_gpu, self.v_gpu)
        if separate:  # as after the fused prologue
            ops.store_kvcache(k, v, *caches, common.slot_mapping)
            self.backend.update_page_bounds(self.k_gpu, self.bounds_gpu, plan)
            out = self.backend.forward(q.to(self.gpu), k, v, *caches, plan, page_bounds=self.bounds_gpu)
        else:
            out = self.backend.forward_with_kv_store(q.to(self.gpu), k, v, *caches, common.slot_mapping, plan,
                                                     page_bounds=self.bounds_gpu)
        self.check(out, q, new, prefills)
        return plan


@pytest.mark.parametrize("hq,hkv,dtype", [(16, 8, BF16), (32, 4, FP16), (8, 1, BF16), (9, 3, BF16)])
def test_prefill_decode_and_mixed_steps(gpu, hq, hkv, dtype):
    runner = Runner(gpu, hq, hkv, dtype, 120, hq)
    assert runner.step([250, 40, 16], 3).route is AttentionRoute.PREFILL
    for i in range(20):  # a page ends in every row at some step
        assert runner.step([1, 1, 1], 0, separate=i % 2 == 1).route is AttentionRoute.DECODE
    # A chunk of the first sequence's continuation beside the others' decode rows.
    assert runner.step([37, 1, 1], 1).route is AttentionRoute.MIXED_SPLIT
    assert runner.step([100, 300, 1, 1], 2, separate=True).route is AttentionRoute.MIXED_SPLIT
    runner.step([1, 1, 1, 1], 0)


def test_short_rows_attend_as_the_dense_backend_does(gpu):
    # No more pages than are selected: all of them, as on the base.
    batch = make_paged_batch(5, [1] * 9, [1, 16, 17, 300, 2047, 2048, 900, 33, 15], 0, 16, 8, device=gpu,
                             rng_device="cuda")
    bounds = torch.full((len(batch.k_cache), 8, 2, 128), math.nan, dtype=BF16, device=gpu)  # none is read
    backend = MI355XSparseAttentionBackend(16, 8, 128, 16, BF16)
    out = backend.forward(batch.q, None, None, batch.k_cache, batch.v_cache, backend.build_plan(batch.common),
                          page_bounds=bounds)
    want = paged_attention(batch.q.cpu(), batch.k_cache.cpu(), batch.v_cache.cpu(), batch.common.block_tables.cpu(),
                           [1] * 9, batch.kv_lengths)
    assert_attention_close(out, want)


def test_warmup_runs_without_bounds(gpu):
    backend = MI355XSparseAttentionBackend(16, 8, 128, 16, BF16)
    dense = MI355XAttentionBackend(16, 8, 128, 16, BF16)
    common = CommonAttentionMetadata(
        num_prefill_seqs=2, num_decode_seqs=0, num_prefill_tokens=50, num_decode_tokens=0,
        query_start_loc=torch.tensor([0, 20, 50], dtype=torch.int32, device=gpu),
        seq_lens=torch.tensor([20, 30], dtype=torch.int32, device=gpu),
        slot_mapping=torch.full((50,), -1, dtype=torch.int32, device=gpu), max_q_len=30, max_kv_len=30, trusted=True)
    q, k, v = (queries(50, n, BF16, n).to(gpu) for n in (16, 8, 8))
    empty = k.new_empty(0)
    got = backend.forward_with_kv_store(q, k, v, empty, empty, common.slot_mapping, backend.build_plan(common))
    assert torch.equal(got, dense.forward(q, k, v, empty, empty, dense.build_plan(common)))


@pytest.mark.parametrize("stored", [True, False])
def test_captured_decode_steps(gpu, stored):
    """Full-decode graphs: tables, lengths, rows and slots change between replays."""
    hq, hkv, batch, width = 16, 4, 4, 40
    runner = Runner(gpu, hq, hkv, BF16, batch * width + 4, 3)
    backend = runner.backend
    runner.step([200, 16, 333, 31], 4)
    state = backend.create_full_decode_graph_state(batch, batch * width, gpu)
    q = torch.zeros(batch, hq, 128, dtype=BF16, device=gpu)
    k, v = (torch.zeros(batch, hkv, 128, dtype=BF16, device=gpu) for _ in range(2))
    slots = torch.full((batch,), -1, dtype=torch.int32, device=gpu)
    kept_k, kept_v, kept_bounds = (t.clone() for t in (runner.k_gpu, runner.v_gpu, runner.bounds_gpu))
    capture = CommonAttentionMetadata(
        num_prefill_seqs=0, num_decode_seqs=batch, num_prefill_tokens=0, num_decode_tokens=batch,
        query_start_loc=torch.arange(batch + 1, dtype=torch.int32, device=gpu),
        seq_lens=torch.ones(batch, dtype=torch.int32, device=gpu), slot_mapping=slots,
        block_tables=torch.zeros((batch, 1), dtype=torch.int32, device=gpu), max_q_len=1, max_kv_len=1,
        block_counts=(1,) * batch, num_kv_blocks=batch, num_prefill_kv_blocks=0, trusted=True)
    plan = backend.build_plan(capture)
    backend.plan_full_decode_graph(state, plan)
    backend.activate_full_decode_graph(state)

    def run():
        caches = (runner.k_gpu, runner.v_gpu)
        if stored:
            return backend.forward_with_kv_store(q, k, v, *caches, slots, plan, page_bounds=runner.bounds_gpu)
        ops.store_kvcache(k, v, *caches, slots)
        backend.update_page_bounds(runner.k_gpu, runner.bounds_gpu, plan)
        return backend.forward(q, k, v, *caches, plan, page_bounds=runner.bounds_gpu)

    try:
        assert run().data_ptr() == state.output.data_ptr()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
    finally:
        backend.deactivate_full_decode_graph()
    assert same(runner.k_gpu, kept_k) and same(runner.v_gpu, kept_v) and same(runner.bounds_gpu, kept_bounds)
    for turn in range(20):
        common, host_slots = runner.batch([1] * batch, 0)
        step_plan = backend.build_plan(common)
        assert backend.full_decode_graph_metadata_fits(state, step_plan)
        backend.plan_full_decode_graph(state, step_plan)
        new_k, new_v = runner.rows_of(batch)
        new_q = queries(batch, hq, BF16, turn)
        runner.host_store(new_k, new_v, host_slots, [1] * batch)
        for buffer, value in ((q, new_q), (k, new_k), (v, new_v), (slots, common.slot_mapping)):
            buffer.copy_(value)
        graph.replay()
        got = state.output.clone()
        runner.check(got, new_q, [1] * batch, 0)
        # Eager work, and the same step eagerly: the same bits.
        eager = backend.forward(q, k, v, runner.k_gpu, runner.v_gpu, step_plan, page_bounds=runner.bounds_gpu)
        assert torch.equal(got, eager)


def test_steps_on_two_streams(gpu):
    # One backend, decode and prefill steps side by side on two streams: each as alone.
    backend = MI355XSparseAttentionBackend(16, 4, 128, PAGE, BF16, selected_pages=20, recent_pages=2)
    steps = []
    for seed, (q_lens, kv_lens, prefills) in enumerate((([1] * 6, [3000, 40, 900, 16, 2222, 1500], 0),
                                                        ([1] * 6, [2800, 700, 33, 1900, 5, 320], 0),
                                                        ([300, 90], [700, 90], 2), ([120, 250], [120, 900], 2))):
        batch = make_paged_batch(20 + seed, q_lens, kv_lens, prefills, 16, 4, device=gpu, rng_device="cuda")
        steps.append((batch, bounds_of(batch.k_cache).contiguous()))

    def run(batch, bounds, plan):
        return backend.forward(batch.q, None, None, batch.k_cache, batch.v_cache, plan, page_bounds=bounds)

    plans = [backend.build_plan(batch.common) for batch, _ in steps]
    alone = [run(*step, plan).clone() for step, plan in zip(steps, plans)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for pair in ((0, 1), (2, 3), (0, 3)):
            outs = []
            for stream, i in zip(streams, pair):
                with torch.cuda.stream(stream):
                    outs.append(run(*steps[i], plans[i]))
            torch.cuda.synchronize()
            assert all(torch.equal(out, alone[i]) for out, i in zip(outs, pair))


def _steps(gpu, seeds, kinds):
    for seed, (q_lens, kv_lens, prefills) in zip(seeds, kinds):
        batch = make_paged_batch(seed, q_lens, kv_lens, prefills, 16, 4, device=gpu, rng_device="cuda")
        yield batch, bounds_of(batch.k_cache).contiguous()


def _forward(backend, step, plan=None):
    batch, bounds = step
    return backend.forward(batch.q, None, None, batch.k_cache, batch.v_cache, plan or backend.build_plan(batch.common),
                           page_bounds=bounds)


@pytest.mark.parametrize("eager_first", [True, False])
@pytest.mark.parametrize("kind", [([1] * 5, [5000, 17, 90, 1000, 33], 0), ([40, 1, 1], [300, 3000, 2000], 1),
                                  ([40, 70], [300, 3000], 2)])
def test_replays_beside_eager_steps_that_grow_the_buffers(gpu, kind, eager_first):
    step, large = _steps(gpu, (1, 2), (kind, ([1] * 70, [2000 + 7 * i for i in range(70)], 0)))
    numbers = {"selected_pages": 33, "recent_pages": 2}
    backend, other = (MI355XSparseAttentionBackend(16, 4, 128, PAGE, BF16, **numbers) for _ in range(2))
    want, large_want = _forward(other, step).clone(), _forward(other, large).clone()
    plan = backend.build_plan(step[0].common)
    if eager_first:
        assert torch.equal(_forward(backend, step, plan), want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _forward(backend, step, plan).clone()
    assert torch.equal(_forward(backend, large), large_want)
    torch.cuda.synchronize()
    # Whatever was given back is taken by these.
    fresh = [torch.full((n << 20,), 0xa5, dtype=torch.uint8, device=gpu) for n in (1, 1, 2, 4, 8)]
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and all((t == 0xa5).all() for t in fresh)
        assert torch.equal(_forward(backend, large), large_want) and torch.equal(_forward(backend, step), want)


def test_two_graphs_of_one_backend_replay_at_once(gpu):
    # Two layers each, of decode steps whose rows are cut into parts and whose choice counts workgroups in.
    backend = MI355XSparseAttentionBackend(16, 4, 128, PAGE, BF16, selected_pages=60)
    graphs = []
    for step in _steps(gpu, (3, 4), (([1] * 3, [4000, 900, 25000], 0), ([1] * 6, [3000] * 6, 0))):
        batch, bounds = step
        plan = backend.build_plan(batch.common)
        swapped = (type(batch)(**{**batch.__dict__, "k_cache": batch.v_cache, "v_cache": batch.k_cache}),
                   bounds_of(batch.v_cache).contiguous())
        want = [_forward(backend, s, plan).clone() for s in (step, swapped)]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = [_forward(backend, s, plan).clone() for s in (step, swapped)]
        graphs.append((graph, outs, want, torch.cuda.Stream(), (step, swapped, plan)))
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, outs, _, stream, _ in graphs:
            with torch.cuda.stream(stream):
                for _ in range(4):
                    graph.replay()
        torch.cuda.synchronize()
        for _, outs, want, _, (step, _, plan) in graphs:
            assert all(torch.equal(a, b) for a, b in zip(outs, want))
            assert torch.equal(_forward(backend, step, plan), want[0])


def test_a_sequence_that_a_batch_holds_twice(gpu):
    # As padding that repeats a row does: the page that both complete is last in both.
    runner = Runner(gpu, 16, 4, BF16, 60, 9)
    runner.step([319, 100], 2)
    common, slots = runner.batch([1, 1], 0)
    k, v = runner.rows_of(2)
    q = queries(2, 16, BF16, 5)
    runner.host_store(k, v, slots, [1, 1])
    of = torch.tensor([0, 1, 0, 0])
    counts = tuple(common.block_counts[i] for i in of.tolist())
    twice = CommonAttentionMetadata(**{
        **common.__dict__, "num_decode_seqs": 4, "num_decode_tokens": 4, "block_counts": counts,
        "num_kv_blocks": sum(counts), "query_start_loc": torch.arange(5, dtype=torch.int32, device=gpu),
        **{name: getattr(common, name)[of.to(gpu)].contiguous() for name in ("seq_lens", "slot_mapping", "block_tables")}})
    out = runner.backend.forward_with_kv_store(
        q[of].to(gpu), k[of].to(gpu), v[of].to(gpu), runner.k_gpu, runner.v_gpu, twice.slot_mapping,
        runner.backend.build_plan(twice), page_bounds=runner.bounds_gpu)
    assert torch.equal(out[2], out[0]) and torch.equal(out[3], out[0])
    runner.check(out[:2], q, [1, 1], 0)


def test_plans_and_steps_that_do_not_fit_are_refused(gpu):
    batch = make_paged_batch(5, [1, 1], [300, 20], 0, 16, 8, device=gpu, rng_device="cuda")
    sparse, dense = (cls(16, 8, 128, 16, BF16) for cls in (MI355XSparseAttentionBackend, MI355XAttentionBackend))
    bounds = bounds_of(batch.k_cache)
    args = (batch.q, None, None, batch.k_cache, batch.v_cache)
    plan = sparse.build_plan(batch.common)
    with pytest.raises(ValueError, match="selects pages made it"):
        dense.forward(*args, plan)
    with pytest.raises(ValueError, match="needs page_bounds"):
        sparse.forward(*args, plan)
    with pytest.raises(ValueError, match="needs page_bounds"):
        sparse.forward_with_kv_store(batch.q, batch.k_new, batch.v_new, batch.k_cache, batch.v_cache,
                                     batch.common.slot_mapping, plan)
    with pytest.raises(ValueError, match="number of pages"):
        sparse.forward(*args, plan, page_bounds=bounds[1:])
    with pytest.raises(TypeError, match="dtype"):
        sparse.forward(*args, plan, page_bounds=bounds.half())
    with pytest.raises(ValueError, match="contiguous"):
        sparse.forward(*args, plan, page_bounds=bounds.transpose(2, 3).contiguous().transpose(2, 3))
    # A dense backend's plan serves: its pieces are not used.
    want = sparse.forward(*args, plan, page_bounds=bounds).clone()
    assert torch.equal(sparse.forward(*args, dense.build_plan(batch.common), page_bounds=bounds), want)
    assert sparse._page_bounds is None
    # Its MIXED plan does not: one launch, and dense; nor does this one's there.
    mixed = make_paged_batch(6, [20, 1], [40, 300], 1, 16, 8, device=gpu, rng_device="cuda")
    args, bounds = (mixed.q, None, None, mixed.k_cache, mixed.v_cache), bounds_of(mixed.k_cache)
    assert dense.build_plan(mixed.common).route is AttentionRoute.MIXED_UNIFIED
    with pytest.raises(ValueError, match="one dense MIXED launch"):
        sparse.forward(*args, dense.build_plan(mixed.common), page_bounds=bounds)
    with pytest.raises(ValueError, match="selects pages made it"):
        dense.forward(*args, sparse.build_plan(mixed.common))
    with pytest.raises(ValueError, match="needs page_bounds"):
        sparse.forward(*args, sparse.build_plan(mixed.common))
    sparse.forward(*args, sparse.build_plan(mixed.common), page_bounds=bounds)


def _refused(error, message, call, *args, **more):
    with pytest.raises(error, match=message):
        call(*args, **more)


def test_operators_refuse(gpu):
    k = torch.zeros(6, 16, 2, 128, dtype=BF16, device=gpu)
    bounds = torch.zeros(6, 2, 2, 128, dtype=BF16, device=gpu)
    table = torch.zeros(3, 6, dtype=torch.int32, device=gpu)
    lens = torch.zeros(3, dtype=torch.int32, device=gpu)
    starts = torch.arange(4, dtype=torch.int32, device=gpu)
    q = torch.zeros(3, 8, 128, dtype=BF16, device=gpu)
    update, select, attend = ops.update_page_bounds, ops.select_pages, ops.paged_decode_selected
    _refused(TypeError, "bfloat16", update, k.float(), bounds, table, lens)
    _refused(ValueError, "k_cache", update, k[:, :8], bounds, table, lens)
    _refused(ValueError, "overlap", update, k[:1].expand(6, 16, 2, 128), bounds, table, lens)
    _refused(ValueError, "overlap", update, k.transpose(2, 3).contiguous().transpose(2, 3), bounds, table, lens)
    _refused(ValueError, "page_bounds must be", update, k, bounds[:, :1], table, lens)
    _refused(ValueError, "number of pages", update, k, bounds[:5], table, lens)
    _refused(TypeError, "dtype", update, k, bounds.half(), table, lens)
    _refused(ValueError, "contiguous", update, k, bounds.expand(6, 2, 2, 128)[:, :, :1].expand(6, 2, 2, 128), table, lens)
    _refused(TypeError, "int32", update, k, bounds, table.long(), lens)
    _refused(ValueError, "dense", update, k, bounds, table.t().contiguous().t(), lens)
    _refused(ValueError, "one row per", update, k, bounds, table[:2], lens)
    _refused(RuntimeError, "device", update, k, bounds, table.cpu(), lens)
    _refused(ValueError, "num_tokens", update, k, bounds, table, lens, starts)
    _refused(ValueError, "one new token", update, k, bounds, table, lens, None, 4)
    _refused(ValueError, "one more entry", update, k, bounds, table, lens, starts[:3], 3)
    _refused(RuntimeError, "int32", update, k, bounds, table, lens, starts.long(), 3)
    _refused(ValueError, "num_tokens", update, k, bounds, table, lens, starts, -1)
    _refused(TypeError, "bfloat16", select, q.float(), bounds, table, lens, 4)
    _refused(ValueError, "inner stride", select, q.transpose(1, 2), bounds, table, lens, 4)
    _refused(ValueError, "query heads", select, q[:, :7], bounds, table, lens, 4)
    _refused(ValueError, "query heads", select, q[:, :1].expand(3, 34, 128), bounds, table, lens, 4)
    _refused(TypeError, "dtype", select, q, bounds.half(), table, lens, 4)
    _refused(ValueError, "row for every query", select, q[:2], bounds, table, lens, 4)
    _refused(ValueError, "at most", select, q, bounds, table, lens, 4, 3, 2)
    _refused(ValueError, "recent_pages", select, q, bounds, table, lens, 4, 1, 0)
    _refused(ValueError, "sink_pages", select, q, bounds, table, lens, 4, -1, 1)
    _refused(TypeError, "num_selected", select, q, bounds, table, lens, 4.0)
    _refused(ValueError, "needs pages", select, q, bounds, table[:, :0], lens, 4)
    _refused(ValueError, "needs pages", select, q, bounds[:0], table, lens, 4)
    _refused(ValueError, "bytes", select, q, bounds, table, lens, 4,
             workspace=torch.empty(8, dtype=torch.uint8, device=gpu))
    _refused(TypeError, "dtype", select, q, bounds, table, lens, 4, k_cache=k.half())
    _refused(ValueError, "number of pages", select, q, bounds, table, lens, 4, k_cache=k[:5])
    _refused(ValueError, "overlap", select, q, bounds, table, lens, 4, k_cache=k[:1].expand(6, 16, 2, 128))
    _refused(ValueError, "uint8", select, q, bounds, table, lens, 4, workspace=torch.empty(1 << 20, device=gpu))
    lists = table[:, None].expand(3, 2, 6)
    _refused(TypeError, "dtype", attend, q, k.half(), k, lists, lens, 1.0)
    _refused(ValueError, "layout", attend, q, k, k[:5], lists, lens, 1.0)
    _refused(ValueError, "query heads", attend, q[:, :5], k, k, lists, lens, 1.0)
    _refused(TypeError, "int32", attend, q, k, k, lists.long(), lens, 1.0)
    _refused(ValueError, "tables must be", attend, q, k, k, lists[:, :1], lens, 1.0)
    _refused(ValueError, "tables must be", attend, q, k, k, lists[..., :0], lens, 1.0)
    _refused(ValueError, "dense lists", attend, q, k, k, lists.transpose(1, 2).contiguous().transpose(1, 2), lens, 1.0)
    _refused(ValueError, "lens", attend, q, k, k, lists, lens[:2], 1.0)
    _refused(ValueError, "out must", attend, q, k, k, lists, lens, 1.0, out=q[:2])
    _refused(ValueError, "pages", attend, q, k[:0], k[:0], lists, lens, 1.0)
    for scale in (0.0, -1.0, math.nan, math.inf):
        _refused(RuntimeError, "softmax_scale", attend, q, k, k, lists, lens, scale)
    # No rows: nothing to do.
    none = select(q[:0], bounds, table[:0], lens[:0], 4)
    assert none[0].shape == (0, 2, 4) and attend(q[:0], k, k, none[0], none[1], 1.0).shape == (0, 8, 128)
    update(k, bounds, table[:0], lens[:0])
    update(k, bounds, table, lens, torch.zeros(4, dtype=torch.int32, device=gpu), 0)
