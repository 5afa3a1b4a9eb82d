"""MXFP4 operators in the kernel forms that large calls and either type select."""

import pytest
import torch

from my_vllm_amd import ops
from my_vllm_amd.attention_backend import MI355XMXFP4AttentionBackend
from my_vllm_amd.contract import AttentionRoute
from oracle import mxfp4
from tests._mxfp4 import assert_within, attention_bound, poison_stale, random_cache, subnormal_bound
from tests.test_gpu_mxfp4 import _hard_rows, _on
from workloads import make_paged_batch

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


# ---- store and read-back: four rows a thread from 2048 workgroups on ------------------

# (tokens, heads): workgroups of 64 tokens and one head of K or V.  8128 x 8 is 2032 of
# them, the last call of one row a thread; the others leave 1, 1, 17, 40 and 63 tokens in the last.
MANY = [(8128, 8), (8129, 8), (8193, 8), (8209, 8), (1000, 64), (2047, 32)]


def _blocks(n, h):
    return -(-n // 64) * 2 * h


def test_the_sizes_take_both_forms():
    assert [_blocks(*x) >= 2048 for x in MANY] == [False, True, True, True, True, True]
    assert [n % 64 for n, _ in MANY] == [0, 1, 1, 17, 40, 63]


@pytest.mark.parametrize("dtype,wide", [(BF16, False), (FP16, True)])
@pytest.mark.parametrize("n,h", MANY)
def test_large_stores_byte_for_byte(gpu, dtype, wide, n, h):
    pages = n // 16 + 3
    gen = torch.Generator().manual_seed(n)
    slots = torch.randperm(pages * 16, generator=gen)[:n]
    slots[5], slots[n - 2], slots[777] = -1, pages * 16, -9  # skipped
    # V is a slice of a packed projection.
    k = _hard_rows(512, h, dtype, 1).repeat(n // 512 + 1, 1, 1)[:n].to(gpu)
    packed = torch.zeros(n, 2 * h + 1, 128, dtype=dtype, device=gpu)
    packed[:, 1:h + 1] = _hard_rows(511, h, dtype, 2).repeat(n // 511 + 1, 1, 1)[:n].to(gpu)
    v = packed[:, 1:h + 1]
    on_gpu = slots.to(torch.int64 if wide else torch.int32).to(gpu)
    before = torch.randint(0, 256, (2, pages, h, 1088), generator=gen, dtype=torch.uint8)
    got, small = before.to(gpu), before.to(gpu)
    ops.store_kvcache_mxfp4(k, v, got[0], got[1], on_gpu)
    # Call by call of one row a thread, whose bytes the oracle's tests settle.
    step = 500
    assert _blocks(step, h) < 2048
    for first in range(0, n, step):
        part = slice(first, first + step)
        ops.store_kvcache_mxfp4(k[part], v[part], small[0], small[1], on_gpu[part])
    assert torch.equal(got, small)
    # And the oracle's, of the first and the last tokens.
    for rows, cache in ((k, got[0].cpu()), (v, got[1].cpu())):
        for part in (slice(0, 70), slice(n - 150, n)):
            own, want = slots[part].tolist(), cache.clone()
            mxfp4.store(rows[part].cpu(), want, own)
            assert torch.equal(cache, want)


@pytest.mark.parametrize("dtype,wide", [(BF16, True), (FP16, False)])
@pytest.mark.parametrize("n,h", MANY)
def test_large_reads_return_the_values(gpu, dtype, wide, n, h):
    pages = 40
    cache = torch.stack([random_cache(pages, h, s) for s in (n, n + 1)])
    cache[0, 3, h - 1, 1024 + 7] = 255
    gen = torch.Generator().manual_seed(n)
    slots = torch.randint(-16, pages * 16 + 16, (n,), generator=gen)
    dev = cache.to(gpu)
    got = ops.load_kvcache_mxfp4(dev[0], dev[1], slots.to(torch.int64 if wide else torch.int32).to(gpu), dtype)
    inside = (slots >= 0) & (slots < pages * 16)
    assert inside.any() and not inside.all()
    for one, part in zip(got, cache):
        held = mxfp4.values(part).reshape(-1, h, 128).to(dtype)  # exact in both types
        expected = torch.where(inside[:, None, None], held[slots.clamp(0, pages * 16 - 1)], torch.zeros((), dtype=dtype))
        assert one.shape == (n, h, 128) and one.dtype == dtype
        assert torch.equal(one.cpu().nan_to_num(nan=1e4), expected.nan_to_num(nan=1e4))


# ---- prefill: one item a workgroup, items in turns, items claimed -----------------------


def _prefill_case(seed, q_lens, kv_lens, hq, hkv, dtype):
    batch = make_paged_batch(seed, q_lens, kv_lens, len(q_lens), hq, hkv, dtype=dtype)
    caches = [random_cache(batch.k_cache.shape[0], hkv, seed + i) for i in (1, 2)]
    for i, cache in enumerate(caches):
        poison_stale(cache, batch.common.block_tables, kv_lens, seed + i)
    return batch, caches


def _bound(expected, spread, largest, keys, dtype):
    return (attention_bound(expected, spread, largest, keys, dtype, dtype)
            + subnormal_bound(keys, 6.0, dtype))


# Key tiles have 64 tokens: items of one, two, three and more of them, one after the other,
# in workgroups that take several, and their plans' orders.
LENGTHS = [(5, 5), (64, 64), (65, 65), (1, 128), (30, 129), (128, 128), (3, 192), (200, 200), (1, 1), (90, 390),
           (16, 16), (1, 64), (2, 66), (63, 127), (17, 193), (1, 257)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("form,hq,hkv,seqs", [
    ("fixed", 64, 64, 3), ("turns", 64, 64, 7), ("turns", 64, 64, 19), ("claims", 64, 64, 26), ("claims", 64, 64, 48),
    ("turns", 128, 64, 12), ("claims", 128, 64, 40), ("claims", 96, 32, 70), ("turns", 256, 32, 17),
])
def test_prefill_forms(gpu, form, hq, hkv, seqs, dtype):
    lengths = [LENGTHS[(5 * i + seqs) % len(LENGTHS)] for i in range(seqs)]
    q_lens, kv_lens = [list(x) for x in zip(*lengths)]
    batch, caches = _prefill_case(seqs, q_lens, kv_lens, hq, hkv, dtype)
    backend = MI355XMXFP4AttentionBackend(hq, hkv, 128, 16, dtype)
    plan = backend.build_plan(_on(batch.common, gpu))
    assert plan.route is AttentionRoute.PREFILL
    per_head = torch.cuda.get_device_properties(gpu).multi_processor_count // hkv
    tiles = plan.metadata.prefill_max_tiles
    assert form == ("fixed" if tiles <= per_head else "turns" if tiles <= 6 * per_head else "claims")
    q, (kd, vd) = batch.q.to(gpu), (c.to(gpu) for c in caches)
    out = backend.forward(q, None, None, kd, vd, plan).clone()
    expected, spread, largest = mxfp4.attention(batch.q, *caches, batch.common.block_tables, q_lens, kv_lens)
    assert out.dtype == dtype
    assert_within(out, expected, _bound(expected, spread, largest, max(kv_lens), dtype))
    for _ in range(3):  # the same plan again, and a plan of its own again: the same bits
        assert torch.equal(backend.forward(q, None, None, kd, vd, plan), out)
    assert torch.equal(backend.forward(q, None, None, kd, vd, backend.build_plan(_on(batch.common, gpu))), out)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("kv", [64, 65, 128])
def test_prefill_of_many_short_prompts(gpu, dtype, kv):
    # Every item has one or two key tiles, and a successor of as few.
    seqs = 33
    batch, caches = _prefill_case(kv, [kv] * seqs, [kv] * seqs, 64, 64, dtype)
    backend = MI355XMXFP4AttentionBackend(64, 64, 128, 16, dtype)
    plan = backend.build_plan(_on(batch.common, gpu))
    out = backend.forward(batch.q.to(gpu), None, None, caches[0].to(gpu), caches[1].to(gpu), plan)
    expected, spread, largest = mxfp4.attention(batch.q, *caches, batch.common.block_tables, [kv] * seqs, [kv] * seqs)
    assert_within(out, expected, _bound(expected, spread, largest, kv, dtype))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("hq", [8, 16, 32])
def test_prefill_nan_groups(gpu, hq, dtype):
    # A NaN of K reaches the queries that see it and no other; one of V also those before it
    # in its tile of queries (256 rows over a KV head's query heads) and keys (64).
    n, hkv = 300, 8
    batch, caches = _prefill_case(hq, [n], [n], hq, hkv, dtype)
    backend = MI355XMXFP4AttentionBackend(hq, hkv, 128, 16, dtype)
    plan = backend.build_plan(_on(batch.common, gpu))
    q = batch.q.to(gpu)

    def run():
        return backend.forward(q, None, None, caches[0].to(gpu), caches[1].to(gpu), plan).cpu()

    clean = run()
    assert torch.isfinite(clean).all()
    table, group = batch.common.block_tables[0], hq // hkv
    caches[0][table[100 // 16], 3, 1024 + 4 * (100 % 16) + 1] = 255
    out = run()
    heads = torch.zeros(hq, dtype=torch.bool)
    heads[3 * group:4 * group] = True
    assert torch.isnan(out[100:, heads]).all()
    assert torch.equal(out[:100], clean[:100]) and torch.equal(out[100:, ~heads], clean[100:, ~heads])
    caches[0][table[100 // 16], 3, 1024 + 4 * (100 % 16) + 1] = 124
    clean = run()
    caches[1][table[290 // 16], 3, 1024 + 4 * (290 % 16) + 2] = 255
    out, dims = run(), slice(64, 96)
    assert torch.isnan(out[290:, heads, dims]).all()
    # Queries 256 .. 299 are in the last tile, and keys 256 .. 299 in theirs.
    assert torch.equal(out[:256], clean[:256])
    assert torch.equal(out[:, ~heads], clean[:, ~heads])
    rest = [d for d in range(128) if d not in range(64, 96)]
    assert torch.equal(out[:, heads][..., rest], clean[:, heads][..., rest])


# ---- fp16: probabilities in fp16, MIXED steps and captured decode ------------------------

FEW_KEYS = [2, 3, 4, 5, 7, 15, 16, 17, 31, 33, 64, 65]


@pytest.mark.parametrize("schedule", ["shared", "listed"])
@pytest.mark.parametrize("hq,hkv", [(16, 8), (40, 8), (12, 4), (16, 1)])
def test_fp16_decode_rounds_probabilities_to_fp16(gpu, monkeypatch, hq, hkv, schedule):
    # Few keys, so that one probability's rounding shows (see test_mxfp4_bounds_host.py).
    monkeypatch.setattr(MI355XMXFP4AttentionBackend, "decode_schedule_override", schedule)
    batch = make_paged_batch(hq, [1] * len(FEW_KEYS), FEW_KEYS, 0, hq, hkv, dtype=FP16)
    k, v = mxfp4.cache_of(batch.k_cache), mxfp4.cache_of(batch.v_cache)
    backend = MI355XMXFP4AttentionBackend(hq, hkv, 128, 16, FP16)
    out = backend.forward(batch.q.to(gpu), None, None, k.to(gpu), v.to(gpu), backend.build_plan(_on(batch.common, gpu)))
    expected, spread, largest = mxfp4.attention(batch.q, k, v, batch.common.block_tables, batch.query_lengths,
                                                batch.kv_lengths)
    bound = attention_bound(expected, spread, largest, max(FEW_KEYS), FP16, FP16)
    assert_within(out, expected, bound + subnormal_bound(max(FEW_KEYS), float(mxfp4.values(v).abs().max()), FP16))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("hq,hkv", [(32, 8), (12, 4), (8, 1)])
def test_mixed_steps_after_their_store(gpu, hq, hkv, dtype):
    q, kv = [50, 7, 130, 1, 1, 1, 1], [180, 7, 130, 300, 17, 1200, 1]
    batch = make_paged_batch(hq, q, kv, 3, hq, hkv, dtype=dtype)
    k, v = mxfp4.cache_of(batch.k_cache), mxfp4.cache_of(batch.v_cache)
    kd, vd = k.to(gpu), v.to(gpu)
    slots = batch.common.slot_mapping.tolist()
    mxfp4.store(batch.k_new, k, slots)
    mxfp4.store(batch.v_new, v, slots)
    backend = MI355XMXFP4AttentionBackend(hq, hkv, 128, 16, dtype)
    common = _on(batch.common, gpu)
    plan = backend.build_plan(common)
    assert plan.route is AttentionRoute.MIXED_SPLIT
    out = backend.forward_with_kv_store(batch.q.to(gpu), batch.k_new.to(gpu), batch.v_new.to(gpu), kd, vd,
                                        common.slot_mapping, plan)
    assert torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), v)
    expected, spread, largest = mxfp4.attention(batch.q, k, v, batch.common.block_tables, q, kv)
    bound = attention_bound(expected, spread, largest, max(kv), dtype, dtype)
    assert_within(out, expected, bound + subnormal_bound(max(kv), float(mxfp4.values(v).abs().max()), dtype))


@pytest.mark.parametrize("hq,hkv", [(16, 8), (8, 1)])
def test_fp16_decode_graph_replays_both_kinds_of_plan(gpu, hq, hkv):
    n, width = 5, 130
    backend = MI355XMXFP4AttentionBackend(hq, hkv, 128, 16, FP16)
    state = backend.create_full_decode_graph_state(n, n * width, gpu)
    caches = torch.zeros(2, *ops.mxfp4_cache_shape(n * width, hkv), dtype=torch.uint8, device=gpu)
    q = torch.zeros(n, hq, 128, dtype=FP16, device=gpu)
    graph = None
    for seed, (ctx, schedule) in enumerate((([100, 7, 64, 300, 1], "shared"), ([2000, 30, 17, 1000, 1], "listed"),
                                            ([2080, 1, 1, 2, 50], "shared"))):
        backend.decode_schedule_override = schedule
        batch = make_paged_batch(seed, [1] * n, ctx, 0, hq, hkv, dtype=FP16)
        k, v = mxfp4.cache_of(batch.k_cache), mxfp4.cache_of(batch.v_cache)
        caches[0, :len(k)], caches[1, :len(v)] = k.to(gpu), v.to(gpu)
        q.copy_(batch.q)
        plan = backend.build_plan(_on(batch.common, gpu))
        eager = backend.forward(q, None, None, caches[0], caches[1], plan).clone()
        expected, spread, largest = mxfp4.attention(batch.q, k, v, batch.common.block_tables, [1] * n, ctx)
        bound = attention_bound(expected, spread, largest, max(ctx), FP16, FP16)
        assert_within(eager, expected, bound + subnormal_bound(max(ctx), float(mxfp4.values(v).abs().max()), FP16))
        backend.plan_full_decode_graph(state, plan)
        backend.activate_full_decode_graph(state)
        try:
            if graph is None:
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    backend.forward(q, None, None, caches[0], caches[1], plan)
        finally:
            backend.deactivate_full_decode_graph()
        for _ in range(3):
            state.output.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(state.output, eager)
            (torch.randn(64, 64, device=gpu) @ torch.randn(64, 64, device=gpu)).sum().item()
