"""The MXFP4 KV cache and attention over it on gfx950 against the 64-bit oracle.

What the cache holds is compared exactly, bytes and values.  Attention is held
to the bound that tests/_mxfp4.py derives from the roundings made.
"""

import shutil
import subprocess
import sys
import types

import pytest
import torch

from my_vllm_amd import _native, attention_backend, ops
from my_vllm_amd.attention_backend import MI355XMXFP4AttentionBackend, integrate_mxfp4
from my_vllm_amd.contract import AttentionRoute, CommonAttentionMetadata
from my_vllm_amd.custom_op import CustomOpConfig
from my_vllm_amd.layers import MXFP4KVCacheStore
from oracle import mxfp4
from tests._mxfp4 import assert_within, attention_bound, cache_pool, poison_stale
from tests._util import set_decode_planning
from workloads import decode_lengths, make_paged_batch

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


# ---- the cache -------------------------------------------------------------------


def _hard_rows(n, h, dtype, seed=0):
    """Rows whose groups span the type: ties, subnormals, the largest values, infinities and NaN."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(n, h, 4, 32, generator=gen)
    scale = torch.exp2(torch.randint(-20, 14, (n, h, 4, 1), generator=gen).float())
    x = (x * scale).to(dtype)
    flat = x.view(-1, 32)
    info = torch.finfo(dtype)
    grid = torch.arange(32) * 0.25  # every code and every tie
    special = [grid, -grid, grid * info.tiny, torch.full((32,), info.max), torch.full((32,), info.smallest_normal / 3),
               torch.linspace(-info.max, info.max, 32), torch.full((32,), 7.0), torch.full((32,), 7.0625),
               torch.cat((torch.tensor([float("inf")]), torch.ones(31))),
               torch.cat((torch.tensor([1.0, -float("inf")]), torch.ones(30))),
               torch.cat((torch.ones(31), torch.tensor([float("nan")]))), torch.zeros(32), -torch.zeros(32),
               torch.full((32,), info.max * 0.9), torch.full((32,), 1.75), torch.full((32,), 1.7578125)]
    for i, group in enumerate(special):
        flat[(i * 5) % flat.shape[0]] = group.to(dtype)
    return x.view(n, h, 128)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("n,h,wide", [(1, 1, False), (3, 8, True), (16, 2, False), (17, 5, False), (300, 8, False),
                                      (1000, 1, True)])
def test_store_matches_the_oracle_byte_for_byte(gpu, dtype, n, h, wide):
    pages = (n + 15) // 16 + 2
    k, v = _hard_rows(n, h, dtype, 1), _hard_rows(n, h, dtype, 2)
    gen = torch.Generator().manual_seed(n)
    slots = torch.randperm(pages * 16, generator=gen)[:n]
    if n > 2:
        slots[1], slots[2] = -1, pages * 16 + 5  # skipped
    before = torch.randint(0, 256, (2, pages, h, 1088), generator=gen, dtype=torch.uint8)
    caches = before.to(gpu)
    ops.store_kvcache_mxfp4(k.to(gpu), v.to(gpu), caches[0], caches[1],
                            slots.to(torch.int64 if wide else torch.int32).to(gpu))
    for rows, cache, got in ((k, before[0].clone(), caches[0]), (v, before[1].clone(), caches[1])):
        mxfp4.store(rows, cache, slots.tolist())
        assert torch.equal(got.cpu(), cache)


def test_store_takes_views_and_skips_everything_else(gpu):
    n, h = 37, 4
    packed = torch.randn(n, 8 + 2 * h, 128, generator=torch.Generator().manual_seed(4)).to(BF16).to(gpu)
    pool = torch.full((2, 3, 5, h, 1088), 7, dtype=torch.uint8, device=gpu)
    slots = torch.arange(3, 3 + n, dtype=torch.int32, device=gpu)
    store = MXFP4KVCacheStore(CustomOpConfig(platform="cuda"))
    store(packed[:, 8:8 + h], packed[:, 8 + h:], pool[0, 1], pool[1, 1], slots)
    expected = torch.full((2, 3, 5, h, 1088), 7, dtype=torch.uint8)
    for i, first in enumerate((8, 8 + h)):
        mxfp4.store(packed[:, first:first + h].cpu(), expected[i, 1], slots.tolist())
    assert torch.equal(pool.cpu(), expected)
    # Rows that start off 16 bytes, and heads apart from one another.
    odd = torch.empty(n * h * 130 + 1, dtype=BF16, device=gpu)[1:].view(n, h, 130)[..., :128]
    odd.copy_(packed[:, 8:8 + h])
    again = torch.full_like(pool, 7)
    ops.store_kvcache_mxfp4(odd, packed[:, 8 + h:], again[0, 1], again[1, 1], slots.long().view(1, -1))
    assert torch.equal(again, pool)
    ops.store_kvcache_mxfp4(odd[:0], odd[:0], again[0, 1], again[1, 1], slots[:0])
    assert torch.equal(again, pool)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("n,h", [(1, 1), (19, 8), (333, 5)])
def test_load_returns_the_values_the_cache_stands_for(gpu, dtype, n, h):
    pages = 24
    rows = _hard_rows(pages * 16, h, dtype, 3)
    rows[5, 0, 40] = float("nan")
    cache = torch.zeros(2, pages, h, 1088, dtype=torch.uint8)
    mxfp4.store(rows, cache[0], list(range(pages * 16)))
    mxfp4.store(rows.flip(0), cache[1], list(range(pages * 16)))
    slots = torch.randint(0, pages * 16, (n,), generator=torch.Generator().manual_seed(n))  # the same slot twice too
    if n > 2:
        slots[0], slots[1], slots[2] = -1, pages * 16, 5
    dev = cache.to(gpu)
    got = ops.load_kvcache_mxfp4(dev[0], dev[1], slots.to(gpu), dtype)
    for one, part in zip(got, cache):
        held = mxfp4.values(part).reshape(-1, h, 128)
        expected = torch.where(((slots >= 0) & (slots < pages * 16))[:, None, None],
                               held[slots.clamp(0, pages * 16 - 1)], 0.0)
        assert one.dtype == dtype and one.shape == (n, h, 128)
        assert torch.equal(one.cpu().double().nan_to_num(nan=1e300), expected.nan_to_num(nan=1e300))
    k, v = ops.load_kvcache_mxfp4(dev[0], dev[1], slots[:0].to(gpu), dtype)
    assert k.shape == v.shape == (0, h, 128)


def test_every_byte_reads_back(gpu):
    # All scale bytes but the NaN one, all codes, in both types.
    scales = torch.arange(256, dtype=torch.uint8)
    cache = torch.zeros(4, 1, 1088, dtype=torch.uint8)
    cache[..., :1024] = (torch.arange(16) + 16 * torch.arange(15, -1, -1)).to(torch.uint8).repeat(64)
    cache[..., 1024:] = scales.view(4, 1, 64)
    dev = cache.to(gpu)
    held = mxfp4.values(cache).reshape(-1, 1, 128)
    for dtype in (BF16, FP16):
        got = ops.load_kvcache_mxfp4(dev, dev, torch.arange(64, device=gpu), dtype)[0].cpu()
        assert torch.equal(got.nan_to_num(nan=7.7, posinf=9.9, neginf=-9.9),
                           held.to(dtype).nan_to_num(nan=7.7, posinf=9.9, neginf=-9.9))


def test_store_and_load_on_another_stream_and_in_a_graph(gpu):
    n, h = 40, 8
    k = torch.randn(n, h, 128, device=gpu).to(BF16)
    slots = torch.randperm(64, device=gpu)[:n]
    cache = torch.zeros(2, 4, h, 1088, dtype=torch.uint8, device=gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.store_kvcache_mxfp4(k, -k, cache[0], cache[1], slots)
        got = ops.load_kvcache_mxfp4(cache[0], cache[1], slots)
    torch.cuda.current_stream().wait_stream(side)
    want = ops.load_kvcache_mxfp4(cache[0], cache[1], slots)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], -want[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.store_kvcache_mxfp4(k, -k, cache[0], cache[1], slots)
        replayed = ops.load_kvcache_mxfp4(cache[0], cache[1], slots)
    for seed in range(3):
        k.copy_(torch.randn(n, h, 128, device=gpu, generator=torch.Generator(gpu).manual_seed(seed)))
        graph.replay()
        got = replayed[0].clone()
        torch.cuda.synchronize()
        other = torch.zeros_like(cache)
        ops.store_kvcache_mxfp4(k, -k, other[0], other[1], slots)
        assert torch.equal(got, ops.load_kvcache_mxfp4(other[0], other[1], slots)[0])


def test_gpu_refusals(gpu):
    k = torch.zeros(4, 2, 128, dtype=BF16, device=gpu)
    cache = torch.zeros(2, 2, 1088, dtype=torch.uint8, device=gpu)
    slots = torch.zeros(4, dtype=torch.int32, device=gpu)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        ops.store_kvcache_mxfp4(k.float(), k.float(), cache, cache, slots)
    with pytest.raises(ValueError, match="number of KV heads"):
        ops.store_kvcache_mxfp4(k[:, :1], k[:, :1], cache, cache, slots)
    with pytest.raises(ValueError, match="one slot per token"):
        ops.store_kvcache_mxfp4(k, k, cache, cache, slots[:3])
    with pytest.raises(TypeError, match="int32 or int64"):
        ops.store_kvcache_mxfp4(k, k, cache, cache, slots.float())
    with pytest.raises(RuntimeError, match="device"):
        ops.store_kvcache_mxfp4(k, k, cache, cache, slots.cpu())
    with pytest.raises(TypeError, match="reads rows as"):
        ops.load_kvcache_mxfp4(cache, cache, slots, torch.float32)
    backend = MI355XMXFP4AttentionBackend(16, 8, 128, 16, BF16)
    batch = make_paged_batch(1, [1], [40], 0, 16, 8)
    common = _on(batch.common, gpu)
    plan = backend.build_plan(common)
    q = batch.q.to(gpu)
    with pytest.raises(ValueError, match="uint8"):
        backend.forward(q, None, None, batch.k_cache.to(gpu), batch.v_cache.to(gpu), plan)
    wrong = torch.zeros(3, 4, 1088, dtype=torch.uint8, device=gpu)
    with pytest.raises(ValueError, match="shape"):
        backend.forward(q, None, None, wrong, wrong, plan)


# ---- attention -------------------------------------------------------------------


def _on(common, device):
    return type(common)(**{**common.__dict__,
                           "query_start_loc": common.query_start_loc.to(device),
                           "seq_lens": common.seq_lens.to(device),
                           "slot_mapping": common.slot_mapping.to(device),
                           "block_tables": common.block_tables.to(device)})


def _check(out, batch, k, v, dtype, p_dtype=BF16):
    expected, spread, largest = mxfp4.attention(batch.q, k, v, batch.common.block_tables, batch.query_lengths,
                                                batch.kv_lengths)
    assert out.dtype == dtype
    assert_within(out, expected, attention_bound(expected, spread, largest, max(batch.kv_lengths), dtype, p_dtype))


def _forward(batch, device, dtype, poison=True):
    """The backend's output over the batch's caches in MXFP4, and those caches on the CPU."""
    hq, hkv = batch.q.shape[1], batch.k_cache.shape[2]
    kd, vd, k, v = cache_pool(batch, device)
    if poison:
        for cache, on_gpu, seed in ((k, kd, 5), (v, vd, 6)):
            poison_stale(cache, batch.common.block_tables, batch.kv_lengths, seed)
            on_gpu.copy_(cache)
    backend = MI355XMXFP4AttentionBackend(hq, hkv, 128, 16, dtype)
    plan = backend.build_plan(_on(batch.common, device))
    out = backend.forward(batch.q.to(device), None, None, kd, vd, plan)
    return out, backend, plan, (kd, vd, k, v)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("hq,hkv", [(16, 8), (32, 8), (64, 8), (16, 4), (16, 2), (8, 1), (12, 4), (40, 8), (16, 1),
                                    (6, 6), (9, 3)])
def test_decode(gpu, hq, hkv, dtype):
    ctx = [1, 2, 15, 16, 17, 63, 64, 65, 80, 129, 700]
    batch = make_paged_batch(hq + hkv, [1] * len(ctx), ctx, 0, hq, hkv, dtype=dtype, extra_pages=3)
    out, backend, plan, (_, _, k, v) = _forward(batch, gpu, dtype)
    assert plan.route is AttentionRoute.DECODE
    _check(out, batch, k, v, dtype)


@pytest.mark.parametrize("per_group", [4, 12])
@pytest.mark.parametrize("waves", [8, 24, 64, 512])
def test_decode_with_long_piece_lists(gpu, monkeypatch, waves, per_group):
    # Many pieces a wavefront, of every length modulo a tile, with one longer than a run of 256 pages; both
    # workgroup sizes.
    set_decode_planning(monkeypatch, waves=waves)
    monkeypatch.setattr(attention_backend, "_MXFP4_WAVES", ((8, per_group), (12, 12)))
    ctx = [1, 16, 17, 33, 48, 64, 65, 100, 113, 128, 129, 200, 8500, 5, 31, 47]
    batch = make_paged_batch(waves, [1] * len(ctx), ctx, 0, 16, 8)
    out, backend, plan, (_, _, k, v) = _forward(batch, gpu, BF16)
    assert plan.metadata.num_decode_waves <= max(waves, 8)
    assert plan.metadata.decode_waves_per_group == per_group
    if waves == 8:
        assert (plan.metadata.decode_items[:, 2] - plan.metadata.decode_items[:, 1]).max() > 512
    _check(out, batch, k, v, BF16)


@pytest.mark.parametrize("hq,hkv,ctx,dtype", [(32, 8, [9001], BF16), (8, 1, [6000, 3], FP16), (16, 2, [4097] * 3, BF16),
                                              (64, 8, [300] * 70, BF16)])
def test_decode_split_and_wide(gpu, hq, hkv, ctx, dtype):
    batch = make_paged_batch(len(ctx), [1] * len(ctx), ctx, 0, hq, hkv, dtype=dtype)
    out, backend, plan, (kd, vd, k, v) = _forward(batch, gpu, dtype)
    _check(out, batch, k, v, dtype)
    # The same bits again over the same workspace, and from a strided query.
    first = out.clone()
    packed = torch.randn(len(ctx), hq + 5, 128, device=gpu).to(dtype)
    packed[:, 2:2 + hq] = batch.q.to(gpu)
    assert torch.equal(backend.forward(packed[:, 2:2 + hq], None, None, kd, vd, plan), first)


def test_decode_of_large_scores(gpu):
    # Scores of several hundred: the reference maximum moves, most rows underflow.
    ctx = [70, 500, 1300]
    batch = make_paged_batch(9, [1] * 3, ctx, 0, 16, 8)
    batch.q.mul_(40)
    out, _, _, (_, _, k, v) = _forward(batch, gpu, BF16)
    _check(out, batch, k, v, BF16)


def test_decode_of_unlike_value_scales(gpu):
    # V groups from 2^-60 to 2^60: the scaled probabilities leave fp16's range.
    batch = make_paged_batch(10, [1] * 2, [300, 77], 0, 16, 8)
    sizes = torch.exp2(torch.randint(-60, 60, (*batch.v_cache.shape[:3], 4, 1),
                                     generator=torch.Generator().manual_seed(1)).float())
    batch.v_cache.copy_((batch.v_cache.float().unflatten(-1, (4, 32)) * sizes).flatten(-2))
    out, _, _, (_, _, k, v) = _forward(batch, gpu, BF16)
    _check(out, batch, k, v, BF16)


def test_nan_groups_reach_the_rows_that_see_them(gpu):
    ctx = [40, 200]
    batch = make_paged_batch(11, [1, 1], ctx, 0, 16, 8)
    batch.k_cache[batch.common.block_tables[0, 1], 3, 2, 5] = float("nan")  # head 2 of sequence 0
    batch.v_cache[batch.common.block_tables[1, 7], 9, 4, 70] = float("inf")  # group 2 of head 4 of sequence 1
    out, *_ = _forward(batch, gpu, BF16, poison=False)
    nan = torch.isnan(out.cpu())
    expected = torch.zeros_like(nan)
    expected[0, 4:6] = True
    expected[1, 8:10, 64:96] = True
    assert torch.equal(nan, expected)


@pytest.mark.parametrize("schedule", ["shared", "listed"])
def test_nan_groups_pass_the_joins(gpu, monkeypatch, schedule):
    # In one chunk of several: through the joins in LDS and the merge.
    monkeypatch.setattr(MI355XMXFP4AttentionBackend, "decode_schedule_override", schedule)
    batch = make_paged_batch(12, [1, 1, 1], [5000, 5000, 90], 0, 16, 8)
    table = batch.common.block_tables
    batch.k_cache[table[0, 100], 3, 2, 5] = float("nan")
    batch.v_cache[table[1, 311], 9, 4, 70] = float("inf")
    batch.v_cache[table[2, 5], 9, 0, 127] = float("nan")  # the last token
    out, _, plan, _ = _forward(batch, gpu, BF16, poison=False)
    assert plan.metadata.num_decode_merges > 0
    nan = torch.isnan(out.cpu())
    expected = torch.zeros_like(nan)
    expected[0, 4:6] = True
    expected[1, 8:10, 64:96] = True
    expected[2, 0:2, 96:] = True
    assert torch.equal(nan, expected)


@pytest.mark.parametrize("dtype,hq,hkv", [(BF16, 32, 8), (FP16, 16, 8), (BF16, 12, 4), (FP16, 8, 1), (BF16, 16, 1)])
def test_prefill(gpu, dtype, hq, hkv):
    q = [1, 37, 130, 64, 2, 300]
    kv = [1, 37 + 48, 130, 64 + 200, 2 + 15, 300 + 16 * 20]
    batch = make_paged_batch(hq, q, kv, len(q), hq, hkv, dtype=dtype, extra_pages=2)
    out, backend, plan, (kd, vd, k, v) = _forward(batch, gpu, dtype)
    assert plan.route is AttentionRoute.PREFILL
    _check(out, batch, k, v, dtype, dtype)
    # Later layers run the step's tile plan over their own caches.
    first = out.clone()
    assert torch.equal(backend.forward(batch.q.to(gpu), None, None, kd, vd, plan), first)
    backend.forward(batch.q.to(gpu), None, None, vd, kd, plan)
    swapped, spread, largest = mxfp4.attention(batch.q, v, k, batch.common.block_tables, q, kv)
    assert_within(backend.forward(batch.q.to(gpu), None, None, vd, kd, plan), swapped,
                  attention_bound(swapped, spread, largest, max(kv), dtype, dtype))


@pytest.mark.parametrize("q,kv", [([1], [1]), ([1], [4000]), ([1200], [1200]), ([17, 1, 1], [17, 1000, 16]),
                                  ([700] * 5, [1500, 700, 900, 2000, 701])])
def test_prefill_lengths(gpu, q, kv):
    batch = make_paged_batch(sum(q), q, kv, len(q), 32, 8)
    out, _, _, (_, _, k, v) = _forward(batch, gpu, BF16)
    _check(out, batch, k, v, BF16)


def test_mixed_step_after_its_store(gpu):
    """A chunked-prefill step as the model runner drives it: rows in, then attention over them."""
    q, kv = [50, 7, 1, 1, 1], [50 + 130, 7, 300, 17, 1200]
    batch = make_paged_batch(21, q, kv, 2, 32, 8)
    kd, vd, k, v = cache_pool(batch, gpu)
    slots = batch.common.slot_mapping.tolist()
    mxfp4.store(batch.k_new, k, slots)
    mxfp4.store(batch.v_new, v, slots)
    backend = MI355XMXFP4AttentionBackend(32, 8, 128, 16, BF16)
    common = _on(batch.common, gpu)
    plan = backend.build_plan(common)
    assert plan.route is AttentionRoute.MIXED_SPLIT
    out = backend.forward_with_kv_store(batch.q.to(gpu), batch.k_new.to(gpu), batch.v_new.to(gpu), kd, vd,
                                        common.slot_mapping, plan)
    assert torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), v)
    _check(out, batch, k, v, BF16)


def test_generation_of_one_sequence(gpu):
    """Prompt, chunk, then single tokens: every step's cache and attention."""
    hq, hkv, total = 12, 4, 90
    gen = torch.Generator().manual_seed(3)
    rows = [torch.randn(total, n, 128, generator=gen).to(BF16) for n in (hq, hkv, hkv)]
    table = torch.tensor([[4, 1, 5, 0, 3, 2]], dtype=torch.int32)
    host = [torch.zeros(6, hkv, 1088, dtype=torch.uint8) for _ in range(2)]
    dev = [c.to(gpu) for c in host]
    backend = MI355XMXFP4AttentionBackend(hq, hkv, 128, 16, BF16)
    done = 0
    for n in (33, 40, 1, 1, 1, 1, 1, 1, 1, 1, 1):
        end = done + n
        slots = [int(table[0, t // 16]) * 16 + t % 16 for t in range(done, end)]
        pages = (end + 15) // 16
        prefill = n > 1
        common = CommonAttentionMetadata(
            num_prefill_seqs=int(prefill), num_decode_seqs=int(not prefill), num_prefill_tokens=n if prefill else 0,
            num_decode_tokens=0 if prefill else 1,
            query_start_loc=torch.tensor([0, n], dtype=torch.int32, device=gpu),
            seq_lens=torch.tensor([end], dtype=torch.int32, device=gpu),
            slot_mapping=torch.tensor(slots, dtype=torch.int32, device=gpu), block_tables=table.to(gpu), max_q_len=n,
            max_kv_len=end, block_counts=(pages,), num_kv_blocks=pages, num_prefill_kv_blocks=pages * prefill,
            trusted=True)
        q, k, v = (r[done:end] for r in rows)
        out = backend.forward_with_kv_store(q.to(gpu), k.to(gpu), v.to(gpu), *dev, common.slot_mapping,
                                            backend.build_plan(common))
        for new, cache in ((k, host[0]), (v, host[1])):
            mxfp4.store(new, cache, slots)
        expected, spread, largest = mxfp4.attention(q, *host, table, [n], [end])
        assert_within(out, expected, attention_bound(expected, spread, largest, end, BF16, BF16))
        done = end
    assert torch.equal(dev[0].cpu(), host[0]) and torch.equal(dev[1].cpu(), host[1])


def test_warmup_runs_on_the_new_rows(gpu):
    batch = make_paged_batch(31, [20, 33], [20, 33], 2, 16, 8)
    common = type(batch.common)(**{**_on(batch.common, gpu).__dict__, "block_tables": None})
    backend = MI355XMXFP4AttentionBackend(16, 8, 128, 16, BF16)
    plan = backend.build_plan(common)
    assert plan.route is AttentionRoute.WARMUP
    empty = torch.empty(0, dtype=torch.uint8, device=gpu)
    out = backend.forward(batch.q.to(gpu), batch.k_new.to(gpu), batch.v_new.to(gpu), empty, empty, plan)
    assert torch.isfinite(out).all() and out.shape == batch.q.shape


@pytest.mark.parametrize("hq,hkv,batch,width", [(16, 8, 6, 40), (8, 1, 3, 60)])
def test_decode_graph_replays(gpu, hq, hkv, batch, width):
    backend = MI355XMXFP4AttentionBackend(hq, hkv, 128, 16, BF16)
    pages = batch * width
    state = backend.create_full_decode_graph_state(batch, pages, gpu)
    caches = torch.zeros(2, *ops.mxfp4_cache_shape(pages, hkv), dtype=torch.uint8, device=gpu)
    q_static = torch.zeros(batch, hq, 128, dtype=BF16, device=gpu)
    capture = CommonAttentionMetadata(
        num_prefill_seqs=0, num_decode_seqs=batch, num_prefill_tokens=0, num_decode_tokens=batch,
        query_start_loc=torch.arange(batch + 1, dtype=torch.int32, device=gpu),
        seq_lens=torch.ones(batch, dtype=torch.int32, device=gpu),
        slot_mapping=torch.full((batch,), -1, dtype=torch.int32, device=gpu),
        block_tables=torch.zeros((batch, 1), dtype=torch.int32, device=gpu),
        max_q_len=1, max_kv_len=1, block_counts=(1,) * batch, num_kv_blocks=batch, num_prefill_kv_blocks=0,
        trusted=True)
    plan = backend.build_plan(capture)
    backend.plan_full_decode_graph(state, plan)
    backend.activate_full_decode_graph(state)
    try:
        backend.forward(q_static, None, None, caches[0], caches[1], plan)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            backend.forward(q_static, None, None, caches[0], caches[1], plan)
        torch.cuda.synchronize()
    finally:
        backend.deactivate_full_decode_graph()
    for seed in (11, 12, 13):
        ctx = decode_lengths(seed, batch, 1, width * 16)
        ctx[0], ctx[-1] = width * 16, 1
        b = make_paged_batch(seed, [1] * batch, ctx, 0, hq, hkv)
        k, v = mxfp4.cache_of(b.k_cache), mxfp4.cache_of(b.v_cache)
        caches.zero_()
        caches[0, :k.shape[0]].copy_(k)
        caches[1, :v.shape[0]].copy_(v)
        q_static.copy_(b.q)
        step = backend.build_plan(_on(b.common, gpu))
        backend.plan_full_decode_graph(state, step)
        graph.replay()
        got = state.output.clone()
        torch.cuda.synchronize()
        x = torch.randn(256, 256, device=gpu)
        (x @ x).sum().item()
        assert torch.equal(got, backend.forward(q_static, None, None, caches[0], caches[1], step))
        _check(got, b, k, v, BF16)


def test_two_backends_on_two_streams(gpu):
    ctx = [900, 33, 1500]
    batch = make_paged_batch(41, [1] * 3, ctx, 0, 32, 8)
    kd, vd, k, v = cache_pool(batch, gpu)
    q = batch.q.to(gpu)
    common = _on(batch.common, gpu)
    pairs = []
    for _ in range(2):
        backend = MI355XMXFP4AttentionBackend(32, 8, 128, 16, BF16)
        pairs.append((backend, backend.build_plan(common), torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        for backend, plan, stream in pairs:
            with torch.cuda.stream(stream):
                outs.append(backend.forward(q, None, None, kd, vd, plan).clone())
    torch.cuda.synchronize()
    assert all(torch.equal(o, outs[0]) for o in outs)
    _check(outs[0], batch, k, v, BF16)


def test_caches_beyond_32_bit_offsets(gpu):
    """K and V of more than 4 GiB each: rows stored, read back and attended to at their far end."""
    hq, hkv, far = 16, 8, 4 << 30
    pages = far // (hkv * 1088) + 40
    ctx, q_lens = [500, 37], [1, 1]
    batch = make_paged_batch(51, q_lens, ctx, 0, hq, hkv)
    count = batch.k_cache.shape[0]
    first = pages - count
    caches = torch.empty(2, pages, hkv, 1088, dtype=torch.uint8, device=gpu)
    assert first * hkv * 1088 > far - (1 << 20) and (pages - 1) * hkv * 1088 > far
    k, v = mxfp4.cache_of(batch.k_cache), mxfp4.cache_of(batch.v_cache)
    caches[0, first:], caches[1, first:] = k.to(gpu), v.to(gpu)
    common = _on(batch.common, gpu)
    tables = torch.where(common.block_tables >= 0, common.block_tables + first, -1)
    common = type(common)(**{**common.__dict__, "block_tables": tables,
                             "slot_mapping": common.slot_mapping + first * 16})
    backend = MI355XMXFP4AttentionBackend(hq, hkv, 128, 16, BF16)
    out = backend.forward_with_kv_store(batch.q.to(gpu), batch.k_new.to(gpu), batch.v_new.to(gpu), caches[0],
                                        caches[1], common.slot_mapping, backend.build_plan(common))
    slots = batch.common.slot_mapping.tolist()
    mxfp4.store(batch.k_new, k, slots)
    mxfp4.store(batch.v_new, v, slots)
    _check(out, batch, k, v, BF16)
    rows = ops.load_kvcache_mxfp4(caches[0], caches[1], common.slot_mapping)
    for got, cache in zip(rows, (k, v)):
        assert torch.equal(got.cpu().double(), mxfp4.values(cache).reshape(-1, hkv, 128)[slots])
    # A prefill over the same pages.
    chunk = make_paged_batch(51, [20, 37], ctx, 2, hq, hkv)
    chunk_common = _on(chunk.common, gpu)
    chunk_common = type(common)(**{**chunk_common.__dict__, "block_tables": tables})
    out = backend.forward(chunk.q.to(gpu), None, None, caches[0], caches[1], backend.build_plan(chunk_common))
    expected, spread, largest = mxfp4.attention(chunk.q, k, v, batch.common.block_tables, [20, 37], ctx)
    assert_within(out, expected, attention_bound(expected, spread, largest, 500, BF16, BF16))


def test_captured_steps_replay_beside_eager_ones(gpu):
    """A prefill and a decode step captured as they are, replayed between eager steps of the same backend."""
    hq, hkv = 32, 8
    pre = make_paged_batch(61, [70, 200], [70 + 64, 200], 2, hq, hkv)
    dec = make_paged_batch(62, [1] * 5, [300, 17, 90, 1000, 33], 0, hq, hkv)
    backend = MI355XMXFP4AttentionBackend(hq, hkv, 128, 16, BF16)
    steps = []
    for batch in (pre, dec):
        kd, vd, k, v = cache_pool(batch, gpu)
        q = batch.q.to(gpu)
        common = _on(batch.common, gpu)
        plan = backend.build_plan(common)
        eager = backend.forward(q, None, None, kd, vd, plan).clone()
        _check(eager, batch, k, v, BF16)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = backend.forward(q, None, None, kd, vd, plan).clone()
        steps.append((graph, out, eager, lambda q=q, kd=kd, vd=vd, c=common: backend.forward(
            q, None, None, kd, vd, backend.build_plan(c))))
    for _ in range(3):
        for graph, out, eager, again in steps:
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, eager)
            (torch.randn(256, 256, device=gpu) @ torch.randn(256, 256, device=gpu)).sum().item()
            assert torch.equal(again(), eager)


def test_native_and_general_launches_agree(gpu, monkeypatch):
    """Every operator through the native module and through ctypes: the same bits and the same errors."""
    real = _native.host_ops()
    names = [n for n in dir(real) if not n.startswith("_") and callable(getattr(real, n))]
    batch = make_paged_batch(71, [1] * 3, [40, 300, 700], 0, 16, 8)
    chunk = make_paged_batch(72, [30, 9], [100, 9], 2, 16, 8)
    kd, vd, _, _ = cache_pool(batch, gpu)
    kp, vp, _, _ = cache_pool(chunk, gpu)
    rows = torch.randn(6, 8, 128, device=gpu).to(BF16)
    slots = torch.tensor([3, 0, -1, 40, 41, 9], device=gpu)

    def calls():
        store = torch.zeros(2, 4, 8, 1088, dtype=torch.uint8, device=gpu)
        ops.store_kvcache_mxfp4(rows, -rows, store[0], store[1], slots)
        backend = MI355XMXFP4AttentionBackend(16, 8, 128, 16, BF16)
        decode = backend.forward(batch.q.to(gpu), None, None, kd, vd, backend.build_plan(_on(batch.common, gpu)))
        backend = MI355XMXFP4AttentionBackend(16, 8, 128, 16, BF16)
        prefill = backend.forward(chunk.q.to(gpu), None, None, kp, vp, backend.build_plan(_on(chunk.common, gpu)))
        return [store, decode, prefill, *ops.load_kvcache_mxfp4(store[0], store[1], slots, FP16)]

    def errors():
        found = []
        backend = MI355XMXFP4AttentionBackend(16, 8, 128, 16, BF16)
        plan = backend.build_plan(_on(batch.common, gpu))
        q = batch.q.to(gpu)
        odd = torch.empty(3 * 16 * 128 + 1, dtype=BF16, device=gpu)[1:].view(3, 16, 128)
        for call in (lambda: backend.forward(odd, None, None, kd, vd, plan),
                     lambda: backend.forward(q, None, None, kd, vd[:-1], plan),
                     lambda: backend.forward(q.half(), None, None, kd, vd, plan),
                     lambda: ops.store_kvcache_mxfp4(rows, rows[:, :4], kd, vd, slots),
                     lambda: ops.load_kvcache_mxfp4(kd, vd.view(torch.int8), slots)):
            with pytest.raises(Exception) as info:
                call()
            found.append((info.type, str(info.value)))
        return found

    fast, fast_errors = calls(), errors()
    monkeypatch.setattr(_native, "_host", types.SimpleNamespace(
        **{n: (real.capture_id if n == "capture_id" else lambda *a: None) for n in names}))
    for a, b in zip(fast, calls()):
        assert torch.equal(a, b)
    assert errors() == fast_errors


def test_foreign_contract_family(gpu):
    from tests import _foreign_contract as foreign

    registered = {}
    registry = types.SimpleNamespace(register=lambda name, cls: registered.__setitem__(name, cls))
    made = integrate_mxfp4(registry, foreign.ForeignBackendBase, foreign.ForeignPlan, foreign.ForeignRoute,
                           foreign.ForeignBatchType, foreign.ForeignCommon)
    assert registered == {"mi355x_mxfp4": made}
    batch = make_paged_batch(81, [9, 1], [40, 77], 1, 16, 8)
    kd, vd, k, v = cache_pool(batch, gpu)
    common = foreign.ForeignCommon(**_on(batch.common, gpu).__dict__)
    backend = made(16, 8, 128, 16, BF16)
    plan = backend.build_plan(common)
    assert type(plan) is foreign.ForeignPlan and plan.route is foreign.ForeignRoute.MIXED_SPLIT
    _check(backend.forward(batch.q.to(gpu), None, None, kd, vd, plan), batch, k, v, BF16)


@pytest.mark.parametrize("large", [False, True])
@pytest.mark.parametrize("hq,hkv,dtype", [(8, 8, BF16), (16, 8, FP16), (32, 2, BF16), (24, 8, FP16), (5, 1, BF16)])
def test_shared_segments_of_every_length(gpu, monkeypatch, hq, hkv, dtype, large):
    """Four wavefronts a piece: lengths that leave some of them without pages, and long ones that are cut."""
    monkeypatch.setattr(MI355XMXFP4AttentionBackend, "decode_schedule_override", "shared")
    ctx = [1, 15, 16, 17, 32, 33, 64, 65, 95, 96, 97, 128, 129, 300, 2047, 9000]
    batch = make_paged_batch(hq, [1] * len(ctx), ctx, 0, hq, hkv, dtype=dtype)
    k, v = mxfp4.cache_of(batch.k_cache), mxfp4.cache_of(batch.v_cache)
    for cache, seed in ((k, 1), (v, 2)):
        poison_stale(cache, batch.common.block_tables, ctx, seed)
    backend = MI355XMXFP4AttentionBackend(hq, hkv, 128, 16, dtype)
    plan = backend.build_plan(_on(batch.common, gpu))
    metadata = plan.metadata
    assert metadata.num_decode_merges >= hkv and (metadata.decode_items[:, 5] < 0).all()
    q, kd, vd = batch.q.to(gpu), k.to(gpu), v.to(gpu)
    if not large:
        _check(backend.forward(q, None, None, kd, vd, plan), batch, k, v, dtype)
        return
    # The same plan in workgroups of twelve.
    out = torch.full_like(q, float("nan"))
    ops.paged_decode_mxfp4(q, kd, vd, metadata.block_tables, metadata.seq_lens, metadata.decode_items,
                           metadata.num_decode_items, metadata.num_decode_waves, metadata.decode_merges,
                           metadata.num_decode_merges, metadata.num_decode_part_slots, out,
                           torch.zeros(ops.decode_workspace_bytes(metadata.num_decode_part_slots, hkv, hq // hkv),
                                       dtype=torch.uint8, device=gpu),
                           backend.softmax_scale, metadata.decode_wave_extra, 12)
    _check(out, batch, k, v, dtype)
    assert torch.equal(out, backend.forward(q, None, None, kd, vd, plan))


def test_one_graph_replays_shared_and_listed_steps(gpu):
    """Steps of one captured launch whose plans are of either kind."""
    hq, hkv, n, width = 16, 8, 6, 260
    backend = MI355XMXFP4AttentionBackend(hq, hkv, 128, 16, BF16)
    state = backend.create_full_decode_graph_state(n, n * width, gpu)
    caches = torch.zeros(2, *ops.mxfp4_cache_shape(n * width, hkv), dtype=torch.uint8, device=gpu)
    q = torch.zeros(n, hq, 128, dtype=BF16, device=gpu)
    graph, kinds = None, []
    for seed, (ctx, schedule) in enumerate((([100, 7, 64, 300, 16, 1], None), ([4100, 30, 17, 1000, 1, 900], "listed"),
                                            ([500] * 6, "listed"), ([4160] * 6, None), ([4100, 1, 1, 2, 3, 50], None))):
        backend.decode_schedule_override = schedule
        batch = make_paged_batch(seed, [1] * n, ctx, 0, hq, hkv)
        k, v = mxfp4.cache_of(batch.k_cache), mxfp4.cache_of(batch.v_cache)
        caches[0, :len(k)], caches[1, :len(v)] = k.to(gpu), v.to(gpu)
        q.copy_(batch.q)
        plan = backend.build_plan(_on(batch.common, gpu))
        kinds.append((bool((plan.metadata.decode_items[:, 5] < 0).all()), plan.metadata.num_decode_merges > 0))
        eager = backend.forward(q, None, None, caches[0], caches[1], plan).clone()
        _check(eager, batch, k, v, BF16)
        assert backend.full_decode_graph_metadata_fits(state, plan)
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
        for _ in range(2):
            state.output.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(state.output, eager)
    assert kinds == [(True, False), (False, True), (False, True), (True, True), (True, True)]


GIL_CALLS = """
import importlib.machinery, importlib.util, sys
import torch

loader = importlib.machinery.ExtensionFileLoader("mva_host", sys.argv[1])
host = importlib.util.module_from_spec(importlib.util.spec_from_loader("mva_host", loader))
loader.exec_module(host)
i32 = dict(dtype=torch.int32, device="cuda")
q, kv = (torch.zeros(4, n, 128, dtype=torch.bfloat16, device="cuda") for n in (8, 2))
cache, ws = torch.zeros(2, 2, 1088, dtype=torch.uint8, device="cuda"), torch.zeros(64, dtype=torch.uint8, device="cuda")
ints, bt = torch.zeros(8, **i32), torch.zeros(4, 2, **i32)
for name, args in (("store_kvcache_mxfp4", (kv, kv, cache, cache, ints[:4])),
                   ("load_kvcache_mxfp4", (cache, cache, ints, 0)),
                   ("paged_decode_mxfp4", (q, cache, cache, bt, ints, None, ints, 1, 1, ints, 0, 0, q, ws, 0.1, ints, 4)),
                   ("paged_prefill_mxfp4", (q, cache, cache, bt, ints, ints, 1, 1, ws, q, 0.1, False))):
    got = getattr(host, name)(*args)
    assert (got is None) if sys.argv[2] == "absent" else (got is not None), name
print("done")
"""


@pytest.mark.parametrize("library", ["present", "absent"])
def test_launches_release_the_gil(gpu, tmp_path, library):
    # Beside a stand-in for the C library whose entry points fail if their thread holds the GIL.  One
    # without them leaves the calls to the general path.
    names = ("mva_silu_and_mul", "mva_rms_norm", "mva_fused_add_rms_norm", "mva_qk_norm_rope_store",
             "mva_paged_decode", "mva_paged_decode_store", "mva_paged_prefill", "mva_paged_prefill_run",
             "mva_paged_mixed", "mva_paged_mixed_run")
    if library == "present":
        names += ("mva_kv_store_mxfp4", "mva_kv_load_mxfp4", "mva_paged_decode_mxfp4", "mva_paged_prefill_mxfp4")
    source = tmp_path / "stand_in.c"
    source.write_text("extern int PyGILState_Check(void);\n"
                      'const char* mva_last_error(void) { return "the launch holds the GIL"; }\n'
                      + "".join(f"int {name}(void) {{ return PyGILState_Check(); }}\n" for name in names))
    subprocess.run(["gcc", "-shared", "-fPIC", str(source), "-o", str(tmp_path / _native.LIB_PATH.name)], check=True)
    module = shutil.copy(_native.HOST_PATH, tmp_path)
    run = subprocess.run([sys.executable, "-c", GIL_CALLS, str(module), library], capture_output=True, text=True,
                         timeout=100)
    assert "done" in run.stdout, run.stderr


def test_calls_on_two_streams_at_once(gpu):
    """Two backends' decode and prefill steps side by side on two streams: each as alone."""
    sides = []
    for seed, (hq, hkv) in enumerate(((32, 8), (16, 4))):
        dec = make_paged_batch(seed, [1] * 12, decode_lengths(seed, 12, 1, 2000), 0, hq, hkv)
        pre = make_paged_batch(seed, [100, 300], [200, 300], 2, hq, hkv)
        backend = MI355XMXFP4AttentionBackend(hq, hkv, 128, 16, BF16)
        steps = []
        for batch in (dec, pre):
            kd, vd, _, _ = cache_pool(batch, gpu)
            q, plan = batch.q.to(gpu), backend.build_plan(_on(batch.common, gpu))
            alone = backend.forward(q, None, None, kd, vd, plan).clone()
            steps.append((q, kd, vd, plan, alone))
        sides.append((backend, torch.cuda.Stream(), steps))
    torch.cuda.synchronize()
    found = []
    for _ in range(10):
        for which in (0, 1):
            for backend, stream, steps in sides:
                q, kd, vd, plan, alone = steps[which]
                with torch.cuda.stream(stream):
                    found.append((backend.forward(q, None, None, kd, vd, plan).clone(), alone))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in found)


def test_padding_rows_and_rows_behind_the_last_stay(gpu):
    """Slots of -1 and tokens behind a call's last leave the cache and the output buffer alone."""
    rows = torch.randn(70, 8, 128, device=gpu).to(BF16)
    cache = torch.full((2, 6, 8, 1088), 0x5a, dtype=torch.uint8, device=gpu)
    slots = torch.full((70,), -1, dtype=torch.int32, device=gpu)
    slots[:3] = torch.tensor([17, 40, 95])
    ops.store_kvcache_mxfp4(rows, rows, cache[0], cache[1], slots)
    want = torch.full((6, 8, 1088), 0x5a, dtype=torch.uint8)
    mxfp4.store(rows[:3].cpu(), want, [17, 40, 95])
    assert torch.equal(cache[0].cpu(), want) and torch.equal(cache[1].cpu(), want)
    batch = make_paged_batch(5, [1] * 4, [20, 300, 16, 900], 0, 16, 8)
    kd, vd, k, v = cache_pool(batch, gpu)
    backend = MI355XMXFP4AttentionBackend(16, 8, 128, 16, BF16)
    m = backend.build_plan(_on(batch.common, gpu)).metadata
    out = torch.full((7, 16, 128), 2.0, dtype=BF16, device=gpu)
    ops.paged_decode_mxfp4(batch.q.to(gpu), kd, vd, m.block_tables, m.seq_lens, m.decode_items, m.num_decode_items,
                           m.num_decode_waves, m.decode_merges, m.num_decode_merges, m.num_decode_part_slots, out,
                           torch.zeros(ops.decode_workspace_bytes(m.num_decode_part_slots, 8, 2), dtype=torch.uint8,
                                       device=gpu), backend.softmax_scale, m.decode_wave_extra,
                           m.decode_waves_per_group)
    _check(out[:4], batch, k, v, BF16)
    assert (out[4:] == 2.0).all()
