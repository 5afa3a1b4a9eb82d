"""CPU: the MXFP4 format's known answers, and what its operators refuse."""

import numpy as np
import pytest
import torch

from my_vllm_amd import _native, ops
from my_vllm_amd.attention_backend import (
    MI355XMXFP4AttentionBackend,
    mxfp4_decode_ranges,
    plan_decode_shared,
    shared_decode_capacity,
)
from my_vllm_amd.contract import AttentionRoute
from my_vllm_amd.custom_op import CustomOpConfig
from my_vllm_amd.layers import MXFP4KVCacheStore
from oracle import mxfp4
from workloads import make_paged_batch


def _row(values, dtype=torch.bfloat16):
    row = torch.zeros(128, dtype=dtype)
    row[:len(values)] = torch.tensor(values, dtype=dtype)
    return row


@pytest.mark.parametrize("values,codes,byte", [
    ([6.0, 0.25, 0.75, 1.25, -1.75, 2.5, 3.5, -5.0], [7, 0, 2, 2, 12, 4, 6, 14], 127),
    ([7.0, 0.5], [7, 1], 127),  # seven times the scale still fits: stored as six
    ([7.0625, 0.5], [6, 0], 128),  # above it the scale doubles; 3.53 is stored as four, 0.25 as zero
    ([4.0, -0.0], [6, 8], 127),
    ([3.5, 0.0], [7, 0], 126),
    ([0.0], [0], 0),
    ([float("inf"), 1.0], [0, 0], 255),
    ([float("nan"), 1.0], [0, 0], 255),
    ([3.3895313892515355e38], [7], 252),  # the largest bf16: 6 * 2^125
])
def test_known_codes_and_scales(values, codes, byte):
    got, scales = mxfp4.quantise(_row(values))
    assert list(got[:len(values)]) == codes
    assert scales[0] == byte and (scales[1:] == 0).all()


def test_largest_fp16_reads_back_finite():
    codes, scales = mxfp4.quantise(_row([65504.0], torch.float16))
    assert (codes[0], scales[0]) == (7, 140)
    assert 6 * 2.0 ** 13 <= torch.finfo(torch.float16).max


def test_rounding_is_within_half_a_step():
    x = torch.randn(50, 3, 128, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    cache = torch.zeros(4, 3, mxfp4.BLOCK, dtype=torch.uint8)
    mxfp4.store(x, cache, list(range(50)))
    back = mxfp4.values(cache).reshape(-1, 3, 128)[:50]
    unit = torch.from_numpy(np.ldexp(1.0, mxfp4.quantise(x)[1].astype(int) - 127)).repeat_interleave(32, -1)
    size = x.double().abs() / unit
    step = torch.where(size <= 2, 0.25, torch.where(size <= 4, 0.5, 1.0))
    assert (((back - x.double()).abs() / unit) <= step).all()


def test_shape_and_zeros():
    assert ops.mxfp4_cache_shape(5, 3) == (5, 3, 1088) and mxfp4.BLOCK == ops.MXFP4_PAGE_BYTES
    assert (mxfp4.values(torch.zeros(2, 1, 1088, dtype=torch.uint8)) == 0).all()


def _rows(n=4, h=2, dtype=torch.bfloat16):
    return torch.zeros(n, h, 128, dtype=dtype)


def test_store_and_load_refuse_bad_arguments():
    k, kc, slots = _rows(), torch.zeros(2, 2, 1088, dtype=torch.uint8), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="shape"):
        ops.store_kvcache_mxfp4(k, _rows(3), kc, kc, slots)
    with pytest.raises(ValueError, match="shape"):
        ops.store_kvcache_mxfp4(k[..., :64], k[..., :64], kc, kc, slots)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.store_kvcache_mxfp4(k, k, kc, kc, slots)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.load_kvcache_mxfp4(kc, kc, slots)


def test_cache_layout_checks():
    good = torch.zeros(4, 2, 1088, dtype=torch.uint8)
    cpu = good.device
    ops._check_mxfp4_caches(good, good.clone(), cpu)
    ops._check_mxfp4_caches(good[::2], good[1::2], cpu)  # pages apart
    pool = torch.zeros(2, 4, 3, 2, 1088, dtype=torch.uint8)
    ops._check_mxfp4_caches(pool[0, 1], pool[1, 1], cpu)
    with pytest.raises(TypeError, match="uint8"):
        ops._check_mxfp4_caches(good.to(torch.int8), good, cpu)
    with pytest.raises(TypeError, match="uint8"):
        ops._check_mxfp4_caches(good[..., :1024], good, cpu)
    with pytest.raises(ValueError, match="apart"):
        ops._check_mxfp4_caches(good[:1].expand(4, 2, 1088), good[:1].expand(4, 2, 1088), cpu)
    with pytest.raises(ValueError, match="layout"):
        ops._check_mxfp4_caches(good, good[:2], cpu)
    with pytest.raises(ValueError, match="layout"):
        ops._check_mxfp4_caches(good, torch.zeros(2, 4, 1088, dtype=torch.uint8).transpose(0, 1), cpu)
    with pytest.raises(RuntimeError, match="device"):
        ops._check_mxfp4_caches(good, good, torch.device("meta"))


def _abi_store(**change):
    args = dict(key=16, ks=256, khs=128, value=16, vs=256, vhs=128, kc=16, vc=16, pages=4, ps=2176, hs=1088, slots=4,
                wide=0, tokens=3, heads=2, dim=128, dtype=0)
    args.update(change)
    return list(args.values()) + [0]


@pytest.mark.parametrize("change,message", [
    ({"dim": 64}, "head_dim must be 128"),
    ({"dtype": 2}, "bf16 or fp16"),
    ({"tokens": -1}, "invalid sizes"),
    ({"heads": 0}, "invalid sizes"),
    ({"heads": 40000}, "at most 32767 KV heads"),
    ({"tokens": (1 << 40) + 1}, "too many tokens"),
    ({"key": 0}, "null buffer"),
    ({"slots": 0}, "null buffer"),
    ({"kc": 0}, "null buffer"),
    ({"key": 8}, "16-byte aligned"),
    ({"khs": 132}, "16-byte aligned"),
    ({"ps": 2180}, "16-byte aligned"),
    ({"vc": 24}, "16-byte aligned"),
    ({"ps": -2176}, "not be negative"),
])
@pytest.mark.parametrize("name", ["mva_kv_store_mxfp4", "mva_kv_load_mxfp4"])
def test_abi_refuses_before_any_launch(name, change, message):
    with pytest.raises(RuntimeError, match=message):
        _native.call(name, *_abi_store(**change))


def test_abi_takes_no_tokens():
    for name in ("mva_kv_store_mxfp4", "mva_kv_load_mxfp4"):
        _native.call(name, *_abi_store(tokens=0, key=0, value=0, slots=0))
    _native.call("mva_kv_store_mxfp4", *_abi_store(pages=0, kc=0, vc=0))


def _abi_decode(**change):
    args = dict(q=16, qts=2048, qhs=128, kc=16, vc=16, pages=4, ps=2176, hs=1088, bt=4, bts=4, sl=4, counts=0, items=32,
                n=4, waves=4, extra=4, per=4, merges=0, nm=0, slots=0, out=16, ots=2048, ohs=128, ws=256,
                wsb=1 << 30, hq=16, hkv=2, dim=128, page=16, scale=0.1, dtype=0)
    args.update(change)
    return list(args.values()) + [0]


@pytest.mark.parametrize("change,message", [
    ({"extra": 0}, "piece lists"),
    ({"ps": 2184}, "16-byte aligned"),
    ({"hs": 1090}, "16-byte aligned"),
    ({"dtype": 2}, "bf16 or fp16"),
    ({"dim": 64}, "head_dim must be 128"),
    ({"page": 32}, "page_size must be 16"),
    ({"hq": 15}, "multiple of num_kv_heads"),
    ({"hq": 34}, "at most 16 query heads"),
    ({"waves": 5}, "num_waves"),
    ({"nm": 1}, "missing merge list"),
    ({"pages": 0}, "empty KV cache"),
    ({"kc": 8}, "16-byte aligned"),
    ({"out": 4}, "8-byte aligned"),
    ({"wsb": 1024}, "workspace too small"),
    ({"per": 8}, "waves_per_group"),
    ({"ps": 1 << 33}, "less than 4 GiB apart"),
    ({"ps": -2176}, "not be negative"),
    ({"n": 1 << 27, "waves": 1 << 27}, "too many wavefronts"),
])
def test_abi_decode_refuses_before_any_launch(change, message):
    with pytest.raises(RuntimeError, match=message):
        _native.call("mva_paged_decode_mxfp4", *_abi_decode(**change))


def _abi_prefill(**change):
    args = dict(q=16, qts=2048, qhs=128, kc=16, vc=16, pages=4, ps=2176, hs=1088, bt=4, bts=4, sl=4, qsl=4, seqs=2,
                tiles=3, ws=256, wsb=1 << 30, planned=0, out=16, ots=2048, ohs=128, hq=16, hkv=2, dim=128, page=16,
                scale=0.1, dtype=0)
    args.update(change)
    return list(args.values()) + [0]


@pytest.mark.parametrize("change,message", [
    ({"ps": 2184}, "16-byte aligned"),
    ({"hs": 1090}, "16-byte aligned"),
    ({"hs": -1088}, "not be negative"),
    ({"dtype": 2}, "bf16 or fp16"),
    ({"dim": 64}, "head_dim must be 128"),
    ({"page": 32}, "page_size must be 16"),
    ({"hq": 15}, "multiple of num_kv_heads"),
    ({"hq": 34}, "at most 16 query heads"),
    ({"pages": 0}, "empty KV cache"),
    ({"vc": 8}, "16-byte aligned"),
    ({"out": 4}, "8-byte aligned"),
    ({"wsb": 1024}, "workspace too small"),
    ({"ws": 0}, "workspace too small"),
    ({"ws": 8}, "16-byte aligned"),
    ({"tiles": -1}, "invalid tile capacity"),
    ({"seqs": -1}, "invalid sequence count"),
    ({"hq": 256, "hkv": 128}, "at most 127 KV heads"),
])
def test_abi_prefill_refuses_before_any_launch(change, message):
    with pytest.raises(RuntimeError, match=message):
        _native.call("mva_paged_prefill_mxfp4", *_abi_prefill(**change))


def test_decode_ranges():
    # Ranges of four pages or more; twelve wavefronts a CU on large batches.
    assert mxfp4_decode_ranges(3, 8) == (1, 4)
    assert mxfp4_decode_ranges(41, 8) == (10, 4)
    assert mxfp4_decode_ranges(20000, 8) == (256, 4)
    assert mxfp4_decode_ranges(40000, 8) == (384, 12)
    assert mxfp4_decode_ranges(4000, 1) == (1000, 4)
    assert mxfp4_decode_ranges(4000, 8, override=64) == (8, 4)
    assert mxfp4_decode_ranges(4000, 300) == (10, 12)  # 2.6 GB


@pytest.mark.parametrize("counts,hkv,cus", [
    ([5, 1, 40, 8, 1, 129], 5, 256),
    ([1875], 8, 256),
    ([2000, 1, 2, 3], 8, 256),
    ([17] * 300, 8, 256),
    ([9, 8, 7], 2, 1),
    ([2 ** 20, 3], 16, 256),
    ([300] * 37, 4, 304),
])
def test_shared_plans_cover_every_segment(counts, hkv, cus):
    items, wave_extra, waves, slots, merges = plan_decode_shared(counts, 3, 7, hkv, cus, always=True)
    assert items.shape == (waves, 8) and (wave_extra == waves).all() and wave_extra.size == waves + 1
    assert len(items) <= shared_decode_capacity(len(counts), hkv, cus)
    groups = items.reshape(-1, 4, 8)
    assert (groups[:, :, 3:] == groups[:, :1, 3:]).all() and (groups[:, :, 0] == groups[:, :1, 0]).all()
    assert (groups[:, 1:, 1] == groups[:, :-1, 2]).all()  # quarters side by side
    assert (items[:, 1] <= items[:, 2]).all() and (items[:, 6] - items[:, 0] == 4).all()
    sizes = items[:, 2] - items[:, 1]
    pieces = (groups[:, 3, 2] - groups[:, 0, 1] + 1) // 2  # tiles
    assert (sizes.reshape(-1, 4) <= 2 * -(-pieces[:, None] // 4)).all()
    ends = np.array(counts)[items[:, 0] - 3]
    assert (items[:, 1] % 2 == 0).all() or (items[:, 1] <= ends).all()  # whole tiles
    used = []
    for s, pages in enumerate(counts):
        for h in range(hkv):
            own = groups[(groups[:, 0, 0] == s + 3) & (groups[:, 0, 7] == h)]
            own = own[np.argsort(own[:, 0, 3])]
            n = len(own)
            assert own[:, 0, 3].tolist() == list(range(n)) and (own[:, 0, 4] == n).all()
            assert own[0, 0, 1] == 0 and own[-1, 3, 2] == pages and (own[1:, 0, 1] == own[:-1, 3, 2]).all()
            base = ~int(own[0, 0, 5])
            assert base >= 0
            merge = merges[(merges[:, 0] == s + 3) & (merges[:, 7] == h)]
            assert len(merge) == (n > 1)
            if n > 1:
                assert merge[0].tolist() == [s + 3, 0, pages, 0, n, base, s + 7, h]
                if h == 0:
                    used += range(base, base + n)
    assert used == list(range(slots))


def test_shared_plan_order():
    # All at once: every CU's workgroups (4 CUs, places i, i + 4, i + 8) sum to about the same.
    counts = np.array([10, 3, 7, 1, 12, 5, 9, 2, 8, 4], np.int64) * 2

    def pages(cus):
        items, _, waves, _, merges = plan_decode_shared(counts, 0, 0, 1, cus, always=True)
        assert waves == 40 and len(merges) == 0
        return (counts[items[::4, 0]] // 2).tolist()

    assert pages(4) == [8, 9, 10, 12, 7, 5, 4, 3, 1, 2]
    # More than a CU holds: longest first.
    assert pages(3) == sorted((counts // 2).tolist(), reverse=True)


@pytest.mark.parametrize("counts,hkv,pieces", [
    ([1], 8, 8),
    ([19], 8, 8),
    ([63] * 32, 8, 256),
    ([13] * 200, 8, 1600),
    ([75], 8, 80),  # 38 tiles, ten pieces (9.5 to nearest, up)
    ([1876], 8, 256),
    ([500] + [10] * 40, 8, None),
    ([8192] * 56, 8, 0),  # page ranges
    ([750] * 40, 8, 0),
])
def test_plans_taken(counts, hkv, pieces):
    waves = plan_decode_shared(counts, 0, 0, hkv, 256)[2]
    assert waves == 4 * pieces if pieces is not None else 4 * 8 * 41 < waves <= 4 * 768


def test_shared_plan_refusals():
    with pytest.raises(ValueError):
        plan_decode_shared([3, 0], 0, 0, 8, 256)
    with pytest.raises(RuntimeError, match="int32 range"):
        plan_decode_shared([3, 3], 2 ** 31 - 1, 0, 8, 256)
    counts, items = np.array([400], np.int64), np.zeros((4096, 8), np.int32)
    extra, merges, out = np.zeros(4097, np.int32), np.zeros((4, 8), np.int32), np.zeros(4, np.int64)

    def call(hkv=1, cus=256, rows=4096, words=4097, joins=4):
        _native.call("mva_decode_plan_shared", counts.ctypes.data, 1, 0, 0, hkv, cus, 1, items.ctypes.data, rows,
                     extra.ctypes.data, words, merges.ctypes.data, joins, out.ctypes.data)

    for change in ({"hkv": 0}, {"cus": 0}, {"words": 0}):
        with pytest.raises(RuntimeError, match="invalid arguments"):
            call(**change)
    for change in ({"rows": 3}, {"words": 4}, {"joins": 0}, {"hkv": 5}):
        with pytest.raises(RuntimeError, match="capacity too small"):
            call(**change)
    call(hkv=4)
    assert out.tolist() == [4 * 4 * 50, 4 * 4 * 50, 50, 4]


class _HostBackend(MI355XMXFP4AttentionBackend):
    require_device_metadata = False


def test_backend_routes_and_refusals():
    for mode in (None, "split"):
        backend = _HostBackend(32, 8, 128, 16, torch.bfloat16, mode)
        assert not backend.mixed_attention_available
        assert "prefill + decode" in backend.mixed_attention_unavailable_reason
        mixed = make_paged_batch(1, [5, 1, 1], [40, 30, 500], 1, 32, 8).common
        assert backend.build_plan(mixed).route is AttentionRoute.MIXED_SPLIT
    # Piece lists at every size and head count.
    backend = _HostBackend(8, 1, 128, 16, torch.float16)
    big = make_paged_batch(2, [1], [40], 0, 8, 1).common
    plan = backend.build_plan(big)
    assert plan.route is AttentionRoute.DECODE and plan.metadata.decode_wave_extra is not None
    assert backend._decode_schedule(1 << 24) == "listed"
    backend.decode_schedule_override = "claims"
    with pytest.raises(ValueError, match="piece lists"):
        backend.build_plan(big)
    q = torch.zeros(1, 8, 128, dtype=torch.float16)
    cache = torch.zeros(4, 1, 1088, dtype=torch.uint8)
    with pytest.raises(ValueError, match="CUDA"):
        backend.forward(q, None, None, cache, cache, plan)


def test_store_operator_shares_the_kv_store_provider():
    store = MXFP4KVCacheStore(CustomOpConfig(platform="cuda", overrides={"kv_cache_store": "native_triton"}))
    assert store.kv_store_provider_name == "hip"
    with pytest.raises(RuntimeError, match="requires CUDA"):
        MXFP4KVCacheStore(CustomOpConfig(platform="cpu"))
