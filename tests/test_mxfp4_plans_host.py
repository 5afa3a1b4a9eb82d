"""CPU: decode plans and graph states of MXFP4 and of 16-bit caches are kept apart."""

import types

import numpy as np
import pytest
import torch

from my_vllm_amd import _native
from my_vllm_amd.attention_backend import (
    MI355XAttentionBackend,
    MI355XFullDecodeGraphState,
    MI355XMXFP4AttentionBackend,
    plan_decode_listed,
    plan_decode_listed_mxfp4,
)
from tests import _decode_plan_spec
from tests._decode_plan_spec import listed_plan_spec, merge_list_spec
from workloads import make_paged_batch


class _Host16(MI355XAttentionBackend):
    require_device_metadata = False


class _HostFp4(MI355XMXFP4AttentionBackend):
    require_device_metadata = False


def _backends(monkeypatch, mode=None):
    """A backend of either kind whose launches are only recorded."""
    calls = []
    for cls in (_Host16, _HostFp4):
        monkeypatch.setattr(cls, "_validate_inputs", lambda self, q, k, v: None)
        monkeypatch.setattr(cls, "_get_workspace", lambda self, nbytes, device: None)
        monkeypatch.setattr(cls, "_run_prefill", lambda self, *a: calls.append("prefill"))
        monkeypatch.setattr(cls, "_run_decode", lambda self, *a: calls.append("decode"))
        monkeypatch.setattr(cls, "_run_mixed", lambda self, *a: calls.append("mixed"))
    return _Host16(16, 4, 128, 16, torch.bfloat16, mode), _HostFp4(16, 4, 128, 16, torch.bfloat16, mode), calls


@pytest.mark.parametrize("prefills,runs", [(0, ["decode"]), (1, ["prefill", "decode"]), (3, ["prefill"])])
def test_a_decode_plan_for_mxfp4_caches_runs_over_those_only(monkeypatch, prefills, runs):
    wide, fp4, calls = _backends(monkeypatch, "split")
    q_lens = [5] * prefills + [1] * (3 - prefills)
    common = make_paged_batch(1, q_lens, [40, 90, 5000], prefills, 16, 4).common
    plan = fp4.build_plan(common)
    q, cache = torch.zeros(sum(q_lens), 16, 128, dtype=torch.bfloat16), torch.zeros(1)
    fp4.forward(q, None, None, cache, cache, plan)
    assert calls == runs
    if prefills == 3:  # the tile plans are the same
        wide.forward(q, None, None, cache, cache, plan)
        assert calls == 2 * runs
        return
    with pytest.raises(ValueError, match="MXFP4"):
        wide.forward(q, None, None, cache, cache, plan)
    if prefills == 0:  # nor with the store folded in
        kv = torch.zeros(3, 4, 128, dtype=torch.bfloat16)
        with pytest.raises(ValueError, match="MXFP4"):
            wide.forward_with_kv_store(q, kv, kv, cache, cache, common.slot_mapping, plan)
    assert calls == runs
    wide.forward(q, None, None, cache, cache, wide.build_plan(common))
    assert calls == 2 * runs


def _state(mxfp4):
    names = [f for f in MI355XFullDecodeGraphState.__dataclass_fields__ if f not in ("plan", "staging_turn", "mxfp4")]
    return MI355XFullDecodeGraphState(**dict.fromkeys(names), plan=types.SimpleNamespace(), mxfp4=mxfp4)


def test_graph_states_belong_to_one_kind_of_cache(monkeypatch):
    wide, fp4, _ = _backends(monkeypatch)
    for own, other, mxfp4 in ((wide, fp4, False), (fp4, wide, True)):
        with pytest.raises(ValueError, match="another kind of cache"):
            other.activate_full_decode_graph(_state(mxfp4))
        own.activate_full_decode_graph(_state(mxfp4))
        own.deactivate_full_decode_graph()


def test_only_the_mxfp4_planner_leaves_pieces_longer_than_128_pages():
    counts = np.array([300, 2, 900], np.int64)
    unlimited = 2 ** 31 - 1
    with pytest.raises(ValueError, match=r"\[1, 128\]"):
        plan_decode_listed(counts, 0, 0, 8, 2, unlimited)
    assert _native.query("mva_decode_plan_listed_rows", 3, 1202, 8, 2, unlimited) == -1
    items, extra, out = np.zeros((100, 8), np.int32), np.zeros(100, np.int32), np.zeros(4, np.int64)
    with pytest.raises(RuntimeError, match=r"\[1, 128\]"):
        _native.call("mva_decode_plan_listed", counts.ctypes.data, 3, 0, 0, 8, 2, unlimited, items.ctypes.data, 100,
                     extra.ctypes.data, 100, 0, 0, out.ctypes.data)
    assert (plan_decode_listed(counts, 0, 0, 8, 2)[0][:, 2] - plan_decode_listed(counts, 0, 0, 8, 2)[0][:, 1]).max() <= 128


@pytest.mark.parametrize("counts,hkv,groups", [([300, 2, 900], 8, 2), ([1], 1, 5), ([7, 1, 1, 40], 3, 4),
                                               ([5] * 50, 2, 1000), ([100000, 3], 8, 384)])
def test_mxfp4_page_ranges(monkeypatch, counts, hkv, groups):
    monkeypatch.setattr(_decode_plan_spec, "MAX_CHUNK_PAGES", 1 << 30)
    counts = np.array(counts, np.int64)
    items, extra, waves, slots, merges = plan_decode_listed_mxfp4(counts, 4, 9, hkv, groups)
    want = listed_plan_spec(counts, 4, 9, hkv, groups, int(counts.sum()))
    assert np.array_equal(items, want[0]) and np.array_equal(extra, want[1]) and (waves, slots) == want[2:4]
    assert np.array_equal(merges, merge_list_spec(want[0]))
    assert len(items) <= (len(counts) + groups) * hkv
    empty = plan_decode_listed_mxfp4(np.zeros(0, np.int64), 0, 0, hkv, groups)
    assert empty[0].shape == (0, 8) and empty[1].tolist() == [0] and empty[2:4] == (0, 0)


def test_more_ranges_than_pages():
    # As many rows as the pages can need, not as the ranges asked for.
    few = plan_decode_listed_mxfp4([3, 1], 0, 0, 8, 4)
    many = plan_decode_listed_mxfp4([3, 1], 0, 0, 8, 2 ** 31 - 1)
    assert all(np.array_equal(a, b) for a, b in zip(few, many))
