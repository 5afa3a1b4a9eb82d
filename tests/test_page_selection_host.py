"""CPU: the page selection's oracle, what the operators refuse, and the backend's
host side."""

import math
import types

import numpy as np
import pytest
import torch

from my_vllm_amd import _native, ops
from my_vllm_amd import attention_backend as ab
from my_vllm_amd.contract import AttentionRoute, CommonAttentionMetadata
from oracle import selection
from oracle.reference import paged_attention
from tests._foreign_contract import ForeignBackendBase, ForeignBatchType, ForeignCommon, ForeignPlan, ForeignRoute
from tests._selection import bounds_of, keys, page_counts, queries, tables_for
from workloads import make_paged_batch

BF16, FP16 = torch.bfloat16, torch.float16


# ---- the oracle --------------------------------------------------------------------


def test_oracle_bounds_are_the_ends_of_each_sorted_column():
    cache = keys(3, 2, BF16, 1)
    before = torch.full((3, 2, 2, 128), 9.0, dtype=BF16)
    got = selection.page_bounds(cache, before, torch.tensor([[2, 0, 1]]), [40], [25])
    ordered = cache.double().sort(1).values
    assert torch.equal(got[0, :, 0].double(), ordered[0, 0]) and torch.equal(got[0, :, 1].double(), ordered[0, -1])
    assert torch.equal(got[2], torch.stack((cache[2].amin(0), cache[2].amax(0)), 1))  # token 15 is new
    assert (got[1] == 9).all()  # 40 tokens: the third page is not full
    again = selection.page_bounds(cache, before, torch.tensor([[2, 0, 1]]), [40], [24])
    assert (again[2] == 9).all()


def test_oracle_scores_bound_every_key():
    cache, q = keys(20, 1, BF16, 2), queries(1, 6, BF16, 3)
    scores = selection.page_scores(q[0], bounds_of(cache)[:, 0])
    products = torch.einsum("gd,ptd->ptg", q[0].double(), cache[:, :, 0].double()).sum(-1)
    assert (torch.from_numpy(scores) >= products.amax(1) - 1e-9).all()
    # One query: the box's largest product, channel by channel.
    box = bounds_of(cache)[:, 0].double()
    one = torch.maximum(q[0, :1].double() * box[:, 0], q[0, :1].double() * box[:, 1]).sum(-1)
    assert np.allclose(selection.page_scores(q[0, :1], bounds_of(cache)[:, 0]), one.numpy(), rtol=1e-13, atol=0)
    # A mistake in the oracle's parts would be seen.
    swapped = torch.flip(bounds_of(cache)[:, 0], (1,))
    assert not (torch.from_numpy(selection.page_scores(q[0], swapped)) >= products.amax(1)).all()


def test_oracle_scores_of_infinities_are_the_products_of_the_queries():
    # Whole numbers: every finite sum is exact.
    gen = torch.Generator().manual_seed(3)
    values = torch.tensor([-math.inf, -2.0, 0.0, 1.0, 3.0, math.inf])
    box = values[torch.randint(0, 6, (4000, 2, 128), generator=gen)].sort(1).values
    box[:, :, 3:] = torch.randint(-2, 3, (4000, 2, 125), generator=gen).float().sort(1).values
    box[500:, :, 1:3] = box[500:, :, 5:7]  # one channel with an infinity in most
    q = torch.zeros(2, 128)
    kinds = set()
    for a in (-1.0, 0.0, 2.0, math.inf, math.nan):
        for b in (-3.0, 0.0, 1.0, -math.inf):
            q[:, :3] = torch.tensor([[a], [b]])
            q[:, 3:] = torch.randint(-2, 3, (2, 125), generator=gen).float()
            got = selection.page_scores(q.to(BF16), box.to(BF16))
            want = torch.maximum(q[:, None] * box[None, :, 0], q[:, None] * box[None, :, 1]).double().sum((0, 2)).numpy()
            assert np.array_equal(got, want, equal_nan=True)
            kinds |= {(math.isinf(a), *x) for x in zip(np.isnan(got).tolist(), np.isinf(got).tolist())}
    assert len(kinds) == 5  # finite ones too, but of no infinite query
    # A channel's -inf says nothing about a product with a positive query.
    box = torch.zeros(1, 2, 128)
    box[0, 0, 0], box[0, 1, 0] = -math.inf, 2.0
    q = torch.zeros(2, 128)
    q[:, 0] = torch.tensor([1.0, 3.0])
    assert selection.page_scores(q, box).tolist() == [8.0]


def test_oracle_choice_ranks_ties_and_nan():
    nan = math.nan
    assert selection.chosen([1.0, 3.0, 3.0, 2.0, 3.0], 2) == [1, 2]
    assert selection.chosen([1.0, nan, math.inf, 2.0, nan], 3) == [1, 2, 4]
    assert selection.chosen([0.0, -0.0, 0.0], 2) == [0, 1]
    assert selection.chosen([-math.inf, -5.0], 1) == [1]


def test_oracle_tables_keep_ends_and_order():
    lens = [16 * 10 + 3, 40, 0]
    counts = page_counts(lens)
    cache = keys(sum(counts), 2, FP16, 4)
    table = tables_for(counts, sum(counts), 5)
    tables, kept = selection.select_pages(queries(3, 4, FP16, 6), bounds_of(cache), table, lens, 5, 2, 1)
    row = table[0].tolist()
    for h in range(2):
        places = [row.index(p) for p in tables[0, h].tolist()]
        assert places == sorted(places) and places[:2] == [0, 1] and places[-1] == 10
    assert kept.tolist() == [4 * 16 + 3, 40, 0]
    assert tables[1, 0].tolist() == [*table[1, :3].tolist(), -1, -1] and (tables[2] == -1).all()


def test_oracle_attention_over_all_pages_is_dense_attention():
    batch = make_paged_batch(7, [1, 1], [70, 33], 0, 6, 2, dtype=FP16)
    counts = batch.block_counts
    tables = batch.common.block_tables[:, None].expand(2, 2, max(counts))
    got, spread, _ = selection.attention(batch.q, batch.k_cache, batch.v_cache, tables, [70, 33], 1 / math.sqrt(128))
    want = paged_attention(batch.q, batch.k_cache, batch.v_cache, batch.common.block_tables, [1, 1], [70, 33])
    assert torch.allclose(got.float(), want, atol=1e-5) and (spread >= got.abs() - 1e-12).all()


# ---- refusals ----------------------------------------------------------------------


def _select_args(**change):
    args = dict(q=0x1000, q_token_stride=1024, q_head_stride=128, page_bounds=0x1000, num_pages=10,
                block_tables=0x1000, block_table_stride=20, table_width=20, seq_lens=0x1000, num_seqs=2,
                num_selected=4, sink=1, recent=1, tables=0x1000, lens=0x1000, k_cache=0, page_stride=0, token_stride=0,
                workspace=0x1000, bytes=1 << 30,
                hq=8, hkv=2, head_dim=128, page=16, dtype=0, stream=0)
    return list({**args, **change}.values())


@pytest.mark.parametrize("change,message", [
    ({"head_dim": 64}, "head_dim"), ({"page": 32}, "page_size"), ({"dtype": 2}, "dtype"), ({"hq": 7}, "sizes"),
    ({"hq": 34}, "sizes"), ({"num_selected": 0}, "sizes"), ({"num_seqs": -1}, "sizes"), ({"table_width": -1}, "sizes"),
    ({"sink": -1}, "recent_pages"), ({"recent": 0}, "recent_pages"), ({"sink": 3, "recent": 2}, "recent_pages"),
    ({"sink": 1 << 62, "recent": 1 << 62}, "recent_pages"), ({"workspace": 0}, "workspace"), ({"bytes": 64}, "workspace"),
    ({"q": 0}, "null"), ({"tables": 0}, "null"), ({"num_pages": 0}, "empty"), ({"table_width": 0}, "empty"),
    ({"q": 0x1008}, "aligned"), ({"page_bounds": 0x1008}, "aligned"), ({"q_head_stride": 129}, "aligned"),
    ({"num_seqs": 1 << 33}, "sizes"), ({"table_width": 1 << 40}, "sizes"), ({"block_table_stride": -20}, "sizes"),
    ({"k_cache": 0x1008, "page_stride": 4096, "token_stride": 256}, "aligned"),
    ({"k_cache": 0x1000, "page_stride": 4097, "token_stride": 256}, "aligned"),
    ({"k_cache": 0x1000, "page_stride": -4096, "token_stride": 256}, "sizes"),
])
def test_select_entry_refuses(change, message):
    with pytest.raises(RuntimeError, match=message):
        _native.call("mva_select_pages", *_select_args(**change))


def test_entries_of_no_rows_do_nothing():
    _native.call("mva_select_pages", *_select_args(num_seqs=0, q=0, workspace=0))
    _native.call("mva_update_page_bounds", 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 8, 128, 16, 0, 0)
    _native.call("mva_paged_decode_selected", 0, 0, 0, 0, 0, 5, 0, 0, 0, 0, 0, 0, 0, 4, 0, 0, 0, 0, 0, 8, 8, 128, 16,
                 1.0, 0, 0)


@pytest.mark.parametrize("change,message", [
    ({13: 64}, "head_dim"), ({14: 8}, "page_size"), ({15: 7}, "dtype"), ({12: 0}, "sizes"), ({1: -1}, "sizes"),
    ({11: -4}, "sizes"), ({9: 0}, "query_start_loc"), ({0: 0}, "null"), ({0: 0x1002}, "aligned"),
    ({2: -1024}, "sizes"), ({3: -16}, "sizes"), ({4: 0x1008}, "aligned"), ({3: 1023}, "aligned"), ({11: 1 << 40}, "too many"),
])
def test_bounds_entry_refuses(change, message):
    args = [0x1000, 10, 16 * 1024, 1024, 0x1000, 0x1000, 20, 20, 0x1000, 0x1000, 2, 7, 8, 128, 16, 0, 0]
    for at, value in change.items():
        args[at] = value
    with pytest.raises(RuntimeError, match=message):
        _native.call("mva_update_page_bounds", *args)


@pytest.mark.parametrize("change,message", [
    ({21: 64}, "head_dim"), ({22: 8}, "page_size"), ({24: 2}, "dtype"), ({19: 9}, "sizes"), ({13: 0}, "sizes"),
    ({9: -1}, "sizes"), ({6: -1024}, "sizes"), ({5: 0}, "empty"), ({3: 0}, "null"), ({14: 0}, "null"), ({0: 0x1004}, "aligned"),
    ({7: 1 << 27}, "2\\^26"), ({23: 0.0}, "softmax_scale"), ({23: math.nan}, "softmax_scale"),
    ({6: 16 * 1024 + 1}, "aligned"), ({14: 0x1004}, "aligned"), ({17: 0}, "workspace"), ({18: 100}, "workspace"),
])
def test_attention_entry_refuses(change, message):
    args = [0x1000, 1024, 128, 0x1000, 0x1000, 10, 16 * 1024, 1024, 0x1000, 160, 20, 0x1000, 2, 20, 0x1000, 1024, 128,
            0x1000, 1 << 30, 8, 8, 128, 16, 1.0, 0, 0]
    for at, value in change.items():
        args[at] = value
    with pytest.raises(RuntimeError, match=message):
        _native.call("mva_paged_decode_selected", *args)


@pytest.mark.parametrize("tokens", [1 << 31, 1 << 62, (1 << 63) - 15, (1 << 63) - 1])
def test_bounds_entry_refuses_token_counts_whose_grid_overflows(tokens):
    with pytest.raises(RuntimeError, match="too many"):
        _native.call("mva_update_page_bounds", 0x1000, 10, 16 * 1024, 1024, 0x1000, 0x1000, 20, 20, 0x1000, 0x1000, 2,
                     tokens, 8, 128, 16, 0, 0)


def test_attention_entry_refuses_tokens_too_far_apart_from_the_first_on():
    # 2^26 elements, and the largest stride below: that one is refused for its workspace alone.
    for stride, message in ((1 << 26, "2\\^26"), ((1 << 26) - 8, "workspace")):
        with pytest.raises(RuntimeError, match=message):
            _native.call("mva_paged_decode_selected", 0x1000, 1024, 128, 0x1000, 0x1000, 10, 1 << 30, stride, 0x1000,
                         160, 20, 0x1000, 2, 20, 0x1000, 1024, 128, 0, 0, 8, 8, 128, 16, 1.0, 0, 0)


def test_workspace_sizes():
    size = ops.selection_workspace_bytes
    assert size(0, 8, 8, 10, 4) >= 0
    assert size(4, 32, 8, 2048, 128) >= 4 * 8 * 2048 * 8
    assert size(4, 32, 8, 2048, 128) <= size(4, 32, 8, 4096, 128)
    for bad in ((-1, 8, 8, 10, 4), (1, 9, 8, 10, 4), (1, 17, 1, 10, 4), (1, 8, 8, -1, 4), (1, 8, 8, 10, 0),
                (1 << 31, 8, 8, 10, 4), (1, 8, 8, 1 << 30, 4)):
        with pytest.raises(ValueError, match="sizes"):
            size(*bad)


# Enough for fewer rows, heads, pages and columns: fewer rows are cut into more parts.
@pytest.mark.parametrize("change", [{"num_seqs": n} for n in (1, 2, 31, 32, 47, 48, 49, 63)] + [
    {"num_q_heads": 16}, {"num_q_heads": 8}, {"num_kv_heads": 4, "num_seqs": 33}, {"num_kv_heads": 4}, {"table_width": 0},
    {"table_width": 1, "num_seqs": 13}, {"num_selected": 1}, {"num_selected": 17, "num_seqs": 40}])
@pytest.mark.parametrize("width", [0, 200, 2048])
def test_a_workspace_is_enough_for_smaller_sizes(change, width):
    largest = dict(num_seqs=64, num_q_heads=64, num_kv_heads=8, table_width=width, num_selected=128)
    smaller = {**largest, **{k: min(v, largest[k]) for k, v in change.items()}}
    assert ops.selection_workspace_bytes(*smaller.values()) <= ops.selection_workspace_bytes(*largest.values())


@pytest.mark.parametrize("hq,hkv", [(8, 8), (32, 8), (64, 8), (16, 1), (16, 4)])
@pytest.mark.parametrize("selected", [1, 16, 17, 128, 5000])
def test_workspace_sizes_do_not_fall_as_rows_are_added(hq, hkv, selected):
    sizes = [ops.selection_workspace_bytes(n, hq, hkv, 100, selected) for n in range(0, 1600)]
    assert sizes == sorted(sizes)


def test_operators_refuse_cpu_tensors():
    q, cache = torch.zeros(2, 8, 128, dtype=BF16), torch.zeros(4, 16, 2, 128, dtype=BF16)
    bounds, table, lens = torch.zeros(4, 2, 2, 128, dtype=BF16), torch.zeros(2, 4, dtype=torch.int32), torch.ones(
        2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.update_page_bounds(cache, bounds, table, lens)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.select_pages(q, bounds, table, lens, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_decode_selected(q, cache, cache, table[:, None].expand(2, 2, 4), lens, 1.0)
    assert ops.page_bounds_shape(4, 2) == (4, 2, 2, 128)


# ---- the backend -------------------------------------------------------------------


def _common(batch, contract=CommonAttentionMetadata):
    return contract(**batch.common.__dict__)


@pytest.fixture
def host_planning(monkeypatch):
    monkeypatch.setattr(ab.MI355XAttentionBackendMixin, "require_device_metadata", False)


@pytest.mark.parametrize("given,error,message", [
    ({"selected_pages": 0}, ValueError, "selected_pages"), ({"selected_pages": 4.0}, TypeError, "selected_pages"),
    ({"sink_pages": -1}, ValueError, "sink_pages"), ({"recent_pages": 0}, ValueError, "recent_pages"),
    ({"recent_pages": True}, TypeError, "recent_pages"),
    ({"selected_pages": 4, "sink_pages": 1, "recent_pages": 4}, ValueError, "at most"),
])
def test_backend_refuses_page_numbers(given, error, message):
    with pytest.raises(error, match=message):
        ab.MI355XSparseAttentionBackend(16, 8, 128, 16, BF16, **given)


def test_backend_plans_no_decode_pieces(host_planning):
    backend = ab.MI355XSparseAttentionBackend(16, 8, 128, 16, BF16)
    assert (backend.selected_pages, backend.sink_pages, backend.recent_pages) == (128, 1, 4)
    decode = backend.build_plan(_common(make_paged_batch(1, [1, 1], [500, 3], 0, 16, 8)))
    assert decode.route is AttentionRoute.DECODE and decode.metadata.decode_items is None
    mixed = backend.build_plan(_common(make_paged_batch(1, [30, 1], [60, 90], 1, 16, 8)))
    assert mixed.route is AttentionRoute.MIXED_SPLIT and mixed.metadata.decode_items is None
    assert not backend.mixed_attention_available and "selected" in backend.mixed_attention_unavailable_reason


def test_graph_states_belong_to_one_kind_of_decode(host_planning):
    backend, dense = (cls(16, 8, 128, 16, BF16) for cls in (ab.MI355XSparseAttentionBackend, ab.MI355XAttentionBackend))
    names = [f for f in ab.MI355XFullDecodeGraphState.__dataclass_fields__ if f not in ("plan", "selects", "mxfp4")]
    for own, other, selects in ((dense, backend, False), (backend, dense, True)):
        state = ab.MI355XFullDecodeGraphState(**dict.fromkeys(names), plan=types.SimpleNamespace(), mxfp4=False,
                                              selects=selects)
        with pytest.raises(ValueError, match="another kind of decode"):
            other.activate_full_decode_graph(state)
        own.activate_full_decode_graph(state)
        own.deactivate_full_decode_graph()


def test_each_eager_stream_has_buffers_of_its_own(monkeypatch):
    # One backend whose steps run on two streams, played on the CPU: nothing that one writes is the other's.
    backend, cpu = ab.MI355XSparseAttentionBackend(16, 8, 128, 16, BF16), torch.device("cpu")
    stream = [0]
    monkeypatch.setattr(_native, "stream_of", lambda device: stream[0])
    q = torch.zeros(5, 16, 128, dtype=BF16)

    def step(n):
        stream[0] = n
        return (backend._get_reusable_attention_output(q), backend._get_workspace(1 << 20, cpu),
                backend._get_prefill_workspace(4, cpu))

    def addresses(tensors):
        return [t.data_ptr() for t in tensors]

    first, second = step(1), step(2)
    assert not set(addresses(first)) & set(addresses(second))
    # Back on the first: its own again, and no tile plan counts as laid there.
    backend._prefill_planned_for = object()
    assert addresses(step(1)) == addresses(first) and backend._prefill_planned_for is None
    assert addresses(step(1)) == addresses(first) and addresses(step(2)) == addresses(second)
    # A decode step of a graph state has its output from the state.
    taken = []
    monkeypatch.setattr(backend, "_attend", lambda q, *_: taken.append(backend._get_workspace(1 << 20, q.device)))
    stream[0] = 1
    backend._run_decode_graph(q, None, None, types.SimpleNamespace(
        block_tables_buffer=None, seq_lens_buffer=None, output=None))
    assert taken[0] is first[1]
    # As many streams as are in use at a time, not as many as ever were.
    held = [step(n) for n in range(3, 40)]
    assert len(backend._other_streams) <= 8 and addresses(step(38)) == addresses(held[-2])
    assert backend._workspace is None  # the dense decode's, whose words mean something else


def test_integrate_builds_on_another_contract(host_planning):
    registered = {}
    registry = types.SimpleNamespace(register=registered.__setitem__)
    cls = ab.integrate_sparse(registry, ForeignBackendBase, ForeignPlan, ForeignRoute, ForeignBatchType, ForeignCommon,
                              selected_pages=64, sink_pages=2)
    assert registered == {"mi355x_sparse": cls} and cls.backend_name == "mi355x_sparse"
    backend = cls(16, 8, 128, 16, BF16)
    assert (backend.selected_pages, backend.sink_pages, backend.recent_pages) == (64, 2, 4)
    plan = backend.build_plan(_common(make_paged_batch(1, [1, 1], [500, 3], 0, 16, 8), ForeignCommon))
    assert isinstance(plan, ForeignPlan) and plan.route is ForeignRoute.DECODE
