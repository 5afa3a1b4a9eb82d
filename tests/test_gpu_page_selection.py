"""GPU: page bounds, page selection and attention over selected pages against
their 64-bit oracle.  Bounds and selected pages have to be equal; attention is
within the bound of tests/_mxfp4.py::attention_bound (one rounding of P, fp32
sums, one rounding of the result)."""

import math

import pytest
import torch

from my_vllm_amd import ops
from oracle import selection
from tests._mxfp4 import assert_within, attention_bound
from tests._selection import PAGE, bounds_of, keys, page_counts, queries, same, tables_for

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
SCALE = 1 / math.sqrt(128)


def _ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


# ---- bounds ----------------------------------------------------------------------


def _update(gpu, cache, bounds, table, lens, new, gave_starts=True):
    starts = torch.zeros(len(new) + 1, dtype=torch.int32)
    starts[1:] = torch.tensor(new).cumsum(0)
    got = bounds.to(gpu)
    if gave_starts:
        ops.update_page_bounds(cache, got, table.to(gpu), _ints(lens, gpu), starts.to(gpu), sum(new))
    else:
        ops.update_page_bounds(cache, got, table.to(gpu), _ints(lens, gpu))
    return got


@pytest.mark.parametrize("dtype,heads", [(BF16, 8), (FP16, 8), (BF16, 1), (FP16, 3), (BF16, 5)])
@pytest.mark.parametrize("lens,new", [
    ([16], [1]), ([15], [1]), ([17], [1]), ([1], [1]), ([32, 16, 48, 33], [1, 1, 1, 1]),
    ([16], [16]), ([40], [40]), ([100, 37, 16], [100, 5, 16]), ([64, 64], [0, 1]), ([64, 31, 0, 48], [0, 0, 0, 33]),
    ([512, 300], [257, 299]), ([80] * 20, [1, 17, 0, 16, 80] * 4),
])
def test_bounds_of_the_pages_that_a_step_completes(gpu, dtype, heads, lens, new):
    counts = page_counts(lens)
    total = sum(counts) + 3
    cache = keys(total, heads, dtype, 1)
    before = torch.randn(total, heads, 2, 128, generator=torch.Generator().manual_seed(2)).to(dtype)
    table = tables_for(counts, total, 3)
    got = _update(gpu, cache.to(gpu), before, table, lens, new)
    assert torch.equal(got.cpu(), selection.page_bounds(cache, before, table, lens, new))


def test_bounds_of_one_token_a_sequence_without_starts(gpu):
    lens = [16 * (i % 4) + 16 - (i % 3) for i in range(150)]
    counts = page_counts(lens)
    cache = keys(sum(counts), 2, BF16, 4)
    before = torch.zeros(sum(counts), 2, 2, 128, dtype=BF16)
    table = tables_for(counts, sum(counts), 5)
    want = selection.page_bounds(cache, before, table, lens, [1] * len(lens))
    for gave_starts in (False, True):
        got = _update(gpu, cache.to(gpu), before, table, lens, [1] * len(lens), gave_starts)
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_bounds_of_infinities_nan_and_zeros(gpu, dtype):
    cache = keys(4, 2, dtype, 6)
    cache[0, 3, 0, 5], cache[0, 4, 0, 6], cache[0, :, 0, 7] = math.inf, -math.inf, -0.0
    cache[1, 0, 1, 9], cache[1, 15, 1, 10] = math.nan, -math.nan
    cache[1, 2, 0, 11], cache[1, 9, 0, 11], cache[1, 8, 0, 12] = math.nan, -math.inf, torch.finfo(dtype).min
    bits = cache.view(torch.int16)
    bits[2, 7, 1, 100] = -1  # a negative NaN of every bit set
    bits[2, 8, 1, 101] = 0x7fff
    table, lens = torch.arange(4, dtype=torch.int32)[None], [64]
    before = torch.zeros(4, 2, 2, 128, dtype=dtype)
    got = _update(gpu, cache.to(gpu), before, table, lens, [64])
    want = selection.page_bounds(cache, before, table, lens, [64])
    assert want.isnan().any() and want.isinf().any() and same(got, want)


def test_bounds_skip_pages_beyond_table_and_cache(gpu):
    cache = keys(4, 2, BF16, 7)
    before = torch.zeros(4, 2, 2, 128, dtype=BF16)
    table = torch.tensor([[0, -1, 4, 1], [2, 3, -7, 0]], dtype=torch.int32)
    lens, new = [64, 200], [64, 200]
    got = _update(gpu, cache.to(gpu), before, table, lens, new)
    assert torch.equal(got.cpu(), selection.page_bounds(cache, before, table, lens, new))


def test_bounds_of_a_layer_of_a_pool_and_wider_tables(gpu):
    # Pages of a pool that interleaves the layers, block tables of a wider buffer.
    lens, new = [100, 48], [50, 1]
    counts = page_counts(lens)
    pool = torch.full((sum(counts), 3, PAGE, 2, 128), math.nan, dtype=BF16)
    cache = keys(sum(counts), 2, BF16, 8)
    pool[:, 1] = cache
    table = tables_for(counts, sum(counts), 9)
    wide = torch.full((2, 40), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    before = torch.ones(sum(counts), 2, 2, 128, dtype=BF16)
    got = _update(gpu, pool.to(gpu)[:, 1], before, wide.to(gpu)[:, :table.shape[1]], lens, new)
    assert torch.equal(got.cpu(), selection.page_bounds(cache, before, table, lens, new))


def test_bounds_among_many_empty_sequences(gpu):
    # More sequences without new tokens between two with some than the kernel reads starts at a time.
    for seqs, at in ((70, (0, 69)), (300, (3, 150, 299)), (5000, (0, 1, 64, 65, 2500, 4999))):
        new = [0] * seqs
        for i, s in enumerate(at):
            new[s] = 16 + i
        lens = [32 + i % 16 if n else 1 for i, n in enumerate(new)]
        cache = keys(64, 1, BF16, seqs)
        table = torch.randint(0, 64, (seqs, 3), generator=torch.Generator().manual_seed(seqs)).to(torch.int32)
        before = torch.zeros(64, 1, 2, 128, dtype=BF16)
        got = _update(gpu, cache.to(gpu), before, table, lens, new)
        assert torch.equal(got.cpu(), selection.page_bounds(cache, before, table, lens, new))


# ---- selection -------------------------------------------------------------------


def _select(gpu, q, bounds, table, lens, n, sink, recent, **more):
    got = ops.select_pages(q.to(gpu), bounds.to(gpu), table.to(gpu), _ints(lens, gpu), n, sink, recent, **more)
    return [t.cpu() for t in got]


def _check_selection(gpu, q, bounds, table, lens, n, sink, recent):
    got = _select(gpu, q, bounds, table, lens, n, sink, recent)
    want = selection.select_pages(q, bounds, table, lens, n, sink, recent)
    assert torch.equal(got[1], want[1])
    assert torch.equal(got[0], want[0])


@pytest.mark.parametrize("hq,hkv,dtype", [(8, 8, BF16), (16, 8, FP16), (8, 1, BF16), (10, 2, BF16), (48, 3, FP16)])
@pytest.mark.parametrize("n,sink,recent", [(4, 1, 1), (4, 0, 1), (5, 2, 3), (16, 1, 4), (64, 4, 1), (1, 0, 1)])
def test_selected_pages(gpu, hq, hkv, dtype, n, sink, recent):
    # One token, a page short of, at and past the number selected, and long rows.
    lens = [1, 16, 16 * n - 1, 16 * n, 16 * n + 1, 16 * n + 16, 16 * n + 17, 16 * n + 300, 1500, 2049, 0]
    counts = page_counts(lens)
    cache = keys(sum(counts), hkv, dtype, n)
    table = tables_for(counts, sum(counts), n + 1)
    _check_selection(gpu, queries(len(lens), hq, dtype, n + 2), bounds_of(cache), table, lens, n, sink, recent)


@pytest.mark.parametrize("pages", [255, 256, 257, 1000, 2047, 2049, 4100, 9000])
def test_selected_pages_of_long_rows(gpu, pages):
    lens = [16 * pages - 3, 16 * (pages // 2)]
    counts = page_counts(lens)
    cache = keys(sum(counts), 1, BF16, pages)
    table = tables_for(counts, sum(counts), pages + 1)
    for n in (7, 128, pages // 2 + 1):
        _check_selection(gpu, queries(2, 4, BF16, pages + 2), bounds_of(cache), table, lens, n, 1, 2)


# Rows enough that each has one workgroup: its keys in registers, in LDS and in memory.
@pytest.mark.parametrize("pages", [300, 2300, 8300])
def test_selected_pages_of_many_rows(gpu, pages):
    q = queries(3, 2, BF16, pages)
    cache = keys(pages, 1, BF16, pages + 1)
    table = tables_for([pages], pages, pages + 2)
    lens = [16 * pages, 16 * pages - 5, 16 * (pages - pages // 3) + 1]
    want = selection.select_pages(q, bounds_of(cache), table.expand(3, pages), lens, 50, 2, 3)
    rows = torch.arange(3).repeat(180)
    got = _select(gpu, q[rows], bounds_of(cache), table.expand(len(rows), pages).contiguous(),
                  [lens[i] for i in rows.tolist()], 50, 2, 3)
    assert torch.equal(got[0], want[0][rows]) and torch.equal(got[1], want[1][rows])


@pytest.mark.parametrize("n,sink,recent", [(9, 1, 1), (40, 0, 3), (150, 2, 2)])
def test_ties_go_to_the_lowest_place(gpu, n, sink, recent):
    # Small whole numbers in few channels: scores are exact and many are equal.
    gen = torch.Generator().manual_seed(n)
    lens = [16 * 200, 16 * 333 + 5]
    counts = page_counts(lens)
    bounds = torch.zeros(sum(counts), 2, 2, 128)
    bounds[..., :3] = torch.randint(-2, 3, (sum(counts), 2, 2, 3), generator=gen).float()
    q = torch.zeros(2, 4, 128)
    q[..., :3] = torch.randint(-1, 2, (2, 4, 3), generator=gen).float()
    _check_selection(gpu, q.to(BF16), bounds.to(BF16), tables_for(counts, sum(counts), 1), lens, n, sink, recent)
    # All alike, of either sign of zero: the pages after the first ones.
    zero = torch.zeros(sum(counts), 2, 2, 128, dtype=BF16)
    zero[::2] = -0.0
    _check_selection(gpu, q.to(BF16), zero, tables_for(counts, sum(counts), 1), lens, n, sink, recent)


def test_nan_and_infinities_rank(gpu):
    lens = [16 * 50]
    gen = torch.Generator().manual_seed(3)
    bounds = torch.randn(50, 1, 2, 128, generator=gen).to(BF16)
    bounds[7, 0, 0, 3], bounds[30, 0, 1, 4], bounds[31, 0, 0, 3] = math.nan, math.nan, -math.nan
    bounds[9, 0, 1, 5], bounds[12, 0, 1, 5] = math.inf, -math.inf
    bounds[20, 0], bounds[21, 0] = torch.finfo(BF16).max, torch.finfo(BF16).min
    q = queries(1, 4, BF16, 5)
    q[0, :, 5] = 1.0
    table = torch.randperm(50, generator=gen).to(torch.int32)[None]
    bounds = bounds[torch.argsort(table[0].long())].contiguous()
    for n in (3, 4, 5, 6, 7, 8, 20, 49):
        _check_selection(gpu, q, bounds, table, lens, n, 0, 1)
    # A NaN query: every page alike, the lowest places.
    q[0, 1, 7] = math.nan
    _check_selection(gpu, q, bounds, table, lens, 11, 2, 3)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("pages,rows", [(40, 6), (700, 6), (300, 180)])
def test_infinities_count_as_products_with_the_queries(gpu, dtype, pages, rows):
    # Whole numbers, so that finite scores are exact; a few infinite bounds, and queries
    # of one sign, of both, zero, infinite and NaN in those channels.  Rows in several
    # workgroups and in one.
    gen = torch.Generator().manual_seed(pages)
    bounds = torch.randint(-2, 3, (pages, 2, 2, 128), generator=gen).float()
    values = torch.tensor([-math.inf, -2.0, 0.0, 1.0, math.inf])
    odd = torch.randperm(pages, generator=gen)[:pages // 3]
    bounds[odd, :, :, :2] = values[torch.randint(0, 5, (len(odd), 2, 2, 2), generator=gen)]
    bounds = bounds.sort(2).values.to(dtype)
    q = torch.randint(-2, 3, (6, 4, 128), generator=gen).float()  # two queries a KV head
    q[:, :, :2] = torch.tensor([[[1.0, 3.0], [2.0, 1.0]], [[-1.0, 2.0], [-2.0, 0.0]], [[0.0, 1.0], [-1.0, -1.0]],
                                [[-math.inf, 1.0], [1.0, 2.0]], [[math.nan, 1.0], [1.0, 1.0]],
                                [[0.0, 0.0], [0.0, 0.0]]]).repeat(1, 2, 1)
    q[4, :2] = 1.0  # NaN queries of one KV head only
    lens = [16 * pages - s for s in range(6)]
    table = torch.stack([torch.randperm(pages, generator=gen) for _ in range(6)]).to(torch.int32)
    of = torch.arange(rows) % 6
    for n in (4, 11, pages // 3, pages - 2):
        want = selection.select_pages(q.to(dtype), bounds, table, lens, n, 1, 2)
        got = _select(gpu, q[of].to(dtype), bounds, table[of].contiguous(), [lens[i] for i in of.tolist()], n, 1, 2)
        assert torch.equal(got[0], want[0][of]) and torch.equal(got[1], want[1][of])


def test_values_at_the_ends_of_the_types(gpu):
    for dtype in (BF16, FP16):
        top, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
        gen = torch.Generator().manual_seed(9)
        scale = torch.tensor([top, tiny, 1.0, tiny * 2 ** -5])[torch.randint(0, 4, (300, 1, 2, 128), generator=gen)]
        bounds = (torch.rand(300, 1, 2, 128, generator=gen) * scale).to(dtype)
        # One channel each, so that a score is one product and exact.
        bounds = torch.where(torch.arange(128) == 17, bounds, torch.zeros((), dtype=dtype))
        q = torch.zeros(1, 1, 128, dtype=dtype)
        for value in (top, -top, tiny, 1.0):
            q[0, 0, 17] = value
            _check_selection(gpu, q, bounds, torch.arange(300, dtype=torch.int32)[None], [4800], 25, 1, 1)


@pytest.mark.parametrize("hq,hkv,dtype", [(8, 8, BF16), (16, 1, FP16), (9, 3, BF16)])
@pytest.mark.parametrize("rows", [1, 15, 40, 300])
def test_selection_that_brings_the_bounds_up_to_date(gpu, hq, hkv, dtype, rows):
    lens = [16 + 16 * (7 * s % 23) + (0, 0, 1, 15)[s % 4] for s in range(rows)]
    counts = page_counts(lens)
    cache = keys(sum(counts), hkv, dtype, rows)
    table, q = tables_for(counts, sum(counts), rows + 1), queries(rows, hq, dtype, rows + 2)
    # Pages that this step's tokens complete have none yet.
    bounds = bounds_of(cache)
    for s, length in enumerate(lens):
        if length % 16 == 0:
            bounds[table[s, counts[s] - 1].long()] = math.nan
    for given in (cache.to(gpu), torch.stack((cache, cache), 1).to(gpu)[:, 1]):
        got = bounds.to(gpu)
        tables, kept = ops.select_pages(q.to(gpu), got, table.to(gpu), _ints(lens, gpu), 9, 1, 2, k_cache=given)
        assert same(got, selection.page_bounds(cache, bounds, table, lens, [1] * rows)) and not got.isnan().any()
        want = selection.select_pages(q, bounds_of(cache), table, lens, 9, 1, 2)
        assert torch.equal(tables.cpu(), want[0]) and torch.equal(kept.cpu(), want[1])


def test_lengths_beyond_the_tables_count_as_theirs(gpu):
    cache = keys(40, 2, BF16, 1)
    table = tables_for([20, 20], 40, 2)
    long, full = [16 * 20 + 5, 2 ** 31 - 1], [16 * 20, 16 * 20]
    q = queries(2, 4, BF16, 3)
    got = _select(gpu, q, bounds_of(cache), table, long, 6, 1, 1)
    want = selection.select_pages(q, bounds_of(cache), table, full, 6, 1, 1)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # More tokens than a list's pages hold: all of its pages.
    k, v = cache.to(gpu), keys(40, 2, BF16, 4).to(gpu)
    lists = got[0].to(gpu)
    outs = [ops.paged_decode_selected(q.to(gpu), k, v, lists, _ints(lens, gpu), SCALE)
            for lens in ([96, 96], [97, 2 ** 31 - 1])]
    assert torch.equal(*outs)


def test_strided_queries_and_tables(gpu):
    # Queries as a view of the packed projection, tables as columns of a wider buffer.
    lens = [700, 16, 900]
    counts = page_counts(lens)
    cache = keys(sum(counts), 2, BF16, 1)
    table = tables_for(counts, sum(counts), 2)
    packed = queries(3, 8 + 4, BF16, 3).to(gpu)
    wide = torch.full((3, 100), -1, dtype=torch.int32, device=gpu)
    wide[:, 2:2 + table.shape[1]] = table.to(gpu)
    got = ops.select_pages(packed[:, 2:10], bounds_of(cache).to(gpu), wide[:, 2:2 + table.shape[1]], _ints(lens, gpu),
                           20, 1, 2)
    want = selection.select_pages(packed[:, 2:10].cpu(), bounds_of(cache), table, lens, 20, 1, 2)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    # Rows that do not start at multiples of 16 bytes are copied.
    flat = torch.zeros(3 * 8 * 128 + 1, dtype=BF16, device=gpu)
    odd = flat[1:].view(3, 8, 128)
    odd.copy_(packed[:, 2:10])
    again = ops.select_pages(odd, bounds_of(cache).to(gpu), wide[:, 2:2 + table.shape[1]], _ints(lens, gpu), 20, 1, 2)
    assert torch.equal(again[0], got[0])


# ---- attention -------------------------------------------------------------------


def _lists(counts_of_pages, heads, num_pages, n, seed):
    """Tables ``[S, heads, n]`` of distinct pages in a row; unreadable ids behind them."""
    gen = torch.Generator().manual_seed(seed)
    tables = torch.full((len(counts_of_pages), heads, n), 0x7ffffff0, dtype=torch.int32)
    for s, count in enumerate(counts_of_pages):
        for h in range(heads):
            tables[s, h, :count] = torch.randperm(num_pages, generator=gen)[:count]
    return tables


def _check_attention(out, q, k, v, tables, lens, dtype):
    expected, spread, largest = selection.attention(q, k, v, tables, lens, SCALE)
    assert_within(out, expected, attention_bound(expected, spread, largest, max(max(lens), 1), dtype, dtype))


@pytest.mark.parametrize("hq,hkv,dtype", [(8, 8, BF16), (16, 8, FP16), (16, 1, BF16), (10, 2, BF16), (9, 3, FP16),
                                          (64, 8, BF16)])
@pytest.mark.parametrize("lens,n", [([1], 1), ([16, 17, 15], 2), ([100, 1, 0, 128, 127], 8), ([300], 19),
                                    ([16 * 40, 16 * 40 - 15, 33], 40), ([2048, 2000], 128), ([100] * 70, 7)])
def test_attention_over_lists_of_pages(gpu, hq, hkv, dtype, lens, n):
    counts = page_counts(lens)
    total = max(counts) + 5
    k, v = keys(total, hkv, dtype, 1), keys(total, hkv, dtype, 2)
    q, tables = queries(len(lens), hq, dtype, 3), _lists(counts, hkv, total, n, 4)
    out = ops.paged_decode_selected(q.to(gpu), k.to(gpu), v.to(gpu), tables.to(gpu), _ints(lens, gpu), SCALE)
    _check_attention(out, q, k, v, tables, lens, dtype)
    assert all((out[s] == 0).all() for s, length in enumerate(lens) if length == 0)


# One, two and three parts a row, rows of few pages among them, and lists of more
# than 64 pages a wavefront.
@pytest.mark.parametrize("rows,hkv,n", [(100, 8, 300), (97, 8, 40), (45, 8, 61), (30, 8, 70), (257, 1, 33)])
def test_attention_of_many_rows(gpu, rows, hkv, n):
    kinds = [16 * n - 3, 16 * n, 200, 16 * (n // 2) + 9]
    counts = page_counts(kinds)
    total = max(counts) + 20
    k, v = keys(total, hkv, FP16, 1), keys(total, hkv, FP16, 2)
    q, tables = queries(4, 2 * hkv, FP16, 3), _lists(counts, hkv, total, n, 4)
    of = torch.arange(rows) % 4
    out = ops.paged_decode_selected(q[of].to(gpu), k.to(gpu), v.to(gpu), tables[of].to(gpu),
                                    _ints([kinds[i] for i in of.tolist()], gpu), SCALE)
    _check_attention(out[:4], q, k, v, tables, kinds, FP16)
    assert torch.equal(out, out[:4][of.to(gpu)])


def test_rows_behind_the_last_token_do_not_show(gpu):
    # Whatever an earlier use of the last page left there.
    lens, n = [1, 16 * 3 + 5, 200], 13
    k, v = keys(30, 2, BF16, 5), keys(30, 2, BF16, 6)
    tables = _lists(page_counts(lens), 2, 30, n, 7)
    q = queries(3, 8, BF16, 8)
    clean = ops.paged_decode_selected(q.to(gpu), k.to(gpu), v.to(gpu), tables.to(gpu), _ints(lens, gpu), SCALE)
    for s, length in enumerate(lens):
        alone_k, alone_v = k.clone(), v.clone()
        for h in range(2):
            last = int(tables[s, h, (length - 1) // PAGE])
            for value, cache in ((math.nan, alone_k), (math.inf, alone_v)):
                cache[last, length % PAGE:, h] = value if length % PAGE else cache[last, length % PAGE:, h]
        out = ops.paged_decode_selected(q.to(gpu), alone_k.to(gpu), alone_v.to(gpu), tables.to(gpu), _ints(lens, gpu),
                                        SCALE)
        assert torch.equal(out[s], clean[s])


def test_out_strides_layers_of_a_pool_and_shared_lists(gpu):
    # One list for all heads (an expanded view), a pool that interleaves layers, out with rows apart.
    lens, n = [150, 16], 10
    pool = torch.full((2, 12, 3, PAGE, 4, 128), math.nan, dtype=BF16)
    k, v = keys(12, 4, BF16, 1), keys(12, 4, BF16, 2)
    pool[0, :, 2], pool[1, :, 2] = k, v
    pool = pool.to(gpu)
    lists = _lists(page_counts(lens), 1, 12, n, 3)
    tables = lists.to(gpu).expand(2, 4, n)
    q = queries(2, 8, BF16, 4)
    whole = torch.full((2, 20, 128), 7.0, dtype=BF16, device=gpu)
    got = ops.paged_decode_selected(q.to(gpu), pool[0, :, 2], pool[1, :, 2], tables, _ints(lens, gpu), SCALE,
                                    out=whole[:, 4:12])
    assert got.data_ptr() == whole[:, 4:12].data_ptr()
    _check_attention(got, q, k, v, lists.expand(2, 4, n), lens, BF16)
    assert (whole[:, :4] == 7).all() and (whole[:, 12:] == 7).all()


@pytest.mark.parametrize("rows,n", [(1, 128), (3, 40), (200, 20)])
def test_out_may_be_the_queries(gpu, rows, n):
    lens = [16 * n - s % 5 for s in range(rows)]
    k, v = keys(n, 4, BF16, 1).to(gpu), keys(n, 4, BF16, 2).to(gpu)
    tables = _lists([n], 4, n, n, 3).to(gpu).expand(rows, 4, n)
    q = queries(rows, 16, BF16, 4).to(gpu)
    want = ops.paged_decode_selected(q, k, v, tables, _ints(lens, gpu), SCALE)
    assert torch.equal(ops.paged_decode_selected(q, k, v, tables, _ints(lens, gpu), SCALE, out=q), want)


@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_a_nan_or_infinite_key_or_value_shows(gpu, value):
    lens, n = [100, 90], 8
    k, v = keys(20, 1, BF16, 1), keys(20, 1, BF16, 2)
    tables = _lists(page_counts(lens), 1, 20, n, 3)
    q = queries(2, 4, BF16, 4)
    page = int(tables[0, 0, 2])
    for cache in (k, v):
        bad = cache.clone()
        bad[page, 3, 0, 5] = value
        caches = (bad, v) if cache is k else (k, bad)
        out = ops.paged_decode_selected(q.to(gpu), caches[0].to(gpu), caches[1].to(gpu), tables.to(gpu),
                                        _ints(lens, gpu), SCALE).cpu()
        want = selection.attention(q, *caches, tables, lens, SCALE)[0]
        if cache is v:
            assert torch.equal(out[0, :, 5].isfinite(), want[0, :, 5].isfinite())
            assert out[0, :, :5].isfinite().all()
        elif math.isnan(value):
            assert out[0].isnan().all()
        if page not in tables[1, 0, :page_counts(lens)[1]].tolist():
            assert out[1].isfinite().all()


def test_large_caches(gpu):
    # Pages, bounds and tables whose byte offsets pass 32 bits.
    heads, pages = 8, 150_000  # 4.9 GB a cache
    k = torch.zeros(pages, PAGE, heads, 128, dtype=BF16, device=gpu)
    v = torch.zeros_like(k)
    ids = [3, 149_999, 70_001, 140_000, 149_990]
    rows = keys(len(ids), heads, BF16, 1), keys(len(ids), heads, BF16, 2)
    k[ids], v[ids] = rows[0].to(gpu), rows[1].to(gpu)
    lens = [16 * 4 + 3]
    tables = torch.tensor(ids, dtype=torch.int32).expand(1, heads, len(ids)).contiguous()
    q = queries(1, 16, BF16, 3)
    out = ops.paged_decode_selected(q.to(gpu), k, v, tables.to(gpu), _ints(lens, gpu), SCALE)
    small = torch.arange(len(ids), dtype=torch.int32).expand(1, heads, len(ids))
    _check_attention(out, q, *rows, small, lens, BF16)
    del v
    # Bounds past 4 GiB: 1.2 million pages of 8 heads.
    bounds = torch.zeros(1_200_000, heads, 2, 128, dtype=BF16, device=gpu)
    far = [1_199_999 - 7 * i for i in range(60)]
    cache = keys(60, heads, BF16, 4)
    bounds[far] = bounds_of(cache).to(gpu)
    table = torch.tensor([far], dtype=torch.int32)
    got = ops.select_pages(q.to(gpu), bounds, table.to(gpu), _ints([16 * 60], gpu), 20, 1, 1)[0].cpu()
    places = selection.select_pages(q, bounds_of(cache), torch.arange(60, dtype=torch.int32)[None], [16 * 60], 20, 1, 1)
    assert torch.equal(got, table[0][places[0].long()])
    del bounds
    bounds = torch.zeros(pages, heads, 2, 128, dtype=BF16, device=gpu)
    ops.update_page_bounds(k, bounds, _ints([ids], gpu), _ints([80], gpu), _ints([0, 80], gpu), 80)
    assert torch.equal(bounds[ids].cpu(), bounds_of(rows[0])) and int((bounds != 0).any(-1).sum()) == len(ids) * heads * 2


# ---- together ----------------------------------------------------------------------


def test_one_workspace_serves_calls_of_other_sizes(gpu):
    lens = [900, 16, 400]
    counts = page_counts(lens)
    k, v = keys(sum(counts), 2, BF16, 1), keys(sum(counts), 2, BF16, 2)
    table, q = tables_for(counts, sum(counts), 3), queries(3, 8, BF16, 4)
    nbytes = ops.selection_workspace_bytes(3, 8, 2, table.shape[1], 20)
    workspace = torch.full((nbytes + 4096,), 0xff, dtype=torch.uint8, device=gpu)
    workspace[:ops.SELECTION_HEADER_BYTES] = 0
    outs = []
    for n in (20, 7, 20):
        tables, kept = ops.select_pages(q.to(gpu), bounds_of(k).to(gpu), table.to(gpu), _ints(lens, gpu), n, 1, 1,
                                        workspace=workspace)
        outs.append(ops.paged_decode_selected(q.to(gpu), k.to(gpu), v.to(gpu), tables, kept, SCALE,
                                              workspace=workspace))
        want = selection.select_pages(q, bounds_of(k), table, lens, n, 1, 1)
        assert torch.equal(tables.cpu(), want[0]) and torch.equal(kept.cpu(), want[1])
        _check_attention(outs[-1], q, k, v, *want, BF16)
    assert torch.equal(outs[0], outs[2])
    assert (workspace[nbytes:] == 0xff).all() and (workspace[:ops.SELECTION_HEADER_BYTES] == 0).all()


def test_one_workspace_serves_a_batch_that_drains(gpu):
    # Fewer rows are cut into more parts: 52 and 49 rows of 8 heads in one, 48 in two, 3 in eight.
    lens = [16 * 130 - 7 * s for s in range(52)]
    counts = page_counts(lens)
    k, v = keys(max(counts), 8, BF16, 1), keys(max(counts), 8, BF16, 2)
    table, q = torch.arange(max(counts), dtype=torch.int32).expand(52, -1).contiguous(), queries(52, 8, BF16, 3)
    nbytes = ops.selection_workspace_bytes(52, 8, 8, table.shape[1], 120)
    workspace = torch.full((nbytes + 4096,), 0xff, dtype=torch.uint8, device=gpu)
    workspace[:ops.SELECTION_HEADER_BYTES] = 0
    on_gpu = [t.to(gpu) for t in (q, bounds_of(k), k, v, table, _ints(lens, gpu))]
    for rows in (52, 49, 48, 33, 3):
        few = on_gpu[0][:rows], *on_gpu[1:4], on_gpu[4][:rows], on_gpu[5][:rows]
        out = ops.sparse_decode(*few, SCALE, 120, 1, 4, out=torch.empty_like(few[0]), workspace=workspace[:nbytes])
        assert torch.equal(out, ops.sparse_decode(*few, SCALE, 120, 1, 4))
        if rows == 3:
            want = selection.select_pages(q[:3], bounds_of(k), table[:3], lens[:3], 120, 1, 4)
            _check_attention(out, q[:3], k, v, *want, BF16)
    assert (workspace[nbytes:] == 0xff).all() and (workspace[:ops.SELECTION_HEADER_BYTES] == 0).all()


def test_calls_on_two_streams_and_captured_ones(gpu):
    sets = []
    for seed in (1, 2):
        lens = [3000 - 100 * seed, 500, 16]
        counts = page_counts(lens)
        k, v = keys(sum(counts), 2, BF16, seed), keys(sum(counts), 2, BF16, seed + 5)
        table, q = tables_for(counts, sum(counts), seed), queries(3, 8, BF16, seed + 7)
        want = selection.select_pages(q, bounds_of(k), table, lens, 30, 1, 2)
        bounds = torch.zeros(sum(counts), 2, 2, 128, dtype=BF16, device=gpu)
        sets.append((q.to(gpu), k.to(gpu), v.to(gpu), bounds, table.to(gpu), _ints(lens, gpu),
                     _ints([0, *torch.tensor(lens).cumsum(0).tolist()], gpu), sum(lens), want))

    def step(q, k, v, bounds, table, lens, starts, tokens, _):
        ops.update_page_bounds(k, bounds, table, lens, starts, tokens)
        tables, kept = ops.select_pages(q, bounds, table, lens, 30, 1, 2)
        return tables, ops.paged_decode_selected(q, k, v, tables, kept, SCALE)

    alone = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams, graphs, outs = [torch.cuda.Stream() for _ in sets], [], []
    for _ in range(5):
        got = []
        for stream, s in zip(streams, sets):
            with torch.cuda.stream(stream):
                got.append(step(*s))
        torch.cuda.synchronize()
        for (tables, out), (want_tables, want_out), s in zip(got, alone, sets):
            assert torch.equal(tables, want_tables) and torch.equal(out, want_out)
            assert torch.equal(tables.cpu(), s[-1][0])
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(*s))
        graphs.append(graph)
    for turn in range(4):
        for s, (tables, out) in zip(sets, outs):
            s[3].zero_()
            tables.zero_()
            out.zero_()
        torch.cuda.synchronize()
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(outs, alone):
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        # Eager work between the replays.
        assert all(torch.equal(step(*s)[1], want[1]) for s, want in zip(sets, alone))
