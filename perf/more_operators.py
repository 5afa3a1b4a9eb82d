"""The measured operators: decode attention over the cache pages that a cheap score selects.

A 16-bit paged KV cache (``[pages, 16, KV heads, 128]``) carries, for every page
that is full, the smallest and the largest value of each channel of its keys:
``page_bounds [pages, KV heads, 2, 128]``, minima then maxima.  A decode step
bounds each page's scores with them and attends to the best pages only.

* ``bounds``: the bounds of the pages that a step's new tokens have completed
  (a decode step's single tokens, or the chunks of a prefill step);
* ``select``: for each sequence and KV head the first and the last pages and,
  of the others, those of the highest score, as a table of page ids;
* ``attend``: attention of each sequence's query over its tables' pages;
* ``step``: one layer of a decode step, selection and attention.

The score of a page is the sum over channels and the KV head's query heads of
``max(q * min, q * max)``, which no key of the page exceeds.  Lengths are drawn
per case (``lengths`` seeds them), values and page permutations from the seed.
Head counts, contexts and batch sizes are those of the repository's benchmark
configurations (Qwen3-0.6B, 8B and 32B layers and their tensor-parallel shards,
page 16, head_dim 128) and of the steps between them.
"""

import math

import numpy as np
import torch

own = False

PAGE = 16
DIM = 128
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
HEADS = ((16, 8), (32, 8), (64, 8), (16, 4), (32, 4), (16, 2), (8, 1), (40, 8), (24, 8))
# A drawn case costs no more than the largest listed one of its kind.
MAX_SCORED = 56 * 2048 * 8  # (page, KV head) pairs, padded
MAX_ATTENDED = 64 * 256 * 8
MAX_NEW_TOKENS = 16384


def listed():
    return [
        # A decode step's new rows: 61 sequences of which a few complete a page.
        {"name": "bounds_61seq_1tok", "kind": "bounds", "dtype": "bf16", "hkv": 8, "seqs": 61, "q_lo": 1, "q_hi": 1,
         "prefix_lo": 127, "prefix_hi": 2047, "lengths": 3},
        # A full prefill step: chunks that begin and end inside pages.
        {"name": "bounds_prefill_16384tok", "kind": "bounds", "dtype": "bf16", "hkv": 8, "seqs": 8, "q_lo": 2048,
         "q_hi": 2048, "prefix_lo": 0, "prefix_hi": 1024, "lengths": 4},
        # A few interactive users: launch latency.
        {"name": "select_8seq_4k", "kind": "select", "dtype": "bf16", "hq": 16, "hkv": 8, "batch": 8, "ctx_lo": 1024,
         "ctx_hi": 4096, "pages": 64, "sink": 1, "recent": 2, "lengths": 11},
        # One user with a long document.
        {"name": "select_1seq_30k", "kind": "select", "dtype": "bf16", "hq": 32, "hkv": 8, "batch": 1,
         "ctx_lo": 30001, "ctx_hi": 30001, "pages": 128, "sink": 1, "recent": 4, "lengths": 0},
        # Half of an 8B layer's heads (tensor parallelism over two GPUs), fp16; short
        # contexts keep all of their pages.
        {"name": "select_37seq_6k_shard_fp16", "kind": "select", "dtype": "fp16", "hq": 16, "hkv": 4, "batch": 37,
         "ctx_lo": 300, "ctx_hi": 6000, "pages": 77, "sink": 1, "recent": 1, "lengths": 5},
        # Long-context decode at the 32B shape.
        {"name": "select_56seq_32k", "kind": "select", "dtype": "bf16", "hq": 64, "hkv": 8, "batch": 56,
         "ctx_lo": 8192, "ctx_hi": 32768, "pages": 128, "sink": 1, "recent": 4, "lengths": 4},
        # One user: the split of 128 pages over the GPU.
        {"name": "attend_1seq_128pages", "kind": "attend", "dtype": "bf16", "hq": 32, "hkv": 8, "batch": 1,
         "ctx_lo": 30001, "ctx_hi": 30001, "pages": 128, "lengths": 0},
        # Contexts around the table's size, fp16: some rows hold fewer pages.
        {"name": "attend_37seq_77pages_shard_fp16", "kind": "attend", "dtype": "fp16", "hq": 16, "hkv": 4, "batch": 37,
         "ctx_lo": 300, "ctx_hi": 6000, "pages": 77, "lengths": 5},
        # A large batch that keeps 4096 tokens a sequence, at the 32B shape.
        {"name": "attend_64seq_256pages", "kind": "attend", "dtype": "bf16", "hq": 64, "hkv": 8, "batch": 64,
         "ctx_lo": 8192, "ctx_hi": 16384, "pages": 256, "lengths": 6},
        # One layer of a decode step: one user with a long document, and the
        # long-context batch.
        {"name": "step_1seq_30k", "kind": "step", "dtype": "bf16", "hq": 32, "hkv": 8, "batch": 1, "ctx_lo": 30001,
         "ctx_hi": 30001, "pages": 128, "sink": 1, "recent": 4, "lengths": 0},
        {"name": "step_56seq_32k", "kind": "step", "dtype": "bf16", "hq": 64, "hkv": 8, "batch": 56, "ctx_lo": 8192,
         "ctx_hi": 32768, "pages": 128, "sink": 1, "recent": 4, "lengths": 4},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choices(("select", "attend", "step", "bounds"), (30, 30, 25, 15))[0]
    hq, hkv = rng.choice(HEADS)
    case = {"kind": kind, "dtype": rng.choice(("bf16", "bf16", "fp16")), "hkv": hkv, "lengths": rng.randrange(1 << 16)}
    if kind == "bounds":
        case["seqs"] = _log_int(rng, 1, 256)
        case["q_hi"] = rng.choice((1, _log_int(rng, 1, 4096), _log_int(rng, 16, 4096)))
        case["q_hi"] = max(1, min(case["q_hi"], MAX_NEW_TOKENS // case["seqs"]))
        case["q_lo"] = max(1, case["q_hi"] // rng.choice((1, 2, 8)))
        case["prefix_hi"] = rng.choice((0, _log_int(rng, 1, 4096)))
        case["prefix_lo"] = rng.choice((0, case["prefix_hi"] // 2))
        return case
    case["hq"] = hq
    case["batch"] = _log_int(rng, 1, 256)
    hi = _log_int(rng, 1, 32768)
    case["ctx_hi"] = max(1, min(hi, MAX_SCORED // hkv // case["batch"] * PAGE))
    case["ctx_lo"] = max(1, case["ctx_hi"] // rng.choice((1, 2, 4, 16)))
    case["pages"] = min(_log_int(rng, 4, 512), max(4, MAX_ATTENDED // hkv // case["batch"]))
    if kind != "attend":
        case["recent"] = rng.choice((1, 2, _log_int(rng, 1, case["pages"] // 2)))
        case["sink"] = rng.choice((0, 1, case["pages"] // 4))
    return case


def _lengths(case):
    """(new tokens, context lengths with them) of each sequence."""
    rng = np.random.default_rng(case["lengths"])
    if case["kind"] != "bounds":
        ctx = rng.integers(case["ctx_lo"], case["ctx_hi"] + 1, size=case["batch"])
        return np.ones_like(ctx), ctx
    q = rng.integers(case["q_lo"], case["q_hi"] + 1, size=case["seqs"])
    return q, q + rng.integers(case["prefix_lo"], case["prefix_hi"] + 1, size=case["seqs"])


def _page_counts(lengths):
    return (lengths + PAGE - 1) // PAGE


# ---- the plain form ------------------------------------------------------------


def _plain_bounds(s):
    q_len = s["query_start_loc"][1:] - s["query_start_loc"][:-1]
    first, last = (s["seq_lens"] - q_len) // PAGE, s["seq_lens"] // PAGE  # the complete pages, before and after
    count = last - first
    seq = torch.repeat_interleave(torch.arange(len(count), device="cuda"), count, output_size=s["completed"])
    place = torch.arange(s["completed"], device="cuda") - (torch.cumsum(count, 0) - count)[seq]
    page = s["block_tables"][seq, first[seq] + place].long()
    rows = s["k_cache"][page].float()
    dtype = s["k_cache"].dtype
    s["page_bounds"][page] = torch.stack((rows.amin(1).to(dtype), rows.amax(1).to(dtype)), 2)
    return s["page_bounds"]


def _plain_select(s):
    """Scores in 64 bits: which pages are taken depends on values next to each other."""
    case = s["case"]
    hkv, pages = case["hkv"], case["pages"]
    table = s["block_tables"]
    seqs, width = table.shape
    n = (s["seq_lens"].long() + PAGE - 1) // PAGE
    heads = s["q"].double().view(seqs, hkv, -1, DIM)
    up, down = heads.clamp(min=0).sum(2), heads.clamp(max=0).sum(2)
    bounds = s["page_bounds"][table.long().clamp_min(0)]  # [S, W, H, 2, 128]
    scores = (bounds[:, :, :, 1].double() * up[:, None]).sum(-1) + (bounds[:, :, :, 0].double() * down[:, None]).sum(-1)
    place = torch.arange(width, device="cuda")
    kept = (place < case["sink"]) | (place >= n[:, None] - case["recent"])
    scores = scores.masked_fill_(kept[:, :, None], math.inf)
    scores = scores.masked_fill_((place >= n[:, None])[:, :, None], -math.inf).transpose(1, 2)
    order = torch.sort(scores, dim=-1, descending=True, stable=True).indices  # ties: the lowest page first
    if width < pages:
        order = torch.nn.functional.pad(order, (0, pages - width), value=width)
    taken = torch.minimum(n, torch.full_like(n, pages))
    rank = torch.arange(pages, device="cuda")
    order = order[:, :, :pages].masked_fill((rank >= taken[:, None])[:, None], width).sort(-1).values
    ids = table[torch.arange(seqs, device="cuda")[:, None, None], order.clamp_max(width - 1)]
    ids = ids.masked_fill((rank >= taken[:, None])[:, None], -1).to(torch.int32)
    return [ids, (s["seq_lens"] - PAGE * (n - taken)).to(torch.int32)]


def _plain_attend(s, ids, lens):
    """Attention of one query a sequence over the pages of its tables, padded to their width."""
    case = s["case"]
    hq, hkv = case["hq"], case["hkv"]
    seqs = ids.shape[0]
    pages, head = ids.long().clamp_min(0), torch.arange(hkv, device="cuda")[None, :, None]
    q = s["q"].float().view(seqs, hkv, hq // hkv, DIM)
    rows = s["k_cache"][pages, :, head].float().flatten(2, 3)  # [S, H, pages * 16, 128]
    scores = torch.matmul(q, rows.transpose(-1, -2).contiguous()).mul_(1 / math.sqrt(DIM))
    hidden = torch.arange(rows.shape[2], device="cuda") >= lens[:, None]
    scores = scores.masked_fill_(hidden[:, None, None], -math.inf)
    scores = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    scores = scores.div_(scores.sum(-1, keepdim=True))
    rows = s["v_cache"][pages, :, head].float().flatten(2, 3)
    return torch.matmul(scores, rows).view(seqs, hq, DIM).to(s["q"].dtype)


# ---- inputs --------------------------------------------------------------------


def _generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _keys(gen, case, pages):
    """Pages of keys: channels of unlike size, and a centre that a page's tokens share."""
    dtype, hkv = DTYPES[case["dtype"]], case["hkv"]
    channels = torch.exp(0.5 * torch.randn(hkv, DIM, generator=gen, device="cuda"))
    rows = torch.empty(pages, PAGE, hkv, DIM, dtype=dtype, device="cuda")
    step = 1 << 14  # pages at a time: the fp32 values take twice the cache's room
    for a in range(0, pages, step):
        part = rows[a: a + step]
        centre = torch.randn(len(part), 1, hkv, DIM, generator=gen, device="cuda") * 0.5
        part.copy_((torch.randn(part.shape, generator=gen, device="cuda") + centre) * channels)
    return rows


def _bounds_of(keys):
    return torch.stack((keys.amin(1), keys.amax(1)), 2)


def _tables(gen, counts):
    """Block tables of pages in a random order, -1 behind a sequence's last page."""
    total, width = int(counts.sum()), int(counts.max())
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    used = torch.arange(width, device="cuda")[None] < torch.from_numpy(counts).to("cuda")[:, None]
    table = torch.full((len(counts), width), -1, dtype=torch.int32, device="cuda")
    table[used] = order
    return table


def _selection(gen, case, table, counts):
    """Tables as a selection leaves them: a sequence's first and last page and random ones between."""
    n = torch.from_numpy(counts).to("cuda")
    seqs, width = table.shape
    pages = case["pages"]
    value = torch.rand(seqs, case["hkv"], width, generator=gen, device="cuda")
    place = torch.arange(width, device="cuda")
    value = value.masked_fill(((place == 0) | (place == n[:, None] - 1))[:, None], 2.0)
    value = value.masked_fill((place >= n[:, None])[:, None], -1.0)
    order = torch.topk(value, min(pages, width), -1).indices
    taken = n.clamp_max(pages)
    off = torch.arange(order.shape[2], device="cuda") >= taken[:, None]
    order = order.masked_fill(off[:, None], width).sort(-1).values
    ids = table[torch.arange(seqs, device="cuda")[:, None, None], order.clamp_max(width - 1)]
    ids = torch.nn.functional.pad(ids.masked_fill(off[:, None], -1), (0, pages - order.shape[2]), value=-1)
    lens = torch.from_numpy(_lengths(case)[1]).to("cuda") - PAGE * (n - taken)
    return ids.to(torch.int32).contiguous(), lens.to(torch.int32)


def _inputs(case, seed):
    gen = _generator(seed)
    dtype, hkv = DTYPES[case["dtype"]], case["hkv"]
    q_len, kv_len = _lengths(case)
    counts = _page_counts(kv_len)
    total = int(counts.sum())
    state = {"case": case, "block_tables": _tables(gen, counts),
             "seq_lens": torch.from_numpy(kv_len.astype(np.int32)).to("cuda")}
    if case["kind"] == "bounds":
        state["query_start_loc"] = torch.from_numpy(np.concatenate(([0], np.cumsum(q_len))).astype(np.int32)).to("cuda")
        state["num_tokens"] = int(q_len.sum())
        state["completed"] = int((kv_len // PAGE - (kv_len - q_len) // PAGE).sum())
        state["k_cache"] = _keys(gen, case, total)
        # What an earlier use of the pages left there.
        state["page_bounds"] = torch.randn(total, hkv, 2, DIM, generator=gen, device="cuda").to(dtype)
        return state
    state["q"] = torch.randn((case["batch"], case["hq"], DIM), generator=gen, device="cuda").to(dtype)
    if case["kind"] == "select":
        centre = torch.randn(total, hkv, DIM, generator=gen, device="cuda") * 0.6
        spread = 1.77 + 0.5 * torch.randn(total, hkv, DIM, generator=gen, device="cuda").abs()
        state["page_bounds"] = torch.stack((centre - spread, centre + spread), 2).to(dtype)
        return state
    state["k_cache"] = _keys(gen, case, total)
    if case["kind"] == "step":
        state["page_bounds"] = _bounds_of(state["k_cache"])
    else:
        state["tables"], state["lens"] = _selection(gen, case, state["block_tables"], counts)
    state["v_cache"] = _keys(gen, case, total)
    return state


def _backend(state):
    """The backend and the step's plan, which serve all layers of a model."""
    from my_vllm_amd.attention_backend import MI355XSparseAttentionBackend
    from my_vllm_amd.contract import CommonAttentionMetadata

    case = state["case"]
    kv_len = _lengths(case)[1]
    batch = len(kv_len)
    counts = tuple(int(n) for n in _page_counts(kv_len))
    common = CommonAttentionMetadata(
        num_prefill_seqs=0, num_decode_seqs=batch, num_prefill_tokens=0, num_decode_tokens=batch,
        query_start_loc=torch.arange(batch + 1, dtype=torch.int32, device="cuda"), seq_lens=state["seq_lens"],
        slot_mapping=torch.full((batch,), -1, dtype=torch.int32, device="cuda"), block_tables=state["block_tables"],
        max_q_len=1, max_kv_len=int(kv_len.max()), block_counts=counts, num_kv_blocks=sum(counts),
        num_prefill_kv_blocks=0, trusted=True,
    )
    backend = MI355XSparseAttentionBackend(
        case["hq"], case["hkv"], DIM, PAGE, DTYPES[case["dtype"]], selected_pages=case["pages"],
        sink_pages=case["sink"], recent_pages=case["recent"])
    return backend, backend.build_plan(common)


def prepare(case, seed):
    state = _inputs(case, seed)
    if own:
        if case["kind"] == "step":
            state["backend"], state["plan"] = _backend(state)
        elif case["kind"] != "bounds":
            from my_vllm_amd import ops

            # The layers of a program share one workspace, zeroed when it is made.
            nbytes = ops.selection_workspace_bytes(case["batch"], case["hq"], case["hkv"],
                                                   state["block_tables"].shape[1], case["pages"])
            state["workspace"] = torch.zeros(nbytes, dtype=torch.uint8, device="cuda")
    return state


def run(state):
    s, case = state, state["case"]
    kind = case["kind"]
    if not own:
        if kind == "bounds":
            return _plain_bounds(s)
        if kind == "attend":
            return _plain_attend(s, s["tables"], s["lens"])
        selection = _plain_select(s)
        return selection if kind == "select" else _plain_attend(s, *selection)
    if kind == "step":
        return s["backend"].forward(s["q"], None, None, s["k_cache"], s["v_cache"], s["plan"],
                                    page_bounds=s["page_bounds"])
    from my_vllm_amd import ops

    if kind == "bounds":
        ops.update_page_bounds(s["k_cache"], s["page_bounds"], s["block_tables"], s["seq_lens"], s["query_start_loc"],
                               s["num_tokens"])
        return s["page_bounds"]
    if kind == "select":
        return list(ops.select_pages(s["q"], s["page_bounds"], s["block_tables"], s["seq_lens"], case["pages"],
                                     case["sink"], case["recent"], workspace=s["workspace"]))
    return ops.paged_decode_selected(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["lens"], 1 / math.sqrt(DIM),
                                     workspace=s["workspace"])


def work(case):
    """Each input read and each output written once.  Bounds: the rows and the
    bounds of the pages completed.  Selection: the bounds of the pages that are
    neither kept anyway nor all taken, one multiply and add a bound; its table.
    Attention: each selected row, query, output and page id, and two products a
    (query head, token)."""
    q_len, kv_len = _lengths(case)
    counts = _page_counts(kv_len)
    if case["kind"] == "bounds":
        pages = int((kv_len // PAGE - (kv_len - q_len) // PAGE).sum())
        moved = pages * case["hkv"] * (PAGE + 2) * DIM * 2 + 4 * (pages + 2 * len(q_len))
        return {"bytes": moved, "flops": pages * case["hkv"] * 2 * (PAGE - 1) * DIM}
    queries = case["batch"] * case["hq"] * DIM * 2
    taken = np.minimum(counts, case["pages"])
    table = 4 * (int(taken.sum()) * case["hkv"] + case["batch"])
    moved = flops = 0
    if case["kind"] != "attend":
        scored = np.where(counts > case["pages"], counts - case["sink"] - case["recent"], 0)
        scored = int(scored.sum()) * case["hkv"]
        moved += scored * 2 * DIM * 2 + queries + 4 * int(counts.sum()) + table
        flops += scored * 4 * DIM
    if case["kind"] != "select":
        tokens = int((kv_len - PAGE * (counts - taken)).sum())
        moved += tokens * case["hkv"] * 2 * DIM * 2 + queries * (2 if case["kind"] == "attend" else 1)
        moved += table if case["kind"] == "attend" else -table  # within a step the table is the path's own
        flops += tokens * case["hq"] * 4 * DIM
    return {"bytes": moved, "flops": flops}


# ---- the definition, in 64 bits -------------------------------------------------


def _exact_selection(case, s):
    """Page places of each (sequence, KV head): score by score from the bounds."""
    q_len, kv_len = _lengths(case)
    counts = _page_counts(kv_len)
    hkv, pages = case["hkv"], case["pages"]
    found = []
    for i, n in enumerate(int(x) for x in counts):
        if n <= pages:
            found.append(torch.arange(n, device="cuda").expand(hkv, n))
            continue
        box = s["page_bounds"][s["block_tables"][i, :n].long()].double()  # [n, H, 2, 128]
        q = s["q"][i].double().view(hkv, -1, DIM)
        score = torch.zeros(n, hkv, dtype=torch.float64, device="cuda")
        for g in range(q.shape[1]):
            score += torch.maximum(q[:, g] * box[:, :, 0], q[:, g] * box[:, :, 1]).sum(-1)
        middle = torch.arange(case["sink"], n - case["recent"], device="cuda")
        best = torch.sort(score[middle], dim=0, descending=True, stable=True).indices
        best = middle[best[: pages - case["sink"] - case["recent"]]]
        ends = torch.cat((torch.arange(case["sink"], device="cuda"),
                          torch.arange(n - case["recent"], n, device="cuda")))
        found.append(torch.cat((best.t(), ends.expand(hkv, -1)), 1).sort(1).values)
    return found


def _exact_attention(case, s, ids, lens):
    """``ids[i]``: page ids ``[H, pages]`` of sequence i; ``lens[i]``: their tokens."""
    hkv, group = case["hkv"], case["hq"] // case["hkv"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, (page, n) in enumerate(zip(ids, lens)):
        head = torch.arange(hkv, device="cuda")[:, None]
        k = s["k_cache"][page.long(), :, head].double().flatten(1, 2)[:, :n]
        v = s["v_cache"][page.long(), :, head].double().flatten(1, 2)[:, :n]
        q = s["q"][i].double().view(hkv, group, DIM)
        scores = torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(DIM)
        out[i] = torch.matmul(torch.softmax(scores, -1), v).view(-1, DIM)
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    q_len, kv_len = _lengths(case)
    counts = _page_counts(kv_len)
    if case["kind"] == "bounds":
        for i, (new, kv) in enumerate(zip(q_len.tolist(), kv_len.tolist())):
            page = s["block_tables"][i, (kv - new) // PAGE: kv // PAGE].long()
            ordered = s["k_cache"][page].double().sort(1).values
            s["page_bounds"][page] = torch.stack((ordered[:, 0], ordered[:, -1]), 2).to(s["page_bounds"].dtype)
        return s["page_bounds"].double()
    taken = np.minimum(counts, case["pages"])
    lens = [int(x) for x in kv_len - PAGE * (counts - taken)]
    if case["kind"] == "attend":
        ids = [s["tables"][i, :, :n] for i, n in enumerate(taken.tolist())]
        return _exact_attention(case, s, ids, lens)
    places = _exact_selection(case, s)
    ids = [s["block_tables"][i][place] for i, place in enumerate(places)]
    if case["kind"] == "step":
        return _exact_attention(case, s, ids, lens)
    table = torch.full((case["batch"], case["hkv"], case["pages"]), -1, dtype=torch.int32, device="cuda")
    for i, page in enumerate(ids):
        table[i, :, : page.shape[1]] = page
    return [table, torch.tensor(lens, dtype=torch.int32, device="cuda")]
