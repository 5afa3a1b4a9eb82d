"""The measured operators: a KV cache held in four bits and the attention over it.

The cache is in the OCP microscaling format MXFP4: e2m1 elements (0, 0.5, 1,
1.5, 2, 3, 4, 6 and their negatives) with one power-of-two scale, an E8M0 byte,
for 32 of them.  Each of K and V is a ``uint8 [pages, KV heads, 1088]`` tensor:
the 16 tokens of a page and head at 64 bytes each (element 2i in the low four
bits of byte i), then their scales at four bytes each.

* ``write``: a step's K/V rows quantised into the cache by ``slot_mapping``, and
  read back from it (what the cache holds is compared as the values it stands
  for);
* ``read``: cached rows read back by slot, as a prefix leaves for a host copy or
  for another server;
* ``decode``: one layer's attention of a pure-decode step;
* ``prefill``: one layer's attention of a prefill step, over new tokens that
  follow cached ones (a prefix hit, or the earlier chunks of a long prompt).

A step's plan is built once for all of a model's layers, so it is part of what
``prepare`` hands over; lengths are drawn per case (``lengths`` seeds them),
values and page permutations from the seed.  Head counts, contexts and batch
sizes are those of the repository's benchmark configurations (Qwen3-0.6B, 8B
and 32B layers and their tensor-parallel shards, page 16, head_dim 128) and of
the steps between them.
"""

import math

import numpy as np
import torch

own = False

PAGE = 16
DIM = 128
GROUP = 32
ROW = DIM // 2  # bytes of a token's elements
SCALES = DIM // GROUP  # scale bytes of a token
BLOCK = PAGE * (ROW + SCALES)  # bytes of one page of one KV head
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
# Largest scale byte: every value read back is finite in the row's type.
MAX_SCALE = {"bf16": 252, "fp16": 140}
HEADS = ((16, 8), (32, 8), (64, 8), (16, 4), (32, 4), (16, 2), (8, 1), (40, 8), (24, 8))
# A drawn case costs no more than the largest listed one of its kind.
MAX_DECODE_ROWS = 56 * 32768 * 8  # padded (token, KV head) rows
MAX_PREFILL_FLOPS = 3.3e11
MAX_PREFILL_SCORES = 16 * 32 * 2048 * 2048


def listed():
    return [
        # A decode step's new rows: one token of each of 61 sequences, so the
        # rows land on 61 pages; the smallest call.
        {"name": "write_61tok", "kind": "write", "dtype": "bf16", "hq": 32, "hkv": 8, "tokens": 61, "run": 1},
        # A full prefill step's rows, as the packed projection leaves them.
        {"name": "write_16384tok", "kind": "write", "dtype": "bf16", "hq": 32, "hkv": 8, "tokens": 16384,
         "run": 1024},
        # A short cached prompt read back, fp16.
        {"name": "read_333tok_fp16", "kind": "read", "dtype": "fp16", "hkv": 8, "tokens": 333, "run": 333},
        # A long document's rows read back.
        {"name": "read_30001tok", "kind": "read", "dtype": "bf16", "hkv": 8, "tokens": 30001, "run": 30001},
        # A decode step of a few interactive users: launch latency.
        {"name": "decode_8seq_1k", "kind": "decode", "dtype": "bf16", "hq": 16, "hkv": 8, "batch": 8,
         "ctx_lo": 256, "ctx_hi": 1024, "lengths": 11},
        # One user with a long document: the split along the context.
        {"name": "decode_1seq_30k", "kind": "decode", "dtype": "bf16", "hq": 32, "hkv": 8, "batch": 1,
         "ctx_lo": 30001, "ctx_hi": 30001, "lengths": 0},
        # The benchmark's decode batch.
        {"name": "decode_64seq_2k", "kind": "decode", "dtype": "bf16", "hq": 16, "hkv": 8, "batch": 64,
         "ctx_lo": 128, "ctx_hi": 2048, "lengths": 1},
        # Half of an 8B layer's heads (tensor parallelism over two GPUs), fp16.
        {"name": "decode_37seq_6k_shard_fp16", "kind": "decode", "dtype": "fp16", "hq": 16, "hkv": 4, "batch": 37,
         "ctx_lo": 300, "ctx_hi": 6000, "lengths": 5},
        # Long-context decode at the 32B shape: the largest cache read.
        {"name": "decode_56seq_32k", "kind": "decode", "dtype": "bf16", "hq": 64, "hkv": 8, "batch": 56,
         "ctx_lo": 8192, "ctx_hi": 32768, "lengths": 4},
        # One short prompt without a cached prefix (time to first token), fp16.
        {"name": "prefill_1seq_333_fp16", "kind": "prefill", "dtype": "fp16", "hq": 16, "hkv": 8, "seqs": 1,
         "q_lo": 333, "q_hi": 333, "prefix_lo": 0, "prefix_hi": 0, "lengths": 0},
        # A 512-token chunk late in a long prompt.
        {"name": "prefill_chunk_512_over_7k", "kind": "prefill", "dtype": "bf16", "hq": 32, "hkv": 8, "seqs": 1,
         "q_lo": 512, "q_hi": 512, "prefix_lo": 7168, "prefix_hi": 7168, "lengths": 0},
        # The benchmark's batch of prompts with cached prefixes.
        {"name": "prefill_16seq_prefix", "kind": "prefill", "dtype": "bf16", "hq": 32, "hkv": 8, "seqs": 16,
         "q_lo": 64, "q_hi": 2048, "prefix_lo": 0, "prefix_hi": 1024, "lengths": 2},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choices(("decode", "prefill", "write", "read"), (40, 30, 15, 15))[0]
    hq, hkv = rng.choice(HEADS)
    case = {"kind": kind, "dtype": rng.choice(("bf16", "bf16", "fp16")), "hkv": hkv}
    if kind != "read":
        case["hq"] = hq
    if kind in ("write", "read"):
        case["tokens"] = _log_int(rng, 1, 16384 if kind == "write" else 30001)
        case["run"] = rng.choice((1, _log_int(rng, 1, case["tokens"]), case["tokens"]))
        return case
    case["lengths"] = rng.randrange(1 << 16)
    if kind == "decode":
        case["batch"] = _log_int(rng, 1, 256)
        hi = _log_int(rng, 1, 32768)
        case["ctx_hi"] = max(1, min(hi, MAX_DECODE_ROWS // hkv // case["batch"]))
        case["ctx_lo"] = max(1, case["ctx_hi"] // rng.choice((1, 2, 4, 16)))
        return case
    case["seqs"] = _log_int(rng, 1, 24)
    case["q_hi"] = _log_int(rng, 1, 6000)
    case["q_lo"] = max(1, case["q_hi"] // rng.choice((1, 2, 8, 32)))
    case["prefix_hi"] = rng.choice((0, _log_int(rng, 16, 8192), _log_int(rng, 16, 16384)))
    case["prefix_lo"] = rng.choice((0, case["prefix_hi"]))
    while (work(case)["flops"] > MAX_PREFILL_FLOPS or case["seqs"] * hq * case["q_hi"] *
           (case["q_hi"] + case["prefix_hi"]) > MAX_PREFILL_SCORES):
        case["q_hi"] = max(1, case["q_hi"] * 3 // 4)
        case["q_lo"] = min(case["q_lo"], case["q_hi"])
        case["prefix_hi"] = case["prefix_hi"] * 7 // 8
        case["prefix_lo"] = min(case["prefix_lo"], case["prefix_hi"])
    return case


def _lengths(case):
    """(query lengths, context lengths) of an attention case."""
    rng = np.random.default_rng(case["lengths"])

    def uniform(lo, hi, n):
        return [int(x) for x in rng.integers(lo, hi + 1, size=n)]

    if case["kind"] == "decode":
        ctx = uniform(case["ctx_lo"], case["ctx_hi"], case["batch"])
        return [1] * len(ctx), ctx
    q = uniform(case["q_lo"], case["q_hi"], case["seqs"])
    # Cached prefixes are whole pages.
    prefix = [PAGE * x for x in uniform(case["prefix_lo"] // PAGE, case["prefix_hi"] // PAGE, case["seqs"])]
    return q, [a + b for a, b in zip(q, prefix)]


# ---- the plain form ------------------------------------------------------------


def _power(byte):
    """2 ** (byte - 127) in fp32, NaN for 255."""
    power = torch.ldexp(torch.ones((), dtype=torch.float32, device=byte.device), byte.to(torch.int32) - 127)
    return torch.where(byte == 255, torch.full_like(power, math.nan), power)


def _quantise(x, max_byte):
    """(codes ``uint8 [..., 128]``, scale bytes ``uint8 [..., 4]``) of rows.

    The scale is the smallest power of two with amax <= 7 * scale, so that no
    element is rounded by more than the last step's half, 1 * scale."""
    groups = x.float().unflatten(-1, (SCALES, GROUP))
    size = groups.abs()
    amax = size.amax(-1)
    # The exponent of amax, one more where its mantissa is above 1.75; 6 and 7
    # lie two binades above 1.
    byte = (((amax.view(torch.int32) + 0x1FFFFF) >> 23) - 2).clamp(0, max_byte)
    bad = ~torch.isfinite(amax)
    byte = torch.where(bad, torch.full_like(byte, 255), byte)
    up = torch.ldexp(torch.ones_like(amax), 127 - byte.clamp(max=max_byte))
    size = torch.where(bad[..., None], torch.zeros_like(size), size * up[..., None])
    # Nearest, halfway to the even code.
    code = ((size > 0.25).to(torch.uint8) + (size >= 0.75) + (size > 1.25) + (size >= 1.75) + (size > 2.5)
            + (size >= 3.5) + (size > 5.0))
    sign = (torch.signbit(groups) & ~bad[..., None]).to(torch.uint8)
    return (code + 8 * sign).to(torch.uint8).flatten(-2), byte.to(torch.uint8)


def _pairs(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _dequantise(elements, scales):
    """fp32 rows ``[..., 128]`` of packed elements ``[..., 64]`` and scales ``[..., 4]``."""
    size = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=elements.device)
    value = torch.cat((size, -size))
    table = torch.stack((value.repeat(16), value.repeat_interleave(16)), -1)  # of a byte's two codes
    rows = torch.nn.functional.embedding(elements.to(torch.int32), table).flatten(-2)
    return rows.unflatten(-1, (SCALES, GROUP)).mul_(_power(scales)[..., None]).flatten(-2)


def _parts(cache):
    """A cache's elements ``[P, H, 16, 64]`` and scales ``[P, H, 16, 4]``, as views."""
    return (cache[..., : PAGE * ROW].unflatten(-1, (PAGE, ROW)),
            cache[..., PAGE * ROW:].unflatten(-1, (PAGE, SCALES)))


def _plain_write(s):
    slots = s["slots"].long()
    pages, offsets = slots // PAGE, slots % PAGE
    for rows, cache in ((s["k"], s["k_cache"]), (s["v"], s["v_cache"])):
        codes, scales = _quantise(rows, MAX_SCALE[s["case"]["dtype"]])
        elements, held = _parts(cache)
        elements[pages, :, offsets] = _pairs(codes)
        held[pages, :, offsets] = scales


def _plain_read(s):
    slots = s["slots"].long()
    pages, offsets = slots // PAGE, slots % PAGE
    dtype = DTYPES[s["case"]["dtype"]]

    def rows(cache):
        elements, scales = _parts(cache)
        return _dequantise(elements[pages, :, offsets], scales[pages, :, offsets]).to(dtype)

    return [rows(s["k_cache"]), rows(s["v_cache"])]


def _plain_attention(s):
    """Causal attention of every sequence over its pages, padded to the longest."""
    case = s["case"]
    hq, hkv = case["hq"], case["hkv"]
    group = hq // hkv
    starts, kv_len = s["query_start_loc"].long(), s["seq_lens"].long()
    q_len = starts[1:] - starts[:-1]
    seqs, longest = len(kv_len), s["longest_query"]
    pages = s["block_tables"].long().clamp_min(0)

    def gathered(cache):
        elements, scales = _parts(cache[pages])  # [S, W, H, 16, .]
        rows = _dequantise(elements.transpose(1, 2).flatten(2, 3), scales.transpose(1, 2).flatten(2, 3))
        return rows  # [S, H, W * 16, 128]

    place = torch.arange(longest, device="cuda")
    real = place[None, :] < q_len[:, None]
    at = (starts[:-1, None] + place).clamp_max(s["q"].shape[0] - 1)
    q = s["q"][at].float().view(seqs, longest, hkv, group, DIM).permute(0, 2, 3, 1, 4)
    q = q.reshape(seqs, hkv, group * longest, DIM)
    scores = torch.matmul(q, gathered(s["k_cache"]).transpose(-1, -2).contiguous()).mul_(1 / math.sqrt(DIM))
    last = (kv_len - q_len)[:, None] + place  # a query's own position
    hidden = torch.arange(scores.shape[-1], device="cuda") > last[:, :, None]
    scores = scores.view(seqs, hkv, group, longest, -1).masked_fill_(hidden[:, None, None], -math.inf)
    scores = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    scores = scores.div_(scores.sum(-1, keepdim=True)).view(seqs, hkv, group * longest, -1)
    out = torch.matmul(scores, gathered(s["v_cache"])).view(seqs, hkv, group, longest, DIM)
    out = out.permute(0, 3, 1, 2, 4).reshape(seqs, longest, hq, DIM)
    return out[real].to(s["q"].dtype)


# ---- inputs --------------------------------------------------------------------


def _generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _rows(gen, dtype, hkv, *lead):
    """K/V rows ``[*lead, hkv, 128]``: normal, with channels of unlike size."""
    channels = torch.exp(0.5 * torch.randn(hkv, DIM, generator=gen, device="cuda"))
    return (torch.randn((*lead, hkv, DIM), generator=gen, device="cuda") * channels).to(dtype)


def _cache(gen, case, pages):
    """A cache of written pages."""
    codes, scales = _quantise(_rows(gen, DTYPES[case["dtype"]], case["hkv"], pages, PAGE).transpose(1, 2),
                              MAX_SCALE[case["dtype"]])
    return torch.cat((_pairs(codes).flatten(-2), scales.flatten(-2)), -1).contiguous()


def _slots(gen, case):
    """(slots, pages): runs of ``run`` tokens over whole pages of their own, the pages permuted."""
    run, tokens = case["run"], case["tokens"]
    per_run = -(-run // PAGE)
    pages = -(-tokens // run) * per_run
    order = torch.randperm(pages, generator=gen, device="cuda")
    token = torch.arange(tokens, device="cuda")
    within = token % run
    slots = order[token // run * per_run + within // PAGE] * PAGE + within % PAGE
    return slots.to(torch.int32), pages


def _inputs(case, seed):
    gen = _generator(seed)
    dtype, hkv = DTYPES[case["dtype"]], case["hkv"]
    if case["kind"] in ("write", "read"):
        slots, pages = _slots(gen, case)
        state = {"case": case, "slots": slots, "k_cache": _cache(gen, case, pages), "v_cache": _cache(gen, case, pages)}
        if case["kind"] == "write":
            # k comes out of the rotary embedding, v is a view of the projection.
            heads = case["hq"] + 2 * hkv
            state["k"] = _rows(gen, dtype, hkv, case["tokens"])
            state["v"] = _rows(gen, dtype, heads, case["tokens"])[:, heads - hkv:]
        return state
    q_len, kv_len = _lengths(case)
    counts = [(n + PAGE - 1) // PAGE for n in kv_len]
    order = torch.randperm(sum(counts), generator=gen, device="cuda").to(torch.int32)
    used = torch.arange(max(counts), device="cuda")[None, :] < torch.tensor(counts, device="cuda")[:, None]
    table = torch.full((len(counts), max(counts)), -1, dtype=torch.int32, device="cuda")
    table[used] = order
    starts = torch.from_numpy(np.concatenate(([0], np.cumsum(q_len))).astype(np.int32)).to("cuda")
    return {
        "case": case, "longest_query": max(q_len), "query_start_loc": starts, "block_tables": table,
        "seq_lens": torch.tensor(kv_len, dtype=torch.int32, device="cuda"),
        "q": torch.randn((sum(q_len), case["hq"], DIM), generator=gen, device="cuda").to(dtype),
        "k_cache": _cache(gen, case, sum(counts)), "v_cache": _cache(gen, case, sum(counts)),
    }


def _plan(state):
    """The backend and the step's plan, which serve all layers of a model."""
    from my_vllm_amd.attention_backend import MI355XMXFP4AttentionBackend
    from my_vllm_amd.contract import CommonAttentionMetadata

    case = state["case"]
    q_len, kv_len = _lengths(case)
    counts = tuple((n + PAGE - 1) // PAGE for n in kv_len)
    prefills = len(q_len) if case["kind"] == "prefill" else 0
    decodes = len(q_len) - prefills
    common = CommonAttentionMetadata(
        num_prefill_seqs=prefills, num_decode_seqs=decodes, num_prefill_tokens=sum(q_len) - decodes,
        num_decode_tokens=decodes, query_start_loc=state["query_start_loc"], seq_lens=state["seq_lens"],
        slot_mapping=torch.full((sum(q_len),), -1, dtype=torch.int32, device="cuda"),
        block_tables=state["block_tables"], max_q_len=max(q_len), max_kv_len=max(kv_len), block_counts=counts,
        num_kv_blocks=sum(counts), num_prefill_kv_blocks=sum(counts[:prefills]), trusted=True,
    )
    backend = MI355XMXFP4AttentionBackend(case["hq"], case["hkv"], DIM, PAGE, DTYPES[case["dtype"]])
    return backend, backend.build_plan(common)


def prepare(case, seed):
    state = _inputs(case, seed)
    if own and case["kind"] in ("decode", "prefill"):
        state["backend"], state["plan"] = _plan(state)
    return state


def run(state):
    s = state
    kind = s["case"]["kind"]
    if not own:
        if kind == "write":
            _plain_write(s)
        return _plain_read(s) if kind in ("write", "read") else _plain_attention(s)
    if kind in ("write", "read"):
        from my_vllm_amd import ops

        if kind == "write":
            ops.store_kvcache_mxfp4(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"])
        return list(ops.load_kvcache_mxfp4(s["k_cache"], s["v_cache"], s["slots"], DTYPES[s["case"]["dtype"]]))
    return s["backend"].forward(s["q"], None, None, s["k_cache"], s["v_cache"], s["plan"])


def work(case):
    """Rows: each input read and each output written once, the cache's bytes
    among them.  Attention: each cached row, query, output and page id once; two
    products per visible (query, key) pair and head."""
    if case["kind"] in ("write", "read"):
        rows = 2 * case["tokens"] * case["hkv"]
        moved = 2 * DIM + ROW + SCALES  # out of the cache, and into the result
        if case["kind"] == "write":
            moved += 2 * DIM
        return {"bytes": rows * moved + 4 * case["tokens"], "flops": rows * DIM}
    q_len, kv_len = _lengths(case)
    pairs = sum(q * (n - q) + q * (q + 1) // 2 for q, n in zip(q_len, kv_len))
    moved = sum(kv_len) * 2 * case["hkv"] * (ROW + SCALES) + 2 * sum(q_len) * case["hq"] * DIM * 2
    moved += 4 * sum((n + PAGE - 1) // PAGE for n in kv_len)
    return {"bytes": moved, "flops": 4 * DIM * case["hq"] * pairs}


# ---- the definition, in 64 bits -------------------------------------------------


def _value(nibble):
    """The e2m1 value of a code: sign, two exponent bits, one mantissa bit."""
    exponent, mantissa = (nibble >> 1) & 3, (nibble & 1).double()
    size = torch.where(exponent == 0, mantissa / 2, (1 + mantissa / 2) * torch.exp2(exponent.double() - 1))
    return torch.where(nibble >= 8, -size, size)


def _exact_rows(block):
    """float64 ``[..., 16, 128]`` of page blocks ``uint8 [..., 1088]``."""
    elements = block[..., : PAGE * ROW]
    rows = torch.stack((_value(elements & 15), _value(elements >> 4)), -1).reshape(*block.shape[:-1], PAGE, DIM)
    scales = torch.exp2(block[..., PAGE * ROW:].double() - 127).reshape(*block.shape[:-1], PAGE, SCALES)
    return rows * scales.repeat_interleave(GROUP, -1)


def _exact_rounded(x, largest):
    """The value that the cache holds for each element of finite rows."""
    groups = x.double().reshape(-1, GROUP)
    amax = groups.abs().amax(-1, keepdim=True)
    # amax = m * 2 ** p with 0.5 <= m < 1: at most 7 units of 2 ** (p - 3) where m <= 0.875.
    mantissa, power = torch.frexp(amax)
    exponent = torch.clamp(power - torch.where(mantissa <= 0.875, 3, 2), min=-127, max=largest - 127)
    unit = torch.ldexp(torch.ones_like(amax), exponent)
    size = (groups / unit).abs()
    # Steps of 0.5 below 2, of 1 below 4, of 2 from there; round() takes ties to even.
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0)).double()
    size = torch.clamp(torch.round(size / step) * step, max=6.0)
    return (torch.copysign(size, groups) * unit).reshape(x.shape)


def _exact_attention(case, s):
    hkv, group = case["hkv"], case["hq"] // case["hkv"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for i, (n, kv) in enumerate(zip(*_lengths(case))):
        pages = s["block_tables"][i, : (kv + PAGE - 1) // PAGE].long()

        def rows(cache):
            return _exact_rows(cache[pages]).transpose(1, 2).reshape(-1, hkv, DIM)[:kv]

        k = rows(s["k_cache"]).permute(1, 2, 0).contiguous()
        v = rows(s["v_cache"]).permute(1, 0, 2).contiguous()
        for a in range(0, n, 256):
            b = min(a + 256, n)
            q = s["q"][first + a: first + b].double().reshape(b - a, hkv, group, DIM)
            q = q.permute(1, 2, 0, 3).reshape(hkv, group * (b - a), DIM).contiguous()
            scores = torch.matmul(q, k).view(hkv, group, b - a, kv) / math.sqrt(DIM)
            last = torch.arange(kv - n + a, kv - n + b, device="cuda")
            scores.masked_fill_(torch.arange(kv, device="cuda")[None, :] > last[:, None], -math.inf)
            part = torch.matmul(torch.softmax(scores, -1).view(hkv, -1, kv), v)
            out[first + a: first + b] = part.view(hkv, group, b - a, DIM).permute(2, 0, 1, 3).reshape(b - a, -1, DIM)
        first += n
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "write":
        return [_exact_rounded(s[name], MAX_SCALE[case["dtype"]]) for name in ("k", "v")]
    if case["kind"] == "read":
        slots = s["slots"].long()
        return [_exact_rows(s[name]).transpose(1, 2).reshape(-1, case["hkv"], DIM)[slots]
                for name in ("k_cache", "v_cache")]
    return _exact_attention(case, s)
