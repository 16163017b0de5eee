"""What serving in 8-bit integers is measured on: the paged cache with a scale for each token and head, attention of new
tokens over it, and the matrix product with scales for each token and channel.

A case is one of three kinds.

``cache``      one layer's cache in a step: the step's keys and values (two column ranges of the fused projection's rows)
               are quantised into their slots, then rows of the cache are read back (the new ones, or whole sequences, as
               a program does that hands a cached prefix on).
``attention``  one layer's attention in a step: every sequence brings one token (decoding), a few (drafted tokens) or a
               portion of a prompt, and its tokens attend to the keys of the sequence, causally, perhaps inside a window.
``linear``     one product of a step: the tokens' rows are quantised, each with a scale of its own, and multiplied with a
               weight that was quantised when it was loaded.

Row quantisation, everywhere: with a = max(max |x|, 2^-100) of the row, code = rint(x * (127 / a)), scale = a / 127.
"""

from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

FLOOR = 2.0 ** -100          # the least magnitude a row is scaled by
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ---- the cases ----------------------------------------------------------------------------------

def _cache(name, new, context=0, seqs=1, whole=False, kv_heads=8, dim=128, heads=16, page=16, dtype="bfloat16"):
    return {"name": name, "kind": "cache", "new": new, "context": context, "seqs": seqs, "whole": whole, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype}


def _attention(name, decode=0, context=0, ragged=False, draft=1, portion=0, prefix=0, heads=16, kv_heads=8, dim=128, page=16,
               window=0, dtype="bfloat16"):
    return {"name": name, "kind": "attention", "decode": decode, "context": context, "ragged": ragged, "draft": draft,
            "portion": portion, "prefix": prefix, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "window": window, "dtype": dtype}


def _linear(name, rows, n, k, dtype="bfloat16"):
    return {"name": name, "kind": "linear", "rows": rows, "n": n, "k": k, "dtype": dtype}


def listed() -> list:
    return [
        # eight users decode a token each: the latency of a step's smallest piece of work
        _cache("cache_decode_8", new=1, context=2048, seqs=8),
        # a long portion of a prompt, written and read back
        _cache("cache_prompt_8000", new=8000),
        # the 32-bit path: small portions of ragged length behind cached tokens, the sequences read back whole
        _cache("cache_whole_float32", new=33, context=1500, seqs=12, whole=True, dtype="float32"),
        # one user in a conversation
        _attention("attention_decode_1", decode=1, context=2048),
        # a busy server: many requests of all lengths, the larger models' head count
        _attention("attention_decode_64_ragged", decode=64, context=4096, ragged=True, heads=32),
        # a few very long contexts
        _attention("attention_decode_4_long", decode=4, context=32000, heads=64),
        # sixteen requests with five drafted tokens each
        _attention("attention_draft_16x5", decode=16, context=1500, ragged=True, draft=5),
        # the benchmark's prompt
        _attention("attention_prompt_2048", portion=2048, heads=32),
        # continuous batching: decoding requests beside a later portion of a long prompt
        _attention("attention_mixed_24_and_3000", decode=24, context=1500, ragged=True, portion=3000, prefix=5000, heads=32),
        # decoding: the up and gate projection of the benchmark's second model for eight requests, and its output
        # projection for one, unrounded
        _linear("linear_decode_8", rows=8, n=24576, k=4096),
        _linear("linear_decode_1_float32", rows=1, n=4096, k=4096, dtype="float32"),
        # a prompt's portion through the up and gate projection
        _linear("linear_prompt_2048", rows=2048, n=24576, k=4096),
    ]


def _log_uniform(rng, lo: int, hi: int) -> int:
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


HEADS = [(16, 8), (16, 8), (32, 8), (64, 8), (8, 8), (12, 4), (6, 2)]
DIMS = [128, 128, 128, 64, 96]


def draw(rng) -> dict:
    kind = rng.choice(["cache", "attention", "attention", "attention", "attention", "linear", "linear", "linear"])
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    heads, kv_heads = rng.choice(HEADS)
    dim, page = rng.choice(DIMS), rng.choice([16, 16, 32, 8, 64])
    if kind == "cache":
        seqs = _log_uniform(rng, 1, 32)
        new = _log_uniform(rng, 1, 4000 // seqs)
        case = _cache("", new, _log_uniform(rng, 16, 12000 // seqs), seqs, rng.random() < 0.4, kv_heads, dim, heads, page, dtype)
    elif kind == "attention":
        case = _attention("", heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype)
        how = rng.choice(["decode", "decode", "draft", "prompt", "mixed"])
        if how != "prompt":
            case["decode"] = _log_uniform(rng, 1, 64 if how != "mixed" else 24)
            case["context"] = _log_uniform(rng, 16, min(32000, 120000 // case["decode"]) if how == "decode" else 4000)
            case["ragged"] = rng.random() < 0.7
        if how == "draft":
            case["draft"] = rng.randrange(2, 9)
        if how in ("prompt", "mixed"):
            case["portion"] = _log_uniform(rng, 9, 1500 if dtype == "float32" else 2500)
            case["prefix"] = rng.choice([0, _log_uniform(rng, 16, 2000 if dtype == "float32" else 5000)])
        if rng.random() < 0.25:
            case["window"] = _log_uniform(rng, 32, 4096)
    else:
        k = rng.choice([1024, 2048, 4096, 5120, 12288, _log_uniform(rng, 100, 12288)])
        n = rng.choice([1024, 4096, 5120, 6144, _log_uniform(rng, 100, 24576)])
        case = _linear("", _log_uniform(rng, 1, 2048), n, k, dtype)
    del case["name"]
    return case


# ---- what a program has in hand -------------------------------------------------------------------

def _lengths(case: dict, gen) -> list:
    """(new tokens, keys after the step) of every sequence; those with one new token come first, as in a step."""
    out = []
    for _ in range(case["decode"]):
        n = case["context"]
        if case["ragged"]:
            n = int(torch.randint(max(1, n // 8), n + 1, (1,), generator=gen))
        out.append((case["draft"], max(n, case["draft"])))
    if case["portion"]:
        out.append((case["portion"], case["prefix"] + case["portion"]))
    return sorted(out, key=lambda x: x[0] != 1)


def _codes(rows: torch.Tensor):
    a = rows.abs().amax(-1).clamp(min=FLOOR)
    return torch.round(rows * (127.0 / a)[..., None]).to(torch.int8), a / 127.0


def _pool(pages: int, case: dict, device_gen):
    """A cache in use: keys with a few wide channels, values; a page at a time's worth of rows is quantised."""
    hkv, page, d = case["kv_heads"], case["page"], case["dim"]
    data = torch.empty(pages, 2, hkv, page, d, dtype=torch.int8, device="cuda")
    scales = torch.empty(pages, 2, hkv, page, dtype=torch.float32, device="cuda")
    wide = torch.ones(2, hkv, 1, d, device="cuda")
    wide[0, :, :, ::17] = 4.0
    step = max(1, (1 << 26) // (2 * hkv * page * d))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        x = torch.randn(n, 2, hkv, page, d, device="cuda", generator=device_gen) * wide
        data[p:p + n], scales[p:p + n] = _codes(x)
    return data, scales


def _tables(key_counts: list, page: int, gen):
    """Pages of every sequence, in no order; page 0 belongs to nobody."""
    per = [-(-n // page) for n in key_counts]
    order = (torch.randperm(sum(per), generator=gen) + 1).to(torch.int32)
    return list(order.split(per)), sum(per) + 1


def _slots(table, positions, page: int):
    return table[positions // page].long() * page + positions % page


def _prepare_cache(case: dict, gen, device_gen):
    lengths = [(case["new"], case["context"] + case["new"])] * case["seqs"]
    tables, pages = _tables([n for _, n in lengths], case["page"], gen)
    write, read = [], []
    for table, (new, n) in zip(tables, lengths):
        write.append(_slots(table, torch.arange(n - new, n), case["page"]))
        read.append(_slots(table, torch.arange(0 if case["whole"] else n - new, n), case["page"]))
    st = SimpleNamespace(case=case)
    st.write, st.read = torch.cat(write).to("cuda", torch.int32), torch.cat(read).to("cuda", torch.int32)
    t, d, hq, hkv = st.write.numel(), case["dim"], case["heads"], case["kv_heads"]
    qkv = torch.randn(t, (hq + 2 * hkv) * d, device="cuda", generator=device_gen).to(DTYPES[case["dtype"]])
    st.k = qkv[:, hq * d:(hq + hkv) * d].view(t, hkv, d)
    st.v = qkv[:, (hq + hkv) * d:].view(t, hkv, d)
    st.data, st.scales = _pool(pages, case, device_gen)
    return st


def _prepare_attention(case: dict, gen, device_gen):
    lengths = _lengths(case, gen)
    tables, pages = _tables([n for _, n in lengths], case["page"], gen)
    st = SimpleNamespace(case=case, q_lens=[a for a, _ in lengths], kv_lens=[b for _, b in lengths])
    t = sum(st.q_lens)
    st.q = torch.randn(t, case["heads"], case["dim"], device="cuda", generator=device_gen).to(DTYPES[case["dtype"]])
    st.scale, st.window = case["dim"] ** -0.5, case["window"]
    st.data, st.scales = _pool(pages, case, device_gen)
    st.table = torch.zeros(len(lengths), max(x.numel() for x in tables), dtype=torch.int32)
    for i, x in enumerate(tables):
        st.table[i, :x.numel()] = x
    st.table = st.table.cuda()
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    st.cu = ints([0] + torch.tensor(st.q_lens).cumsum(0).tolist())
    st.lens = ints(st.kv_lens)
    st.token_seq = torch.repeat_interleave(torch.arange(len(lengths), dtype=torch.int32, device="cuda"),
                                           torch.tensor(st.q_lens, device="cuda"))
    st.positions = torch.cat([torch.arange(n - q, n, dtype=torch.int32) for q, n in lengths]).cuda()
    return st


def _prepare_linear(case: dict, gen, device_gen):
    st = SimpleNamespace(case=case)
    x = torch.randn(case["rows"], case["k"], device="cuda", generator=device_gen)
    x[:, ::61] *= 12.0                     # activations have a few wide channels
    st.x = x.to(DTYPES[case["dtype"]])
    w = torch.randn(case["n"], case["k"], device="cuda", generator=device_gen) * 0.02
    st.codes, st.scales = _codes(w)
    return st


def prepare(case: dict, seed: int):
    gen = torch.Generator().manual_seed(seed)
    device_gen = torch.Generator("cuda").manual_seed(seed)
    st = {"cache": _prepare_cache, "attention": _prepare_attention, "linear": _prepare_linear}[case["kind"]](
        case, gen, device_gen)
    if own:
        from deterministic_inference_b200.engine.batch import AttentionMeta
        from deterministic_inference_b200.kernels import ops
        st.ops = ops
        if case["kind"] == "linear":
            st.weight = ops.Int8Weight(st.codes, st.scales)
        else:
            st.cache = ops.Int8Cache(st.data, st.scales)
        if case["kind"] == "attention":
            st.meta = AttentionMeta(
                block_table=st.table, slot_mapping=torch.zeros_like(st.token_seq), token_seq=st.token_seq,
                positions=st.positions, cu_q_lens=st.cu, seq_lens=st.lens, q_lens=st.q_lens, kv_lens=st.kv_lens,
                num_decode=sum(1 for n in st.q_lens if n == 1))
    return st


# ---- one pass ---------------------------------------------------------------------------------------

def _plain_cache(st):
    page = st.case["page"]
    at = st.write.long()
    for kv, x in ((0, st.k), (1, st.v)):
        st.data[at // page, kv, :, at % page], st.scales[at // page, kv, :, at % page] = _codes(x.float())
    at = st.read.long()
    rows = [st.data[at // page, kv, :, at % page].float() * st.scales[at // page, kv, :, at % page][..., None]
            for kv in (0, 1)]
    return [x.to(st.k.dtype) for x in rows]


ROWS_AT_ONCE = 1 << 28        # scores held at a time


def _plain_attention(st):
    out = torch.zeros_like(st.q)
    hq, hkv, d, page = st.case["heads"], st.case["kv_heads"], st.case["dim"], st.case["page"]
    start = 0
    for b, (n, keys) in enumerate(zip(st.q_lens, st.kv_lens)):
        pages = st.table[b, :-(-keys // page)].long()
        rows = st.data[pages].float() * st.scales[pages][..., None]                     # [pages, 2, Hkv, page, D]
        k, v = rows.permute(1, 2, 0, 3, 4).reshape(2, hkv, -1, d)[:, :, :keys]
        at = torch.arange(keys, device="cuda")
        step = max(1, ROWS_AT_ONCE // (hq * keys))
        for r in range(0, n, step):
            m = min(step, n - r)
            q = st.q[start + r:start + r + m].float().view(m, hkv, hq // hkv, d).permute(1, 2, 0, 3).reshape(hkv, -1, d)
            s = (q @ k.transpose(1, 2)).view(hkv, hq // hkv, m, keys) * st.scale
            pos = st.positions[start + r:start + r + m, None]
            seen = at <= pos
            if st.window:
                seen &= at > pos - st.window
            s = s.masked_fill(~seen, -math.inf)
            p = torch.exp(s - s.amax(-1, keepdim=True))
            o = p.view(hkv, -1, keys) @ v / p.sum(-1).view(hkv, -1, 1)
            out[start + r:start + r + m] = o.view(hkv, hq // hkv, m, d).permute(2, 0, 1, 3).reshape(m, hq, d).to(out.dtype)
        start += n
    return out


def _plain_linear(st):
    codes, scales = _codes(st.x.float())
    y = codes.float() @ st.codes.float().t()
    return (y * scales[:, None] * st.scales).to(st.x.dtype)


@torch.inference_mode()
def run(st):
    kind = st.case["kind"]
    if not own:
        return {"cache": _plain_cache, "attention": _plain_attention, "linear": _plain_linear}[kind](st)
    if kind == "cache":
        st.ops.int8_cache_write(st.k, st.v, st.cache, st.write)
        return list(st.ops.int8_cache_read(st.cache, st.read, st.k.dtype))
    if kind == "attention":
        return st.ops.int8_paged_attention(st.q, st.cache, st.meta, st.scale, st.window or None)
    return st.ops.int8_linear(st.x, st.weight)


# ---- what a pass cannot do without --------------------------------------------------------------------

def work(case: dict) -> dict:
    size = 2 if case["dtype"] == "bfloat16" else 4
    if case["kind"] == "linear":
        m, n, k = case["rows"], case["n"], case["k"]
        return {"bytes": m * k * size + n * (k + 4) + m * n * size, "flops": 2 * m * n * k}
    hkv, d = case["kv_heads"], case["dim"]
    if case["kind"] == "cache":
        new = case["seqs"] * case["new"]
        read = case["seqs"] * (case["new"] + (case["context"] if case["whole"] else 0))
        return {"bytes": 2 * hkv * (new + read) * (d * size + d + 4) + 4 * (new + read),
                "flops": 2 * hkv * d * (3 * new + read)}
    tokens = keys = pairs = 0
    for _ in range(case["decode"]):          # of a ragged step, its mean length
        n = case["context"] * (9 / 16 if case["ragged"] else 1)
        seen = min(n, case["window"] + case["draft"] - 1) if case["window"] else n
        tokens, keys = tokens + case["draft"], keys + seen
        pairs += case["draft"] * (min(n, case["window"]) if case["window"] else n)
    if case["portion"]:
        n, p, w = case["portion"], case["prefix"], case["window"] or case["portion"] + case["prefix"]
        tokens, keys = tokens + n, keys + min(n + p, w + n - 1)
        short = max(0, min(n, w - p))        # rows whose window reaches back to the first key
        pairs += short * p + short * (short + 1) / 2 + (n - short) * w
    return {"bytes": int(2 * tokens * case["heads"] * d * size + 2 * hkv * keys * (d + 4)),
            "flops": int(4 * case["heads"] * d * pairs)}


# ---- the definition in 64 bits --------------------------------------------------------------------------

def _rounded64(x: torch.Tensor) -> torch.Tensor:
    """The values that the codes of the last axis' rows stand for."""
    x = x.double()
    unit = torch.clamp(x.abs().max(dim=-1, keepdim=True).values, min=FLOOR) / 127
    return torch.round(x / unit) * unit


def _exact_attention(st):
    case, result = st.case, []
    page, group = case["page"], case["heads"] // case["kv_heads"]
    at = 0
    for b in range(len(st.q_lens)):
        n, length = st.q_lens[b], st.kv_lens[b]
        place = torch.arange(length, device="cuda")
        page_of, row = st.table[b].long()[place // page], place % page
        first = length - n
        q = st.q[at:at + n].double()
        heads = []
        for h in range(case["heads"]):
            g = h // group
            key = st.data[page_of, 0, g, row].double() * st.scales[page_of, 0, g, row, None].double()
            value = st.data[page_of, 1, g, row].double() * st.scales[page_of, 1, g, row, None].double()
            logits = torch.mm(q[:, h], key.t()) * st.scale
            query_pos = torch.arange(first, length, device="cuda").unsqueeze(1)
            hidden = place.unsqueeze(0) > query_pos
            if case["window"]:
                hidden = hidden | (query_pos - place.unsqueeze(0) >= case["window"])
            heads.append(torch.softmax(logits.masked_fill(hidden, -math.inf), dim=1).mm(value))
        result.append(torch.stack(heads, dim=1))
        at += n
    return torch.cat(result)


@torch.inference_mode()
def exact(case: dict, seed: int):
    gen, device_gen = torch.Generator().manual_seed(seed), torch.Generator("cuda").manual_seed(seed)
    if case["kind"] == "linear":
        st = _prepare_linear(case, gen, device_gen)
        return torch.mm(_rounded64(st.x), (st.codes.double() * st.scales.double()[:, None]).t())
    if case["kind"] == "attention":
        return _exact_attention(_prepare_attention(case, gen, device_gen))
    st = _prepare_cache(case, gen, device_gen)
    values = st.data.double() * st.scales.double().unsqueeze(-1)          # what the cache stands for
    by_slot = values.permute(0, 3, 1, 2, 4).reshape(-1, 2, case["kv_heads"], case["dim"])
    by_slot[st.write.long()] = torch.stack([_rounded64(st.k), _rounded64(st.v)], dim=1)
    rows = by_slot[st.read.long()]
    return [rows[:, 0], rows[:, 1]]
