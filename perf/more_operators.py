"""What serving in 4-bit floating point is measured on: rows in 4 bits, the matrix product of two such matrices, the paged
cache of keys and values in 4 bits, and attention of new tokens over it.

A case is one of four kinds.

``rows``       a matrix is quantised row by row, and what its codes stand for is read back (a weight that is being loaded, the
               activations of a step, a check of what quantising loses).
``linear``     one product of a step: the tokens' rows are quantised and multiplied with a weight that was quantised when it
               was loaded.
``cache``      one layer's cache in a step: the step's keys and values (two column ranges of the fused projection's rows) are
               quantised into their slots, then rows of the cache are read back (the new ones, or whole sequences, as a
               program does that hands a cached prefix on).
``attention``  one layer's attention in a step: every sequence brings one token (decoding), a few (drafted tokens) or a portion
               of a prompt, and its tokens attend to the keys of the sequence, causally, perhaps inside a window.

A row in 4 bits, everywhere.  With a = max(max |x|, 2^-100) of the row: its exponent E is the least with a <= 2688 * 2^E (kept
as the byte E + 127; 255 for a row that holds no finite numbers); every block of 16 values has the scale
b = e4m3(max |x| of the block / (6 * 2^E)), a value the code e2m1(x / (2^E * b)), 0 where b is 0.  Both roundings go to the
nearest, ties to even.  The code stands for code * b * 2^E.  e2m1 holds 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives; a byte
holds two codes, the first in its low half.
"""

from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

FLOOR = 2.0 ** -100          # the least magnitude a row is scaled by
BLOCK = 16
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
CODES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]


# ---- the cases ----------------------------------------------------------------------------------

def _rows(name, rows, k, dtype="bfloat16"):
    return {"name": name, "kind": "rows", "rows": rows, "k": k, "dtype": dtype}


def _linear(name, rows, n, k, dtype="bfloat16"):
    return {"name": name, "kind": "linear", "rows": rows, "n": n, "k": k, "dtype": dtype}


def _cache(name, new, context=0, seqs=1, whole=False, kv_heads=8, dim=128, heads=16, page=16, dtype="bfloat16"):
    return {"name": name, "kind": "cache", "new": new, "context": context, "seqs": seqs, "whole": whole, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype}


def _attention(name, decode=0, context=0, ragged=False, draft=1, portion=0, prefix=0, heads=16, kv_heads=8, dim=128, page=16,
               window=0, dtype="bfloat16"):
    return {"name": name, "kind": "attention", "decode": decode, "context": context, "ragged": ragged, "draft": draft,
            "portion": portion, "prefix": prefix, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "window": window, "dtype": dtype}


def listed() -> list:
    return [
        # eight users decode a token each: what stands in front of each of their products
        _rows("rows_decode_8", rows=8, k=4096),
        # the up and gate projection of the benchmark's second model while it is loaded
        _rows("rows_weight", rows=24576, k=4096),
        # decoding: that projection for eight requests, and the output projection for one, unrounded
        _linear("linear_decode_8", rows=8, n=24576, k=4096),
        _linear("linear_decode_1_float32", rows=1, n=4096, k=4096, dtype="float32"),
        # a prompt's portion through the up and gate projection
        _linear("linear_prompt_2048", rows=2048, n=24576, k=4096),
        # small portions of ragged length behind cached tokens, their sequences read back whole, on the 32-bit path
        _cache("cache_whole_float32", new=33, context=1500, seqs=12, whole=True, dtype="float32"),
        # a long portion of a prompt, written and read back
        _cache("cache_prompt_8000", new=8000),
        # one user in a conversation
        _attention("attention_decode_1", decode=1, context=2048),
        # a busy server: many requests of all lengths, the larger models' head count
        _attention("attention_decode_64_ragged", decode=64, context=4096, ragged=True, heads=32),
        # a few very long contexts, which a cache in 4 bits is for
        _attention("attention_decode_4_long", decode=4, context=32000, heads=64),
        # sixteen requests with five drafted tokens each
        _attention("attention_draft_16x5", decode=16, context=1500, ragged=True, draft=5),
        # continuous batching: decoding requests beside a later portion of a long prompt
        _attention("attention_mixed_24_and_3000", decode=24, context=1500, ragged=True, portion=3000, prefix=5000, heads=32),
    ]


def _log_uniform(rng, lo: int, hi: int) -> int:
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


HEADS = [(16, 8), (16, 8), (32, 8), (64, 8), (8, 8), (12, 4), (6, 2)]
DIMS = [128, 128, 128, 64, 96]


def draw(rng) -> dict:
    kind = rng.choice(["rows", "linear", "linear", "linear", "cache", "attention", "attention", "attention", "attention"])
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    heads, kv_heads = rng.choice(HEADS)
    dim, page = rng.choice(DIMS), rng.choice([16, 16, 32, 8, 64])
    if kind == "rows":
        k = rng.choice([1024, 4096, 12288, _log_uniform(rng, 100, 12288)])
        case = _rows("", _log_uniform(rng, 1, min(24576, 50000000 // k)), k, dtype)
    elif kind == "linear":
        k = rng.choice([1024, 2048, 4096, 5120, 12288, _log_uniform(rng, 100, 12288)])
        n = rng.choice([1024, 4096, 5120, 6144, _log_uniform(rng, 100, 24576)])
        case = _linear("", _log_uniform(rng, 1, 2048), n, k, dtype)
    elif kind == "cache":
        seqs = _log_uniform(rng, 1, 32)
        new = _log_uniform(rng, 1, 4000 // seqs)
        case = _cache("", new, _log_uniform(rng, 16, 12000 // seqs), seqs, rng.random() < 0.4, kv_heads, dim, heads, page, dtype)
    else:
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
    del case["name"]
    return case


# ---- rows in 4 bits, plainly ----------------------------------------------------------------------

def _exponents(top: torch.Tensor) -> torch.Tensor:
    """E of rows whose largest magnitude is ``top``, as float32; NaN where that is no finite number."""
    share, e = torch.frexp(top.clamp(min=FLOOR))               # top = share * 2^e, share in [0.5, 1); 2688 = 0.65625 * 2^12
    e = e - 12 + (share > 0.65625)
    return torch.where(torch.isfinite(top), e.float(), math.nan)


def _power(e: torch.Tensor) -> torch.Tensor:
    return torch.where(e.isnan(), math.nan, torch.ldexp(torch.ones_like(e), e.nan_to_num().int()))


def _quantised(x: torch.Tensor):
    """Rows [.., K] in float32 -> (values of the codes [.., K], block scales [.., ceil(K / 16)], E [..])."""
    k = x.shape[-1]
    blocks = torch.nn.functional.pad(x, (0, -k % BLOCK)).unflatten(-1, (-1, BLOCK))
    tops = blocks.abs().amax(-1)
    e = _exponents(tops.amax(-1))
    down = _power(-e)[..., None]
    six = torch.full_like(tops, 6.0)                           # (by a plain number it would be a product with 1 / 6)
    scales = (tops * down / six).nan_to_num(0.0, 0.0, 0.0).to(torch.float8_e4m3fn).float()
    y = blocks * down[..., None] / scales[..., None]
    step = torch.where(y.abs() < 2.0, 0.5, torch.where(y.abs() < 4.0, 1.0, 2.0))
    y = (torch.round(y / step) * step).clamp(-6.0, 6.0)
    y = torch.where((scales == 0.0)[..., None] | e.isnan()[..., None, None], 0.0, y)
    return y.flatten(-2)[..., :k], scales, e


def _packed(x: torch.Tensor):
    """The same as it is kept: codes uint8 [.., ceil(K / 2)], block scales float8_e4m3fn, exponent bytes uint8 [..]."""
    y, scales, e = _quantised(x)
    y = torch.nn.functional.pad(y, (0, y.shape[-1] % 2))
    m = y.abs()
    code = torch.where(m < 2.0, m * 2.0, torch.where(m < 4.0, m + 2.0, m / 2.0 + 4.0)).to(torch.uint8)
    code += torch.signbit(y).to(torch.uint8) * 8
    code = code.unflatten(-1, (-1, 2))
    byte = torch.where(e.isnan(), 255.0, e + 127.0).to(torch.uint8)
    return code[..., 0] + code[..., 1] * 16, scales.to(torch.float8_e4m3fn), byte


def _values(codes: torch.Tensor, scales: torch.Tensor, exponents: torch.Tensor, k: int) -> torch.Tensor:
    """What packed rows stand for, float32 [.., K]."""
    table = torch.tensor(CODES, device=codes.device)
    y = table[torch.stack([codes & 15, codes >> 4], -1).int()].flatten(-2)[..., :k]
    e = torch.where(exponents == 255, math.nan, exponents.float() - 127.0)
    return y * scales.float().repeat_interleave(BLOCK, -1)[..., :k] * _power(e)[..., None]


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


def _pool(st, pages: int, case: dict, device_gen) -> None:
    """A cache in use: keys with a few wide channels, values; a page at a time's worth of rows is quantised."""
    hkv, page, d = case["kv_heads"], case["page"], case["dim"]
    st.data = torch.empty(pages, 2, hkv, page, d // 2, dtype=torch.uint8, device="cuda")
    st.scales = torch.empty(pages, 2, hkv, page, d // BLOCK, dtype=torch.float8_e4m3fn, device="cuda")
    st.exponents = torch.empty(pages, 2, hkv, page, dtype=torch.uint8, device="cuda")
    wide = torch.ones(2, hkv, 1, d, device="cuda")
    wide[0, :, :, ::17] = 4.0
    step = max(1, (1 << 26) // (2 * hkv * page * d))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        x = torch.randn(n, 2, hkv, page, d, device="cuda", generator=device_gen) * wide
        st.data[p:p + n], st.scales[p:p + n], st.exponents[p:p + n] = _packed(x)


def _tables(key_counts: list, page: int, gen):
    """Pages of every sequence, in no order; page 0 belongs to nobody."""
    per = [-(-n // page) for n in key_counts]
    order = (torch.randperm(sum(per), generator=gen) + 1).to(torch.int32)
    return list(order.split(per)), sum(per) + 1


def _slots(table, positions, page: int):
    return table[positions // page].long() * page + positions % page


def _activations(rows: int, k: int, dtype: str, device_gen) -> torch.Tensor:
    x = torch.randn(rows, k, device="cuda", generator=device_gen)
    x[:, ::61] *= 12.0                     # activations have a few wide channels
    return x.to(DTYPES[dtype])


def _prepare_rows(case: dict, gen, device_gen):
    st = SimpleNamespace(case=case)
    if case["rows"] > 2048:                # a weight
        st.x = torch.randn(case["rows"], case["k"], device="cuda", generator=device_gen).mul_(0.02).to(DTYPES[case["dtype"]])
    else:
        st.x = _activations(case["rows"], case["k"], case["dtype"], device_gen)
    return st


def _prepare_linear(case: dict, gen, device_gen):
    st = SimpleNamespace(case=case)
    st.x = _activations(case["rows"], case["k"], case["dtype"], device_gen)
    w = torch.randn(case["n"], case["k"], device="cuda", generator=device_gen) * 0.02
    st.codes, st.scales, st.exponents = _packed(w)
    return st


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
    _pool(st, pages, case, device_gen)
    return st


def _prepare_attention(case: dict, gen, device_gen):
    lengths = _lengths(case, gen)
    tables, pages = _tables([n for _, n in lengths], case["page"], gen)
    st = SimpleNamespace(case=case, q_lens=[a for a, _ in lengths], kv_lens=[b for _, b in lengths])
    t = sum(st.q_lens)
    st.q = torch.randn(t, case["heads"], case["dim"], device="cuda", generator=device_gen).to(DTYPES[case["dtype"]])
    st.scale, st.window = case["dim"] ** -0.5, case["window"]
    _pool(st, pages, case, device_gen)
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


_PREPARE = {"rows": _prepare_rows, "linear": _prepare_linear, "cache": _prepare_cache, "attention": _prepare_attention}


def prepare(case: dict, seed: int):
    gen = torch.Generator().manual_seed(seed)
    device_gen = torch.Generator("cuda").manual_seed(seed)
    st = _PREPARE[case["kind"]](case, gen, device_gen)
    if own:
        from deterministic_inference_b200.engine.batch import AttentionMeta
        from deterministic_inference_b200.kernels import ops
        st.ops = ops
        if case["kind"] == "linear":
            st.weight = ops.Fp4Weight(st.codes, st.scales, st.exponents, case["k"])
        elif case["kind"] != "rows":
            st.cache = ops.Fp4Cache(st.data, st.scales, st.exponents)
        if case["kind"] == "attention":
            st.meta = AttentionMeta(
                block_table=st.table, slot_mapping=torch.zeros_like(st.token_seq), token_seq=st.token_seq,
                positions=st.positions, cu_q_lens=st.cu, seq_lens=st.lens, q_lens=st.q_lens, kv_lens=st.kv_lens,
                num_decode=sum(1 for n in st.q_lens if n == 1))
    return st


# ---- one pass ---------------------------------------------------------------------------------------

def _plain_rows(st):
    return _values(*_packed(st.x.float()), st.case["k"]).to(st.x.dtype)


def _plain_linear(st):
    y, scales, e = _quantised(st.x.float())
    k = st.case["k"]
    x = y * scales.repeat_interleave(BLOCK, -1)[..., :k] * _power(e)[..., None]
    return (x @ _values(st.codes, st.scales, st.exponents, k).t()).to(st.x.dtype)


def _plain_cache(st):
    page, d = st.case["page"], st.case["dim"]
    at = st.write.long()
    for kv, x in ((0, st.k), (1, st.v)):
        to = (at // page, kv, slice(None), at % page)
        st.data[to], st.scales[to], st.exponents[to] = _packed(x.float())
    at = st.read.long()
    out = []
    for kv in (0, 1):
        of = (at // page, kv, slice(None), at % page)
        out.append(_values(st.data[of], st.scales[of], st.exponents[of], d).to(st.k.dtype))
    return out


ROWS_AT_ONCE = 1 << 28        # scores held at a time


def _plain_attention(st):
    out = torch.zeros_like(st.q)
    hq, hkv, d, page = st.case["heads"], st.case["kv_heads"], st.case["dim"], st.case["page"]
    start = 0
    for b, (n, keys) in enumerate(zip(st.q_lens, st.kv_lens)):
        pages = st.table[b, :-(-keys // page)].long()
        rows = _values(st.data[pages], st.scales[pages], st.exponents[pages], d)               # [pages, 2, Hkv, page, D]
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


_PLAIN = {"rows": _plain_rows, "linear": _plain_linear, "cache": _plain_cache, "attention": _plain_attention}


@torch.inference_mode()
def run(st):
    kind = st.case["kind"]
    if not own:
        return _PLAIN[kind](st)
    if kind == "rows":
        return st.ops.fp4_quantize_rows(st.x).tensor(st.x.dtype)
    if kind == "linear":
        return st.ops.fp4_linear(st.x, st.weight)
    if kind == "cache":
        st.ops.fp4_cache_write(st.k, st.v, st.cache, st.write)
        return list(st.ops.fp4_cache_read(st.cache, st.read, st.k.dtype))
    return st.ops.fp4_paged_attention(st.q, st.cache, st.meta, st.scale, st.window or None)


# ---- what a pass cannot do without --------------------------------------------------------------------

def work(case: dict) -> dict:
    size = 2 if case["dtype"] == "bfloat16" else 4
    held = lambda k: -(-k // 2) + -(-k // BLOCK) + 1          # bytes of a row of k values in 4 bits
    if case["kind"] == "rows":
        m, k = case["rows"], case["k"]
        return {"bytes": 2 * m * (k * size + held(k)), "flops": 6 * m * k}
    if case["kind"] == "linear":
        m, n, k = case["rows"], case["n"], case["k"]
        return {"bytes": m * k * size + n * held(k) + m * n * size, "flops": 2 * m * n * k}
    hkv, d = case["kv_heads"], case["dim"]
    if case["kind"] == "cache":
        new = case["seqs"] * case["new"]
        read = case["seqs"] * (case["new"] + (case["context"] if case["whole"] else 0))
        return {"bytes": 2 * hkv * (new + read) * (d * size + held(d)) + 4 * (new + read),
                "flops": 2 * hkv * d * (4 * new + 2 * read)}
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
    return {"bytes": int(2 * tokens * case["heads"] * d * size + 2 * hkv * keys * held(d)),
            "flops": int(4 * case["heads"] * d * pairs)}


# ---- the definition in 64 bits --------------------------------------------------------------------------

def _nearest(x: torch.Tensor, least_exponent: int, digits: int, largest: float) -> torch.Tensor:
    """The nearest number of a small floating-point format with ``digits`` binary digits behind the point, ties to even."""
    exponent = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** least_exponent)))
    unit = torch.exp2(exponent - digits)
    return (torch.round(x / unit) * unit).clamp(min=-largest, max=largest)


def _rounded64(x: torch.Tensor) -> torch.Tensor:
    """The values that the rows' codes stand for, from the rule."""
    x = x.double()
    k = x.shape[-1]
    top = x.abs().max(dim=-1, keepdim=True).values.clamp(min=FLOOR)
    unit = torch.exp2(torch.ceil(torch.log2(top / 2688.0)))
    parts = []
    for at in range(0, k, BLOCK):
        part = x[..., at:at + BLOCK]
        scale = _nearest(part.abs().max(dim=-1, keepdim=True).values / (6.0 * unit), -6, 3, 448.0) * unit
        codes = _nearest(part / torch.where(scale > 0, scale, 1.0), 0, 1, 6.0)
        parts.append(codes * scale)
    return torch.cat(parts, dim=-1)


def _held64(codes, scales, exponents, k: int) -> torch.Tensor:
    """What kept rows stand for."""
    halves = torch.stack([torch.remainder(codes, 16), torch.div(codes, 16, rounding_mode="floor")], dim=-1).flatten(-2).double()
    sign = torch.where(halves >= 8, -1.0, 1.0).double()
    code = torch.remainder(halves, 8)
    e = torch.clamp(torch.div(code, 2, rounding_mode="floor"), min=1.0)
    m = torch.where(code < 2, code / 2, 1 + torch.remainder(code, 2) / 2)      # (0 and 0.5 have no leading one)
    number = (sign * m * torch.exp2(e - 1))[..., :k]
    block = torch.arange(k, device=codes.device) // BLOCK
    return number * scales.double()[..., block] * torch.exp2(exponents.double() - 127).unsqueeze(-1)


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
        query_pos = torch.arange(first, length, device="cuda").unsqueeze(1)
        hidden = place.unsqueeze(0) > query_pos
        if case["window"]:
            hidden = hidden | (query_pos - place.unsqueeze(0) >= case["window"])
        heads = []
        for g in range(case["kv_heads"]):
            key, value = (_held64(st.data[page_of, i, g, row], st.scales[page_of, i, g, row], st.exponents[page_of, i, g, row],
                                  case["dim"]) for i in (0, 1))
            for h in range(g * group, (g + 1) * group):
                logits = torch.mm(q[:, h], key.t()) * st.scale
                heads.append(torch.softmax(logits.masked_fill(hidden, -math.inf), dim=1).mm(value))
        result.append(torch.stack(heads, dim=1))
        at += n
    return torch.cat(result)


@torch.inference_mode()
def exact(case: dict, seed: int):
    gen, device_gen = torch.Generator().manual_seed(seed), torch.Generator("cuda").manual_seed(seed)
    st = _PREPARE[case["kind"]](case, gen, device_gen)
    if case["kind"] == "rows":
        return _rounded64(st.x)
    if case["kind"] == "linear":
        return torch.mm(_rounded64(st.x), _held64(st.codes, st.scales, st.exponents, case["k"]).t())
    if case["kind"] == "attention":
        return _exact_attention(st)
    # what the cache stands for, a row a slot
    d, hkv = case["dim"], case["kv_heads"]
    kept = lambda t: t.movedim(3, 1).flatten(0, 1)
    rows = _held64(kept(st.data)[st.read.long()], kept(st.scales)[st.read.long()], kept(st.exponents)[st.read.long()], d)
    place = torch.full((st.data.shape[0] * case["page"],), -1, dtype=torch.long, device="cuda")
    place[st.write.long()] = torch.arange(st.write.numel(), device="cuda")
    new = place[st.read.long()]
    fresh = torch.stack([_rounded64(st.k), _rounded64(st.v)], dim=1)
    rows = torch.where((new >= 0)[:, None, None, None], fresh[new.clamp(min=0)], rows)
    return [rows[:, 0], rows[:, 1]]
