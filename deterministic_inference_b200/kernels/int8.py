"""Serving in 8-bit integers: weights and activations with a scale for each output channel and each token, and a paged
cache of keys and values with a scale for each token and head.  ``ops`` exports what is here.

One rule quantises every row (a token's activations, an output channel of a weight, a token's key or value of one head):

    a = max(max |x|, 2^-100),  code = rint(x * (127 * (1 / a))) (ties to even),  scale = a * (1 / 127),  value = scale * code

in float32, whatever the row's type.  A row that holds an infinity or a NaN has the scale NaN and reads back as NaN.

``Int8Weight``          a weight [N, K], quantised once (``Int8Weight.of``) or given as codes and scales
``quantize_rows``       activations [M, K] -> ``Int8Rows``; ``int8_linear`` takes either
``int8_linear``         y = x @ weight^T: an exact 32-bit sum of products of codes, times the two scales
``Int8Cache``           the cache of one layer: data int8 [pages, 2, Hkv, page_size, D], scales float32 [.., page_size]
``int8_cache_write``    keys and values into their slots
``int8_qk_norm_rope_cache``  the same from the fused projection's rows, q and k normed and rotated on the way
``int8_cache_read``     what the rows of given slots stand for
``int8_paged_attention``  attention of a step's new tokens over the cache
"""

from __future__ import annotations

import ctypes
from ctypes import c_float, c_int, c_longlong, c_void_p

import torch

MAX_K = 133144          # 127^2 * K stays below 2^31
MAX_HEAD_DIM = 256


# A decoded token's operators take the GPU a few microseconds: what the host does in front of a launch is kept short.  The C
# functions are looked up once, with their argument types (pointers and numbers are passed as Python integers); an argument
# is looked at in one expression, and the check that words the error runs only where that fails.
_P, _I, _L, _F = c_void_p, c_int, c_longlong, c_float
_SIGNATURES = {
    "dib_quantize_rows": ("cache_int8", (_P, _L, _P, _P, _L, _I, _I, _P)),
    "dib_int8_cache_write": ("cache_int8", (_P, _P, _L, _L, _P, _P, _P, _I, _I, _I, _I, _L, _I, _P)),
    "dib_int8_cache_read": ("cache_int8", (_P, _P, _P, _P, _P, _I, _I, _I, _I, _L, _I, _P)),
    "dib_int8_qk_norm_rope_cache": ("cache_int8", (_P, _P, _P, _P, _P, _P, _F, _P, _I, _I, _P, _P, _I, _I, _I, _I, _I, _L, _I, _P)),
    "dib_gemm_int8": ("gemm_int8", (_P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _P)),
    "dib_int8_linear": ("gemm_int8", (_P, _P, _L, _I, _I, _P, _P, _P, _P, _I, _I, _I, _I, _P)),
    "dib_int8_attention_split": ("attention_int8", (_P, _P, _P, _P, _L, _P, _I, _P, _P, _P, _I, _I, _I, _I, _P, _P, _I, _I, _I, _I,
                                                    _I, _I, _F, _I, _I, _I, _P)),
    "dib_int8_attention_any": ("attention_int8", (_P, _P, _P, _P, _P, _I, _P, _P, _P, _I, _I, _I, _I, _I, _L, _F, _I, _I, _P)),
    "dib_int8_attention_prompt": ("attention_int8_prompt", (_P, _P, _P, _P, _L, _P, _I, _P, _P, _P, _I, _I, _P, _I, _I, _I, _P, _P,
                                                            _I, _I, _I, _I, _I, _I, _F, _I, _P)),
}
_functions: dict = {}
_ops_module = None


def _ops():
    global _ops_module
    if _ops_module is None:
        from . import ops
        _ops_module = ops
    return _ops_module


def _fn(name: str):
    fn = _functions.get(name)
    if fn is None:
        library, types = _SIGNATURES[name]
        fn = getattr(_ops()._lib(library), name)
        fn.argtypes, fn.restype = types, c_int
        _functions[name] = fn
    return fn


def _stream() -> int:
    """The current stream.  (There are tensors on the GPU: torch has been set up.)"""
    raw = _ops()._raw_stream
    return raw(torch._C._cuda_getDevice()) if raw is not None else torch.cuda.current_stream().cuda_stream


def _done(status: int, what: str, detail, kernels: int = 1) -> None:
    """``detail``: called for the error's text."""
    if status == 0:
        _ops()._launched(kernels)
    else:
        _ops()._check(status, what, detail(), kernels)


def _require(t, name: str, dtype, ndim: int) -> None:
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.is_cuda and t.dim() == ndim and t.is_contiguous()):
        _ops()._need(t, name, dtype, ndim)


def _require_entries(t, name: str, n: int) -> None:
    _require(t, name, torch.int32, 1)
    if t.shape[0] < n:
        raise _ops().KernelError(f"int8_paged_attention: {name} has {t.shape[0]} entries, the step needs {n}")


def _code(dtype, name: str) -> int:
    code = _ops()._DT.get(dtype)
    if code is None:
        raise _ops().KernelError(f"{name}: dtype {dtype} is not supported (float32 or bfloat16)")
    return code


def _same_device(what: str, first, *others) -> None:
    device = first.device
    for t in others:
        if t.device != device:
            raise _ops().KernelError(f"{what}: tensors on different devices "
                                     f"({sorted({str(x.device) for x in (first, *others)})})")


def _padded(k: int) -> int:
    return -(-k // 16) * 16


class Int8Rows:
    """Rows [M, K] in 8 bits: ``codes`` int8 [M, K rounded up to 16] (zeros behind K), ``scales`` float32 [M]; ``dtype`` is
    the type of the tensor they were made from, which a product's output takes."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, k: int, dtype: torch.dtype):
        ops = _ops()
        ops._need(codes, "codes", torch.int8, 2)
        ops._need(scales, "scales", torch.float32, 1)
        if not 1 <= k <= MAX_K or codes.shape[1] != _padded(k) or scales.shape[0] != codes.shape[0]:
            raise ops.KernelError(f"Int8Rows: codes {tuple(codes.shape)}, scales {tuple(scales.shape)} for rows of {k} values "
                                  f"(K from 1 to {MAX_K}, codes of K rounded up to 16)")
        if codes.data_ptr() % 16:
            raise ops.KernelError("Int8Rows: codes must lie on 16 bytes")
        _same_device("Int8Rows", codes, scales)
        _code(dtype, "Int8Rows")
        self._set(codes, scales, int(k), dtype)

    def _set(self, codes, scales, k, dtype) -> "Int8Rows":
        self.codes, self.scales, self.k, self.dtype = codes, scales, k, dtype
        return self

    @property
    def shape(self):
        return torch.Size((self.codes.shape[0], self.k))

    @property
    def device(self):
        return self.codes.device

    def tensor(self) -> torch.Tensor:
        """The values the codes stand for, float32."""
        return self.codes[:, :self.k].float() * self.scales[:, None]


class Int8Weight:
    """A weight [N, K] in 8 bits with a scale for each output channel: ``codes`` int8 [N, K rounded up to 16] on 16 bytes,
    ``scales`` float32 [N].  ``Int8Weight(codes [N, K], scales [N])`` lays out codes that were made elsewhere, -128 not
    among them.  A constant, like every weight: the products read it ahead of their wait for the kernel in front."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        ops = _ops()
        ops._need(codes, "codes", torch.int8, 2)
        ops._need(scales, "scales", torch.float32, 1)
        n, k = codes.shape
        if scales.shape[0] != n or k < 1 or k > MAX_K:
            raise ops.KernelError(f"Int8Weight: codes {tuple(codes.shape)}, scales {tuple(scales.shape)} "
                                  f"(K from 1 to {MAX_K})")
        _same_device("Int8Weight", codes, scales)
        if _padded(k) != k or codes.data_ptr() % 16:
            padded = torch.zeros(n, _padded(k), dtype=torch.int8, device=codes.device)
            padded[:, :k] = codes
            codes = padded
        self._set(codes, scales, k)

    @classmethod
    def of(cls, weight: torch.Tensor) -> "Int8Weight":
        """Quantises a float32 or bfloat16 weight [N, K]."""
        rows = _quantize(weight, "weight")
        return cls.__new__(cls)._set(rows.codes, rows.scales, rows.k)

    def _set(self, codes, scales, k) -> "Int8Weight":
        # The copy stands between the kernel of this package that may have made the codes, which lets the next one start beside
        # it, and a product, which reads its weight ahead of its wait for the kernel in front: a copy waits for all of it.
        self.codes, self.scales, self.k = codes, scales.clone(), k
        return self

    @property
    def shape(self):
        return torch.Size((self.codes.shape[0], self.k))

    @property
    def device(self):
        return self.codes.device

    def tensor(self) -> torch.Tensor:
        """The values the codes stand for, float32."""
        return self.codes[:, :self.k].float() * self.scales[:, None]


def _check_rows(x, name: str) -> int:
    """The type's code of a matrix whose rows are consecutive values, at any distance from one another."""
    ops = _ops()
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ops.KernelError(f"{name} must be a CUDA tensor: this package has no CPU path")
    if x.dim() != 2 or (x.shape[1] > 1 and x.stride(1) != 1):
        raise ops.KernelError(f"{name} must be rows of consecutive values (shape {tuple(x.shape)}, stride {x.stride()})")
    if not 1 <= x.shape[1] <= MAX_K:
        raise ops.KernelError(f"{name} has rows of {x.shape[1]} values (1 to {MAX_K})")
    return _code(x.dtype, name)


def _quantize(x: torch.Tensor, name: str) -> Int8Rows:
    code = _check_rows(x, name)
    m, k = x.shape
    codes = torch.empty(m, _padded(k), dtype=torch.int8, device=x.device)
    scales = torch.empty(m, dtype=torch.float32, device=x.device)
    st = _fn("dib_quantize_rows")(x.data_ptr(), x.stride(0), codes.data_ptr(), scales.data_ptr(), m, k, code, _stream())
    _done(st, "quantize_rows", lambda: f"rows {m} x {k}")
    return Int8Rows.__new__(Int8Rows)._set(codes, scales, k, x.dtype)


def quantize_rows(x) -> Int8Rows:
    """Rows [M, K] (float32 or bfloat16, any distance between rows; or the partial sums of a product) in 8 bits."""
    return _quantize(_ops().as_tensor(x), "x")


def int8_linear(x, weight: Int8Weight, out_dtype=None) -> torch.Tensor:
    """y = x @ weight^T, [M, N]: ``x`` [M, K] is quantised row by row (or is an ``Int8Rows``); the sum of the codes'
    products is exact in 32 bits, so a row's bits depend on the row and the weight alone; times the token's and the
    channel's scale in float32, rounded once to ``out_dtype`` (float32 or bfloat16; x's type if not given)."""
    if not isinstance(weight, Int8Weight):
        raise _ops().KernelError("int8_linear: weight must be an Int8Weight")
    rows = isinstance(x, Int8Rows)
    if not rows:
        if not isinstance(x, torch.Tensor):
            x = _ops().as_tensor(x)
        code = _check_rows(x, "x")
    m, k = x.shape
    if k != weight.k:
        raise _ops().KernelError(f"int8_linear: x {tuple(x.shape)} against weight {tuple(weight.shape)}")
    codes = weight.codes
    device = codes.device
    if x.device != device:
        _same_device("int8_linear", x, weight)
    n = codes.shape[0]
    out_dtype = out_dtype or x.dtype
    out_code = _code(out_dtype, "out")
    out = torch.empty(m, n, dtype=out_dtype, device=device)
    if rows:
        if x.codes.shape[1] != codes.shape[1]:
            raise _ops().KernelError(f"int8_linear: codes {tuple(x.codes.shape)} against the weight's {tuple(codes.shape)}")
        st = _fn("dib_gemm_int8")(x.codes.data_ptr(), x.scales.data_ptr(), codes.data_ptr(), weight.scales.data_ptr(),
                                  out.data_ptr(), m, n, x.codes.shape[1], out_code, _sms(device), _stream())
    else:
        work = torch.empty(m * (_padded(k) + 4), dtype=torch.int8, device=device)      # codes, then scales
        st = _fn("dib_int8_linear")(_address("dib_quantize_rows"), x.data_ptr(), x.stride(0), code, k, work.data_ptr(),
                                    codes.data_ptr(), weight.scales.data_ptr(), out.data_ptr(), m, n, out_code,
                                    _sms(device), _stream())
    _done(st, "int8_linear", lambda: f"M={m} N={n} K={k}", 1 if rows else 2)
    return out


_addresses: dict = {}


def _address(name: str) -> int:
    got = _addresses.get(name)
    if got is None:
        got = _addresses[name] = ctypes.cast(_fn(name), c_void_p).value
    return got


def force_product_form(form: int) -> None:
    """Measurement and test switch of the product: mma.sync on a streamed weight (0), tiles of 128 x 64, 128 x 128 or
    128 x 256 (1, 2, 3), the pair of CTAs (4), clusters that share k on tiles of 128 x 64 or 128 x 128 (5, 6), whatever the
    sizes; -1: the library's own choice.  All give the same bits."""
    _ops()._lib("gemm_int8").dib_gemm_int8_force_form(c_int(form))


_sm_counts: dict = {}


def _sms(device) -> int:
    n = _sm_counts.get(device)
    if n is None:
        n = _sm_counts[device] = torch.cuda.get_device_properties(device).multi_processor_count
    return n


class Int8Cache:
    """One layer's paged cache in 8 bits: ``data`` int8 [pages, 2, Hkv, page_size, D], ``scales`` float32
    [pages, 2, Hkv, page_size]; [:, 0] are keys, [:, 1] values.  D a multiple of 16, at most 256."""

    def __init__(self, data: torch.Tensor, scales: torch.Tensor):
        ops = _ops()
        ops._need(data, "data", torch.int8, 5)
        ops._need(scales, "scales", torch.float32, 4)
        pages, two, hkv, page_size, d = data.shape
        if tuple(scales.shape) != (pages, two, hkv, page_size) or two != 2 or hkv < 1 or page_size < 1:
            raise ops.KernelError(f"Int8Cache: data {tuple(data.shape)}, scales {tuple(scales.shape)}")
        if d < 16 or d > MAX_HEAD_DIM or d % 16:
            raise ops.KernelError(f"Int8Cache: heads of {d} (a multiple of 16, at most {MAX_HEAD_DIM})")
        if data.data_ptr() % 16:
            raise ops.KernelError("Int8Cache: data must lie on 16 bytes")
        _same_device("Int8Cache", data, scales)
        self.data, self.scales = data, scales

    @classmethod
    def zeros(cls, num_pages: int, num_kv_heads: int, page_size: int, head_dim: int, device="cuda") -> "Int8Cache":
        return cls(torch.zeros(num_pages, 2, num_kv_heads, page_size, head_dim, dtype=torch.int8, device=device),
                   torch.zeros(num_pages, 2, num_kv_heads, page_size, dtype=torch.float32, device=device))

    @property
    def shape(self):
        return self.data.shape

    @property
    def device(self):
        return self.data.device


def _row_stride(x, name: str, hkv: int, d: int) -> int:
    """Distance of a token's rows [Hkv, D], which lie together (a column range of a fused projection, say)."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise _ops().KernelError(f"{name} must be a CUDA tensor: this package has no CPU path")
    shape, stride = x.shape, x.stride()
    if len(shape) != 3 or shape[1] != hkv or shape[2] != d:
        raise _ops().KernelError(f"{name} has shape {tuple(shape)}, the cache's heads are [{hkv}, {d}]")
    if stride[2] != 1 or (hkv > 1 and stride[1] != d):
        raise _ops().KernelError(f"{name}: a token's heads must lie together (stride {stride})")
    return stride[0]


def int8_cache_write(k: torch.Tensor, v: torch.Tensor, cache: Int8Cache, slot_mapping: torch.Tensor) -> None:
    """k, v [T, Hkv, D] (float32 or bfloat16; column ranges of wider rows too) into the rows ``slot_mapping`` (int32 [T],
    page * page_size + offset) of the cache; a negative slot is skipped.  Slots are distinct."""
    data = cache.data
    pages, _, hkv, page_size, d = data.shape
    ks, vs = _row_stride(k, "k", hkv, d), _row_stride(v, "v", hkv, d)
    _require(slot_mapping, "slot_mapping", torch.int32, 1)
    t = k.shape[0]
    if v.shape[0] != t or v.dtype is not k.dtype or slot_mapping.shape[0] < t:
        raise _ops().KernelError(f"int8_cache_write: k {tuple(k.shape)} {k.dtype}, v {tuple(v.shape)} {v.dtype}, "
                                 f"{slot_mapping.shape[0]} slots")
    device = data.get_device()
    if k.get_device() != device or v.get_device() != device or slot_mapping.get_device() != device:
        _same_device("int8_cache_write", data, k, v, slot_mapping)
    st = _fn("dib_int8_cache_write")(k.data_ptr(), v.data_ptr(), ks, vs, data.data_ptr(), cache.scales.data_ptr(),
                                     slot_mapping.data_ptr(), t, hkv, d, page_size, pages, _code(k.dtype, "k"), _stream())
    _done(st, "int8_cache_write", lambda: f"heads {hkv} x {d}")


def int8_qk_norm_rope_cache(qkv, num_heads: int, num_kv_heads: int, head_dim: int, q_norm_weight, k_norm_weight, eps: float,
                            cos_sin, positions: torch.Tensor, cache: Int8Cache, slot_mapping: torch.Tensor) -> torch.Tensor:
    """``ops.qk_norm_rope_cache`` with an 8-bit cache: q [T, Hq, D] normed and rotated; k, treated alike, and v are rounded to
    the activations' type, quantised and written to the tokens' slots."""
    ops = _ops()
    qkv = ops.as_tensor(qkv)
    ops._need(qkv, "qkv", None, 2)
    t, width = qkv.shape
    pages, _, hkv, page_size, d = cache.shape
    if (hkv, d) != (num_kv_heads, head_dim) or width != (num_heads + 2 * hkv) * d:
        raise ops.KernelError(f"int8_qk_norm_rope_cache: rows of {width} for heads {num_heads}/{num_kv_heads} x {head_dim}, "
                              f"cache {tuple(cache.shape)}")
    for x, name in ((positions, "positions"), (slot_mapping, "slot_mapping")):
        ops._need(x, name, torch.int32, 1)
        if x.shape[0] < t:
            raise ops.KernelError(f"int8_qk_norm_rope_cache: {x.shape[0]} {name} for {t} tokens")
    for w, name in ((q_norm_weight, "q_norm_weight"), (k_norm_weight, "k_norm_weight")):
        if w is not None:
            ops._need(w, name, torch.float32, 1)
            if w.shape[0] != d:
                raise ops.KernelError(f"{name} has {w.shape[0]} elements, head_dim is {d}")
    rotary_dim, max_pos = 0, 0
    if cos_sin is not None:
        ops._need(cos_sin, "cos_sin", torch.float32, 2)
        max_pos, rotary_dim = cos_sin.shape
    _same_device("int8_qk_norm_rope_cache", qkv, cache.data, positions, slot_mapping)
    q = torch.empty(t, num_heads, d, dtype=qkv.dtype, device=qkv.device)
    st = _fn("dib_int8_qk_norm_rope_cache")(
        qkv.data_ptr(), q.data_ptr(), cache.data.data_ptr(), cache.scales.data_ptr(), _pointer(q_norm_weight),
        _pointer(k_norm_weight), float(eps), _pointer(cos_sin), rotary_dim, max_pos, positions.data_ptr(),
        slot_mapping.data_ptr(), t, num_heads, hkv, d, page_size, pages, _code(qkv.dtype, "qkv"), _stream())
    _done(st, "int8_qk_norm_rope_cache", lambda: f"head_dim {d}, rotary_dim {rotary_dim}")
    return q


def _pointer(t) -> int:
    return 0 if t is None else t.data_ptr()


def int8_cache_read(cache: Int8Cache, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16):
    """(k, v) [T, Hkv, D] in ``dtype``: what the rows ``slots`` (int32 [T]) of the cache stand for; zeros for a negative
    slot."""
    data = cache.data
    pages, _, hkv, page_size, d = data.shape
    _require(slots, "slots", torch.int32, 1)
    if slots.get_device() != data.get_device():
        _same_device("int8_cache_read", data, slots)
    code = _code(dtype, "out")
    t = slots.shape[0]
    k, v = torch.empty(2, t, hkv, d, dtype=dtype, device=data.device).unbind(0)
    st = _fn("dib_int8_cache_read")(data.data_ptr(), cache.scales.data_ptr(), slots.data_ptr(), k.data_ptr(), v.data_ptr(), t,
                                    hkv, d, page_size, pages, code, _stream())
    _done(st, "int8_cache_read", lambda: f"heads {hkv} x {d}")
    return k, v


# ---- a step's work: one launch of the split form for the sequences with one new token, one for those with a few, one of the
# prompt form for those with many

def _pages_fit(page_size: int) -> bool:
    """Page sizes that the split form takes: a block of 32 keys is whole pages, or lies in one."""
    return page_size >= 4 and page_size & (page_size - 1) == 0


def _most_runs(kv_len: int, group: int) -> int:
    """The most runs of a sequence of at most ``kv_len`` keys and ``group`` rows or more (the lengths on the device may be less
    than the host's, so a token's rows are all that is certain)."""
    runs, keys = 1, _lib().dib_int8_attention_split_keys
    for n in {min(kv_len, 2048), min(kv_len, 4096), min(kv_len, 16384), kv_len}:
        runs = max(runs, -(-n // keys(n, group)))
    return runs


def _lib():
    return _ops()._lib("attention_int8")


def _split_work(seqs: list, q_lens: list, kv_lens: list, group: int, hkv: int, tile_rows: int, runs: int) -> int:
    """The most work that the split form's kernel counts, in tiles of 128 keys (a work item: its run's, the last run counted as
    a whole one, and one; of 512 keys at least)."""
    return sum(hkv * -(-q_lens[s] * group // tile_rows) * (2 * (kv_lens[s] // 128 + 3) + runs) for s in seqs)


class _SplitPart:
    """The sequences of one launch: their number, the most rows of one, rows a tile, the most work items of one."""

    def __init__(self, seqs: list, q_lens: list, kv_lens: list, group: int, hkv: int, wide: bool, device):
        first, count = seqs[0], len(seqs)
        self.first, self.count, self.list = first, count, None
        if seqs != list(range(first, first + count)):
            self.list = torch.tensor(seqs, dtype=torch.int32).to(device, non_blocking=True)
        self.max_rows = max(q_lens[s] for s in seqs) * group
        self.tile_rows = next(r for r in ((8, 16) if wide else (4, 8, 16, 24, 32)) if self.max_rows <= r or r == (16 if wide else 32))
        runs = _most_runs(max(kv_lens[s] for s in seqs), group)
        tiles, per32 = -(-self.max_rows // self.tile_rows), 32 // self.tile_rows
        longest = max(kv_lens[s] for s in seqs)
        if count * hkv * tiles * (2 * (longest // 128 + 3) + runs) >= 1 << 31 \
                and _split_work(seqs, q_lens, kv_lens, group, hkv, self.tile_rows, runs) >= 1 << 31:
            raise _ops().KernelError(f"int8_paged_attention: {sum(q_lens[s] for s in seqs)} new tokens of up to {longest} keys, "
                                     f"{group} heads a kv head, are more than a launch counts: smaller portions")
        # (runs get longer with the rows: tiles * runs is largest at 64 rows, or the tiles' own number is)
        self.items = hkv * min(tiles * runs, max(2 * per32 * runs, per32 * (runs + 1) + tiles))
        # (rows of partial results: none where every sequence has one run)
        self.rows = count * self.items * self.tile_rows if runs > 1 else 0
        self.list_pointer = _pointer(self.list)


# Rows (new tokens x query heads of a kv head) of a sequence of drafted tokens above which they take the prompt form (bfloat16),
# whose query tiles have 128 rows.  By the sequence's own rows, so that its bits do not depend on the step: 16 sequences of 4,096
# keys and 48 rows take 76 us there and 210 in the split form, of 1,500 keys and 64 rows 36 and 111, one of 4,096 keys 72 and 37.
# A prompt's portions take it whatever their rows: the scheduler cuts a prompt where the step has room, and in a captured step
# the host knows a portion's bucket only, so a line between two forms would show in a request's bits.  (One of 5 tokens on 4,096
# keys, 10 rows, takes 70 us there, where the split form takes 16; sixteen on 1,500 32 and 29.)
PROMPT_ROWS = 32
# Bytes of partial results that a launch of the prompt form may take, where rows have several chunks of keys: 8,192 tokens of 64
# heads on 65,536 keys would take 4.4 GB at once; those of a few thousand rows fill the GPU.
SCRATCH_BYTES = 1 << 30


class _PromptPart:
    """The sequences of the prompt form's launches: the list of query-tile pairs (and chunks of keys, and places of partial
    results), longest last in a launch; ``launches``: (first unit, units, first entry, entries, tokens of the longest entry),
    an entry being tokens of a sequence whose chunks are added up; ``rows``: tokens that partial results are held of."""

    def __init__(self, seqs: list, q_lens: list, kv_lens: list, group: int, hkv: int, window: int, device):
        from . import attention_bf16
        chosen = set(seqs)
        new = [n if s in chosen else 0 for s, n in enumerate(q_lens)]
        keys = [max(n, kv) for n, kv in zip(new, kv_lens)]
        tokens = 128 // group
        self.chunks = -(-max(keys[s] for s in seqs) // (attention_bf16.CHUNK_TILES * 128))
        self.chunk_tiles = attention_bf16.CHUNK_TILES if self.chunks > 1 else 0
        self.max_tokens, self.rows = max(new), 0
        if self.chunks > 1:
            units = list(zip(*attention_bf16.extend_chunk_units(new, keys, 0, tokens, attention_bf16.CHUNK_TILES)))
            entries, place = self._entries(seqs, new, 2 * tokens, group * hkv * self.chunks * 520)
        else:
            # how tiles are paired depends on the step, the arithmetic of a tile does not (see ``extend_tile_pairs``)
            ctas = (sum(-(-n // tokens) for n in new) + 1) // 2 * hkv
            sms = _sms(device)
            units = [(*u, 0) for u in zip(*attention_bf16.extend_tile_pairs(new, keys, 0, tokens, window, alone=2 * ctas <= sms,
                                                                            neighbours=ctas > sms))]
            entries, place = [[(s, 0, new[s], 0) for s in seqs]], lambda s, t: (0, 0)
        units = [(*place(s, a), s, a, b, c) for s, a, b, c in units]
        units.sort(key=lambda u: u[0])          # by launch, in their order
        self.count, self.launches, at = len(units), [], 0
        for i, own in enumerate(entries):
            count = sum(1 for u in units if u[0] == i)
            self.launches.append((sum(n for _, n, *_ in self.launches), count, at, len(own), max(hi - lo for _, lo, hi, _ in own)))
            at += len(own)
        flat = [e for own in entries for e in own]
        lists = torch.tensor([u[i] for i in (2, 3, 4, 5, 1) for u in units] + [e[i] for i in range(4) for e in flat],
                             dtype=torch.int32).to(device, non_blocking=True)
        self.units, self.entries = lists[:4 * self.count], lists[5 * self.count:]
        self.entry_count = len(flat)
        self.seq_list = self.entries[:self.entry_count]

    def _entries(self, seqs: list, new: list, pair: int, token_bytes: int):
        """The launches' entries (sequence, first token, end, place of its first token's partial results), cut between pairs of
        query tiles where a launch's partial results are full, and the launch and place of a pair."""
        room = max(1, SCRATCH_BYTES // (token_bytes * pair)) * pair
        entries, where, used = [[]], {}, 0
        for s in seqs:
            at = 0
            while at < new[s]:
                if used >= room:
                    entries.append([])
                    used = 0
                end = min(new[s], at + room - used)
                entries[-1].append((s, at, end, used))
                for t in range(at, end, pair):
                    where[s, t] = (len(entries) - 1, used + t - at)
                used += -(-(end - at) // pair) * pair
                self.rows = max(self.rows, used)
                at = end
        return entries, lambda s, t: where[s, t]


def _parts(meta, group: int, hkv: int, wide: bool, window: int, portions: bool, device) -> list:
    """The step's launches: the sequences with one new token, those of the prompt form (bfloat16: all others that are portions
    of prompts, or those with many drafted tokens), the rest."""
    key = ("int8", group, hkv, wide, window, portions)
    parts = meta.scratch.get(key)
    if parts is None:
        q_lens, kv_lens = meta.q_lens, meta.kv_lens
        if not len(q_lens) == len(kv_lens) <= meta.block_table.shape[0]:
            raise _ops().KernelError(f"int8_paged_attention: {len(q_lens)} q_lens and {len(kv_lens)} kv_lens for a block table "
                                     f"of {meta.block_table.shape[0]} sequences")
        one = [s for s, n in enumerate(q_lens) if n == 1]
        more = [s for s, n in enumerate(q_lens) if n > 1]
        many = [s for s in more if not wide and (portions or q_lens[s] * group > PROMPT_ROWS) and group <= 128]
        few = [s for s in more if s not in set(many)]
        parts = [_SplitPart(x, q_lens, kv_lens, group, hkv, wide, device) for x in (one, few) if x]
        if many:
            parts.append(_PromptPart(many, q_lens, kv_lens, group, hkv, window, device))
        meta.scratch[key] = parts
    return parts


def _prompt(q, out, cache: Int8Cache, meta, part: _PromptPart, scale: float, window: int) -> None:
    pages, _, hkv, page_size, d = cache.data.shape
    hq = q.shape[1]
    rows = part.rows * hq * part.chunks
    held = torch.empty(rows * 130, dtype=torch.float32, device=q.device) if rows else None      # outputs, then (maximum, sum)
    partial = _pointer(held)
    units, entries = part.units.data_ptr(), part.entries.data_ptr()
    for first, count, first_entry, num_entries, max_tokens in part.launches:
        st = _fn("dib_int8_attention_prompt")(
            q.data_ptr(), out.data_ptr(), cache.data.data_ptr(), cache.scales.data_ptr(), pages, meta.block_table.data_ptr(),
            meta.block_table.shape[1], meta.cu_q_lens.data_ptr(), meta.seq_lens.data_ptr(), units + 4 * first, count, part.count,
            entries + 4 * first_entry, num_entries, part.entry_count, max_tokens, partial, partial + rows * 512, part.chunk_tiles,
            part.chunks, hq, hkv, d, page_size, scale, window, _stream())
        _done(st, "int8_paged_attention", lambda: f"head_dim {d}, heads {hq}/{hkv}", 2 if part.chunks > 1 else 1)


def _split(q, out, cache: Int8Cache, meta, part: _SplitPart, scale: float, window: int) -> None:
    pages, _, hkv, page_size, d = cache.data.shape
    hq = q.shape[1]
    rows = part.rows
    held = torch.empty(rows * (d + 2), dtype=torch.float32, device=q.device) if rows else None      # outputs, (maximum, sum)
    partial = _pointer(held)
    st = _fn("dib_int8_attention_split")(
        q.data_ptr(), out.data_ptr(), cache.data.data_ptr(), cache.scales.data_ptr(), pages, meta.block_table.data_ptr(),
        meta.block_table.shape[1], meta.cu_q_lens.data_ptr(), meta.seq_lens.data_ptr(), part.list_pointer, part.first, part.count,
        part.max_rows, part.tile_rows, partial, partial + rows * d * 4, part.items, 1 if rows else 0, hq, hkv, d, page_size, scale,
        window, _ops()._DT[q.dtype], _sms(q.device), _stream())
    _done(st, "int8_paged_attention", lambda: f"head_dim {d}, heads {hq}/{hkv}", 2 if rows else 1)


def int8_paged_attention(q: torch.Tensor, cache: Int8Cache, meta, scale: float, window=None,
                         portions: bool = False) -> torch.Tensor:
    """Causal attention of every token of the step over its sequence's keys in the cache, as ``ops.paged_attention``: q
    [T, Hq, D] float32 or bfloat16, ``meta`` the step's ``AttentionMeta``.  A sequence's new tokens are its last ones
    (``seq_lens`` counts them); each sees the keys up to its own position, the last ``window`` of them if given.  The
    codes of keys and values enter the products as they are, the scales join scores and probabilities in float32.  A
    token that sees no key gives zeros.

    ``portions``: the sequences with more than one new token bring portions of prompts.  In bfloat16 they then all take one
    form, so that a token's bits depend neither on where its prompt was cut (a portion of one token aside) nor on whether
    ``meta`` holds the lengths or upper bounds of them.  Otherwise they count as drafted tokens, few of which are faster in
    another form, chosen by their number."""
    ops = _ops()
    if not (isinstance(q, torch.Tensor) and q.is_cuda and q.dim() == 3 and q.is_contiguous()):
        ops._need(q, "q", None, 3)
    code = _code(q.dtype, "q")
    t, hq, d = q.shape
    data = cache.data
    pages, _, hkv, page_size, d2 = data.shape
    if d2 != d or hq < 1 or hq % hkv:
        raise ops.KernelError(f"int8_paged_attention: q {tuple(q.shape)} vs cache {tuple(cache.shape)}")
    table, token_seq, cu, lens = meta.block_table, meta.token_seq, meta.cu_q_lens, meta.seq_lens
    _require(table, "block_table", torch.int32, 2)
    b = table.shape[0]
    _require_entries(token_seq, "token_seq", t)
    _require_entries(cu, "cu_q_lens", b + 1)
    _require_entries(lens, "seq_lens", b)
    win = int(window) if window else 0
    if win < 0:
        raise ops.KernelError(f"int8_paged_attention: a window of {win} keys")
    device = data.get_device()
    if q.get_device() != device or table.get_device() != device or token_seq.get_device() != device \
            or cu.get_device() != device or lens.get_device() != device:
        _same_device("int8_paged_attention", data, q, table, token_seq, cu, lens)
    out = torch.empty_like(q)
    if t == 0:
        return out
    if d <= 128 and _pages_fit(page_size) and q.data_ptr() % 16 == 0 and cache.scales.data_ptr() % 16 == 0 \
            and pages * 2 * hkv * page_size < 1 << 31:
        for part in _parts(meta, hq // hkv, hkv, code == 0, win, bool(portions), q.device):
            run = _prompt if isinstance(part, _PromptPart) else _split
            run(q, out, cache, meta, part, float(scale), win)
        return out
    st = _fn("dib_int8_attention_any")(
        q.data_ptr(), out.data_ptr(), data.data_ptr(), cache.scales.data_ptr(), table.data_ptr(), table.shape[1],
        token_seq.data_ptr(), cu.data_ptr(), lens.data_ptr(), t, hq, hkv, d, page_size, pages, float(scale), win, code, _stream())
    _done(st, "int8_paged_attention", lambda: f"head_dim {d}, heads {hq}/{hkv}")
    return out
