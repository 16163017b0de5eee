"""Serving in 4-bit floating point: weights and activations as rows of 4-bit codes with a scale for each 16 of them, and a paged
cache of keys and values held the same way.  ``ops`` exports what is here.

One rule quantises every row (a token's activations, an output channel of a weight, a token's key or value of one head).  With
a = max(max |x|, 2^-100) of the row:

    E = the least exponent with a <= 2688 * 2^E;  b = e4m3(max |x| of a block of 16 values / (6 * 2^E));
    code = e2m1(x / (2^E * b)), 0 where b is 0;   value = code * b * 2^E

whatever the row's type; quotients are rounded to float32, b and the code to the nearest, ties to even.  A row that holds an
infinity or a NaN reads back as NaN.  Rows are given and kept as codes (uint8, two a byte, the first in the low half; e2m1 is 0,
0.5, 1, 1.5, 2, 3, 4, 6 and, from 8 on, their negatives), block scales (float8_e4m3fn, not negative) and exponents (uint8,
E + 127; 255: no numbers).

``Fp4Rows``             activations [M, K] in 4 bits (``fp4_quantize_rows``), in the tensor cores' layout
``Fp4Weight``           a weight [N, K], quantised once (``Fp4Weight.of``) or given as codes, scales and exponents
``fp4_linear``          y = x @ weight^T on codes and scales, sums in float32
``Fp4Cache``            the cache of one layer: data [pages, 2, Hkv, page_size, D / 2], scales [.., D / 16], exponents [..]
``fp4_cache_write``     keys and values into their slots
``fp4_qk_norm_rope_cache``  the same from the fused projection's rows, q and k normed and rotated on the way
``fp4_cache_read``      what the rows of given slots stand for
``fp4_paged_attention``  attention of a step's new tokens over the cache
"""

from __future__ import annotations

import ctypes
import functools
from ctypes import c_float, c_int, c_longlong, c_void_p
from types import SimpleNamespace

import torch

MAX_K = 1 << 24
MAX_HEAD_DIM = 256
BLOCK = 16


# What the host does in front of a launch is kept short, as in the 8-bit operators: the C functions are looked up once, with their
# argument types; an argument is looked at in one expression, and the check that words the error runs only where that fails.
_P, _I, _L, _F = c_void_p, c_int, c_longlong, c_float
_SIGNATURES = {
    "dib_fp4_quantize_rows": ("rows_fp4", (_P, _L, _P, _P, _P, _L, _I, _I, _I, _P)),
    "dib_fp4_read_rows": ("rows_fp4", (_P, _P, _P, _P, _L, _I, _I, _P)),
    "dib_fp4_layout_rows": ("rows_fp4", (_P, _P, _P, _P, _P, _P, _L, _I, _P)),
    "dib_gemm_fp4": ("gemm_fp4", (_P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _P)),
    "dib_fp4_linear": ("gemm_fp4", (_P, _P, _L, _I, _I, _P, _P, _P, _P, _P, _I, _I, _I, _I, _P)),
    "dib_fp4_cache_write": ("cache_fp4", (_P, _P, _L, _L, _P, _P, _P, _P, _I, _I, _I, _I, _L, _I, _P)),
    "dib_fp4_cache_read": ("cache_fp4", (_P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _L, _I, _P)),
    "dib_fp4_qk_norm_rope_cache": ("cache_fp4", (_P, _P, _P, _P, _P, _P, _P, _F, _P, _I, _I, _P, _P, _I, _I, _I, _I, _I, _L, _I, _P)),
    "dib_fp4_unpack_pages": ("cache_fp4", (_P, _P, _P, _L, _P, _I, _P, _P, _P, _P, _I, _I, _P, _I, _I, _I, _I, _P)),
    "dib_fp4_finish_portions": ("cache_fp4", (_P, _L, _P, _I, _P, _P, _P, _I, _I, _P, _I, _I, _I, _I, _I, _P)),
    "dib_fp4_attention_split": ("attention_fp4", (_P, _P, _P, _P, _P, _L, _P, _I, _P, _P, _P, _I, _I, _I, _I, _P, _P, _I, _I, _I, _I,
                                                  _I, _I, _F, _I, _I, _I, _P)),
    "dib_fp4_attention_stream": ("attention_fp4_stream", (_P, _P, _P, _P, _P, _L, _P, _I, _P, _P, _P, _I, _I, _I, _I, _P, _P, _I, _I, _I,
                                                          _I, _I, _I, _F, _I, _I, _I, _P)),
    "dib_fp4_attention_any": ("attention_fp4", (_P, _P, _P, _P, _P, _P, _I, _P, _P, _P, _I, _I, _I, _I, _I, _L, _F, _I, _I, _P)),
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


_addresses: dict = {}


def _address(name: str) -> int:
    got = _addresses.get(name)
    if got is None:
        got = _addresses[name] = ctypes.cast(_fn(name), c_void_p).value
    return got


def _stream(what: str, device: torch.device) -> int:
    """The current stream of the current device, which the tensors must be on: kernels are launched there."""
    current = torch._C._cuda_getDevice()
    if device.index != current:
        raise _ops().KernelError(f"{what}: tensors on {device}, the current device is cuda:{current}")
    raw = _ops()._raw_stream
    return raw(current) if raw is not None else torch.cuda.current_stream().cuda_stream


def _done(status: int, what: str, detail, kernels: int = 1) -> None:
    """``detail``: called for the error's text."""
    if status == 0:
        _ops()._launched(kernels)
    else:
        _ops()._check(status, what, detail(), kernels)


def _require(t, name: str, dtype, ndim: int) -> None:
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.is_cuda and t.dim() == ndim and t.is_contiguous()):
        _ops()._need(t, name, dtype, ndim)


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


def _pointer(t) -> int:
    return 0 if t is None else t.data_ptr()


_sm_counts: dict = {}


def _sms(device) -> int:
    n = _sm_counts.get(device)
    if n is None:
        n = _sm_counts[device] = torch.cuda.get_device_properties(device).multi_processor_count
    return n


# ---- rows of a matrix

def _code_bytes(k: int) -> int:
    """Bytes of a row's codes in the tensor cores' layout."""
    return -(-k // 32) * 16


def _tile_bytes(rows: int, k: int) -> int:
    """Bytes of the block scales of ``rows`` rows: 512 for each 128 rows x 64 values, the latter rounded up to 256."""
    return -(-rows // 128) * -(-k // 256) * 2048


class _Rows:
    """Rows [R, K] in the tensor cores' layout: ``codes`` uint8 [R, K rounded up to 32, / 2] (zeros behind K), ``tiles``
    uint8, the block scales in tiles of 128 rows x 64 values, ``units`` float32 [R], 2^E (NaN: no numbers).  They lie in one
    tensor, ``held``: the block scales, the codes, the units."""

    def _allocate(self, rows: int, k: int, device) -> None:
        codes_at = _tile_bytes(rows, k)
        units_at = codes_at + rows * _code_bytes(k)
        self.rows, self.k, self._at = rows, k, (codes_at, units_at)
        self.held = torch.empty(units_at + 4 * rows, dtype=torch.uint8, device=device)

    def _pointers(self) -> tuple:
        """Addresses of the codes, the block scales and the units."""
        tiles, (codes_at, units_at) = self.held.data_ptr(), self._at
        return tiles + codes_at, tiles, tiles + units_at

    def _quantize(self, x: torch.Tensor, name: str) -> None:
        code = _check_rows(x, name)
        m, k = x.shape
        device = x.device
        self._allocate(m, k, device)
        st = _fn("dib_fp4_quantize_rows")(x.data_ptr(), x.stride(0), *self._pointers(), m, k, code, _sms(device),
                                          _stream("fp4_quantize_rows", device))
        _done(st, "fp4_quantize_rows", lambda: f"rows {m} x {k}")

    @property
    def tiles(self) -> torch.Tensor:
        return self.held[:self._at[0]]

    @property
    def codes(self) -> torch.Tensor:
        return self.held[self._at[0]:self._at[1]].view(self.rows, _code_bytes(self.k))

    @property
    def units(self) -> torch.Tensor:
        return self.held[self._at[1]:].view(torch.float32)

    @property
    def shape(self):
        return torch.Size((self.rows, self.k))

    @property
    def device(self):
        return self.held.device

    def tensor(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values the codes stand for [R, K]; exact in float32, rounded once in bfloat16."""
        code, m, k, device = _code(dtype, "tensor"), self.rows, self.k, self.held.device
        out = torch.empty(m, k, dtype=dtype, device=device)
        st = _fn("dib_fp4_read_rows")(*self._pointers(), out.data_ptr(), m, k, code, _stream("tensor", device))
        _done(st, "Fp4 rows as a tensor", lambda: f"rows {m} x {k}")
        return out

    def block_scales(self) -> torch.Tensor:
        """The block scales, float8_e4m3fn [R, ceil(K / 16)]."""
        m, k = self.shape
        t = self.tiles.view(-(-m // 128), -(-k // 256) * 4, 32, 4, 4).permute(0, 3, 2, 1, 4)       # 128-rows, 32-rows, row, 64s, 16s
        return t.reshape(-1, -(-k // 256) * 16)[:m, :-(-k // BLOCK)].contiguous().view(torch.float8_e4m3fn)

    def exponents(self) -> torch.Tensor:
        """The rows' exponents, uint8 [R]: E + 127; 255 for a row without numbers."""
        return (self.units.view(torch.int32) >> 23).to(torch.uint8)


class Fp4Rows(_Rows):
    """Activations in 4 bits, as ``fp4_quantize_rows`` makes them; ``dtype`` is the type of the tensor they were made from, which
    a product's output takes."""

    def __init__(self, x: torch.Tensor):
        self._quantize(x, "x")
        self.dtype = x.dtype


class Fp4Weight(_Rows):
    """A weight [N, K] in 4 bits.  ``Fp4Weight(codes, block_scales, exponents, k)`` lays out rows that were quantised elsewhere:
    codes uint8 [N, ceil(K / 2)], block scales float8_e4m3fn [N, ceil(K / 16)], not negative, exponents uint8 [N].  A
    constant, like every weight: the products read it ahead of their wait for the kernel in front."""

    def __init__(self, codes: torch.Tensor, block_scales: torch.Tensor, exponents: torch.Tensor, k: int):
        ops = _ops()
        ops._need(codes, "codes", torch.uint8, 2)
        ops._need(block_scales, "block_scales", torch.float8_e4m3fn, 2)
        ops._need(exponents, "exponents", torch.uint8, 1)
        n, k = codes.shape[0], int(k)
        if not 1 <= k <= MAX_K or codes.shape[1] != -(-k // 2) or tuple(block_scales.shape) != (n, -(-k // BLOCK)) \
                or exponents.shape[0] != n:
            raise ops.KernelError(f"Fp4Weight: codes {tuple(codes.shape)}, block scales {tuple(block_scales.shape)}, exponents "
                                  f"{tuple(exponents.shape)} for rows of {k} values (1 to {MAX_K}; two codes a byte, a scale "
                                  f"for each {BLOCK})")
        _same_device("Fp4Weight", codes, block_scales, exponents)
        self._allocate(n, k, codes.device)
        st = _fn("dib_fp4_layout_rows")(codes.data_ptr(), block_scales.data_ptr(), exponents.data_ptr(), *self._pointers(), n, k,
                                        _stream("Fp4Weight", codes.device))
        _done(st, "Fp4Weight", lambda: f"rows {n} x {k}")
        self._settle()

    @classmethod
    def of(cls, weight: torch.Tensor) -> "Fp4Weight":
        """Quantises a float32 or bfloat16 weight [N, K]."""
        made = cls.__new__(cls)
        made._quantize(weight, "weight")
        made._settle()
        return made

    def _settle(self) -> None:
        # A copy stands between the kernel of this package that made the codes, which lets the next one start beside it, and a
        # product, which reads its weight ahead of its wait for the kernel in front: a copy waits for all of it.
        units = self.units
        units.copy_(units.clone())


def _check_rows(x, name: str) -> int:
    """The type's code of a matrix whose rows are consecutive values, at any distance from one another."""
    ops = _ops()
    if isinstance(x, torch.Tensor) and x.is_cuda and x.dim() == 2 and x.stride(1) == 1 and 1 <= x.shape[1] <= MAX_K:
        code = ops._DT.get(x.dtype)
        if code is not None:
            return code
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ops.KernelError(f"{name} must be a CUDA tensor: this package has no CPU path")
    if x.dim() != 2 or (x.shape[1] > 1 and x.stride(1) != 1):
        raise ops.KernelError(f"{name} must be rows of consecutive values (shape {tuple(x.shape)}, stride {x.stride()})")
    if not 1 <= x.shape[1] <= MAX_K:
        raise ops.KernelError(f"{name} has rows of {x.shape[1]} values (1 to {MAX_K})")
    return _code(x.dtype, name)


def fp4_quantize_rows(x) -> Fp4Rows:
    """Rows [M, K] (float32 or bfloat16, any distance between rows; or the partial sums of a product) in 4 bits."""
    return Fp4Rows(_ops().as_tensor(x))


def fp4_linear(x, weight: Fp4Weight, out_dtype=None) -> torch.Tensor:
    """y = x @ weight^T, [M, N]: ``x`` [M, K] is quantised row by row (or is an ``Fp4Rows``); the products of codes and block
    scales are added up in float32 in one order of k whatever the other sizes, so a row's bits depend on the row and the
    weight alone; times the two rows' powers of two, rounded once to ``out_dtype`` (float32 or bfloat16; x's type if not given)."""
    if not isinstance(weight, Fp4Weight):
        raise _ops().KernelError("fp4_linear: weight must be an Fp4Weight")
    rows = isinstance(x, Fp4Rows)
    if not rows:
        if not isinstance(x, torch.Tensor):
            x = _ops().as_tensor(x)
        code = _check_rows(x, "x")
    m, k = x.shape
    if k != weight.k:
        raise _ops().KernelError(f"fp4_linear: x {tuple(x.shape)} against weight {tuple(weight.shape)}")
    n, device = weight.rows, weight.held.device
    if x.device != device:
        _same_device("fp4_linear", x, weight)
    out_dtype = out_dtype or x.dtype
    out_code = _code(out_dtype, "out")
    out = torch.empty(m, n, dtype=out_dtype, device=device)
    if rows:
        st = _fn("dib_gemm_fp4")(*x._pointers(), *weight._pointers(), out.data_ptr(), m, n, k, out_code, _sms(device),
                                 _stream("fp4_linear", device))
    else:
        # block scales, codes, units
        work = torch.empty(_tile_bytes(m, k) + m * (_code_bytes(k) + 4), dtype=torch.uint8, device=device)
        st = _fn("dib_fp4_linear")(_address("dib_fp4_quantize_rows"), x.data_ptr(), x.stride(0), code, k, work.data_ptr(),
                                   *weight._pointers(), out.data_ptr(), m, n, out_code, _sms(device), _stream("fp4_linear", device))
    _done(st, "fp4_linear", lambda: f"M={m} N={n} K={k}", 1 if rows else 2)
    return out


def force_product_form(form: int) -> None:
    """Measurement and test switch of the product: tiles of 128 x 64, 128 x 128 or 128 x 192 (0, 1, 2), the pair of CTAs (3),
    clusters that share k (4, up to 128 rows), whatever the sizes; -1: the library's own choice.  All give the same bits."""
    _ops()._lib("gemm_fp4").dib_gemm_fp4_force_form(c_int(form))


# ---- the cache

class Fp4Cache:
    """One layer's paged cache in 4 bits: ``data`` uint8 [pages, 2, Hkv, page_size, D / 2], ``scales`` float8_e4m3fn
    [pages, 2, Hkv, page_size, D / 16], finite and not negative in the rows that are read, ``exponents`` uint8
    [pages, 2, Hkv, page_size]; [:, 0] are keys, [:, 1] values.  D a multiple of 16, at most 256."""

    def __init__(self, data: torch.Tensor, scales: torch.Tensor, exponents: torch.Tensor):
        ops = _ops()
        ops._need(data, "data", torch.uint8, 5)
        ops._need(scales, "scales", torch.float8_e4m3fn, 5)
        ops._need(exponents, "exponents", torch.uint8, 4)
        pages, two, hkv, page_size, half = data.shape
        d = 2 * half
        if tuple(exponents.shape) != (pages, two, hkv, page_size) or tuple(scales.shape) != (pages, two, hkv, page_size, d // BLOCK) \
                or two != 2 or hkv < 1 or page_size < 1:
            raise ops.KernelError(f"Fp4Cache: data {tuple(data.shape)}, scales {tuple(scales.shape)}, exponents "
                                  f"{tuple(exponents.shape)}")
        if d < 16 or d > MAX_HEAD_DIM or d % 16:
            raise ops.KernelError(f"Fp4Cache: heads of {d} (a multiple of 16, at most {MAX_HEAD_DIM})")
        if data.data_ptr() % 16:
            raise ops.KernelError("Fp4Cache: data must lie on 16 bytes")
        _same_device("Fp4Cache", data, scales, exponents)
        self.data, self.scales, self.exponents = data, scales, exponents
        self.shape = torch.Size((pages, 2, hkv, page_size, d))

    @classmethod
    def zeros(cls, num_pages: int, num_kv_heads: int, page_size: int, head_dim: int, device="cuda") -> "Fp4Cache":
        rows = (num_pages, 2, num_kv_heads, page_size)
        return cls(torch.zeros(*rows, head_dim // 2, dtype=torch.uint8, device=device),
                   torch.zeros(*rows, head_dim // BLOCK, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn),
                   torch.zeros(rows, dtype=torch.uint8, device=device))

    @property
    def device(self):
        return self.data.device

    def _pointers(self) -> tuple:
        return self.data.data_ptr(), self.scales.data_ptr(), self.exponents.data_ptr()


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


def fp4_cache_write(k: torch.Tensor, v: torch.Tensor, cache: Fp4Cache, slot_mapping: torch.Tensor) -> None:
    """k, v [T, Hkv, D] (float32 or bfloat16; column ranges of wider rows too) into the rows ``slot_mapping`` (int32 [T],
    page * page_size + offset) of the cache; a negative slot is skipped.  Slots are distinct."""
    pages, _, hkv, page_size, d = cache.shape
    ks, vs = _row_stride(k, "k", hkv, d), _row_stride(v, "v", hkv, d)
    _require(slot_mapping, "slot_mapping", torch.int32, 1)
    t = k.shape[0]
    if v.shape[0] != t or v.dtype is not k.dtype or slot_mapping.shape[0] < t:
        raise _ops().KernelError(f"fp4_cache_write: k {tuple(k.shape)} {k.dtype}, v {tuple(v.shape)} {v.dtype}, "
                                 f"{slot_mapping.shape[0]} slots")
    device = cache.device
    if k.device != device or v.device != device or slot_mapping.device != device:
        _same_device("fp4_cache_write", cache.data, k, v, slot_mapping)
    st = _fn("dib_fp4_cache_write")(k.data_ptr(), v.data_ptr(), ks, vs, *cache._pointers(), slot_mapping.data_ptr(), t, hkv, d,
                                    page_size, pages, _code(k.dtype, "k"), _stream("fp4_cache_write", device))
    _done(st, "fp4_cache_write", lambda: f"heads {hkv} x {d}")


def fp4_qk_norm_rope_cache(qkv, num_heads: int, num_kv_heads: int, head_dim: int, q_norm_weight, k_norm_weight, eps: float,
                           cos_sin, positions: torch.Tensor, cache: Fp4Cache, slot_mapping: torch.Tensor) -> torch.Tensor:
    """``ops.qk_norm_rope_cache`` with a 4-bit cache: q [T, Hq, D] normed and rotated; k, treated alike, and v are rounded to
    the activations' type, quantised and written to the tokens' slots."""
    ops = _ops()
    qkv = ops.as_tensor(qkv)
    ops._need(qkv, "qkv", None, 2)
    t, width = qkv.shape
    pages, _, hkv, page_size, d = cache.shape
    if (hkv, d) != (num_kv_heads, head_dim) or width != (num_heads + 2 * hkv) * d:
        raise ops.KernelError(f"fp4_qk_norm_rope_cache: rows of {width} for heads {num_heads}/{num_kv_heads} x {head_dim}, "
                              f"cache {tuple(cache.shape)}")
    for x, name in ((positions, "positions"), (slot_mapping, "slot_mapping")):
        ops._need(x, name, torch.int32, 1)
        if x.shape[0] < t:
            raise ops.KernelError(f"fp4_qk_norm_rope_cache: {x.shape[0]} {name} for {t} tokens")
    for w, name in ((q_norm_weight, "q_norm_weight"), (k_norm_weight, "k_norm_weight")):
        if w is not None:
            ops._need(w, name, torch.float32, 1)
            if w.shape[0] != d:
                raise ops.KernelError(f"{name} has {w.shape[0]} elements, head_dim is {d}")
    rotary_dim, max_pos = 0, 0
    if cos_sin is not None:
        ops._need(cos_sin, "cos_sin", torch.float32, 2)
        max_pos, rotary_dim = cos_sin.shape
    _same_device("fp4_qk_norm_rope_cache", qkv, cache.data, positions, slot_mapping,
                 *(x for x in (q_norm_weight, k_norm_weight, cos_sin) if x is not None))
    q = torch.empty(t, num_heads, d, dtype=qkv.dtype, device=qkv.device)
    st = _fn("dib_fp4_qk_norm_rope_cache")(
        qkv.data_ptr(), q.data_ptr(), *cache._pointers(), _pointer(q_norm_weight), _pointer(k_norm_weight), float(eps),
        _pointer(cos_sin), rotary_dim, max_pos, positions.data_ptr(), slot_mapping.data_ptr(), t, num_heads, hkv, d, page_size,
        pages, _code(qkv.dtype, "qkv"), _stream("fp4_qk_norm_rope_cache", qkv.device))
    _done(st, "fp4_qk_norm_rope_cache", lambda: f"head_dim {d}, rotary_dim {rotary_dim}")
    return q


def fp4_cache_read(cache: Fp4Cache, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16):
    """(k, v) [T, Hkv, D] in ``dtype``: what the rows ``slots`` (int32 [T]) of the cache stand for; zeros for a negative
    slot."""
    pages, _, hkv, page_size, d = cache.shape
    _require(slots, "slots", torch.int32, 1)
    device = cache.device
    if slots.device != device:
        _same_device("fp4_cache_read", cache.data, slots)
    code = _code(dtype, "out")
    t = slots.shape[0]
    k, v = torch.empty(2, t, hkv, d, dtype=dtype, device=device).unbind(0)
    st = _fn("dib_fp4_cache_read")(*cache._pointers(), slots.data_ptr(), k.data_ptr(), v.data_ptr(), t, hkv, d, page_size, pages,
                                   code, _stream("fp4_cache_read", device))
    _done(st, "fp4_cache_read", lambda: f"heads {hkv} x {d}")
    return k, v


# ---- attention: a step's work is one launch of the split form for the sequences with one new token, one for those with a
# few, and the prompt form for those with many

# Rows (new tokens x query heads of a kv head) of a sequence of drafted tokens above which they take the prompt form (bfloat16).  By
# the sequence's own rows, so that its bits do not depend on the step; a prompt's portions take it whatever their rows.
PROMPT_ROWS = 32
# Bytes of bfloat16 pages that a launch of the prompt form makes of its sequences' keys and values, one sequence at least (and all
# with 4,096 new tokens or more).
PAGES_BYTES = 1 << 30
PAGE = 128
SPLIT_SEQS = 4096      # sequences of a launch of the stream and split forms, whose CTAs keep their lengths in shared memory
# Bytes of partial results up to which a launch takes sequences of any sizes.  Every sequence of a launch has the room of the one with the most;
# beyond this, sequences whose own room is less than half of that are launched by themselves.
PARTIAL_BYTES = 1 << 28
PARTIAL_ROW = 528      # bytes: 128 sums, two references, a sum of weights


def _split_fits(d: int, page_size: int) -> bool:
    """Shapes that the split form takes: four keys lie in one page, their block scales on 8 bytes."""
    return d <= 128 and d % 32 == 0 and page_size >= 4 and page_size & (page_size - 1) == 0


@functools.lru_cache(maxsize=1 << 16)
def _most_runs(kv_len: int) -> int:
    """The most runs of a sequence of at most ``kv_len`` keys, whatever its rows (the lengths on the device may be less than the
    host's)."""
    keys = _ops()._lib("attention_fp4").dib_fp4_attention_split_keys
    return max(1, max(-(-n // keys(n, 1)) for n in (min(kv_len, 2048), kv_len)))


class _SplitPart:
    """The sequences of one launch: their number, the most rows of one, rows a tile, the most work items of one."""

    def __init__(self, seqs: list, q_lens: list, kv_lens: list, group: int, hkv: int, stream: bool, device, sizes=None):
        self.form = "dib_fp4_attention_stream" if stream else "dib_fp4_attention_split"
        self.first, self.count, self.list = seqs[0], len(seqs), None
        if seqs != list(range(seqs[0], seqs[0] + len(seqs))):
            self.list = torch.tensor(seqs, dtype=torch.int32).to(device, non_blocking=True)
        self.list_pointer = _pointer(self.list)
        self.max_rows, self.tile_rows, self.items, self.runs = sizes or _split_sizes(seqs, q_lens, kv_lens, group, hkv, stream)
        self.rows = self.count * self.items * self.tile_rows if self.runs else 0


def _split_sizes(seqs: list, q_lens: list, kv_lens: list, group: int, hkv: int, stream: bool) -> tuple:
    """Of a launch: the most rows of a sequence, rows a tile, the most work items of a sequence, the most runs of one (0: all have
    one, and there is nothing to add up)."""
    longest: dict = {}      # keys, by new tokens: the bounds below grow with both
    for s in seqs:
        n, keys = q_lens[s], kv_lens[s]
        if keys > longest.get(n, -1):
            longest[n] = keys
    max_rows = max(longest) * group
    tile_rows = 4 if stream and max_rows <= 4 else 8 if max_rows <= 8 else 16
    items = most = 1
    for n, keys in longest.items():
        tiles, runs = -(-n * group // tile_rows), _most_runs(keys)
        # (runs get longer with the rows: tiles times runs is at most the tiles' number and twice that of the shortest runs)
        items, most = max(items, hkv * min(tiles * runs, tiles + 2 * runs)), max(most, runs)
    return max_rows, tile_rows, items, most if most > 1 else 0


def _split_launches(seqs: list, q_lens: list, kv_lens: list, group: int, hkv: int, stream: bool) -> list:
    """Every launch's sequences and sizes: one launch, but for sequences that would only widen the others' partial results."""
    def measured(some: list) -> tuple:      # sizes, bytes of partial results
        sizes = _split_sizes(some, q_lens, kv_lens, group, hkv, stream)
        return sizes, len(some) * sizes[2] * sizes[1] * PARTIAL_ROW if sizes[3] else 0

    launches = []
    for i in range(0, len(seqs), SPLIT_SEQS):
        some = seqs[i:i + SPLIT_SEQS]
        sizes, room = measured(some)
        while room > PARTIAL_BYTES:
            own = {s: measured([s])[1] for s in some}
            half = max(own.values()) // 2
            large, rest = [s for s in some if own[s] > half], [s for s in some if own[s] <= half]
            if not rest:
                break
            launches.append((large, measured(large)[0]))
            some, (sizes, room) = rest, measured(rest)
        launches.append((some, sizes))
    return launches


class _PromptPart:
    """The sequences of one launch of the prompt form: the pages that hold their keys and values in bfloat16, and what the
    attention over them needs to know of the step."""

    def __init__(self, seqs: list, q_lens: list, kv_lens: list, meta, device):
        pages = [-(-max(kv_lens[s], 1) // PAGE) for s in seqs]
        first = [0]
        for n in pages:
            first.append(first[-1] + n)
        self.count, self.most, self.pages = len(seqs), max(pages), first[-1]
        b = len(q_lens)
        table = torch.zeros(b, self.most, dtype=torch.int32)
        for s, at, n in zip(seqs, first, pages):
            table[s, :n] = torch.arange(at, at + n, dtype=torch.int32)
        chosen = set(seqs)
        own = [n if s in chosen else 0 for s, n in enumerate(q_lens)]
        ints = torch.cat([torch.tensor(seqs + first, dtype=torch.int32), table.flatten(),
                          torch.tensor([s in chosen for s in range(b)], dtype=torch.int32)]).to(device, non_blocking=True)
        self.ints, n = ints, len(seqs)
        self.seqs, self.first = ints[:n].data_ptr(), ints[n:2 * n + 1].data_ptr()
        # The attention adds up the chunks of long rows of every token that has some: those of other sequences must not, so
        # their lengths are 0 there.
        self.mask = None if len(chosen) == b else ints[2 * n + 1 + b * self.most:]
        self.meta = SimpleNamespace(block_table=ints[2 * n + 1:2 * n + 1 + b * self.most].view(b, self.most), q_lens=own,
                                    kv_lens=[n if s in chosen else 0 for s, n in enumerate(kv_lens)], num_decode=0, scratch={})


class _Parts(list):
    """A step's launches.  Their lists, and those that the prompt attention keeps with them, are copied to the device by the first call
    on the step, on its stream: calls on other streams wait for ``ready``."""
    stream, ready = None, None

    def wait(self, stream: int) -> None:
        if self.stream != stream and self.ready is not None and not torch.cuda.is_current_stream_capturing():
            torch.cuda.current_stream().wait_event(self.ready)      # (a capture begins when the device is idle)

    def made(self, stream: int) -> None:
        self.stream = stream
        if any(isinstance(p, _PromptPart) or p.list is not None for p in self) and not torch.cuda.is_current_stream_capturing():
            self.ready = torch.cuda.Event()
            self.ready.record()


def _parts(meta, group: int, hkv: int, d: int, page_size: int, prompts: bool, stream: bool, portions: bool, device) -> list:
    """The step's launches: the sequences with one new token, those with a few, those of the prompt form (bfloat16: all others
    that are portions of prompts, or those with many drafted tokens)."""
    key = ("fp4", group, hkv, d, page_size, prompts, stream, portions)
    parts = meta.scratch.get(key)
    if parts is None:
        from . import attention_bf16
        q_lens, kv_lens = list(meta.q_lens), [max(a, b) for a, b in zip(meta.q_lens, meta.kv_lens)]
        if not len(q_lens) == len(meta.kv_lens) <= meta.block_table.shape[0]:
            raise _ops().KernelError(f"fp4_paged_attention: {len(q_lens)} q_lens and {len(meta.kv_lens)} kv_lens for a block table "
                                     f"of {meta.block_table.shape[0]} sequences")
        prompts = prompts and attention_bf16.supports(group * hkv, hkv, d, PAGE)
        one = [s for s, n in enumerate(q_lens) if n == 1]
        many = [s for s, n in enumerate(q_lens) if n > 1 and prompts and (portions or n * group > PROMPT_ROWS)]
        few = sorted({s for s, n in enumerate(q_lens) if n > 1} - set(many))
        # A launch's attention adds up chunks of keys of every token of the step, and takes those of the other launches, whose
        # sequences have no key there, for tokens in front of the first key: fewer than a chunk's number of them lie in the first
        # chunk and are left alone.  Sequences of more are all in the last launch that adds up chunks.  Those of more keys than it
        # adds up take another kernel, which is by the launch's longest: they follow in launches of their own.
        far = [s for s in many if kv_lens[s] > attention_bf16.MAX_CHUNKS * attention_bf16.CHUNK_TILES * PAGE]
        long = [s for s in many if q_lens[s] >= attention_bf16.CHUNK_TILES * PAGE and s not in far]
        parts, some, used = _Parts(), [], 0
        room = max(1, PAGES_BYTES // (4 * hkv * PAGE * d))
        for s in [s for s in many if s not in long and s not in far] + long + far:
            n = -(-kv_lens[s] // PAGE)
            if some and (used + n > room and s not in long[1:] or s in far[:1]):
                parts.append(_PromptPart(some, q_lens, kv_lens, meta, device))
                some, used = [], 0
            some.append(s)
            used += n
        if some:
            parts.append(_PromptPart(some, q_lens, kv_lens, meta, device))
        parts += [_SplitPart(x, q_lens, kv_lens, group, hkv, stream, device, sizes)
                  for y in (one, few) for x, sizes in _split_launches(y, q_lens, kv_lens, group, hkv, stream)]
        meta.scratch[key] = parts
    return parts


def _prompt(q, out, cache: Fp4Cache, meta, part: _PromptPart, scale: float, window: int, stream: int) -> None:
    from . import attention_bf16
    pages, _, hkv, page_size, d = cache.shape
    held = torch.empty(part.pages, 2, hkv, PAGE, d, dtype=torch.bfloat16, device=q.device)
    own = SimpleNamespace(**vars(part.meta), cu_q_lens=meta.cu_q_lens, token_seq=meta.token_seq, seq_lens=meta.seq_lens)
    if part.mask is not None and max(own.kv_lens) > attention_bf16.CHUNK_TILES * PAGE:
        own.seq_lens = meta.seq_lens[:len(own.q_lens)] * part.mask
    st = _fn("dib_fp4_unpack_pages")(*cache._pointers(), pages, meta.block_table.data_ptr(), meta.block_table.shape[1],
                                     meta.cu_q_lens.data_ptr(), meta.seq_lens.data_ptr(), part.seqs, part.first, part.count, part.most,
                                     held.data_ptr(), hkv, d, page_size, window, stream)
    _done(st, "fp4_paged_attention", lambda: f"head_dim {d}, kv heads {hkv}, {part.pages} pages")
    attention_bf16.run(q, out, held, own, scale, window)
    # (tokens in front of the first key, and those that see a row that is no number)
    st = _fn("dib_fp4_finish_portions")(cache.exponents.data_ptr(), pages, meta.block_table.data_ptr(), meta.block_table.shape[1],
                                        meta.cu_q_lens.data_ptr(), meta.seq_lens.data_ptr(), part.seqs, part.count, part.most,
                                        out.data_ptr(), q.shape[1], hkv, d, page_size, window, stream)
    _done(st, "fp4_paged_attention", lambda: f"head_dim {d}, heads {q.shape[1]}")


def _split(q, out, cache: Fp4Cache, meta, part: _SplitPart, scale: float, window: int, stream: int) -> None:
    pages, _, hkv, page_size, d = cache.shape
    hq, rows = q.shape[1], part.rows
    held = torch.empty(rows * PARTIAL_ROW, dtype=torch.uint8, device=q.device) if rows else None      # sums, (references, sum of weights)
    partial = _pointer(held)
    st = _fn(part.form)(
        q.data_ptr(), out.data_ptr(), *cache._pointers(), pages, meta.block_table.data_ptr(), meta.block_table.shape[1],
        meta.cu_q_lens.data_ptr(), meta.seq_lens.data_ptr(), part.list_pointer, part.first, part.count, part.max_rows, part.tile_rows,
        partial, partial + rows * 512, part.items, part.runs, hq, hkv, d, page_size, scale, window, _ops()._DT[q.dtype],
        _sms(q.device), stream)
    _done(st, "fp4_paged_attention", lambda: f"head_dim {d}, heads {hq}/{hkv}, {part.count} sequences", 2 if rows else 1)


def _require_entries(t, name: str, n: int) -> None:
    _require(t, name, torch.int32, 1)
    if t.shape[0] < n:
        raise _ops().KernelError(f"fp4_paged_attention: {name} has {t.shape[0]} entries, the step needs {n}")


def fp4_paged_attention(q: torch.Tensor, cache: Fp4Cache, meta, scale: float, window=None,
                        portions: bool = False) -> torch.Tensor:
    """Causal attention of every token of the step over its sequence's keys in the cache, as ``ops.paged_attention``: q
    [T, Hq, D] float32 or bfloat16, ``meta`` the step's ``AttentionMeta`` (lists that it keeps for later calls are the same for
    all of them; calls on one step may run on several streams).  A sequence's new tokens are its last ones (``seq_lens`` counts
    them); each sees the keys up to its own position, the last ``window`` of them if given.  Keys and values enter the products
    as what their codes and block scales stand for, exactly; the rows' powers of two join scores and probabilities in float32.
    A token that sees no key gives zeros.

    ``portions``: the sequences with more than one new token bring portions of prompts.  In bfloat16 they then all take one
    form, which makes bfloat16 pages of their keys and values and runs the prompt attention of the unquantised cache over
    them.  Otherwise they count as drafted tokens, few of which are faster in another form, chosen by their number."""
    ops = _ops()
    if not (isinstance(q, torch.Tensor) and q.is_cuda and q.dim() == 3 and q.is_contiguous()):
        ops._need(q, "q", None, 3)
    if not isinstance(cache, Fp4Cache):
        raise ops.KernelError("fp4_paged_attention: cache must be an Fp4Cache")
    code = _code(q.dtype, "q")
    t, hq, d = q.shape
    pages, _, hkv, page_size, d2 = cache.shape
    if d2 != d or hq < 1 or hq % hkv:
        raise ops.KernelError(f"fp4_paged_attention: q {tuple(q.shape)} vs cache {tuple(cache.shape)}")
    table, token_seq, cu, lens = meta.block_table, meta.token_seq, meta.cu_q_lens, meta.seq_lens
    device, whole = cache.data.device, torch.int32
    _require(table, "block_table", whole, 2)
    b = table.shape[0]
    if not (isinstance(token_seq, torch.Tensor) and token_seq.dtype is whole and token_seq.dim() == 1 and token_seq.shape[0] >= t
            and isinstance(cu, torch.Tensor) and cu.dtype is whole and cu.dim() == 1 and cu.shape[0] > b
            and isinstance(lens, torch.Tensor) and lens.dtype is whole and lens.dim() == 1 and lens.shape[0] >= b
            and q.device == device and table.device == device and token_seq.device == device and cu.device == device
            and lens.device == device and token_seq.is_contiguous() and cu.is_contiguous() and lens.is_contiguous()):
        _require_entries(token_seq, "token_seq", t)
        _require_entries(cu, "cu_q_lens", b + 1)
        _require_entries(lens, "seq_lens", b)
        _same_device("fp4_paged_attention", cache.data, q, table, token_seq, cu, lens)
    win = int(window) if window else 0
    if win < 0:
        raise ops.KernelError(f"fp4_paged_attention: a window of {win} keys")
    if win >= table.shape[1] * page_size:      # every key that the table has room for (and what is beyond 32 bits is cut there)
        win = 0
    out = torch.empty_like(q)
    if t == 0:
        return out
    stream = _stream("fp4_paged_attention", device)
    if _split_fits(d, page_size) and q.data_ptr() % 16 == 0 and cache.scales.data_ptr() % 8 == 0 and cache.exponents.data_ptr() % 4 == 0 \
            and pages * 2 * hkv * page_size < 1 << 31:
        # (scores on the cache's codes as they are: bfloat16 queries, heads that are whole steps of 64 values)
        stream_form = code == 1 and d % 64 == 0 and cache.scales.data_ptr() % 16 == 0
        # (the prompt attention masks scores before it scales them)
        parts = _parts(meta, hq // hkv, hkv, d, page_size, code == 1 and scale > 0, stream_form, bool(portions), device)
        if parts.stream != stream:
            parts.wait(stream)
        for part in parts:
            run = _prompt if isinstance(part, _PromptPart) else _split
            run(q, out, cache, meta, part, float(scale), win, stream)
        if parts.stream is None:
            parts.made(stream)
        return out
    st = _fn("dib_fp4_attention_any")(
        q.data_ptr(), out.data_ptr(), *cache._pointers(), table.data_ptr(), table.shape[1], token_seq.data_ptr(), cu.data_ptr(),
        lens.data_ptr(), t, hq, hkv, d, page_size, pages, float(scale), win, code, stream)
    _done(st, "fp4_paged_attention", lambda: f"head_dim {d}, heads {hq}/{hkv}")
    return out
