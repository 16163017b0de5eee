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
from ctypes import c_float, c_int, c_longlong, c_void_p

import torch

MAX_K = 1 << 24
MAX_HEAD_DIM = 256
BLOCK = 16


# What the host does in front of a launch is kept short, as in the 8-bit operators: the C functions are looked up once, with their
# argument types; an argument is looked at in one expression, and the check that words the error runs only where that fails.
_P, _I, _L, _F = c_void_p, c_int, c_longlong, c_float
_SIGNATURES = {
    "dib_fp4_quantize_rows": ("rows_fp4", (_P, _L, _P, _P, _P, _L, _I, _I, _P)),
    "dib_fp4_read_rows": ("rows_fp4", (_P, _P, _P, _P, _L, _I, _I, _P)),
    "dib_fp4_layout_rows": ("rows_fp4", (_P, _P, _P, _P, _P, _P, _L, _I, _P)),
    "dib_gemm_fp4": ("gemm_fp4", (_P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _P)),
    "dib_fp4_linear": ("gemm_fp4", (_P, _P, _L, _I, _I, _P, _P, _P, _P, _P, _I, _I, _I, _I, _P)),
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
    uint8, the block scales in tiles of 128 rows x 64 values, ``units`` float32 [R], 2^E (NaN: no numbers)."""

    def _allocate(self, rows: int, k: int, device) -> None:
        self.codes = torch.empty(rows, _code_bytes(k), dtype=torch.uint8, device=device)
        self.tiles = torch.empty(_tile_bytes(rows, k), dtype=torch.uint8, device=device)
        self.units = torch.empty(rows, dtype=torch.float32, device=device)
        self.k = k

    def _quantize(self, x: torch.Tensor, name: str) -> None:
        code = _check_rows(x, name)
        m, k = x.shape
        self._allocate(m, k, x.device)
        st = _fn("dib_fp4_quantize_rows")(x.data_ptr(), x.stride(0), self.codes.data_ptr(), self.tiles.data_ptr(),
                                          self.units.data_ptr(), m, k, code, _stream("fp4_quantize_rows", x.device))
        _done(st, "fp4_quantize_rows", lambda: f"rows {m} x {k}")

    @property
    def shape(self):
        return torch.Size((self.codes.shape[0], self.k))

    @property
    def device(self):
        return self.codes.device

    def tensor(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values the codes stand for [R, K]; exact in float32, rounded once in bfloat16."""
        code, (m, k) = _code(dtype, "tensor"), self.shape
        out = torch.empty(m, k, dtype=dtype, device=self.device)
        st = _fn("dib_fp4_read_rows")(self.codes.data_ptr(), self.tiles.data_ptr(), self.units.data_ptr(), out.data_ptr(), m, k,
                                      code, _stream("tensor", self.device))
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
        st = _fn("dib_fp4_layout_rows")(codes.data_ptr(), block_scales.data_ptr(), exponents.data_ptr(), self.codes.data_ptr(),
                                        self.tiles.data_ptr(), self.units.data_ptr(), n, k, _stream("Fp4Weight", codes.device))
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
        self.units = self.units.clone()


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
    codes = weight.codes
    device = codes.device
    if x.device != device:
        _same_device("fp4_linear", x, weight)
    n = codes.shape[0]
    out_dtype = out_dtype or x.dtype
    out_code = _code(out_dtype, "out")
    out = torch.empty(m, n, dtype=out_dtype, device=device)
    if rows:
        st = _fn("dib_gemm_fp4")(x.codes.data_ptr(), x.tiles.data_ptr(), x.units.data_ptr(), codes.data_ptr(),
                                 weight.tiles.data_ptr(), weight.units.data_ptr(), out.data_ptr(), m, n, k, out_code, _sms(device),
                                 _stream("fp4_linear", device))
    else:
        # block scales, codes, units
        work = torch.empty(_tile_bytes(m, k) + m * (_code_bytes(k) + 4), dtype=torch.uint8, device=device)
        st = _fn("dib_fp4_linear")(_address("dib_fp4_quantize_rows"), x.data_ptr(), x.stride(0), code, k, work.data_ptr(),
                                   codes.data_ptr(), weight.tiles.data_ptr(), weight.units.data_ptr(), out.data_ptr(), m, n,
                                   out_code, _sms(device), _stream("fp4_linear", device))
    _done(st, "fp4_linear", lambda: f"M={m} N={n} K={k}", 1 if rows else 2)
    return out


def force_product_form(form: int) -> None:
    """Measurement and test switch of the product: tiles of 128 x 64, 128 x 128 or 128 x 192 (0, 1, 2), the pair of CTAs (3),
    clusters that share k (4, up to 128 rows), whatever the sizes; -1: the library's own choice.  All give the same bits."""
    _ops()._lib("gemm_fp4").dib_gemm_fp4_force_form(c_int(form))
