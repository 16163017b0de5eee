"""The operators in 4-bit floating point by themselves: rows, product, cache and attention against plain forms in 64 bits."""

from __future__ import annotations

import pytest
import torch

from deterministic_inference_b200.kernels import fp4, ops
from tests.fp4_util import Fp4Case, quantised, rounded, values

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _rand(*shape, seed=0, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).cuda().to(dtype)


def _same_rows(rows, x):
    codes, scales, exponents = quantised(x)
    k = x.shape[1]
    assert torch.equal(rows.codes[:, :codes.shape[1]], codes) and not rows.codes[:, codes.shape[1]:].any()
    assert torch.equal(rows.block_scales().view(torch.uint8), scales.view(torch.uint8))
    assert torch.equal(rows.exponents(), exponents)
    want = values(codes, scales, exponents, k)
    for dtype in (F32, BF16):
        assert torch.equal(rows.tensor(dtype).nan_to_num(7.0), want.to(dtype).nan_to_num(7.0))


# ---- rows

@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,k", [(1, 1), (3, 15), (2, 16), (5, 17), (130, 33), (9, 256), (7, 257), (4, 1000), (300, 64), (2, 4096),
                                 (1, 12288), (3, 8208), (2, 20000), (1, 32768), (2, 33001)])
def test_rows(m, k, dtype):
    x = _rand(m, k, seed=m + k, dtype=dtype) * torch.exp2(torch.randint(-20, 20, (m, 1), generator=torch.Generator().manual_seed(k))).cuda().to(dtype)
    x[:, ::7] *= 0.01
    _same_rows(ops.fp4_quantize_rows(x), x)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("extra,at", [(1, 1), (16, 0), (5, 3)])
def test_rows_that_lie_apart(extra, at, dtype):
    wide = _rand(9, 96 + extra, seed=extra, dtype=dtype)
    x = wide[:, at:at + 96]
    _same_rows(ops.fp4_quantize_rows(x), x)
    _same_rows(ops.fp4_quantize_rows(wide[::2, at:at + 96]), wide[::2, at:at + 96])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,k", [(10000, 48), (2500, 1000), (700, 4096), (300, 20000), (300, 33000)])
def test_more_rows_than_are_worked_on_at_once(m, k, dtype):
    x = _rand(m, k, seed=k, dtype=dtype) * (1 + torch.arange(m, device="cuda")[:, None] % 7).to(dtype)
    _same_rows(ops.fp4_quantize_rows(x), x)


def test_rows_next_to_borders():
    """Values on a border between two codes, and a float32 step to either side; blocks whose scale is rounded up and down, and
    blocks too small beside the row's largest for a scale of their own."""
    b = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    near = torch.cat([b, torch.nextafter(b, b * 0), torch.nextafter(b, b * 9), -b])       # 28 values
    rows = []
    for unit in (1.0, 1.125, 1.875, 2.0 ** -7, 448.0, 0.3):
        block = torch.cat([torch.tensor([6.0]), near[:15]]) * unit, torch.cat([torch.tensor([-6.0]), near[13:28]]) * unit
        rows.append(torch.cat([*block, torch.full((16,), unit * 2.0 ** -9), torch.full((16,), unit * 2.0 ** -20)]))
    x = torch.stack(rows).cuda()
    _same_rows(ops.fp4_quantize_rows(x), x)
    _same_rows(ops.fp4_quantize_rows(x.to(BF16)), x.to(BF16))


def test_every_code_of_every_block_scale():
    """All finite block scales against multiples of a 64th of their units: what a code is rounded to, ties among them, does not
    depend on whether its quotient is one of 8 or of 24 digits."""
    scales = torch.arange(1, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    at = torch.arange(-390, 391).float() / 64
    blocks = (scales[:, None, None] * torch.cat([at, torch.full((15 * 53 - at.numel(),), 0.125)]).reshape(1, 53, 15))
    blocks = torch.cat([(scales * 6.0)[:, None, None].expand(-1, 53, 1), blocks.clamp(-6 * scales[:, None, None], 6 * scales[:, None, None])], 2)
    x = torch.cat([torch.full((126, 16), 2688.0), blocks.reshape(126, 53 * 16)], 1).cuda()
    for unit in (2.0 ** -90, 1.0, 2.0 ** 100):
        _same_rows(ops.fp4_quantize_rows(x * unit), x * unit)
        _same_rows(ops.fp4_quantize_rows((x * unit).to(BF16)), (x * unit).to(BF16))


def test_rows_of_no_numbers_zeros_and_extremes():
    x = _rand(8, 80, seed=4)
    x[1, 7], x[2, 33], x[3] = float("nan"), -float("inf"), 0.0
    x[4], x[5], x[6], x[7] = x[4] * 1e-37, x[5] * 3e-45, x[6] * 2.0 ** 100, -0.0
    rows = ops.fp4_quantize_rows(x)
    _same_rows(rows, x)
    back = rows.tensor()
    assert back[1:3].isnan().all() and not back[3].any() and back[6].isfinite().all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n,k", [(1, 16), (130, 33), (257, 1000), (128, 256), (64, 4112)])
def test_weights(n, k, dtype):
    w = _rand(n, k, seed=n, dtype=dtype)
    made = ops.Fp4Weight.of(w)
    _same_rows(made, w)
    given = ops.Fp4Weight(*quantised(w), k)
    for a, b in ((made.codes, given.codes), (made.units, given.units), (made.block_scales().view(torch.uint8), given.block_scales().view(torch.uint8))):
        assert torch.equal(a, b)
    assert made.shape == given.shape == (n, k)


# ---- product

def _check_product(y, x, w, out_dtype):
    """Sums in float32 on exact products: a rounding of at most 2^-23 of the sum of magnitudes for each 64 values (the tensor
    core's own way of adding 64 products in float32, two steps), each part of k and each power of two; then the output's."""
    a, b = rounded(x), values(w.codes, torch.nn.functional.pad(w.block_scales().float(), (0, 0)).to(torch.float8_e4m3fn), w.exponents(), x.shape[1])
    want, mass = a @ b.t(), a.abs() @ b.abs().t()
    tol = (2 * (x.shape[1] / 64 + 1) + 8 + 2) * 2.0 ** -23 * mass
    if out_dtype == BF16:
        tol = tol + 2.0 ** -8 * want.abs()
    off = (y.double() - want).abs()
    assert y.dtype == out_dtype and (off <= tol).all(), (off - tol).max().item()


SIZES = [(1, 1, 1), (1, 8, 64), (3, 33, 100), (8, 128, 256), (9, 200, 2048), (16, 1000, 4096), (31, 70, 333), (32, 4096, 1024),
         (33, 96, 5000), (64, 384, 12288), (127, 129, 2064), (128, 640, 4100), (129, 257, 300), (256, 192, 4096), (300, 1000, 2500),
         (520, 64, 512), (1, 24576, 512)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product(m, n, k, dtype):
    x, w = _rand(m, k, seed=m, dtype=dtype), ops.Fp4Weight.of(_rand(n, k, seed=n, scale=0.05))
    x[:, ::61] *= 12
    _check_product(ops.fp4_linear(x, w), x, w, dtype)
    rows = ops.fp4_quantize_rows(x)
    other = BF16 if dtype == F32 else F32
    y = ops.fp4_linear(rows, w, other)
    _check_product(y, x, w, other)
    assert torch.equal(ops.linear(x, w, other), y)
    ops.check_kernel_status()


@pytest.mark.parametrize("m,n,k", SIZES)
def test_every_form_gives_the_same_bits(m, n, k):
    """Tiles, pairs and clusters; rows of values that leave sums that float32 has to round."""
    x, w = _rand(m, k, seed=m + 1), ops.Fp4Weight.of(_rand(n, k, seed=n + 1))
    x *= torch.exp2(torch.randint(-6, 6, (m, k), generator=torch.Generator().manual_seed(k))).cuda()
    try:
        fp4.force_product_form(0)
        want = ops.fp4_linear(x, w)
        for form in (1, 2, 3, 4):
            fp4.force_product_form(form)
            assert torch.equal(ops.fp4_linear(x, w), want), f"form {form}"
            ops.check_kernel_status()
    finally:
        fp4.force_product_form(-1)
    assert torch.equal(ops.fp4_linear(x, w), want)


@pytest.mark.parametrize("n,k", [(1000, 4096), (4096, 1300)])
def test_a_row_has_the_same_bits_in_any_batch(n, k):
    x, w = _rand(700, k, seed=3, dtype=BF16), ops.Fp4Weight.of(_rand(n, k, seed=4))
    whole = ops.fp4_linear(x, w, F32)
    for a, b in ((0, 1), (5, 13), (0, 40), (100, 228), (300, 600), (699, 700)):
        assert torch.equal(ops.fp4_linear(x[a:b], w, F32), whole[a:b])


def test_product_of_rows_that_are_no_numbers():
    x, w = _rand(20, 512, seed=1), _rand(300, 512, seed=2)
    good = ops.fp4_linear(x, ops.Fp4Weight.of(w))
    x[3, 100], x[17, 0], w[7, 5] = float("nan"), float("inf"), float("nan")
    y = ops.fp4_linear(x, ops.Fp4Weight.of(w))
    bad = torch.zeros(20, 300, dtype=torch.bool, device="cuda")
    bad[3], bad[17], bad[:, 7] = True, True, True
    assert torch.equal(y.isnan(), bad) and torch.equal(y[~bad], good[~bad])


@pytest.mark.parametrize("m", [3, 200])
@pytest.mark.parametrize("x_scale,w_scale", [(2.0 ** 110, 2.0 ** -105), (2.0 ** -95, 2.0 ** 115), (2.0 ** 60, 2.0 ** 40), (2.0 ** -60, 2.0 ** -50)])
def test_product_of_large_and_small_rows(m, x_scale, w_scale):
    """Rows and channels whose powers of two are far apart: no step on the way overflows or vanishes where the result does not."""
    x, w = _rand(m, 300, seed=m) * x_scale, ops.Fp4Weight.of(_rand(130, 300, seed=5) * w_scale)
    y = ops.fp4_linear(x, w)
    a, b = values(*quantised(x), 300, torch.float64), w.tensor().double()
    want, mass = a @ b.t(), a.abs() @ b.abs().t()
    assert y.isfinite().all() and ((y.double() - want).abs() <= 30 * 2.0 ** -23 * mass).all()      # as in _check_product
    swapped = ops.fp4_linear(ops.fp4_quantize_rows(w.tensor()), ops.Fp4Weight.of(x))
    assert ((swapped.double() - want.t()).abs() <= 30 * 2.0 ** -23 * mass.t()).all()


def test_product_with_no_rows():
    w = ops.Fp4Weight.of(_rand(32, 64))
    assert ops.fp4_linear(torch.empty(0, 64, device="cuda"), w).shape == (0, 32)
    rows = ops.fp4_quantize_rows(torch.empty(0, 5, device="cuda", dtype=BF16))
    assert rows.shape == (0, 5) and rows.tensor().shape == (0, 5)


def test_gated_product():
    x, w = _rand(70, 128, dtype=BF16), ops.Fp4Weight.of(_rand(512, 128, seed=5))
    assert torch.equal(ops.as_tensor(ops.gated_linear(x, w)), ops.silu_mul(ops.fp4_linear(x, w)))


# ---- cache

def _held(cache, slots, page):
    at = slots.long()
    return [(cache.data[at // page, kv, :, at % page], cache.scales[at // page, kv, :, at % page], cache.exponents[at // page, kv, :, at % page])
            for kv in (0, 1)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("t,hkv,d,page", [(1, 1, 16, 1), (1, 8, 128, 16), (7, 3, 48, 5), (33, 2, 64, 8), (130, 8, 128, 16),
                                          (9, 4, 256, 32), (5, 1, 144, 64), (1000, 2, 96, 16)])
def test_cache_write_and_read(t, hkv, d, page, dtype):
    cache = ops.Fp4Cache.zeros(t // page + 4, hkv, page, d)
    cache.exponents.fill_(255)
    slots = torch.randperm(cache.shape[0] * page, generator=torch.Generator().manual_seed(t))[:t].to(torch.int32).cuda()
    k, v = _rand(t, hkv, d, seed=1, dtype=dtype), _rand(t, hkv, d, seed=2, dtype=dtype, scale=30.0)
    ops.fp4_cache_write(k, v, cache, slots)
    again = ops.Fp4Cache.zeros(*[cache.shape[i] for i in (0, 2, 3, 4)])
    again.exponents.fill_(255)
    got = ops.fp4_cache_read(cache, slots, dtype)
    at = slots.long()
    for kv, x in ((0, k), (1, v)):
        held = quantised(x)
        for a, b in zip(_held(cache, slots, page)[kv], held):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        assert torch.equal(got[kv], values(*held, d).to(dtype))
        for whole, part in zip((again.data, again.scales.view(torch.uint8), again.exponents), held):
            whole[at // page, kv, :, at % page] = part.view(torch.uint8)
    for a, b in ((cache.data, again.data), (cache.scales.view(torch.uint8), again.scales.view(torch.uint8)), (cache.exponents, again.exponents)):
        assert torch.equal(a, b)                    # nothing beside the slots
    ops.reshape_and_cache(k, v, again, slots)
    assert torch.equal(cache.data, again.data)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("extra", [0, 16, 8, 3])
def test_cache_write_of_column_ranges(extra, dtype):
    """Keys and values as column ranges of the fused projection's rows, at any distance and alignment."""
    hkv, d, t = 2, 64, 11
    rows = _rand(t, extra + 5 * d + 2 * hkv * d, seed=extra, dtype=dtype)
    k = rows[:, extra + 4 * d:extra + (4 + hkv) * d].view(t, hkv, d)
    v = rows[:, extra + (4 + hkv) * d:extra + (4 + 2 * hkv) * d].view(t, hkv, d)
    a, b = ops.Fp4Cache.zeros(3, hkv, 8, d), ops.Fp4Cache.zeros(3, hkv, 8, d)
    slots = torch.arange(t, dtype=torch.int32, device="cuda") + 2
    ops.fp4_cache_write(k, v, a, slots)
    ops.fp4_cache_write(k.contiguous(), v.contiguous(), b, slots)
    assert torch.equal(a.data, b.data) and torch.equal(a.exponents, b.exponents) and a.data.any()
    assert torch.equal(a.scales.view(torch.uint8), b.scales.view(torch.uint8))


def test_cache_skips_slots_that_are_none():
    cache = ops.Fp4Cache.zeros(4, 2, 8, 64)
    x = _rand(4, 2, 64, seed=4)
    slots = torch.tensor([-1, 9, 32, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    ops.fp4_cache_write(x, x, cache, slots)
    assert cache.exponents.count_nonzero() == 4 and cache.data[1, :, :, 1].any()
    k, v = ops.fp4_cache_read(cache, slots, F32)
    assert not k[0].any() and not k[2:].any() and torch.equal(k, v) and k[1].any()
    ops.fp4_cache_write(x[:0], x[:0], cache, slots)
    assert ops.fp4_cache_read(cache, slots[:0])[0].shape == (0, 2, 64)


def test_cache_rows_that_are_no_numbers():
    cache = ops.Fp4Cache.zeros(2, 1, 8, 32)
    k = _rand(3, 1, 32, seed=8)
    k[1, 0, 4] = float("nan")
    v = k.clone()
    v[2, 0, 0] = -float("inf")
    slots = torch.arange(3, dtype=torch.int32, device="cuda")
    ops.fp4_cache_write(k, v, cache, slots)
    rk, rv = ops.fp4_cache_read(cache, slots, F32)
    assert rk[1].isnan().all() and rv[1:].isnan().all() and rk[[0, 2]].isfinite().all() and rv[0].isfinite().all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("t,hq,hkv,d,rotary,norm", [(1, 16, 8, 128, 128, True), (70, 4, 2, 64, 64, True), (33, 6, 3, 48, 32, True),
                                                    (5, 2, 1, 256, 256, True), (9, 3, 3, 144, 96, False), (200, 8, 1, 128, 0, True)])
def test_norm_rotation_and_write(t, hq, hkv, d, rotary, norm, dtype):
    """Queries as the kernel with an 8-bit cache gives them, whose norm and rotation are the same code, and the cache the
    quantisation of what the kernel with an unquantised cache stores.  (Heads of 128: the same operations in the same order; others:
    another order of the norm's sum, 2^-20 of a value in 32 bits, a step in 16, and then now and then a code or scale next to it.)"""
    g = torch.Generator().manual_seed(t + d)
    qkv = torch.randn(t, (hq + 2 * hkv) * d, generator=g).cuda().to(dtype)
    weights = [(1 + 0.1 * torch.randn(d, generator=g)).cuda() if norm else None for _ in range(2)]
    table = torch.randn(64, rotary, generator=g).cuda() if rotary else None
    pos, page = torch.randint(0, 64, (t,), generator=g).to(torch.int32).cuda(), 16
    slots = torch.randperm(t + 40, generator=g)[:t].to(torch.int32).cuda()
    if t > 1:
        slots[t // 2] = -1
    pages = (t + 40) // page + 1
    kv = torch.zeros(pages, 2, hkv, page, d, dtype=dtype, device="cuda")
    cache, eight = ops.Fp4Cache.zeros(pages, hkv, page, d), ops.Int8Cache.zeros(pages, hkv, page, d)
    args = (hq, hkv, d, *weights, 1e-6, table, pos)
    ops.qk_norm_rope_cache(qkv, *args, kv, slots, page)
    want = ops.qk_norm_rope_cache(qkv, *args, eight, slots, page)
    got = ops.qk_norm_rope_cache(qkv, *args, cache, slots, page)
    assert torch.equal(got, want)
    written = torch.zeros(pages * page, dtype=torch.bool, device="cuda")
    written[slots[slots >= 0].long()] = True
    written = written.view(pages, 1, 1, page).expand_as(cache.exponents)
    assert not cache.data[~written].any() and not cache.exponents[~written].any()
    codes, scales, exponents = (x[written] for x in quantised(kv))
    differ = cache.data[written] != codes
    assert differ.double().mean() < (0.04 if d != 128 else 2.0 ** -60)
    if d == 128:
        assert torch.equal(cache.scales.view(torch.uint8)[written], scales.view(torch.uint8)) and torch.equal(cache.exponents[written], exponents)


# ---- attention

def _attend(case, q, q_lens, scale, window=None, kv_lens=None, portions=False):
    out = ops.fp4_paged_attention(q, case.cache(), case.meta(q_lens, kv_lens), scale, window, portions)
    ops.check_kernel_status()
    return out


def _check_attention(case, q_lens, hq, dtype, window=None, kv_lens=None, seed=0, scale=None, q_scale=1.0, portions=False):
    """A score's error: float32 sums of at most 24 steps, 2^-18 of its magnitudes; with bfloat16 queries in four parts of 4 bits,
    each of which leaves at most 0.1771 of a block's largest (half of e2m1's widest step, a sixth of the largest, and e4m3's rounding
    of the scale, a sixteenth): 0.1771^4 < 2^-9.9 of them.  A weight's: float16's half step 2^-11, bfloat16's 2^-8 in the
    prompt form; in two parts of float16 (float32 queries) 2^-21, and sums of at most 40 steps.  Then the output's rounding."""
    q = _rand(sum(q_lens), hq, case.d, seed=seed + 100, dtype=dtype, scale=q_scale)
    scale = case.d ** -0.5 / 32 if scale is None else scale
    out = _attend(case, q, q_lens, scale, window, kv_lens, portions)
    want, vmax, smax = case.attention(q, q_lens, scale, window, kv_lens)
    assert out.dtype == dtype and out.shape == q.shape
    if dtype == F32:
        tol = (2 * smax * 2.0 ** -18 + 2.0 ** -17) * vmax
    else:
        blocks = q.float().unflatten(-1, (-1, 16)).abs().amax(-1, keepdim=True).expand(-1, -1, -1, 16).flatten(-2)
        _, _, most = case.attention(blocks, q_lens, scale, window, kv_lens)
        tol = (2 * (smax * 2.0 ** -18 + most * 2.0 ** -9.9) + 2.0 ** -8) * vmax + 2.0 ** -8 * want.abs()
    err = (out.double() - want).abs()
    assert (err <= tol).all(), f"{(err - tol).max().item()} over, at {(err > tol).nonzero()[:4].tolist()}"
    return out, want


LAYOUTS = [  # (query heads, kv heads, head size, page size)
    (16, 8, 128, 16), (8, 1, 128, 16), (32, 2, 128, 32), (5, 5, 128, 8), (12, 4, 96, 16), (6, 2, 64, 64), (4, 2, 16, 16),
    (6, 3, 48, 24), (20, 1, 128, 256), (40, 1, 64, 16), (2, 1, 256, 16), (4, 4, 32, 1), (7, 1, 144, 48), (3, 1, 96, 4), (8, 2, 128, 4)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hq,hkv,d,page", LAYOUTS)
def test_attention_of_one_token(hq, hkv, d, page, dtype):
    case = Fp4Case([1, 2, 16, 17, 31, 33, 127, 128, 129, 255, 256, 257, 700, 1025], hkv, d, page, seed=d + page)
    _check_attention(case, [1] * len(case.lens), hq, dtype)


@pytest.mark.parametrize("portions", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hq,hkv,d,page", LAYOUTS)
def test_attention_of_mixed_steps(hq, hkv, d, page, dtype, portions):
    case = Fp4Case([40, 1, 300, 5, 70, 9, 520, 64, 130, 333], hkv, d, page, seed=d + page)
    _check_attention(case, [1, 1, 2, 5, 3, 9, 4, 64, 129, 200], hq, dtype, portions=portions)


@pytest.mark.parametrize("portions", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("window", [1, 7, 32, 100, 128, 1000])
@pytest.mark.parametrize("hq,hkv,d,page", [(16, 8, 128, 16), (4, 2, 64, 8), (8, 1, 128, 64), (4, 2, 96, 16)])
def test_attention_in_a_window(hq, hkv, d, page, window, dtype, portions):
    case = Fp4Case([1, 200, 517, 6, 300, 450], hkv, d, page, seed=window)
    _check_attention(case, [1, 1, 1, 6, 77, 300], hq, dtype, window=window, portions=portions)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hq,hkv,d,page", [(16, 8, 128, 16), (4, 2, 64, 8), (2, 1, 80, 4), (4, 2, 96, 8)])
def test_attention_rows_that_see_nothing(hq, hkv, d, page, dtype):
    """More new tokens than keys: the first ones lie before the first key.  A sequence with no key, and one with no token."""
    case = Fp4Case([3, 0, 20, 1], hkv, d, page, seed=9)
    out, _ = _check_attention(case, [5, 2, 0, 6], hq, dtype)
    assert not out[:2].any() and not out[5:7].any() and not out[7:12].any() and out[2].any() and out[12].any()


@pytest.mark.parametrize("portions", [False, True])
@pytest.mark.parametrize("window", [None, 100])
@pytest.mark.parametrize("lens,q_lens", [([20], [50]), ([300, 0, 70], [40, 50, 71]), ([0, 1, 130], [300, 400, 600]),
                                         ([4200, 5], [4500, 40])])
def test_portions_in_front_of_the_first_key(lens, q_lens, window, portions):
    """More new tokens than keys, in numbers for which keys and values become bfloat16 pages; what those lay in before is no
    number."""
    case = Fp4Case(lens, 2, 128, 16, seed=9)
    torch.full((1 << 26,), float("nan"), dtype=BF16, device="cuda")
    out, _ = _check_attention(case, q_lens, 8, BF16, window=window, portions=portions)
    at = 0
    for keys, n in zip(lens, q_lens):
        assert not out[at:at + max(0, n - keys)].any() and (keys == 0 or out[at + n - 1].any())
        at += n


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("q_len", [1, 3, 9, 40])
def test_attention_of_uneven_value_exponents(q_len, dtype):
    """Values over sixty powers of two: against the largest value seen, and (one key alone visible) each by itself."""
    units = lambda n, hkv, g: torch.randint(97, 157, (n, hkv), generator=g).to(torch.uint8)
    case = Fp4Case([q_len + 300, q_len + 37], 2, 128, 16, seed=q_len, exponents=units)
    _check_attention(case, [q_len, q_len], 4, dtype)
    _check_attention(case, [q_len, q_len], 4, dtype, window=1)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("scale", [0.0, -0.003])
def test_attention_of_zero_and_negative_scales(scale, dtype):
    case = Fp4Case([500, 300, 77], 2, 128, 16, seed=8)
    _check_attention(case, [200, 4, 1], 8, dtype, scale=scale)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("q_scale", [1e-30, 3e4, 1e8])
def test_attention_of_small_and_large_queries(q_scale, dtype):
    case = Fp4Case([100, 5], 2, 128, 16, seed=3)
    _check_attention(case, [1, 4], 4, dtype, q_scale=q_scale, scale=0.003 / q_scale)


@pytest.mark.parametrize("d,dtype", [(128, BF16), (64, BF16), (96, BF16), (128, F32), (48, BF16)])
def test_attention_is_off_by_its_rounding(d, dtype):
    """In the root mean square: bfloat16's rounding is 2^-9 of an element at most, 2^-9 / sqrt(3) = 0.0011 to 0.0023 of a row's norm by
    where the elements lie in their binade; the weights' float16 and the queries' parts add 2^-11.  float32: some 2^-20."""
    case = Fp4Case([900, 1500, 300, 64], 2, d, 16, seed=1)
    for q_lens in ([1, 1, 1, 1], [5, 3, 8, 2]):
        q = _rand(sum(q_lens), 8, d, seed=2, dtype=dtype)
        out = _attend(case, q, q_lens, d ** -0.5 / 32)
        want, _, _ = case.attention(q, q_lens, d ** -0.5 / 32)
        off = (out.double() - want).norm(dim=-1) / want.norm(dim=-1)
        assert off.max() < (2.0 ** -8 if dtype == BF16 else 2.0 ** -18)


@pytest.mark.parametrize("d,dtype", [(128, BF16), (64, BF16), (96, BF16), (128, F32)])
@pytest.mark.parametrize("q_len", [1, 8])
def test_attention_query_rows_that_are_no_numbers(q_len, d, dtype):
    case = Fp4Case([260, 260], 2, d, 16, seed=2)
    q = _rand(2 * q_len, 4, d, seed=5, dtype=dtype)
    good = _attend(case, q, [q_len] * 2, 0.003)
    for bad_value in (float("nan"), float("inf")):
        bad = q.clone()
        bad[0, 1, 3] = bad_value
        out = _attend(case, bad, [q_len] * 2, 0.003)
        keep = torch.ones(2 * q_len, 4, dtype=torch.bool)
        keep[0, 1] = False
        assert out[0, 1].isnan().all() and torch.equal(out[keep], good[keep])


@pytest.mark.parametrize("d,dtype,page", [(128, BF16, 16), (64, BF16, 16), (96, BF16, 16), (128, F32, 16), (48, BF16, 5)])
@pytest.mark.parametrize("kv", [0, 1])
@pytest.mark.parametrize("q_len", [1, 5, 16])
def test_attention_rows_of_the_cache_that_are_no_numbers(q_len, kv, d, dtype, page):
    """A key or value row that is no number shows in every row that sees it and in no other."""
    case = Fp4Case([300], 1, d, page, seed=2)
    at = 300 - q_len // 2 - 1
    place = (case.tables[0][at // page], kv, 0, at % page)
    case.exponents[place] = 255
    case.data[place], case.scales[place] = 0, 0            # (as it is written)
    q = _rand(q_len, 2, d, seed=5, dtype=dtype)
    out = _attend(case, q, [q_len], 0.003)
    sees = torch.arange(300 - q_len, 300) >= at
    assert torch.equal(out.isnan().all(-1).all(-1).cpu(), sees) and not out[~sees.cuda()].isnan().any()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kv", [0, 1])
@pytest.mark.parametrize("window", [None, 50])
@pytest.mark.parametrize("q_len", [2, 60, 250])
@pytest.mark.parametrize("hkv,d,page", [(1, 128, 16), (2, 128, 8), (1, 144, 16)])
def test_portions_beside_rows_of_the_cache_that_are_no_numbers(hkv, d, page, q_len, window, kv, dtype):
    """As above for portions of prompts: in the first and the last head's row of a key that some of the tokens see, and of one that a
    window has left."""
    case = Fp4Case([300], hkv, d, page, seed=2)
    q = _rand(q_len, 2 * hkv, d, seed=5, dtype=dtype)
    good = _attend(case, q, [q_len], 0.003, window, portions=True)
    for at, head in ((300 - q_len // 2 - 1, 0), (299, hkv - 1), (300 - q_len - 10, 0), (0, hkv - 1)):
        place = (case.tables[0][at // page], kv, head, at % page)
        held = case.exponents[place].clone()
        case.exponents[place] = 255
        out = _attend(case, q, [q_len], 0.003, window, portions=True)
        case.exponents[place] = held
        pos = torch.arange(300 - q_len, 300)
        sees = torch.zeros(q_len, 2 * hkv, dtype=torch.bool)
        sees[:, 2 * head:2 * head + 2] = ((pos >= at) & (pos < at + (window or 1000)))[:, None]
        sees = sees.cuda()
        assert out[sees].isnan().all() and torch.equal(out[~sees], good[~sees]), (at, head)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("q_len", [1, 5, 90])
@pytest.mark.parametrize("hkv,d,page", [(2, 128, 16), (2, 64, 4), (2, 96, 16), (2, 144, 16), (2, 64, 24)])
def test_pages_that_are_none_of_the_pools(hkv, d, page, q_len, dtype):
    """They are pages of zeros."""
    case = Fp4Case([200, 100], hkv, d, page, seed=5)
    q = _rand(2 * q_len, 2 * hkv, d, seed=4, dtype=dtype)
    zeros = Fp4Case.__new__(Fp4Case)
    zeros.__dict__.update(case.__dict__)
    zeros.scales = case.scales.clone()
    zeros.scales[case.tables[0][2]] = 0
    zeros.exponents = case.exponents.clone()
    zeros.exponents[case.tables[0][2]] = 0
    want = _attend(zeros, q, [q_len] * 2, 0.003)
    for entry in (-1, case.data.shape[0], 2 ** 31 - 1):
        meta = case.meta([q_len] * 2)
        meta.block_table[0, 2] = entry
        assert torch.equal(ops.fp4_paged_attention(q, case.cache(), meta, 0.003), want)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("q_len", [1, 4])
@pytest.mark.parametrize("lens", [[2048, 100, 256, 257], [2049, 2048, 4096], [4096, 4097, 2048, 500], [4600, 4, 4608, 4609]])
def test_attention_of_few_and_many_runs(lens, q_len, dtype):
    """Sequences to either side of the lengths at which a run gets longer, and of those whose runs are added up in another way;
    in steps of any of them alone, too, the same bits."""
    case = Fp4Case(lens, 2, 128, 16, seed=len(lens))
    out, _ = _check_attention(case, [q_len] * len(lens), 6, dtype, window=None)
    _check_attention(case, [q_len] * len(lens), 6, dtype, window=1500)
    q = _rand(q_len * len(lens), 6, 128, seed=100, dtype=dtype)
    for s in range(len(lens)):
        rows = slice(s * q_len, (s + 1) * q_len)
        assert torch.equal(_attend(case.alone(s), q[rows], [q_len], 128 ** -0.5 / 32), out[rows])
    # lengths of the device below the host's, as of a graph that is played again later
    meta = case.meta([q_len] * len(lens))
    short = [max(q_len, n - 1900) for n in lens]
    meta.seq_lens.copy_(torch.tensor(short, dtype=torch.int32))
    less = ops.fp4_paged_attention(q, case.cache(), meta, 128 ** -0.5 / 32)
    assert torch.equal(less, _attend(case, q, [q_len] * len(lens), 128 ** -0.5 / 32, kv_lens=short))


def test_attention_of_long_contexts():
    case = Fp4Case([20000, 9001, 17011], 2, 128, 16, seed=1)
    _check_attention(case, [1, 1, 5], 16, BF16)
    _check_attention(case, [1, 3, 300], 16, BF16)
    _check_attention(case, [1, 1, 2], 16, F32)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_of_more_sequences_than_a_launch_takes(dtype, monkeypatch):
    monkeypatch.setattr(fp4, "SPLIT_SEQS", 40)
    case = Fp4Case([1 + i % 7 * 50 for i in range(150)], 1, 64, 4, seed=1)
    _check_attention(case, [2 if i % 3 == 0 else 1 for i in range(150)], 2, dtype)


def test_attention_of_thousands_of_sequences():
    n = fp4.SPLIT_SEQS + 5
    _check_attention(Fp4Case([1 + i % 7 for i in range(n)], 1, 64, 4, seed=1), [1] * n, 2, BF16)


def test_attention_beyond_32_bits():
    """A cache of more than 2^32 bytes, the sequences on its last pages."""
    first = 2 ** 32 // (2 * 8 * 64 * 64) + 100
    case = Fp4Case([70, 300, 200], 8, 128, 64, seed=4, first_page=first)
    assert case.data.numel() > 2 ** 32 and min(min(t) for t in case.tables) >= first
    _check_attention(case, [1, 4, 150], 16, BF16)
    _check_attention(case, [1, 1, 2], 16, F32)
    cache = case.cache()
    slots = torch.tensor([(case.data.shape[0] - 1) * 64 + 63], dtype=torch.int32, device="cuda")
    x = _rand(1, 8, 128, seed=9)
    ops.fp4_cache_write(x, x, cache, slots)
    assert torch.equal(cache.data[-1, 1, :, 63], quantised(x)[0][0])
    assert torch.equal(ops.fp4_cache_read(cache, slots, F32)[1], rounded(x, F32))


def test_on_another_stream():
    case = Fp4Case([300, 40], 2, 128, 16, seed=1)
    q, w = _rand(9, 4, 128, seed=3, dtype=BF16), ops.Fp4Weight.of(_rand(512, 512, seed=4))
    want, y = _attend(case, q, [1, 8], 0.003), ops.fp4_linear(q.view(9, 512), w)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.fp4_paged_attention(q, case.cache(), case.meta([1, 8]), 0.003)
        z = ops.fp4_linear(q.view(9, 512), w)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(z, y)


# ---- refusals

def _refused(call, *words):
    with pytest.raises(ops.KernelError) as e:
        call()
    for word in words:
        assert word in str(e.value), e.value


def test_refusals():
    cache = ops.Fp4Cache.zeros(3, 2, 16, 64)
    x = _rand(4, 2, 64)
    slots = torch.zeros(4, dtype=torch.int32, device="cuda")
    weight = _rand(32, 64)
    codes, scales, exponents = quantised(weight)
    w = ops.Fp4Weight.of(weight)
    _refused(lambda: ops.fp4_quantize_rows(x[0].cpu()), "CUDA")
    _refused(lambda: ops.fp4_quantize_rows(x[0].half()), "float16")
    _refused(lambda: ops.fp4_quantize_rows(x[0].t()), "consecutive")
    _refused(lambda: ops.fp4_quantize_rows(x[0]).tensor(torch.float16), "float16")
    _refused(lambda: ops.Fp4Weight(codes.int(), scales, exponents, 64), "uint8")
    _refused(lambda: ops.Fp4Weight(codes, scales.float(), exponents, 64), "float8")
    _refused(lambda: ops.Fp4Weight(codes, scales, exponents[:5], 64), "exponents")
    _refused(lambda: ops.Fp4Weight(codes, scales, exponents, 66), "66 values")
    _refused(lambda: ops.Fp4Weight(codes, scales[:, :3].contiguous(), exponents, 64), "block scales")
    _refused(lambda: ops.Fp4Weight(codes.cpu(), scales, exponents, 64), "CUDA")
    _refused(lambda: ops.Fp4Weight.of(torch.zeros(1, 0, device="cuda")), "0 values")
    _refused(lambda: ops.fp4_linear(_rand(2, 65), w), "against weight")
    _refused(lambda: ops.fp4_linear(_rand(2, 64), weight), "Fp4Weight")
    _refused(lambda: ops.fp4_linear(_rand(2, 64), w, torch.float16), "float16")
    _refused(lambda: ops.Fp4Cache(cache.data, cache.scales, cache.exponents[:2]), "exponents")
    _refused(lambda: ops.Fp4Cache(cache.data, cache.scales[:2], cache.exponents), "scales")
    _refused(lambda: ops.Fp4Cache(cache.data, cache.scales.view(torch.uint8), cache.exponents), "float8")
    _refused(lambda: ops.Fp4Cache.zeros(3, 2, 16, 40), "multiple of 16")
    _refused(lambda: ops.Fp4Cache.zeros(3, 2, 16, 272), "at most 256")
    _refused(lambda: ops.fp4_cache_write(x[:, :1], x[:, :1], cache, slots), "heads")
    _refused(lambda: ops.fp4_cache_write(x, x.bfloat16(), cache, slots), "bfloat16")
    _refused(lambda: ops.fp4_cache_write(x, x, cache, slots[:2]), "slots")
    _refused(lambda: ops.fp4_cache_write(x, x, cache, slots.long()), "int32")
    _refused(lambda: ops.fp4_cache_write(x.transpose(1, 2).contiguous().transpose(1, 2), x, cache, slots), "together")
    _refused(lambda: ops.fp4_cache_read(cache, slots, torch.float16), "float16")
    case = Fp4Case([20], 2, 64, 16)
    meta, cache = case.meta([4]), case.cache()
    q = _rand(4, 4, 64)
    _refused(lambda: ops.fp4_paged_attention(q[:, :3].contiguous(), cache, meta, 1.0), "cache")
    _refused(lambda: ops.fp4_paged_attention(q[..., :32].contiguous(), cache, meta, 1.0), "cache")
    _refused(lambda: ops.fp4_paged_attention(q.half(), cache, meta, 1.0), "float16")
    _refused(lambda: ops.fp4_paged_attention(_rand(5, 4, 64), cache, meta, 1.0), "token_seq")
    _refused(lambda: ops.fp4_paged_attention(q, cache, meta, 1.0, window=-3), "window")
    _refused(lambda: ops.fp4_paged_attention(q.cpu(), cache, meta, 1.0), "CUDA")
    _refused(lambda: ops.fp4_paged_attention(q, cache.data, meta, 1.0), "Fp4Cache")
    for q_lens, kv_lens in (([1, 1], [20, 20]), ([4], [20, 20]), ([1, 1, 1], [20])):
        meta = case.meta([4])
        meta.q_lens, meta.kv_lens = q_lens, kv_lens
        _refused(lambda: ops.fp4_paged_attention(q, cache, meta, 0.1), "block table")
