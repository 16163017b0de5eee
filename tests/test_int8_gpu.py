"""Serving in 8-bit integers against plain implementations in 64 bits.

Tolerances, before any run:
  codes, scales, read-back     every operation is a correctly rounded one: equal bits.
  product                      the integer sum is exact; the conversion to float32 and the two scales are a rounding of
                               2^-24 each, the output's rounding 2^-8 (bfloat16) comes on top: relative 2^-22, and 2^-8
                               more.
  attention                    scores: products of codes and queries summed in float32, of queries given by 22 bits or
                               more: scale sum|q||k| (2^-21 + sqrt(D) 2^-23) off.  An error e of the scores is one of 2 e
                               of the output, relative to the largest value seen, probabilities of 22 bits or more
                               (float32) another 2^-20, those rounded to bfloat16 (bfloat16) 2^-8 and the exponential's
                               2^-12; the bfloat16 output's rounding is 2^-8 of itself.
                               (The kernels keep bfloat16 queries to 15 bits of a row's largest element and their
                               probabilities to 15 bits of a tile's largest weight: the 2^-8 holds both.)
"""

from __future__ import annotations

import pytest
import torch

from deterministic_inference_b200.kernels import ops
from tests.int8_util import Int8Case, codes_of

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _rand(*shape, seed=0, dtype=F32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).cuda().to(dtype)


# ---- rows

@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 16), (3, 17), (5, 64), (2, 1000), (33, 1024), (7, 2056), (2, 4104), (4, 8200),
                                 (2, 16384), (2, 20000), (3, 12289), (300, 40)])
def test_rows(m, k, dtype):
    x = _rand(m, k, seed=m * k, dtype=dtype, scale=3.0)
    got = ops.quantize_rows(x)
    codes, scales = codes_of(x)
    assert got.shape == (m, k) and got.codes.shape[1] % 16 == 0
    assert torch.equal(got.codes[:, :k], codes) and torch.equal(got.scales, scales)
    assert not got.codes[:, k:].any()
    assert torch.equal(ops.Int8Weight.of(x).codes, got.codes)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("offset,width", [(0, 300), (8, 296), (3, 200), (5, 1)])
def test_rows_of_wider_rows(offset, width, dtype):
    x = _rand(9, 304, seed=offset, dtype=dtype)[:, offset:offset + width]
    got, (codes, scales) = ops.quantize_rows(x), codes_of(x)
    assert torch.equal(got.codes[:, :width], codes) and torch.equal(got.scales, scales)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_of_odd_values(dtype):
    x = _rand(12, 64, seed=1, dtype=dtype)
    x[0] = 0
    x[1] *= 2.0 ** -99
    x[2] *= 2.0 ** -120
    x[3, 5] = float("nan")
    x[4, 9] = float("inf")
    x[5, 63] = -float("inf")
    x[6] *= 2.0 ** 100
    x[7] = 0
    x[7, 3] = 2.0 ** -126 if dtype == F32 else 2.0 ** -120
    x[8] = torch.arange(64, device="cuda").to(dtype) - 32      # ties
    x[8, 0] = 63.5
    got, (codes, scales) = ops.quantize_rows(x), codes_of(x)
    assert torch.equal(got.codes, codes)
    assert torch.equal(got.scales.isnan(), scales.isnan()) and got.scales.isnan().sum() == 3
    assert torch.equal(got.scales.nan_to_num(), scales.nan_to_num())


# ---- product

def _check_product(y, x, codes, scales, dtype):
    xc, xs = codes_of(x)
    want = (xc.double() @ codes.double().t()) * xs.double()[:, None] * scales.double()
    tol = 2.0 ** -22 + (2.0 ** -8 if dtype == BF16 else 0.0)
    assert y.dtype == dtype and y.shape == want.shape
    assert ((y.double() - want).abs() <= tol * want.abs()).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,n,k", [
    (1, 1, 1), (1, 16, 16), (1, 1024, 1024), (2, 17, 33), (5, 100, 130), (8, 4096, 4096), (9, 257, 1000), (16, 512, 2048),
    (17, 640, 128), (31, 129, 5120), (32, 96, 64), (33, 200, 300), (64, 1024, 512), (65, 1000, 272), (100, 321, 77),
    (127, 128, 4096), (128, 256, 64), (129, 255, 1024), (200, 4100, 130), (256, 2048, 1024), (300, 24, 500),
    (513, 777, 1040), (700, 6144, 256), (1025, 2305, 144), (2048, 4096, 128), (1, 24577, 96), (40, 8, 12288)])
def test_product(m, n, k, dtype):
    x = _rand(m, k, seed=m + n + k, dtype=dtype, scale=2.0)
    w = ops.Int8Weight.of(_rand(n, k, seed=n, scale=0.05))
    y = ops.int8_linear(x, w)
    _check_product(y, x, w.codes[:, :k], w.scales, dtype)
    assert torch.equal(ops.linear(x, w), y)
    assert torch.equal(ops.int8_linear(ops.quantize_rows(x), w), y)


def test_product_of_the_largest_codes():
    """127 * 127 * K at the widest K that stays below 2^31, and the sign of it."""
    k = 133144
    x = torch.ones(3, k, device="cuda")
    x[1] = -1
    w = ops.Int8Weight(torch.full((130, k), 127, dtype=torch.int8, device="cuda"), torch.ones(130, device="cuda"))
    xc, xs = codes_of(x)
    assert (xc.abs() == 127).all()
    y = ops.int8_linear(x, w)
    want = torch.tensor([1, -1, 1], device="cuda").double() * (127 * 127 * k) * xs.double()
    assert ((y.double() - want[:, None]).abs() <= 2.0 ** -22 * want.abs()[:, None]).all()
    y = ops.int8_linear(x[:1].expand(200, k).contiguous(), w)
    assert ((y.double() - want[0]).abs() <= 2.0 ** -22 * want[0]).all()


@pytest.mark.parametrize("m", [4, 70, 300])
def test_product_output_type_and_rows_that_are_no_numbers(m):
    x = _rand(m, 256, seed=m, dtype=BF16)
    w = ops.Int8Weight.of(_rand(384, 256, seed=3))
    y = ops.int8_linear(x, w, torch.float32)
    _check_product(y, x, w.codes, w.scales, F32)
    bad = x.clone()
    bad[2, 7] = float("inf")
    z = ops.int8_linear(bad, w, torch.float32)
    assert z[2].isnan().all()
    keep = [i for i in range(m) if i != 2]
    assert torch.equal(z[keep], y[keep])


@pytest.mark.parametrize("n,k", [(1024, 1024), (24576, 256), (200, 4096)])
def test_a_row_of_a_product_does_not_depend_on_the_others(n, k):
    x = _rand(700, k, seed=k, dtype=BF16)
    w = ops.Int8Weight.of(_rand(n, k, seed=n))
    all_rows = ops.int8_linear(x, w, F32)
    for m in (1, 8, 9, 30, 64, 65, 128, 200, 300):
        assert torch.equal(ops.int8_linear(x[:m], w, F32), all_rows[:m])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,n,k", [(1, 17, 40), (129, 257, 130), (300, 1000, 520), (513, 513, 1040), (256, 24, 16)])
def test_every_form_of_a_product_gives_the_same_bits(m, n, k, dtype):
    from deterministic_inference_b200.kernels import int8
    x, w = _rand(m, k, seed=m, dtype=dtype), ops.Int8Weight.of(_rand(n, k, seed=n))
    want = ops.int8_linear(x, w)
    _check_product(want, x, w.codes[:, :k], w.scales, dtype)
    try:
        for form in range(5):
            int8.force_product_form(form)
            got = ops.int8_linear(x, w)
            ops.check_kernel_status()
            assert torch.equal(got, want), f"form {form}"
    finally:
        int8.force_product_form(-1)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,n,k", [(1, 17, 40), (16, 1024, 1024), (33, 1000, 2064), (65, 130, 4112), (128, 2048, 300),
                                   (129, 257, 1300), (256, 200, 8192), (40, 4096, 1056)])
def test_clusters_that_share_k_give_the_same_bits(m, n, k, dtype):
    from deterministic_inference_b200.kernels import int8
    x, w = _rand(m, k, seed=m + 1, dtype=dtype), ops.Int8Weight.of(_rand(n, k, seed=n + 1))
    try:
        int8.force_product_form(2)
        want = ops.int8_linear(x, w)
        for form in (5, 6):
            int8.force_product_form(form)
            got = ops.int8_linear(x, w)
            ops.check_kernel_status()
            assert torch.equal(got, want), f"form {form}"
    finally:
        int8.force_product_form(-1)
    _check_product(ops.int8_linear(x, w), x, w.codes[:, :k], w.scales, dtype)


def test_product_with_no_rows():
    w = ops.Int8Weight.of(_rand(32, 64))
    assert ops.int8_linear(torch.empty(0, 64, device="cuda"), w).shape == (0, 32)
    assert ops.quantize_rows(torch.empty(0, 5, device="cuda", dtype=BF16)).codes.shape == (0, 16)


def test_gated_product():
    x = _rand(70, 128, dtype=BF16)
    w = ops.Int8Weight.of(_rand(512, 128, seed=5))
    y = ops.int8_linear(x, w)
    assert torch.equal(ops.as_tensor(ops.gated_linear(x, w)), ops.silu_mul(y))


# ---- cache

@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("t,hkv,d,page", [(1, 1, 16, 1), (1, 8, 128, 16), (7, 3, 48, 5), (33, 2, 64, 8), (130, 8, 128, 16),
                                          (9, 4, 256, 32), (5, 1, 144, 64), (1000, 2, 96, 16)])
def test_cache_write_and_read(t, hkv, d, page, dtype):
    cache = ops.Int8Cache.zeros(t // page + 4, hkv, page, d)
    cache.scales.fill_(float("nan"))
    g = torch.Generator().manual_seed(t)
    slots = torch.randperm(cache.shape[0] * page, generator=g)[:t].to(torch.int32).cuda()
    k, v = _rand(t, hkv, d, seed=1, dtype=dtype), _rand(t, hkv, d, seed=2, dtype=dtype, scale=30.0)
    before = cache.data.clone()
    ops.int8_cache_write(k, v, cache, slots)
    at = slots.long()
    for kv, x in ((0, k), (1, v)):
        codes, scales = codes_of(x)
        assert torch.equal(cache.data[at // page, kv, :, at % page], codes)
        assert torch.equal(cache.scales[at // page, kv, :, at % page], scales)
        before[at // page, kv, :, at % page] = codes
    assert torch.equal(cache.data, before)                    # nothing beside the slots
    got = ops.int8_cache_read(cache, slots, dtype)
    for kv, x in ((0, k), (1, v)):
        codes, scales = codes_of(x)
        assert torch.equal(got[kv], (codes.float() * scales[..., None]).to(dtype))
    again = ops.Int8Cache.zeros(*[cache.shape[i] for i in (0, 2, 3, 4)])
    again.scales.fill_(float("nan"))
    ops.reshape_and_cache(k, v, again, slots)
    assert torch.equal(again.data, cache.data)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("extra", [0, 8, 3])
def test_cache_write_of_column_ranges(extra, dtype):
    """Keys and values as column ranges of the fused projection's rows, at any distance and alignment."""
    hkv, d, t = 2, 64, 11
    rows = _rand(t, extra + 5 * d + 2 * hkv * d, seed=extra, dtype=dtype)
    k = rows[:, extra + 4 * d:extra + (4 + hkv) * d].view(t, hkv, d)
    v = rows[:, extra + (4 + hkv) * d:extra + (4 + 2 * hkv) * d].view(t, hkv, d)
    a, b = ops.Int8Cache.zeros(3, hkv, 8, d), ops.Int8Cache.zeros(3, hkv, 8, d)
    slots = torch.arange(t, dtype=torch.int32, device="cuda") + 2
    ops.int8_cache_write(k, v, a, slots)
    ops.int8_cache_write(k.contiguous(), v.contiguous(), b, slots)
    assert torch.equal(a.data, b.data) and torch.equal(a.scales, b.scales) and a.data.any()


def test_cache_skips_slots_that_are_none():
    cache = ops.Int8Cache.zeros(4, 2, 8, 64)
    x = _rand(4, 2, 64, seed=4)
    slots = torch.tensor([-1, 9, 32, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    ops.int8_cache_write(x, x, cache, slots)
    assert cache.data.flatten(3).any(-1).sum() == 4 and cache.data[1, :, :, 1].any()
    k, v = ops.int8_cache_read(cache, slots, F32)
    assert not k[0].any() and not k[2:].any() and torch.equal(k, v) and k[1].any()
    ops.int8_cache_write(x[:0], x[:0], cache, slots)
    assert ops.int8_cache_read(cache, slots[:0])[0].shape == (0, 2, 64)


def test_cache_rows_that_are_no_numbers():
    cache = ops.Int8Cache.zeros(2, 1, 8, 32)
    k = _rand(3, 1, 32, seed=8)
    k[1, 0, 4] = float("nan")
    v = k.clone()
    v[2, 0, 0] = -float("inf")
    slots = torch.arange(3, dtype=torch.int32, device="cuda")
    ops.int8_cache_write(k, v, cache, slots)
    rk, rv = ops.int8_cache_read(cache, slots, F32)
    assert rk[1].isnan().all() and rv[1:].isnan().all() and rk[[0, 2]].isfinite().all() and rv[0].isfinite().all()


# ---- attention

def _check_attention(case, q_lens, hq, dtype, window=None, kv_lens=None, seed=0, scale=None, q_scale=1.0):
    q = _rand(sum(q_lens), hq, case.d, seed=seed + 100, dtype=dtype, scale=q_scale)
    scale = case.d ** -0.5 if scale is None else scale
    cache = ops.Int8Cache(case.data, case.scales)
    out = ops.int8_paged_attention(q, cache, case.meta(q_lens, kv_lens), scale, window)
    ops.check_kernel_status()
    want, vmax, smax = case.attention(q, q_lens, scale, window, kv_lens)
    assert out.dtype == dtype and out.shape == q.shape
    p_err = 2.0 ** -20 if dtype == F32 else 2.0 ** -8 + 2.0 ** -12
    tol = (2 * smax * (2.0 ** -21 + case.d ** 0.5 * 2.0 ** -23) + p_err) * vmax
    if dtype == BF16:
        tol = tol + 2.0 ** -8 * want.abs()
    err = (out.double() - want).abs()
    assert (err <= tol).all(), f"{(err - tol).max().item()} over, at {(err > tol).nonzero()[:4].tolist()}"
    return out


LAYOUTS = [  # (query heads, kv heads, head size, page size)
    (16, 8, 128, 16), (8, 1, 128, 16), (32, 2, 128, 32), (5, 5, 128, 8), (12, 4, 96, 16), (6, 2, 64, 64), (4, 2, 16, 16),
    (6, 3, 48, 24), (20, 1, 128, 128), (40, 1, 64, 16), (2, 1, 256, 16), (4, 4, 32, 1), (7, 1, 144, 48), (3, 1, 80, 4)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hq,hkv,d,page", LAYOUTS)
def test_attention_of_one_token(hq, hkv, d, page, dtype):
    case = Int8Case([1, 2, 16, 17, 31, 33, 127, 128, 129, 255, 256, 257, 700, 1025], hkv, d, page, seed=d + page)
    _check_attention(case, [1] * len(case.lens), hq, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hq,hkv,d,page", LAYOUTS)
def test_attention_of_mixed_chunks(hq, hkv, d, page, dtype):
    case = Int8Case([40, 1, 300, 5, 70, 9, 520, 64, 130, 333], hkv, d, page, seed=d + page)
    _check_attention(case, [1, 1, 2, 5, 3, 9, 4, 64, 129, 200], hq, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("window", [1, 7, 32, 100, 128, 1000])
@pytest.mark.parametrize("hq,hkv,d,page", [(16, 8, 128, 16), (4, 2, 64, 8), (8, 1, 128, 64)])
def test_attention_in_a_window(hq, hkv, d, page, window, dtype):
    case = Int8Case([1, 200, 517, 6, 300, 450], hkv, d, page, seed=window)
    _check_attention(case, [1, 1, 1, 6, 77, 300], hq, dtype, window=window)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hq,hkv,d,page", [(16, 8, 128, 16), (4, 2, 64, 8), (2, 1, 80, 4)])
def test_attention_rows_that_see_nothing(hq, hkv, d, page, dtype):
    """More new tokens than keys: the first ones lie before the first key.  A sequence with no key, and one with no token."""
    case = Int8Case([3, 0, 20, 1], hkv, d, page, seed=9)
    out = _check_attention(case, [5, 2, 0, 40], hq, dtype)
    assert not out[:2].any() and not out[5:7].any() and not out[7:46].any() and out[2].any() and out[46].any()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("q_len", [1, 3, 40, 200])
def test_attention_of_uneven_value_scales(q_len, dtype):
    """Value scales over sixty powers of two: against the largest value seen, and (one key alone visible) each by itself."""
    scales = lambda n, hkv, g: 2.0 ** (torch.rand(n, hkv, generator=g) * 60 - 30)
    case = Int8Case([q_len + 300, q_len + 37], 2, 128, 16, seed=q_len, value_scales=scales)
    _check_attention(case, [q_len, q_len], 4, dtype)
    _check_attention(case, [q_len, q_len], 4, dtype, window=1)


@pytest.mark.parametrize("step", [1 / 24, -1 / 24, 1 / 400])
@pytest.mark.parametrize("keys,q_len", [(700, 1), (700, 300), (4500, 200)])
def test_attention_of_value_scales_that_drift(keys, q_len, step):
    """Scales that leave the first keys' range along the sequence, within it and across its chunks."""
    scales = lambda n, hkv, g: (2.0 ** (torch.arange(n) * step).clamp(-40, 40))[:, None].expand(n, hkv).contiguous()
    case = Int8Case([keys, keys // 2], 2, 128, 16, seed=q_len, value_scales=scales)
    _check_attention(case, [q_len, q_len], 4, BF16)
    _check_attention(case, [q_len, q_len], 4, BF16, window=64)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("scale", [0.0, -0.07])
def test_attention_of_zero_and_negative_scales(scale, dtype):
    case = Int8Case([500, 300, 77], 2, 128, 16, seed=8)
    _check_attention(case, [200, 4, 1], 8, dtype, scale=scale)


@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (6, 2, 64)])
def test_a_prompt_attends_the_same_in_any_portion(hq, hkv, d):
    """The bits of a prompt's rows do not depend on where its portions begin."""
    case = Int8Case([900], hkv, d, 16, seed=6)
    q = _rand(500, hq, d, seed=7, dtype=BF16)
    cache = ops.Int8Cache(case.data, case.scales)
    whole = ops.int8_paged_attention(q, cache, case.meta([500]), 0.1)
    for n in (450, 333, 128, 70):
        got = ops.int8_paged_attention(q[500 - n:].contiguous(), cache, case.meta([n]), 0.1)
        assert torch.equal(got, whole[500 - n:])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("q_len", [1, 150])
@pytest.mark.parametrize("q_scale", [1e-30, 3e4, 1e8])
def test_attention_of_small_and_large_queries(q_len, q_scale, dtype):
    case = Int8Case([q_len + 99, q_len], 2, 128, 16, seed=3)
    _check_attention(case, [q_len] * 2, 4, dtype, q_scale=q_scale, scale=1.0 / q_scale)


@pytest.mark.parametrize("q_len", [1, 8, 200])
def test_attention_query_rows_that_are_no_numbers(q_len):
    case = Int8Case([260, 260], 2, 128, 16, seed=2)
    q = _rand(2 * q_len, 4, 128, seed=5, dtype=BF16)
    cache, meta = ops.Int8Cache(case.data, case.scales), case.meta([q_len] * 2)
    good = ops.int8_paged_attention(q, cache, meta, 0.1)
    bad = q.clone()
    bad[0, 1, 3] = float("nan")
    out = ops.int8_paged_attention(bad, cache, meta, 0.1)
    assert out[0, 1].isnan().all()
    keep = torch.ones(2 * q_len, 4, dtype=torch.bool)
    keep[0, 1] = False
    assert torch.equal(out[keep], good[keep])


@pytest.mark.parametrize("q_len", [1, 5, 100])
def test_attention_key_rows_that_are_no_numbers(q_len):
    """A key row that is no number shows in every row that sees it and in no other."""
    case = Int8Case([300], 1, 128, 16, seed=2)
    at = 300 - q_len // 2 - 1
    case.scales[case.tables[0][at // 16], 0, 0, at % 16] = float("nan")
    q = _rand(q_len, 2, 128, seed=5, dtype=BF16)
    out = ops.int8_paged_attention(q, ops.Int8Cache(case.data, case.scales), case.meta([q_len]), 0.1)
    sees = torch.arange(300 - q_len, 300) >= at
    assert torch.equal(out.isnan().all(-1).all(-1).cpu(), sees) and not out[~sees.cuda()].isnan().any()


def test_attention_of_long_contexts():
    case = Int8Case([20000, 9001, 17011], 2, 128, 16, seed=1)
    _check_attention(case, [1, 1, 5], 16, BF16)
    _check_attention(case, [1, 3, 300], 16, BF16)


def test_attention_beyond_32_bits():
    """A cache of more than 2^32 bytes, the sequences on its last pages."""
    page_bytes = 2 * 8 * 64 * 128
    first = 2 ** 32 // page_bytes + 100
    case = Int8Case([70, 300, 200], 8, 128, 64, seed=4, first_page=first)
    assert case.data.numel() > 2 ** 32 and min(min(t) for t in case.tables) >= first
    _check_attention(case, [1, 4, 150], 16, BF16)
    cache = ops.Int8Cache(case.data, case.scales)
    slots = torch.tensor([(case.data.shape[0] - 1) * 64 + 63], dtype=torch.int32, device="cuda")
    x = _rand(1, 8, 128, seed=9)
    ops.int8_cache_write(x, x, cache, slots)
    codes, scales = codes_of(x)
    assert torch.equal(cache.data[-1, 1, :, 63], codes[0]) and torch.equal(cache.scales[-1, 0, :, 63], scales[0])
    assert torch.equal(ops.int8_cache_read(cache, slots, F32)[1], codes.float() * scales[..., None])


@pytest.mark.parametrize("hq,hkv,d", [(16, 8, 128), (4, 2, 64)])
def test_a_token_attends_the_same_in_any_step(hq, hkv, d):
    """The bits of a sequence's rows do not depend on the other sequences of the step."""
    case = Int8Case([900, 333, 1500, 40, 700], hkv, d, 16, seed=6)
    q_lens = [1, 1, 4, 40, 300]
    q = _rand(sum(q_lens), hq, d, seed=7, dtype=BF16)
    cache = ops.Int8Cache(case.data, case.scales)
    whole = ops.int8_paged_attention(q, cache, case.meta(q_lens), 0.1)
    at = 0
    for s, n in enumerate(q_lens):
        alone = Int8Case.__new__(Int8Case)
        alone.__dict__.update(case.__dict__)
        alone.tables, alone.lens = [case.tables[s]], [case.lens[s]]
        got = ops.int8_paged_attention(q[at:at + n].contiguous(), cache, alone.meta([n]), 0.1)
        assert torch.equal(got, whole[at:at + n])
        at += n


def test_on_another_stream():
    case = Int8Case([300, 40], 2, 128, 16, seed=1)
    q = _rand(9, 4, 128, seed=3, dtype=BF16)
    meta, cache = case.meta([1, 8]), ops.Int8Cache(case.data, case.scales)
    want = ops.int8_paged_attention(q, cache, meta, 0.1)
    w = ops.Int8Weight.of(_rand(512, 512, seed=4))
    y = ops.int8_linear(q.view(9, 512), w)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.int8_paged_attention(q, cache, case.meta([1, 8]), 0.1)
        z = ops.int8_linear(q.view(9, 512), w)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(z, y)


# ---- refusals

def _refused(call, *words):
    with pytest.raises(ops.KernelError) as e:
        call()
    for word in words:
        assert word in str(e.value)


def test_refusals():
    cache = ops.Int8Cache.zeros(3, 2, 16, 64)
    x = _rand(4, 2, 64)
    slots = torch.zeros(4, dtype=torch.int32, device="cuda")
    w = ops.Int8Weight.of(_rand(32, 64))
    _refused(lambda: ops.quantize_rows(x[0].cpu()), "CUDA")
    _refused(lambda: ops.quantize_rows(x[0].half()), "float16")
    _refused(lambda: ops.quantize_rows(x[0].t()), "consecutive")
    _refused(lambda: ops.Int8Weight(torch.zeros(3, 4, device="cuda"), torch.ones(3, device="cuda")), "int8")
    _refused(lambda: ops.Int8Weight(w.codes, torch.ones(3, device="cuda")), "scales")
    _refused(lambda: ops.Int8Weight.of(torch.zeros(1, 133145, device="cuda")), "133145")
    _refused(lambda: ops.int8_linear(_rand(2, 65), w), "against weight")
    _refused(lambda: ops.int8_linear(_rand(2, 64), w.codes), "Int8Weight")
    _refused(lambda: ops.int8_linear(_rand(2, 64), w, torch.float16), "float16")
    _refused(lambda: ops.Int8Cache(cache.data, cache.scales[:2]), "scales")
    _refused(lambda: ops.Int8Cache.zeros(3, 2, 16, 40), "multiple of 16")
    _refused(lambda: ops.Int8Cache.zeros(3, 2, 16, 272), "at most 256")
    _refused(lambda: ops.int8_cache_write(x[:, :1], x[:, :1], cache, slots), "heads")
    _refused(lambda: ops.int8_cache_write(x, x.bfloat16(), cache, slots), "bfloat16")
    _refused(lambda: ops.int8_cache_write(x, x, cache, slots[:2]), "slots")
    _refused(lambda: ops.int8_cache_write(x, x, cache, slots.long()), "int32")
    _refused(lambda: ops.int8_cache_write(x.transpose(1, 2).contiguous().transpose(1, 2), x, cache, slots), "together")
    _refused(lambda: ops.int8_cache_read(cache, slots, torch.float16), "float16")
    case = Int8Case([20], 2, 64, 16)
    meta, cache = case.meta([4]), ops.Int8Cache(case.data, case.scales)
    q = _rand(4, 4, 64)
    _refused(lambda: ops.int8_paged_attention(q[:, :3].contiguous(), cache, meta, 1.0), "cache")
    _refused(lambda: ops.int8_paged_attention(q[..., :32].contiguous(), cache, meta, 1.0), "cache")
    _refused(lambda: ops.int8_paged_attention(q.half(), cache, meta, 1.0), "float16")
    _refused(lambda: ops.int8_paged_attention(_rand(5, 4, 64), cache, meta, 1.0), "token_seq")
    _refused(lambda: ops.int8_paged_attention(q, cache, meta, 1.0, window=-3), "window")
    _refused(lambda: ops.int8_paged_attention(q.cpu(), cache, meta, 1.0), "CUDA")
