"""Attention over the cache in 4-bit floating point where its numbers lie far from one another: scores of any size, values of
zero and next to nothing, values over every power of two that a cache holds."""

from __future__ import annotations

import pytest
import torch

from deterministic_inference_b200.kernels import ops
from tests.fp4_util import Fp4Case
from tests.test_fp4_gpu import _attend, _rand

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
# (query heads, kv heads, head size, page size, type): the stream form in tiles of 4, 8 and 16 rows (with several tokens), the split
# form, the form for every shape
FORMS = [(8, 2, 128, 16, BF16), (16, 2, 64, 64, BF16), (12, 4, 96, 32, BF16), (8, 2, 128, 16, F32), (4, 2, 32, 8, F32), (2, 1, 144, 16, BF16)]


@pytest.mark.parametrize("hq,hkv,d,page,dtype", FORMS)
@pytest.mark.parametrize("q_len", [1, 3])
@pytest.mark.parametrize("size", [1e15, 1e17])
def test_scores_far_below_zero(hq, hkv, d, page, dtype, q_len, size):
    """Keys that are all alike: every one has the same weight, however far below zero the scores are.  (-1e32 to -1e35 here; the mean of
    the values a row sees, off by the weights' rounding, 2^-11 in 16 bits, 2^-21 in 32, sums of 40 steps and the output's rounding.)"""
    case = Fp4Case([700, 40], hkv, d, page, seed=d)
    one = torch.randint(1, 8, (hkv, d // 2), generator=torch.Generator().manual_seed(d)).to(torch.uint8).cuda() * 17      # above zero
    case.data[:, 0], case.scales[:, 0], case.exponents[:, 0] = one[:, None], 0x40, 127 + 50
    q = -_rand(2 * q_len, hq, d, seed=1, dtype=dtype).abs() * size
    out = _attend(case, q, [q_len] * 2, 1.0)
    assert out.isfinite().all()
    at = 0
    for s, n in enumerate(case.lens):
        values = case.rows(s, n)[1].repeat_interleave(hq // hkv, 1)
        for i in range(q_len):
            seen = values[:n - q_len + 1 + i]
            want, most = seen.mean(0), seen.abs().amax()
            tol = (2.0 ** -10 * most + 2.0 ** -8 * want.abs()) if dtype == BF16 else 2.0 ** -18 * most
            assert ((out[at].double() - want).abs() <= tol).all(), (s, i)
            at += 1


def _agrees(case, q, q_lens, scale, window=None, want_of=None, portions=False):
    """Against 64 bits, by what _check_attention of the other tests allows: of the largest visible value, twice a score's error and the
    weights' rounding; of the output, its own."""
    out = _attend(case, q, q_lens, scale, window, portions=portions)
    want, vmax, smax = (want_of or case).attention(q, q_lens, scale, window)
    assert out.isfinite().all()
    if q.dtype == F32:
        tol = (2 * smax * 2.0 ** -18 + 2.0 ** -17) * vmax
    else:
        blocks = q.float().unflatten(-1, (-1, 16)).abs().amax(-1, keepdim=True).expand(-1, -1, -1, 16).flatten(-2)
        _, _, most = (want_of or case).attention(blocks, q_lens, scale, window)
        tol = (2 * (smax * 2.0 ** -18 + most * 2.0 ** -9.9) + 2.0 ** -8) * vmax + 2.0 ** -8 * want.abs()
    err = (out.double() - want).abs()
    assert (err <= tol).all(), f"{(err / vmax).max().item()} of the largest value, at {(err > tol).nonzero()[:4].tolist()}"


def _values_of(case, s, keys, codes=None, scales=None, exponents=None):
    """Sets what the value rows ``keys`` of sequence s hold."""
    at = torch.as_tensor(list(keys))
    page, row = torch.tensor(case.tables[s])[at // case.page_size].cuda(), (at % case.page_size).cuda()
    for held, x in ((case.data, codes), (case.scales, scales), (case.exponents, exponents)):
        if x is not None:
            held[page, 1, :, row] = x


@pytest.mark.parametrize("hq,hkv,d,page,dtype", FORMS)
@pytest.mark.parametrize("q_lens", [[1, 1, 1, 1], [4, 3, 4, 2], [40, 3, 1, 50]])
@pytest.mark.parametrize("exponent", [16, 0])
def test_values_of_zero(hq, hkv, d, page, dtype, q_lens, exponent):
    """Keys whose values are zero take their share of the weights: a run of them, several, one warp's, the first and the last, with
    the exponent that the rule writes (16) and that of a row that nothing was written to (0).  Scores that differ little."""
    case = Fp4Case([2100, 700, 300, 70], hkv, d, page, seed=d)
    for s, keys in ((0, range(512)), (0, range(1536, 1570)), (1, range(100, 700)), (2, range(32)), (2, range(256, 300)), (3, range(69))):
        _values_of(case, s, keys, 0, 0, exponent)
    q = _rand(sum(q_lens), hq, d, seed=2, dtype=dtype)
    for scale in (0.0, d ** -0.5 / 2048, d ** -0.5 / 32):
        _agrees(case, q, q_lens, scale)
        _agrees(case, q, q_lens, scale, portions=True)
        _agrees(case, q, q_lens, scale, window=600)


@pytest.mark.parametrize("hq,hkv,d,page,dtype", FORMS)
@pytest.mark.parametrize("q_lens", [[1, 1], [5, 3], [40, 60]])
def test_values_next_to_nothing(hq, hkv, d, page, dtype, q_lens):
    """The smallest rows that the rule makes, some 2^-100, alone and in front of and behind ordinary ones."""
    for keys in (range(1300), range(700), range(600, 1300)):
        case = Fp4Case([1300, 1300], hkv, d, page, seed=d)
        for s in (0, 1):
            _values_of(case, s, keys, exponents=16)
        q = _rand(sum(q_lens), hq, d, seed=2, dtype=dtype)
        for scale in (0.0, d ** -0.5 / 32):
            _agrees(case, q, q_lens, scale)


@pytest.mark.parametrize("hq,hkv,d,page,dtype", FORMS)
@pytest.mark.parametrize("q_len", [1, 4, 60])
@pytest.mark.parametrize("few", [False, True])
def test_values_over_every_power_of_two(hq, hkv, d, page, dtype, q_len, few):
    """Exponent bytes from 16 to 244 (``few``: of one key in a hundred, the others next to one another): against the largest value
    seen, and (windows of one key) each by itself."""
    def units(n, hkv, g):
        wide = torch.randint(16, 245, (n, hkv), generator=g)
        return torch.where(torch.rand(n, hkv, generator=g) < 0.01, wide, 120 + wide % 4) if few else wide
    case = Fp4Case([900 + q_len, 300], hkv, d, page, seed=q_len, exponents=lambda n, hkv, g: units(n, hkv, g).to(torch.uint8))
    q = _rand(2 * q_len, hq, d, seed=2, dtype=dtype)
    for window in (None, 64, 1):
        for scale in (0.0, d ** -0.5 / 32):
            _agrees(case, q, [q_len] * 2, scale, window)


@pytest.mark.parametrize("hq,hkv,d,dtype", [(8, 2, 128, BF16), (16, 2, 64, BF16), (12, 4, 96, BF16), (8, 2, 128, F32), (4, 2, 32, F32), (2, 1, 144, BF16)])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("q_len", [1, 5, 90])
def test_absent_pages_hold_zeros(hq, hkv, d, dtype, page, q_len):
    """Pages that are none of the pool's, of as many keys as a warp, a tile and a run of them, against 64 bits."""
    case = Fp4Case([1100, 700], hkv, d, page, seed=5)
    zeros = Fp4Case.__new__(Fp4Case)
    zeros.__dict__.update(case.__dict__)
    zeros.data, zeros.scales, zeros.exponents = case.data.clone(), case.scales.clone(), case.exponents.clone()
    meta = case.meta([q_len] * 2)
    for s, places in ((0, range(0, 512 // page)), (0, [800 // page]), (1, range(256 // page, 700 // page))):
        for p in places:
            meta.block_table[s, p] = -1 if p % 2 else case.data.shape[0]
            for held in (zeros.data, zeros.scales, zeros.exponents):
                held[case.tables[s][p]] = 0
    q = _rand(2 * q_len, hq, d, seed=4, dtype=dtype)
    for scale in (0.0, 0.003):
        out = ops.fp4_paged_attention(q, case.cache(), meta, scale)
        want, vmax, smax = zeros.attention(q, [q_len] * 2, scale)
        blocks = q.float().unflatten(-1, (-1, 16)).abs().amax(-1, keepdim=True).expand(-1, -1, -1, 16).flatten(-2)
        _, _, most = zeros.attention(blocks, [q_len] * 2, scale)
        tol = (2 * smax * 2.0 ** -18 + 2.0 ** -17) * vmax if dtype == F32 else \
            (2 * (smax * 2.0 ** -18 + most * 2.0 ** -9.9) + 2.0 ** -8) * vmax + 2.0 ** -8 * want.abs()
        assert ((out.double() - want).abs() <= tol).all()
    ops.check_kernel_status()


@pytest.mark.parametrize("hq,hkv,d,page,dtype", FORMS)
@pytest.mark.parametrize("q_lens", [[1, 1, 1], [4, 3, 2], [60, 40, 50]])
def test_windows_of_any_size(hq, hkv, d, page, dtype, q_lens):
    """Windows as long as the sequences and longer, beyond 32 bits too, are no windows; sequences with fewer keys than new tokens among
    them."""
    case = Fp4Case([700, 2, 30], hkv, d, page, seed=d)
    q = _rand(sum(q_lens), hq, d, seed=2, dtype=dtype)
    for portions in (False, True):
        want = ops.fp4_paged_attention(q, case.cache(), case.meta(q_lens), 0.003, None, portions)
        for window in (700, 5000, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5, 2 ** 40):
            assert torch.equal(ops.fp4_paged_attention(q, case.cache(), case.meta(q_lens), 0.003, window, portions), want), window
