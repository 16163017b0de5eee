"""How far attention over a cache in 8 bits is from 64 bits, against the output's own size.

Bounds, before any run.  bfloat16: an element's rounding is 2^-8 of it at most; over mantissas of every size its root mean square
is 2^-7 / sqrt(12) * 0.72 = 0.0016 to 0.0017, and of a token's elements (512 or more) the norm is within some 15 % of that.  In
front of it each of many terms of either sign is rounded to float16 three times, or to 15 bits of the largest, 2^-12 at most each:
0.0003 of the norm in the root mean square.  So 0.0025 of a token's norm holds, and a key left out of a thousand (3 % of the norm)
or an error of a per cent does not pass.  float32: 28 bits of the largest term, scores of 2^-21 and exponentials of 2^-20, the sums
of 1,000 terms of either sign: 2^-17."""

from __future__ import annotations

import pytest
import torch

from deterministic_inference_b200.kernels import ops
from tests.int8_util import Int8Case

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
BOUND = {BF16: 0.0025, F32: 2.0 ** -17}


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("portions", [False, True])
@pytest.mark.parametrize("lens,q_lens,hq,hkv,d,window", [
    ([1000, 3000, 9000, 20000], [1, 1, 1, 1], 16, 8, 128, None),
    ([1000, 3000, 9000, 17000], [1, 1, 1, 1], 32, 2, 128, None),
    ([1500, 1100, 5000], [5, 3, 2], 16, 8, 128, None),
    ([1500, 4100], [7, 16], 32, 8, 64, None),
    ([1300, 6000], [300, 129], 16, 4, 128, None),
    ([700, 2500, 5000], [1, 6, 200], 16, 4, 128, 600),
    ([1200, 900], [130, 1], 8, 2, 256, None),
    ([1200, 900], [5, 1], 16, 8, 64, None)])
def test_error_of_a_token(lens, q_lens, hq, hkv, d, window, portions, dtype):
    page = 24 if d == 64 and lens[0] == 1200 else 16
    case = Int8Case(lens, hkv, d, page, seed=len(lens) + d)
    g = torch.Generator().manual_seed(3)
    q = torch.randn(sum(q_lens), hq, d, generator=g).cuda().to(dtype)
    cache = ops.Int8Cache(case.data, case.scales)
    out = ops.int8_paged_attention(q, cache, case.meta(q_lens), 0.2 / d ** 0.5, window, portions=portions)
    ops.check_kernel_status()
    want, _, _ = case.attention(q, q_lens, 0.2 / d ** 0.5, window)
    off = (out.double() - want).flatten(1).norm(dim=1) / want.flatten(1).norm(dim=1)
    assert off.max() < BOUND[dtype], off.max().item()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("q_len", [1, 5, 100])
def test_the_bound_sees_a_key_that_is_left_out(q_len, dtype):
    """(The key is left out of the plain implementation.)"""
    case = Int8Case([1100], 2, 128, 16, seed=1)
    g = torch.Generator().manual_seed(3)
    q = torch.randn(q_len, 8, 128, generator=g).cuda().to(dtype)
    out = ops.int8_paged_attention(q, ops.Int8Cache(case.data, case.scales), case.meta([q_len]), 0.02)
    kept = [i for i in range(1100) if i != 500]
    case.rows = lambda s, n, rows=case.rows: tuple(x[kept] for x in rows(s, 1100))
    want, _, _ = case.attention(q, [q_len], 0.02, kv_lens=[1099])
    off = (out.double() - want).flatten(1).norm(dim=1) / want.flatten(1).norm(dim=1)
    assert off.min() > 2 * BOUND[BF16]
