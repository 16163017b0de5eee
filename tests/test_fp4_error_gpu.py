"""How far float32 attention over the 4-bit cache is off, in the root mean square."""

from __future__ import annotations

import pytest
import torch

from tests.fp4_util import Fp4Case
from tests.test_fp4_gpu import _attend, _rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens,q_lens,hq,hkv,d", [([2600], [600], 8, 8, 64), ([3300], [800], 12, 4, 96), ([1500], [1000], 16, 8, 128),
                                                  ([4000] * 4, [1] * 4, 32, 8, 128), ([3000, 900], [5, 3], 32, 8, 128)])
def test_float32_attention_is_off_by_float32_roundings(lens, q_lens, hq, hkv, d):
    """Of a weight: a score's last rounding (at most 2^-20 where it and its value's exponent add up to less than 32), its power of two
    (2^-22), two parts of 11 digits (2^-22), each evenly spread: 2^-20 ln 2 / sqrt(3), 2^-22 / sqrt(3) twice, 4.3e-7 together.  The
    weights' errors are not alike, so the outputs are off by as much of their norm; sums in float32, rounded to the nearest, add less.
    Twice that is allowed.  (Sums that the products' units keep and cut off came to 1.2e-6 to 2.0e-6.)"""
    case = Fp4Case(lens, hkv, d, 16, seed=1)
    q = _rand(sum(q_lens), hq, d, seed=2)
    out = _attend(case, q, q_lens, d ** -0.5 / 32, portions=True)
    want, _, _ = case.attention(q, q_lens, d ** -0.5 / 32)
    assert ((out.double() - want).norm() / want.norm()).item() < 8.6e-7
