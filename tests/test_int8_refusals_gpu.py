"""What the 8-bit operators refuse, or take in good order, beyond the shapes of their calls."""

from __future__ import annotations

import pytest
import torch

from deterministic_inference_b200.kernels import ops
from tests.int8_util import Int8Case

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _rand(*shape, seed=0, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda().to(dtype)


def _refused(call, *words):
    with pytest.raises(ops.KernelError) as e:
        call()
    for word in words:
        assert word in str(e.value)


def test_rows_that_are_not_laid_out_as_rows():
    codes, scales = torch.zeros(4, 64, dtype=torch.int8, device="cuda"), torch.ones(4, device="cuda")
    good = ops.Int8Rows(codes, scales, 50, BF16)
    assert good.shape == (4, 50) and ops.int8_linear(good, ops.Int8Weight.of(_rand(8, 50))).dtype == BF16
    _refused(lambda: ops.Int8Rows(codes, scales, 40, BF16), "rounded up")         # a pitch that is another K's
    _refused(lambda: ops.Int8Rows(codes, scales, 65, BF16), "rounded up")
    _refused(lambda: ops.Int8Rows(codes, scales, 0, BF16), "K from 1")
    _refused(lambda: ops.Int8Rows(codes, scales[:3], 64, BF16), "scales")
    _refused(lambda: ops.Int8Rows(codes, scales.double(), 64, BF16), "float32")
    _refused(lambda: ops.Int8Rows(codes.float(), scales, 64, BF16), "int8")
    _refused(lambda: ops.Int8Rows(codes.t(), scales, 4, BF16), "contiguous")
    _refused(lambda: ops.Int8Rows(codes.cpu(), scales, 64, BF16), "CUDA")
    _refused(lambda: ops.Int8Rows(codes, scales, 64, torch.float16), "float16")
    odd = torch.zeros(4 * 64 + 1, dtype=torch.int8, device="cuda")[1:].view(4, 64)
    _refused(lambda: ops.Int8Rows(odd, scales, 64, BF16), "16 bytes")


def test_a_product_refuses_rows_of_another_pitch():
    rows, weight = ops.quantize_rows(_rand(4, 40)), ops.Int8Weight.of(_rand(8, 40))
    assert ops.int8_linear(rows, weight).shape == (4, 8)
    rows.codes = torch.zeros(4, 64, dtype=torch.int8, device="cuda")
    _refused(lambda: ops.int8_linear(rows, weight), "against the weight's")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("q_len", [1, 5])
@pytest.mark.parametrize("hkv,d,page", [(2, 144, 16), (1, 256, 32), (2, 64, 24), (1, 32, 1)])
def test_pages_that_are_none_of_the_pools_in_the_form_for_every_shape(hkv, d, page, q_len, dtype):
    """Heads above 128 and pages that are no power of two: such pages are pages of zeros there too."""
    case = Int8Case([200, 100], hkv, d, page, seed=5)
    q = _rand(2 * q_len, 2 * hkv, d, seed=4, dtype=dtype)
    zeros = ops.Int8Cache(case.data.clone(), case.scales.clone())
    zeros.scales[case.tables[0][2]] = 0
    want = ops.int8_paged_attention(q, zeros, case.meta([q_len] * 2), 0.1)
    for entry in (-1, case.data.shape[0], 2 ** 31 - 1):
        meta = case.meta([q_len] * 2)
        meta.block_table[0, 2] = entry
        assert torch.equal(ops.int8_paged_attention(q, ops.Int8Cache(case.data, case.scales), meta, 0.1), want)


def test_lengths_of_more_sequences_than_there_are_tables():
    case = Int8Case([200, 100], 2, 64, 16, seed=5)
    q, cache = _rand(2, 4, 64), ops.Int8Cache(case.data, case.scales)
    for q_lens, kv_lens in (([1, 1, 1], [200, 100, 100]), ([1, 1], [200]), ([1], [200, 100])):
        meta = case.meta([1, 1])
        meta.q_lens, meta.kv_lens = q_lens, kv_lens
        _refused(lambda: ops.int8_paged_attention(q, cache, meta, 0.1), "block table")
