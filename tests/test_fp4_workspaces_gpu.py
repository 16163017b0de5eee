"""What attention over the 4-bit cache allocates beside its output."""

from __future__ import annotations

import pytest
import torch

from deterministic_inference_b200.kernels import fp4, ops
from tests.fp4_util import Fp4Case
from tests.test_fp4_gpu import _rand

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F32, 128), (BF16, 96)])
def test_launches_by_size_give_the_same_bits(dtype, d, monkeypatch):
    """Sequences of every size in one launch, and in launches of those that need about the same room."""
    q_lens = [1, 1, 4, 2, 150, 1, 3, 40, 2, 1] if dtype == F32 else [1, 1, 4, 2, 8, 1, 3, 5, 2, 1]
    case = Fp4Case([3000, 40, 700, 2500, 900, 513, 5, 4100, 300, 260], 2, d, 16, seed=1)
    q = _rand(sum(q_lens), 8, d, seed=1, dtype=dtype)
    want = ops.fp4_paged_attention(q, case.cache(), case.meta(q_lens), 0.003)
    monkeypatch.setattr(fp4, "PARTIAL_BYTES", 1)
    meta = case.meta(q_lens)
    assert torch.equal(ops.fp4_paged_attention(q, case.cache(), meta, 0.003), want)
    assert len(next(iter(meta.scratch.values()))) > 4
    ops.check_kernel_status()


def test_room_of_a_long_portion_beside_short_ones():
    """float32: one portion of 2,000 tokens beside 60 of two; 0.02 GB of partial results of its own, 1.1 GB if each of the others had as
    much room."""
    q_lens = [2000] + [2] * 60
    case = Fp4Case([2000] + [300] * 60, 4, 64, 16, seed=1)
    q, cache, meta = _rand(sum(q_lens), 16, 64, seed=2), case.cache(), case.meta(q_lens)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = ops.fp4_paged_attention(q, cache, meta, 0.003)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < out.numel() * 4 + (1 << 28) + (1 << 20)
    want = ops.fp4_paged_attention(q[:2000].contiguous(), cache, case.alone(0).meta([2000]), 0.003)
    assert torch.equal(out[:2000], want)
