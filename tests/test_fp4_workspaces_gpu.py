"""What attention over the 4-bit cache allocates beside its output, and calls that share what a step keeps."""

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


@pytest.mark.parametrize("q_lens,lens", [([300, 1, 90], [9000, 700, 5000]), ([4, 1, 2], [9000, 700, 300])])
def test_two_streams_on_one_step(q_lens, lens):
    """Calls on one step, on two streams at the same time: prompts of more keys than a chunk (partial results), and drafts."""
    case = Fp4Case(lens, 2, 128, 16, seed=1)
    cache, portions = case.cache(), q_lens[0] > 4
    queries = [_rand(sum(q_lens), 8, 128, seed=s, dtype=BF16) for s in (3, 4)]
    want = [ops.fp4_paged_attention(q, cache, case.meta(q_lens), 0.003, None, portions) for q in queries]
    torch.cuda.synchronize()
    for _ in range(5):
        meta, got = case.meta(q_lens), [[], []]
        streams = [torch.cuda.Stream() for _ in (0, 1)]
        torch.cuda.synchronize()
        for _ in range(10):
            for i, s in enumerate(streams):
                with torch.cuda.stream(s):
                    got[i].append(ops.fp4_paged_attention(queries[i], cache, meta, 0.003, None, portions))
        torch.cuda.synchronize()
        for i in (0, 1):
            assert all(torch.equal(y, want[i]) for y in got[i])
    ops.check_kernel_status()


def test_two_captured_graphs_of_one_step_side_by_side():
    """Two graphs of the same step, with other queries, replayed on two streams at the same time."""
    q_lens = [300, 1, 90]
    case = Fp4Case([9000, 700, 5000], 2, 128, 16, seed=1)
    cache, meta = case.cache(), case.meta(q_lens)
    queries = [_rand(sum(q_lens), 8, 128, seed=s, dtype=BF16) for s in (3, 4)]
    want = [ops.fp4_paged_attention(q, cache, meta, 0.003, None, True) for q in queries]
    torch.cuda.synchronize()
    graphs = []
    for q in queries:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = ops.fp4_paged_attention(q, cache, meta, 0.003, None, True)
        graphs.append((graph, y))
    streams = [torch.cuda.Stream() for _ in (0, 1)]
    for _ in range(10):
        torch.cuda.synchronize()
        for (graph, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for i in (0, 1):
            assert torch.equal(graphs[i][1], want[i])
    ops.check_kernel_status()
