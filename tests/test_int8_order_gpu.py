"""8-bit operators one behind the other on a stream, with nothing between them: each reads what the one in front wrote, all of it.
(torch's own kernels wait for everything in front of them and would hide a wait that is missing.)"""

from __future__ import annotations

import pytest
import torch

from deterministic_inference_b200.kernels import ops
from tests.int8_util import Int8Case

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _rand(*shape, seed=0, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda().to(dtype)


# One run a sequence on the device where the host has to reckon with two, so that the merge has nothing to do.
@pytest.mark.parametrize("hq,hkv,lens,q_len", [(64, 8, [300] * 16, 1), (64, 8, [512, 257, 400], 1), (16, 8, [300] * 8, 4),
                                               (40, 1, [511] * 4, 1), (8, 8, [200, 40], 1)])
def test_a_product_behind_attention_reads_all_of_it(hq, hkv, lens, q_len):
    case = Int8Case(lens, hkv, 128, 16, seed=1)
    cache, meta, t = ops.Int8Cache(case.data, case.scales), case.meta([q_len] * len(lens)), q_len * len(lens)
    w = ops.Int8Weight.of(_rand(256, hq * 128, seed=2))
    queries = [_rand(t, hq, 128, seed=s, dtype=BF16) for s in (3, 4)]
    want = []
    for q in queries:
        out = ops.int8_paged_attention(q, cache, meta, 0.1)
        torch.cuda.synchronize()
        want.append(ops.int8_linear(out.view(t, -1), w))
    torch.cuda.synchronize()
    # (the two queries in turn: memory used again holds the other one's results)
    got = [ops.int8_linear(ops.int8_paged_attention(queries[i & 1], cache, meta, 0.1).view(t, -1), w) for i in range(60)]
    ops.check_kernel_status()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i & 1]), f"pass {i}"


@pytest.mark.parametrize("hq,hkv", [(16, 8), (64, 8)])
def test_a_product_behind_attention_in_a_graph_of_longer_sequences(hq, hkv):
    """A graph made for 512 keys a sequence, replayed with 40."""
    case = Int8Case([512] * 8, hkv, 128, 64, seed=1)
    cache, meta = ops.Int8Cache(case.data, case.scales), case.meta([1] * 8)
    w = ops.Int8Weight.of(_rand(256, hq * 128, seed=2))
    queries = [_rand(8, hq, 128, seed=s, dtype=BF16) for s in (3, 4)]
    q = torch.empty_like(queries[0])
    run = lambda: ops.int8_linear(ops.int8_paged_attention(q, cache, meta, 0.1).view(8, -1), w)
    q.copy_(queries[0])
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = run()
    meta.seq_lens.fill_(40)
    short, want = case.meta([1] * 8, [40] * 8), []
    for x in queries:
        out = ops.int8_paged_attention(x, cache, short, 0.1)
        torch.cuda.synchronize()
        want.append(ops.int8_linear(out.view(8, -1), w))
    for i in range(60):
        q.copy_(queries[i & 1])
        graph.replay()
        assert torch.equal(y, want[i & 1]), f"replay {i}"
    ops.check_kernel_status()


@pytest.mark.parametrize("m,n,k", [(4, 4096, 4096), (40, 8192, 2048), (700, 2048, 4096)])
def test_a_weight_made_of_rows_that_are_still_being_quantised(m, n, k):
    """The product reads its weight ahead of its wait for the kernel in front; one made of ``quantize_rows``' codes, and used at
    once, is read when they are there."""
    x = ops.quantize_rows(_rand(m, k, seed=1, dtype=BF16))
    sources = [_rand(n, k, seed=s, dtype=BF16) for s in (2, 3)]
    want = [ops.int8_linear(x, ops.Int8Weight.of(w)) for w in sources]
    torch.cuda.synchronize()
    for i in range(30):
        rows = ops.quantize_rows(sources[i & 1])
        weight = ops.Int8Weight(rows.codes, rows.scales)
        y = ops.int8_linear(x, weight)
        assert weight.scales.data_ptr() != rows.scales.data_ptr()      # (the copy that stands between)
        del rows, weight
        assert torch.equal(y, want[i & 1]), f"pass {i}"
    ops.check_kernel_status()


@pytest.mark.parametrize("m,n,k", [(4, 4096, 4096), (40, 8192, 2048), (700, 2048, 4096)])
def test_a_weight_used_as_soon_as_it_is_quantised(m, n, k):
    x = ops.quantize_rows(_rand(m, k, seed=1, dtype=BF16))
    sources = [_rand(n, k, seed=s, dtype=BF16) for s in (2, 3)]
    want = []
    for w in sources:
        weight = ops.Int8Weight.of(w)
        torch.cuda.synchronize()
        want.append(ops.int8_linear(x, weight))
    del weight
    for i in range(30):
        y = ops.int8_linear(x, ops.Int8Weight.of(sources[i & 1]))
        assert torch.equal(y, want[i & 1]), f"pass {i}"
    ops.check_kernel_status()
