"""What a token's bits over a cache in 4 bits do not depend on: whether its step was launched or replayed, where its prompt was cut, the
other sequences of the step; and operators one behind the other on a stream, with nothing between them."""

from __future__ import annotations

import pytest
import torch

from deterministic_inference_b200.engine.graphs import token_bucket
from deterministic_inference_b200.kernels import fp4, ops
from tests.fp4_util import Fp4Case

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _rand(*shape, seed=0, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda().to(dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 8])
def test_a_portion_attends_the_same_launched_and_captured(group, dtype):
    """``meta`` with a portion's own lengths, and with its bucket's, which are all that the host knows of a captured step."""
    case = Fp4Case([700], 2, 128, 16, seed=group)
    for n in (2, 3, 4, 5, 7, 8, 11, 16, 17, 33):
        q = _rand(n, 2 * group, 128, seed=n, dtype=dtype)
        own, bucket = case.meta([n]), case.meta([n])
        upper, least = token_bucket(n)
        bucket.q_lens, bucket.kv_lens = [upper], [1024 + upper - least]
        want = ops.paged_attention(q, case.cache(), own, 0.003)
        assert torch.equal(ops.paged_attention(q, case.cache(), bucket, 0.003), want), n


@pytest.mark.parametrize("window", [None, 100])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (2, 2, 128), (6, 2, 64)])
def test_a_prompt_attends_the_same_in_any_portion(hq, hkv, d, window):
    """Down to two tokens."""
    case = Fp4Case([900], hkv, d, 16, seed=6)
    q = _rand(500, hq, d, seed=7, dtype=BF16)
    whole = ops.paged_attention(q, case.cache(), case.meta([500]), 0.003, window)
    for n in (450, 333, 128, 33, 17, 5, 2):
        got = ops.paged_attention(q[500 - n:].contiguous(), case.cache(), case.meta([n]), 0.003, window)
        assert torch.equal(got, whole[500 - n:]), n


@pytest.mark.parametrize("window", [None, 5000])
def test_prompts_in_several_launches(window, monkeypatch):
    """The bfloat16 pages limited to a few of them a launch, decoded tokens with many keys among the prompts: the same bits."""
    case, q_lens = Fp4Case([9000, 300, 4500, 14000, 20000], 2, 128, 16, seed=2), [700, 1, 90, 333, 1]
    q = _rand(sum(q_lens), 8, 128, seed=1, dtype=BF16)
    want = ops.paged_attention(q, case.cache(), case.meta(q_lens), 0.003, window)
    ops.check_kernel_status()
    exact, _, _ = case.attention(q, q_lens, 0.003, window)
    # (bfloat16's roundings of the weights and of the output: 2^-9 of each at most)
    assert ((want.double() - exact).norm(dim=-1) < 2.0 ** -7 * exact.norm(dim=-1)).all()
    for pages in (1, 80, 120):
        monkeypatch.setattr(fp4, "PAGES_BYTES", pages * 4 * 2 * 128 * 128)
        meta = case.meta(q_lens)
        assert torch.equal(ops.paged_attention(q, case.cache(), meta, 0.003, window), want)
        parts = next(iter(meta.scratch.values()))
        assert sum(isinstance(p, fp4._PromptPart) for p in parts) == (3 if pages < 120 else 2)


@pytest.mark.parametrize("lens,q_lens", [([66000, 5000, 300], [60, 70, 80]), ([5000, 66000, 4500], [40, 5, 4300])])
def test_portions_beside_one_of_many_keys(lens, q_lens):
    """More than 65,536 keys, which another kernel attends to: the step's other portions keep theirs."""
    case = Fp4Case(lens, 1, 128, 16, seed=2)
    q = _rand(sum(q_lens), 4, 128, seed=1, dtype=BF16)
    got = ops.paged_attention(q, case.cache(), case.meta(q_lens), 0.003, None)
    at = 0
    for s, n in enumerate(q_lens):
        alone = case.alone(s)
        assert torch.equal(got[at:at + n], ops.paged_attention(q[at:at + n].contiguous(), alone.cache(), alone.meta([n]), 0.003, None)), s
        at += n
    ops.check_kernel_status()


@pytest.mark.parametrize("hq,hkv", [(4, 2), (16, 1)])
@pytest.mark.parametrize("long", [4094, 4095, 4096, 4500])
def test_a_long_portion_beside_others_in_several_launches(long, hq, hkv, monkeypatch):
    """Portions of more tokens than a chunk of keys, in front of other launches of the step with many keys: a launch adds up chunks of
    its own sequences' rows alone."""
    case, q_lens = Fp4Case([long, 5000, 130, 4600], hkv, 128, 16, seed=2), [long, 60, 100, 4300 if long == 4500 else 40]
    q = _rand(sum(q_lens), hq, 128, seed=1, dtype=BF16)
    want = ops.paged_attention(q, case.cache(), case.meta(q_lens), 0.003, None)
    assert want.isfinite().all()
    monkeypatch.setattr(fp4, "PAGES_BYTES", 1)
    meta = case.meta(q_lens)
    assert torch.equal(ops.paged_attention(q, case.cache(), meta, 0.003, None), want)
    assert sum(isinstance(p, fp4._PromptPart) for p in next(iter(meta.scratch.values()))) >= 3
    ops.check_kernel_status()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hq,hkv,d", [(16, 8, 128), (4, 2, 64), (6, 2, 96), (8, 1, 128)])
@pytest.mark.parametrize("window", [None, 100])
def test_drafted_tokens_attend_the_same_in_any_step(hq, hkv, d, window, dtype):
    """Steps whose tiles have 4, 8 and 16 rows, by their longest draft."""
    case = Fp4Case([900, 333, 1500, 40, 700, 513], hkv, d, 16, seed=6)
    for q_lens in ([1, 1, 2, 2, 3, 1], [1, 2, 4, 3, 2, 4], [1, 1, 1, 1, 1, 1]):
        q = _rand(sum(q_lens), hq, d, seed=7, dtype=dtype)
        whole = ops.fp4_paged_attention(q, case.cache(), case.meta(q_lens), 0.003, window)
        at = 0
        for s, n in enumerate(q_lens):
            got = ops.fp4_paged_attention(q[at:at + n].contiguous(), case.cache(), case.alone(s).meta([n]), 0.003, window)
            assert torch.equal(got, whole[at:at + n]), (q_lens, s)
            at += n


@pytest.mark.parametrize("hq,hkv,lens,q_len", [(64, 8, [300] * 16, 1), (64, 8, [512, 257, 400], 1), (16, 8, [300] * 8, 4),
                                               (40, 1, [511] * 4, 1), (8, 8, [200, 40], 1)])
def test_a_product_behind_attention_reads_all_of_it(hq, hkv, lens, q_len):
    case = Fp4Case(lens, hkv, 128, 16, seed=1)
    cache, meta, t = case.cache(), case.meta([q_len] * len(lens)), q_len * len(lens)
    w = ops.Fp4Weight.of(_rand(256, hq * 128, seed=2))
    queries = [_rand(t, hq, 128, seed=s, dtype=BF16) for s in (3, 4)]
    want = []
    for q in queries:
        out = ops.fp4_paged_attention(q, cache, meta, 0.003)
        torch.cuda.synchronize()
        want.append(ops.fp4_linear(out.view(t, -1), w))
    torch.cuda.synchronize()
    # (the two queries in turn: memory used again holds the other one's results)
    got = [ops.fp4_linear(ops.fp4_paged_attention(queries[i & 1], cache, meta, 0.003).view(t, -1), w) for i in range(60)]
    ops.check_kernel_status()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i & 1]), f"pass {i}"


def test_a_step_one_operator_behind_the_other():
    """Product, norm and rotation into the cache, attention, product, for steps of a prompt and of single tokens, without a pause
    and with one behind every operator."""
    hq, hkv, d, hidden, page = 8, 2, 128, 512, 16
    w = ops.Fp4Weight.of(_rand((hq + 2 * hkv) * d, hidden, seed=1) * 0.05)
    w_o = ops.Fp4Weight.of(_rand(hidden, hq * d, seed=2) * 0.05)
    norm, table = torch.ones(d, device="cuda"), _rand(600, d, seed=3)
    case = Fp4Case([400, 300], hkv, d, page, seed=4)

    def steps(pause):
        cache = ops.Fp4Cache.zeros(case.data.shape[0], hkv, page, d)
        outs = []
        for lens, news in (([300, 200], [300, 200]), ([301, 201], [1, 1]), ([306, 203], [5, 2]), ([400, 204], [94, 1])):
            meta = case.meta(news, lens)
            slots = torch.cat([torch.tensor([t[p // page] * page + p % page for p in range(n - m, n)], dtype=torch.int32)
                               for t, n, m in zip(case.tables, lens, news)]).cuda()
            x = _rand(sum(news), hidden, seed=sum(lens), dtype=BF16)
            q = ops.qkv_project(x, w, hq, hkv, d, norm, norm, 1e-6, table, meta.positions, cache, slots, page)
            pause()
            o = ops.paged_attention(q, cache, meta, d ** -0.5)
            pause()
            outs.append(ops.linear(o.view(sum(news), -1), w_o))
            pause()
        torch.cuda.synchronize()
        return outs

    want = steps(torch.cuda.synchronize)
    for _ in range(3):
        for a, b in zip(steps(lambda: None), want):
            assert torch.equal(a, b)
    ops.check_kernel_status()


@pytest.mark.parametrize("hq,hkv", [(16, 8), (64, 8)])
def test_a_captured_step_of_shorter_sequences(hq, hkv):
    """A graph made for 2,100 keys a sequence, replayed with 40 and with none; two graphs of the same step in turn."""
    case = Fp4Case([2100] * 8, hkv, 128, 64, seed=1)
    cache, meta = case.cache(), case.meta([1] * 8)
    w = ops.Fp4Weight.of(_rand(256, hq * 128, seed=2))
    queries = [_rand(8, hq, 128, seed=s, dtype=BF16) for s in (3, 4)]
    q = torch.empty_like(queries[0])
    run = lambda: ops.fp4_linear(ops.fp4_paged_attention(q, cache, meta, 0.003).view(8, -1), w)
    q.copy_(queries[0])
    run()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = run()
        graphs.append((graph, y))
    for lens in ([2100] * 8, [40] * 8, [1, 0, 300, 2048, 2049, 77, 129, 1000]):
        meta.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        for x in queries:
            q.copy_(x)
            want = ops.fp4_linear(ops.fp4_paged_attention(x, cache, case.meta([1] * 8, lens), 0.003).view(8, -1), w)
            torch.cuda.synchronize()
            for graph, y in graphs:
                graph.replay()
                torch.cuda.synchronize()
                assert torch.equal(y, want)
    ops.check_kernel_status()


def test_two_streams_at_once():
    """Attention and products on two streams at the same time, of the same cache and weight."""
    case = Fp4Case([900, 3000, 100], 2, 128, 16, seed=1)
    cache, w = case.cache(), ops.Fp4Weight.of(_rand(1024, 1024, seed=2))
    queries = [_rand(n, 8, 128, seed=n, dtype=BF16) for n in (3, 66)]
    q_lens = ([1, 1, 1], [30, 4, 32])
    run = lambda i, meta: ops.fp4_linear(ops.fp4_paged_attention(queries[i], cache, meta, 0.003).view(-1, 1024), w)
    metas = [case.meta(x) for x in q_lens]
    want = [run(i, metas[i]) for i in (0, 1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in (0, 1)]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(i, metas[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(y, want[i]) for y in got[i])
    ops.check_kernel_status()
