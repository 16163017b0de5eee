"""What a token's bits over a cache in 8 bits do not depend on: whether its step was launched or replayed, where its prompt was
cut, the other sequences of the step, and keys that it does not see."""

from __future__ import annotations

import pytest
import torch

from deterministic_inference_b200 import EngineConfig
from deterministic_inference_b200.engine.batch import SequenceInput
from deterministic_inference_b200.engine.graphs import token_bucket
from deterministic_inference_b200.engine.runner import ModelRunner
from deterministic_inference_b200.kernels import ops
from tests.int8_util import Int8Case

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _rand(*shape, seed=0, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda().to(dtype)


# ---- portions

@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 8])
def test_a_portion_attends_the_same_launched_and_captured(group, dtype):
    """``meta`` with a portion's own lengths, and with its bucket's, which are all that the host knows of a captured step."""
    case = Int8Case([700], 2, 128, 16, seed=group)
    cache = ops.Int8Cache(case.data, case.scales)
    for n in (2, 3, 4, 5, 7, 8, 11, 16, 17, 33):
        q = _rand(n, 2 * group, 128, seed=n, dtype=dtype)
        own, bucket = case.meta([n]), case.meta([n])
        upper, least = token_bucket(n)
        bucket.q_lens, bucket.kv_lens = [upper], [1024 + upper - least]
        want = ops.paged_attention(q, cache, own, 0.1)
        assert torch.equal(ops.paged_attention(q, cache, bucket, 0.1), want), n


@pytest.mark.parametrize("window", [None, 100])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (2, 2, 128), (6, 2, 64)])
def test_a_prompt_attends_the_same_in_short_portions(hq, hkv, d, window):
    """Down to two tokens."""
    case = Int8Case([400], hkv, d, 16, seed=6)
    q = _rand(200, hq, d, seed=7, dtype=BF16)
    cache = ops.Int8Cache(case.data, case.scales)
    whole = ops.paged_attention(q, cache, case.meta([200]), 0.1, window)
    for n in (33, 17, 16, 9, 4, 3, 2):
        got = ops.paged_attention(q[200 - n:].contiguous(), cache, case.meta([n]), 0.1, window)
        assert torch.equal(got, whole[200 - n:]), n


def test_a_portion_attends_the_same_at_any_number_of_keys():
    """Around 65,536 keys, where a captured step reckons with more keys than a launched one."""
    case = Int8Case([70000], 1, 128, 64, seed=3)
    cache = ops.Int8Cache(case.data, case.scales)
    for n, keys in ((40, 65530), (5, 65536), (200, 65600), (40, 70000)):
        q = _rand(n, 4, 128, seed=n, dtype=BF16)
        own, bucket = case.meta([n], [keys]), case.meta([n], [keys])
        upper, least = token_bucket(n)
        bucket.q_lens, bucket.kv_lens = [upper], [70000 + upper - least]
        want = ops.paged_attention(q, cache, own, 0.1)
        assert torch.equal(ops.paged_attention(q, cache, bucket, 0.1), want), (n, keys)
        exact, _, _ = case.attention(q, [n], 0.1, kv_lens=[keys])
        # the output's rounding to bfloat16: 2^-8 of an element at most, 0.0017 in the root mean square; of 128 elements, with
        # the roundings to float16 in front of it, well below 2^-8
        off = (want.double() - exact).norm(dim=-1) / exact.norm(dim=-1)
        assert off.max() < 2.0 ** -8
        part = ops.paged_attention(q[n // 2:].contiguous(), cache, case.meta([n - n // 2], [keys]), 0.1)
        assert torch.equal(part, want[n // 2:])


@pytest.mark.parametrize("window", [None, 5000])
def test_partial_results_in_several_launches(window, monkeypatch):
    """The prompt form's partial results limited to a few pairs of query tiles a launch: the same bits."""
    from deterministic_inference_b200.kernels import int8
    case = Int8Case([9000, 300, 4500, 14000], 2, 128, 16, seed=2)
    cache, q_lens = ops.Int8Cache(case.data, case.scales), [700, 1, 90, 333]
    q = _rand(sum(q_lens), 8, 128, seed=1, dtype=BF16)
    want = ops.paged_attention(q, cache, case.meta(q_lens), 0.1, window)
    for pairs in (1, 3, 8):
        monkeypatch.setattr(int8, "SCRATCH_BYTES", pairs * 64 * 8 * 4 * 520)
        meta = case.meta(q_lens)
        assert torch.equal(ops.paged_attention(q, cache, meta, 0.1, window), want)
        part = next(p for p in meta.scratch[next(iter(meta.scratch))] if isinstance(p, int8._PromptPart))
        assert len(part.launches) == -(-(11 + 2 + 6) // pairs) and part.rows <= pairs * 64
    ops.check_kernel_status()


# ---- the other sequences of a step, and keys that a row does not see

def _alone(case, s):
    """Sequence s of a case by itself."""
    alone = Int8Case.__new__(Int8Case)
    alone.__dict__.update(case.__dict__)
    alone.tables, alone.lens = [case.tables[s]], [case.lens[s]]
    return alone


@pytest.mark.parametrize("window", [None, 60, 150])
@pytest.mark.parametrize("step", [4, -4, 13, -13])
def test_a_prompt_with_moving_value_scales_attends_the_same_in_any_step(window, step):
    """Value scales 2^step times larger from each tile of 128 keys to the next; alone, in portions, and beside prompts that make
    query tiles share their keys in another way."""
    scales = lambda n, hkv, g: (2.0 ** (torch.arange(n) // 128 * step) * (1 + torch.arange(n) % 7))[:, None].expand(n, hkv).contiguous()
    case = Int8Case([900, 900, 900, 800], 2, 128, 16, seed=6, value_scales=scales)
    cache, q_lens = ops.Int8Cache(case.data, case.scales), [300, 900, 900, 800]
    q = _rand(sum(q_lens), 8, 128, seed=7, dtype=BF16)
    whole = ops.paged_attention(q, cache, case.meta(q_lens), 0.1, window)
    alone = _alone(case, 0)
    assert torch.equal(ops.paged_attention(q[:300].contiguous(), cache, alone.meta([300]), 0.1, window), whole[:300])
    for n in (200, 131, 33, 2):
        assert torch.equal(ops.paged_attention(q[300 - n:300].contiguous(), cache, alone.meta([n]), 0.1, window), whole[300 - n:300])
    exact, _, _ = alone.attention(q[:300], [300], 0.1, window)
    # (as above)
    assert ((whole[:300].double() - exact).norm(dim=-1) <= 2.0 ** -8 * exact.norm(dim=-1)).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hq,hkv,d", [(16, 8, 128), (4, 2, 64), (6, 2, 128), (8, 1, 128)])
@pytest.mark.parametrize("window", [None, 100])
def test_drafted_tokens_attend_the_same_in_any_step(hq, hkv, d, window, dtype):
    """Steps whose tiles have 4 to 32 rows, by their longest draft."""
    case = Int8Case([900, 333, 1500, 40, 700, 513], hkv, d, 16, seed=6)
    cache = ops.Int8Cache(case.data, case.scales)
    for q_lens in ([1, 1, 2, 2, 3, 1], [1, 2, 4, 3, 2, 5], [1, 1, 8, 2, 16, 3], [2, 1, 5, 20, 2, 2]):
        q = _rand(sum(q_lens), hq, d, seed=7, dtype=dtype)
        whole = ops.int8_paged_attention(q, cache, case.meta(q_lens), 0.1, window)
        at = 0
        for s, n in enumerate(q_lens):
            got = ops.int8_paged_attention(q[at:at + n].contiguous(), cache, _alone(case, s).meta([n]), 0.1, window)
            assert torch.equal(got, whole[at:at + n]), (q_lens, s)
            at += n


def _with_scales(case, s, keys, kv, scale):
    """The case's cache with the scales of some keys of sequence s set."""
    scales = case.scales.clone()
    at = torch.tensor(keys)
    page = torch.tensor(case.tables[s])[at // case.page_size].cuda()
    scales[page, kv, :, (at % case.page_size).cuda()] = scale
    return ops.Int8Cache(case.data, scales)


@pytest.mark.parametrize("kv", [0, 1])
@pytest.mark.parametrize("scale", [float("nan"), float("inf"), 2.0 ** 20, 2.0 ** -40, 0.0])
def test_prompt_rows_do_not_depend_on_keys_before_the_window(kv, scale):
    """Pages that a window has left may be anybody's."""
    case = Int8Case([700], 2, 128, 16, seed=3)
    q = _rand(300, 8, 128, seed=4, dtype=BF16)
    run = lambda cache: ops.paged_attention(q, cache, case.meta([300]), 0.1, 70)
    want = run(ops.Int8Cache(case.data, case.scales))
    assert torch.equal(run(_with_scales(case, 0, range(400 - 69), kv, scale)), want)
    ops.check_kernel_status()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kv", [0, 1])
@pytest.mark.parametrize("q_len", [1, 5])
@pytest.mark.parametrize("scale", [float("nan"), float("inf"), 2.0 ** 20, 2.0 ** -40, 0.0])
def test_few_rows_do_not_depend_on_keys_before_the_window(q_len, kv, scale, dtype):
    case = Int8Case([700, 300], 2, 128, 16, seed=3)
    q = _rand(2 * q_len, 4, 128, seed=4, dtype=dtype)
    run = lambda cache: ops.int8_paged_attention(q, cache, case.meta([q_len] * 2), 0.1, 70)
    want = run(ops.Int8Cache(case.data, case.scales))
    assert want.isfinite().all()
    assert torch.equal(run(_with_scales(case, 0, range(700 - q_len - 69), kv, scale)), want)
    ops.check_kernel_status()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kv", [0, 1])
@pytest.mark.parametrize("portions", [False, True])
@pytest.mark.parametrize("scale", [float("nan"), -float("inf"), 2.0 ** 10, 2.0 ** -5])
def test_rows_do_not_depend_on_later_keys(portions, kv, scale, dtype):
    """The last two of six tokens have another scale: the rows in front keep their bits, and a scale that is no number shows in
    every row that sees it."""
    case = Int8Case([300], 2, 128, 16, seed=5)
    q = _rand(6, 4, 128, seed=4, dtype=dtype)
    run = lambda cache: ops.int8_paged_attention(q, cache, case.meta([6]), 0.1, portions=portions)
    want, got = run(ops.Int8Cache(case.data, case.scales)), run(_with_scales(case, 0, [298, 299], kv, scale))
    assert want.isfinite().all() and torch.equal(got[:4], want[:4])
    assert (got[4:].isnan().all() if scale != scale or abs(scale) == float("inf") else (got[4:] != want[4:]).any())
    ops.check_kernel_status()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("q_len", [1, 4, 40])
def test_a_page_that_is_none_of_the_pools_is_a_page_of_zeros(q_len, dtype):
    """Not what was read before it, and nothing beyond the pool."""
    case = Int8Case([300, 300], 2, 128, 16, seed=5)
    q = _rand(2 * q_len, 4, 128, seed=4, dtype=dtype)
    zeros = ops.Int8Cache(case.data.clone(), case.scales.clone())
    page = case.tables[0][7]
    zeros.scales[page] = 0
    want = ops.int8_paged_attention(q, zeros, case.meta([q_len] * 2), 0.1)
    for entry in (-1, case.data.shape[0], 2 ** 31 - 1):
        meta = case.meta([q_len] * 2)
        meta.block_table[0, 7] = entry
        assert torch.equal(ops.int8_paged_attention(q, ops.Int8Cache(case.data, case.scales), meta, 0.1), want)
    ops.check_kernel_status()


@pytest.mark.parametrize("name", ["d", "e"])
def test_short_portions_replayed_give_the_bits_of_launched_ones(name, tiny_model_dirs):
    """Portions of 3 to 7 tokens behind different prompts, one bucket: from the third on they are replayed."""
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, 300, (40 + i,), generator=g).tolist() for i in range(6)]
    outs = []
    for graphs in (True, False):
        r = ModelRunner(EngineConfig(model_path=str(tiny_model_dirs[name]), dtype="bfloat16", weight_dtype="int8",
                                     cache_dtype="int8", kv_pool_tokens=4096, page_size=32, max_reqs=16, max_seq_len=512,
                                     cuda_graphs=graphs))
        rows = []
        for p, n in zip(prompts, (5, 3, 7, 4, 6, 3)):
            slot = r.cache.allocate_slot()
            for at, m in ((0, len(p) - n), (len(p) - n, n)):
                rows.append(r.step([SequenceInput(slot, p[at:at + m], at, [m - 1])])[0].clone())
                torch.cuda.synchronize()
        if graphs:
            assert r.step_graphs.replays >= 2
        outs.append(rows)
    ops.check_kernel_status()
    for i, (a, b) in enumerate(zip(*outs)):
        assert torch.equal(a, b), i


def test_a_portion_whose_work_is_large():
    """1,024 float32 tokens of 512 heads on one kv head: the count of work items once went beyond 31 bits, and rows were left
    out."""
    case = Int8Case([1024], 1, 16, 16, seed=1)
    cache, q = ops.Int8Cache(case.data, case.scales), _rand(1024, 512, 16, seed=2)
    out = ops.int8_paged_attention(q, cache, case.meta([1024]), 0.25)
    ops.check_kernel_status()
    exact, vmax, smax = case.attention(q, [1024], 0.25)
    tol = (2 * smax * (2.0 ** -21 + 4 * 2.0 ** -23) + 2.0 ** -20) * vmax      # as for every float32 case
    assert ((out.double() - exact).abs() <= tol).all()
