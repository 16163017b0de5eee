"""What attention over the 4-bit cache allocates beside its output, and for whom, as far as the host settles it."""

from __future__ import annotations

import random
from types import SimpleNamespace

import pytest
import torch

from deterministic_inference_b200.kernels import fp4

ROW_BYTES = 528      # of a partial result: 128 sums, two references, a sum of weights


def _parts(q_lens, kv_lens, group=4, hkv=8, stream=False, portions=True):
    meta = SimpleNamespace(q_lens=q_lens, kv_lens=kv_lens, block_table=torch.zeros(len(q_lens), 1, dtype=torch.int32), scratch={})
    return fp4._parts(meta, group, hkv, 128, 16, False, stream, portions, torch.device("cpu"))


def _bytes(parts):
    return sum(p.rows for p in parts) * ROW_BYTES


def _listed(part):
    return part.list.tolist() if part.list is not None else list(range(part.first, part.first + part.count))


STEPS = [([8000] + [5] * 63, [8000] + [300] * 63), ([8000] + [5] * 200, [8000] + [2100] * 200), ([2] * 40 + [6000, 1000, 3], [32000] * 43),
         ([1] * 30 + [4000] + [2] * 30, [500] * 30 + [40000] + [70] * 30)]


@pytest.mark.parametrize("q_lens,kv_lens", STEPS)
@pytest.mark.parametrize("stream", [False, True])
def test_partial_results_follow_the_sequences_own_sizes(q_lens, kv_lens, stream):
    """A long portion beside short ones: at most twice what the sequences take one by one, or the limit of a launch."""
    parts = _parts(q_lens, kv_lens, stream=stream)
    alone = sum(_bytes(_parts([q], [kv], stream=stream)) for q, kv in zip(q_lens, kv_lens))
    assert _bytes(parts) <= 2 * alone + len(parts) * (1 << 28)
    assert max(p.rows for p in parts) * ROW_BYTES <= max(2 * alone, 1 << 28)
    assert len(parts) <= 6
    seen = sorted(s for p in parts for s in _listed(p))
    assert seen == list(range(len(q_lens)))
    for p in parts:      # blocks of the kernel that adds partial results up
        if p.runs:
            assert p.count * p.max_rows * 8 <= p.rows


def test_ordinary_steps_are_one_launch_for_single_tokens_and_one_for_drafts():
    rng = random.Random(1)
    for _ in range(50):
        q_lens = sorted(rng.choice([1, 1, 1, 5]) for _ in range(64))
        parts = _parts(q_lens, [rng.randrange(5, 9000) for _ in range(64)], portions=False)
        assert len(parts) == len(set(q_lens))


def test_a_step_keeps_no_partial_results_of_prompts(monkeypatch):
    """Calls on one step, on two streams or in two captured graphs, must not write the same partial results: what the step keeps between
    calls is lists of whole numbers."""
    from deterministic_inference_b200.kernels import attention_bf16, ops

    calls = []

    class Library:
        def __getattr__(self, name):
            return lambda *args: calls.append((name, args)) or 0

    made = []
    empty = torch.empty
    monkeypatch.setattr(ops, "_lib", lambda name: Library())
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(torch, "empty", lambda *a, **k: made.append(empty(*a, **k)) or made[-1])
    q = torch.zeros(5000, 4, 128, dtype=torch.bfloat16)
    cache = torch.zeros(1, 2, 2, 128, 128, dtype=torch.bfloat16)
    ints = lambda x: torch.tensor(x, dtype=torch.int32)
    meta = SimpleNamespace(block_table=ints([[0]]), token_seq=ints([0]), cu_q_lens=ints([0, 5000]), seq_lens=ints([9000]), q_lens=[5000],
                           kv_lens=[9000], num_decode=0, scratch={})
    for _ in range(2):
        attention_bf16.run(q, torch.zeros_like(q), cache, meta, 0.1, 0)

    def tensors(x):
        if isinstance(x, torch.Tensor):
            yield x
        elif isinstance(x, (list, tuple)):
            for y in x:
                yield from tensors(y)

    assert meta.scratch and not [t for t in tensors(list(meta.scratch.values())) if t.is_floating_point()]
    assert len(calls) == 2 and len(made) == 4 and len({t.data_ptr() for t in made}) == 4       # (held on to by `made`: each its own)
