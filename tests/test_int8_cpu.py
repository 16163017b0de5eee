"""What serving in 8 bits settles on the host: options, page sizes in bytes, the work lists, refusals without a GPU."""

from __future__ import annotations

import random

import pytest
import torch

from deterministic_inference_b200 import EngineConfig, preset
from deterministic_inference_b200.cache.manager import CacheManager, group_page_bytes
from deterministic_inference_b200.kernels import int8, ops
from deterministic_inference_b200.parts.spec import PagedKVSpec


def test_options():
    ok = EngineConfig(model_config=preset("tiny_a"), random_seed=0, weight_dtype="int8", cache_dtype="int8")
    assert ok.weight_dtype == ok.cache_dtype == "int8"
    for name in ("weight_dtype", "cache_dtype"):
        with pytest.raises(ValueError, match=name):
            EngineConfig(model_config=preset("tiny_a"), random_seed=0, **{name: "fp8"})


def test_page_bytes():
    specs = {0: PagedKVSpec(8, 128), 1: PagedKVSpec(8, 128)}
    (_, wide), = group_page_bytes(specs, 16, torch.bfloat16).values()
    (_, narrow), = group_page_bytes(specs, 16, torch.int8).values()
    assert wide == 2 * 8 * 16 * 512 and narrow == 2 * 8 * 16 * (256 + 8)
    manager = CacheManager(specs, 4, 16, 2, 64, dtype=torch.int8, device="cpu", allocate_device=False)
    assert manager.bytes_per_page() == narrow


def test_there_is_no_cpu_path():
    x = torch.zeros(2, 64)
    for call in (lambda: ops.quantize_rows(x), lambda: ops.Int8Weight.of(x),
                 lambda: ops.Int8Weight(x.to(torch.int8), torch.ones(2)), lambda: ops.Int8Cache.zeros(2, 1, 16, 64, device="cpu")):
        with pytest.raises(ops.KernelError, match="CUDA"):
            call()


def test_prompt_units_cover_every_token_once():
    """Every token of a sequence of the prompt form is in one query tile, with the chunks of keys up to its own position."""
    for q_lens, kv_lens in (([1, 3, 200, 70, 500], [9, 50, 200, 4500, 9000]), ([130, 129], [130, 700])):
        many = [s for s, n in enumerate(q_lens) if n * 2 > int8.PROMPT_ROWS]
        part = int8._PromptPart.__new__(int8._PromptPart)
        int8._sm_counts[torch.device("cpu")] = 148
        part.__init__(many, q_lens, kv_lens, 2, 8, 0, torch.device("cpu"))
        seq, a, b, chunk = part.units.view(4, part.count).tolist()
        seen = {}
        for s, t0, t1, c in zip(seq, a, b, chunk):
            for t in (t0, t1):
                if t >= 0:
                    for tok in range(t, min(t + 64, q_lens[s])):
                        assert (s, tok, c) not in seen
                        seen[s, tok, c] = True
        for s in many:
            for tok in range(q_lens[s]):
                last = (kv_lens[s] - q_lens[s] + tok) // 4096 if part.chunk_tiles else 0
                assert all((s, tok, c) in seen for c in range(last + 1))
        assert part.seq_list.tolist() == many and part.max_tokens == max(q_lens[s] for s in many)


def _runs(keys: int, rows: int) -> int:
    return max(1, -(-keys // int8._lib().dib_int8_attention_split_keys(keys, rows)))


@pytest.mark.parametrize("group", [1, 2, 4, 5, 8, 40])
@pytest.mark.parametrize("wide", [False, True])
def test_split_work_covers_the_steps_that_the_lengths_allow(group, wide):
    """Work items and partial results are sized for every step that the host's lengths, upper bounds in a captured step, allow;
    and where none of those has a second run of keys, there are no partial results and no merge."""
    rng = random.Random(group)
    for _ in range(300):
        n = rng.randrange(1, 5)
        q_lens = [rng.choice([1, 1, 2, 3, 7, 32 // group + 1, 200]) for _ in range(n)]
        kv_lens = [rng.choice([1, 100, 256, 257, 300, 512, 513, 4096, 16384, 16385, rng.randrange(1, 40000)]) for _ in range(n)]
        part = int8._SplitPart(list(range(n)), q_lens, kv_lens, group, 8, wide, torch.device("cpu"))
        two = False
        for q, kv in zip(q_lens, kv_lens):
            for _ in range(20):
                q1, kv1 = rng.choice([q, rng.randrange(1, q + 1)]), rng.choice([kv, rng.randrange(1, kv + 1)])
                runs = _runs(kv1, q1 * group)
                assert 8 * -(-q1 * group // part.tile_rows) * runs <= part.items
                two |= runs > 1
            two |= _runs(min(kv, 16384), group) > 1
        assert (part.rows > 0) == two


def _device_work(q: int, kv: int, group: int, hkv: int, tile_rows: int) -> int:
    """What the split form's kernel counts for a sequence."""
    split = int8._lib().dib_int8_attention_split_keys(kv, q * group)
    return -(-q * group // tile_rows) * max(1, -(-kv // split)) * hkv * (-(-min(split, max(kv, 512)) // 128) + 1)


def test_the_work_of_a_step_is_counted_without_overflow():
    """A long float32 portion's work, and that of several, stays below 2^31; a step beyond it is refused."""
    for q, kv, group, hkv in ((23171, 23171, 8, 8), (100000, 100000, 8, 8), (1024, 1024, 512, 1), (8192, 65536, 8, 8)):
        part = int8._SplitPart([0], [q], [kv], group, hkv, True, torch.device("cpu"))
        assert _device_work(q, kv, group, hkv, part.tile_rows) < 1 << 31
    for group in (1, 8):
        int8._SplitPart(list(range(64)), [8192] * 64, [8192] * 64, group, 8, True, torch.device("cpu"))
        with pytest.raises(ops.KernelError, match="smaller portions"):
            int8._SplitPart([0], [1 << 21], [1 << 21], group, 8, True, torch.device("cpu"))
    rng = random.Random(3)
    for _ in range(3000):
        group, tile_rows = rng.choice([1, 2, 5, 8, 64]), rng.choice([4, 8, 16, 24, 32])
        q, kv = int(2 ** rng.uniform(0, 15)), int(2 ** rng.uniform(0, 18))
        runs = int8._most_runs(kv, group)
        most = int8._split_work([0], [q], [kv], group, 8, tile_rows, runs)
        for _ in range(5):
            assert _device_work(rng.randrange(1, q + 1), rng.randrange(1, kv + 1), group, 8, tile_rows) <= most
