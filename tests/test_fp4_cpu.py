"""What serving in 4 bits settles on the host: options, page sizes in bytes, the work lists, refusals without a GPU; and what can be
shown from the kernels' sources."""

from __future__ import annotations

import random
import re

import pytest
import torch

from deterministic_inference_b200 import EngineConfig, preset
from deterministic_inference_b200.cache.manager import CacheManager, group_page_bytes
from deterministic_inference_b200.kernels import fp4, ops
from deterministic_inference_b200.kernels.build import CSRC
from deterministic_inference_b200.parts.spec import PagedKVSpec
from tests import test_kernel_sources_cpu as sources
from tests.fp4_util import quantised, values


def test_options():
    ok = EngineConfig(model_config=preset("tiny_a"), random_seed=0, weight_dtype="fp4", cache_dtype="fp4")
    assert ok.weight_dtype == ok.cache_dtype == "fp4"
    for name in ("weight_dtype", "cache_dtype"):
        with pytest.raises(ValueError, match=name):
            EngineConfig(model_config=preset("tiny_a"), random_seed=0, **{name: "int4"})


def test_page_bytes():
    specs = {0: PagedKVSpec(8, 128), 1: PagedKVSpec(8, 128)}
    (_, narrow), = group_page_bytes(specs, 16, torch.float4_e2m1fn_x2).values()
    assert narrow == 2 * 8 * 16 * 2 * (64 + 8 + 1)
    manager = CacheManager(specs, 4, 16, 2, 64, dtype=torch.float4_e2m1fn_x2, device="cpu", allocate_device=False)
    assert manager.bytes_per_page() == narrow


def test_there_is_no_cpu_path():
    x = torch.zeros(2, 64)
    for call in (lambda: ops.fp4_quantize_rows(x), lambda: ops.Fp4Weight.of(x), lambda: ops.Fp4Weight(*quantised(x), 64),
                 lambda: ops.Fp4Cache.zeros(2, 1, 16, 64, device="cpu")):
        with pytest.raises(ops.KernelError, match="CUDA"):
            call()


def test_the_rule():
    """Every code of every scale comes back as itself, and a value is off by half a step of its code at most, a sixth of its block's
    largest (and, where e4m3 rounds the scale down, by what lies above six of them)."""
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6])
    for bits in range(8, 127):
        scale = torch.tensor(bits, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
        row = torch.cat([torch.cat([table, -table]) * scale, torch.tensor([2688.0] + [0.0] * 15)])[None]
        assert torch.equal(values(*quantised(row), 32, torch.float32), row)
    x = torch.randn(200, 512, generator=torch.Generator().manual_seed(1)) * torch.exp2(torch.arange(200) - 100.0)[:, None]
    off = (values(*quantised(x), 512) - x.double()).abs().unflatten(-1, (-1, 16)).amax(-1)
    assert (off <= x.double().abs().unflatten(-1, (-1, 16)).amax(-1) * 0.1771).all()


def _device_items(q: int, kv: int, group: int, hkv: int, tile_rows: int) -> tuple:
    split = ops._lib("attention_fp4").dib_fp4_attention_split_keys(kv, q * group)
    runs = max(1, -(-kv // split))
    return -(-q * group // tile_rows) * runs * hkv, runs


@pytest.mark.parametrize("group", [1, 2, 4, 5, 8, 40])
@pytest.mark.parametrize("stream", [False, True])
def test_split_work_covers_the_steps_that_the_lengths_allow(group, stream):
    """Work items and partial results are sized for every step that the host's lengths, upper bounds in a captured step, allow;
    and where none of those has a second run of keys, there are no partial results and no merge."""
    rng = random.Random(group)
    for _ in range(300):
        n = rng.randrange(1, 5)
        q_lens = [rng.choice([1, 1, 2, 3, 7, 32 // group + 1, 200]) for _ in range(n)]
        kv_lens = [rng.choice([1, 100, 256, 257, 300, 512, 513, 2048, 2049, 4096, 16385, rng.randrange(1, 40000)]) for _ in range(n)]
        part = fp4._SplitPart(list(range(n)), q_lens, kv_lens, group, 8, stream, torch.device("cpu"))
        for q, kv in zip(q_lens, kv_lens):
            for _ in range(20):
                q1, kv1 = rng.choice([q, rng.randrange(1, q + 1)]), rng.choice([kv, rng.randrange(1, kv + 1)])
                items, runs = _device_items(q1, kv1, group, 8, part.tile_rows)
                assert items <= part.items and (runs == 1 or part.rows > 0), (q1, kv1, part.items, items)
            if _device_items(1, min(kv, 2048), group, 8, part.tile_rows)[1] > 1:
                assert part.rows == part.count * part.items * part.tile_rows


def test_prompt_pages_cover_every_key():
    """Every page of 128 keys of a sequence of the prompt form has a number of its own, the others have no tokens there."""
    q_lens, kv_lens = [1, 3, 200, 70, 500], [9, 50, 200, 4500, 9000]
    part = fp4._PromptPart([2, 3, 4], q_lens, kv_lens, None, torch.device("cpu"))
    assert part.meta.q_lens == [0, 0, 200, 70, 500] and part.meta.kv_lens == [0, 0, 200, 4500, 9000]
    assert part.mask.tolist() == [0, 0, 1, 1, 1] and part.pages == 2 + 36 + 71 and part.most == 71
    table = part.meta.block_table
    seen = [table[s, p].item() for s, n in zip((2, 3, 4), (2, 36, 71)) for p in range(n)]
    assert seen == list(range(part.pages)) and not table[:2].any()


SOURCES = ("rows_fp4.cu", "gemm_fp4.cu", "cache_fp4.cu", "attention_fp4.cu", "attention_fp4_stream.cu")


@pytest.mark.parametrize("name", SOURCES)
def test_no_block_leaves_without_having_waited_for_the_kernel_in_front(name):
    sources.test_no_block_leaves_without_having_waited_for_the_kernel_in_front(name)


@pytest.mark.parametrize("name", ["gemm_fp4.cu", "attention_fp4_stream.cu"])
def test_a_kernel_that_gives_up_waits_for_its_copies(name):
    """After a wait that ran out a kernel waits for the copies it has sent for, with a limit again; and no barrier without a limit
    has warps that may be missing from it."""
    kernels = sources._limited(name)
    assert kernels
    for kernel, body in kernels:
        copies = re.search(r"for \(int (\w) = [^;]*(?:- a?\.?stages|- STAGES|- SH::STAGES)[^;]*; [^;]*; \+\+\w\)\s*"
                           r"mbar_wait_brief\(&full\[", body)
        assert copies, f"{name}: {kernel} leaves with copies in flight"
        assert not re.search(r"bar\.sync", body), f"{name}: {kernel}"


def test_no_source_waits_without_a_limit():
    for name in SOURCES:
        text = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
        assert "while (true)" not in text and "try_wait" not in text, name
