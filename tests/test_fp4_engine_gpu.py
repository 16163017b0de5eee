"""The engine with its matrices and its cache in 4 bits: the model against a restatement in 64 bits with the same quantisation, and
generation that does not depend on the batch or on graph replay."""

from __future__ import annotations

import pytest
import torch

from deterministic_inference_b200 import Engine, EngineConfig, SamplingParams
from deterministic_inference_b200.engine.batch import SequenceInput
from deterministic_inference_b200.engine.runner import ModelRunner
from deterministic_inference_b200.kernels import ops
from tests import plain_qwen3 as plain
from tests.fp4_util import rounded

pytestmark = pytest.mark.gpu


def _plain_layer(cfg, w, i, x):
    """Layer i on the residual stream x of a whole sequence in 64 bits: what it adds to the stream, its weights, the products'
    inputs, keys and values quantised by rows."""
    d, eps, n = cfg["head_dim"], cfg["rms_norm_eps"], x.shape[0]
    product = lambda x, m: rounded(x) @ rounded(m).T
    angles = plain.rope_angles(torch.arange(n), d, cfg["rope_theta"])
    p = f"model.layers.{i}."
    h = plain.rms_norm(x, w[p + "input_layernorm.weight"], eps)
    q, k, v = (product(h, w[p + f"self_attn.{name}_proj.weight"]).view(n, -1, d) for name in "qkv")
    q = plain.apply_rope(plain.rms_norm(q, w[p + "self_attn.q_norm.weight"], eps), angles)
    k = plain.apply_rope(plain.rms_norm(k, w[p + "self_attn.k_norm.weight"], eps), angles)
    o = plain.attention(q, rounded(k), rounded(v), d ** -0.5, plain.layer_window(cfg, i))
    o = product(o.reshape(n, -1), w[p + "self_attn.o_proj.weight"])
    h = plain.rms_norm(x + o, w[p + "post_attention_layernorm.weight"], eps)
    gate, up = product(h, w[p + "mlp.gate_proj.weight"]), product(h, w[p + "mlp.up_proj.weight"])
    return o + product(gate * torch.sigmoid(gate) * up, w[p + "mlp.down_proj.weight"])


@pytest.mark.parametrize("name,page", [("a", 16), ("d", 16), ("e", 32)])
def test_layers_in_4_bits(tiny_model_dirs, name, page):
    """A prompt in one step, its tail in small ones; every layer on the stream that the engine gave it.  A value next to the
    border between two codes may fall to either side, a sixth of its block's largest at most, and moves others behind it in the
    layer; a token has some thousand values in a layer, each within 2^-20 of a border once in 2^17, so most tokens have none: the
    median is float32's own error, and no token is off by more than a few such steps of one value in 64 or more, 1 / 6 / 8 each."""
    cfg, w = plain.read_model_dir(tiny_model_dirs[name], torch.float64)
    ids = torch.randint(0, cfg["vocab_size"], (150,), generator=torch.Generator().manual_seed(4)).tolist()
    runner = ModelRunner(EngineConfig(model_path=str(tiny_model_dirs[name]), dtype="float32", weight_dtype="fp4",
                                      cache_dtype="fp4", kv_pool_tokens=1024, page_size=page, debug_checks=True,
                                      cuda_graphs=False))
    streams = [[] for _ in range(cfg["num_hidden_layers"])]
    runner.model.after_layer = lambda entry, hidden, residual: streams[entry.layer].append(
        (ops.as_tensor(hidden) + residual).double().cpu())
    slot = runner.cache.allocate_slot()
    for at, n in ((0, 140), (140, 4), (144, 1), (145, 1), (146, 4)):
        runner.step([SequenceInput(slot=slot, tokens=ids[at:at + n], num_computed=at, want=list(range(n)))])
    ops.check_kernel_status()
    x = w["model.embed_tokens.weight"][torch.tensor(ids)]
    for i, stream in enumerate(streams):
        got, want = torch.cat(stream) - x, _plain_layer(cfg, w, i, x)
        rel = (got - want).norm(dim=1) / want.norm(dim=1)
        assert rel.max() < 0.1 and rel.median() < 0.01, (i, rel.max(), rel.median())
        x = torch.cat(stream)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("kinds", [("fp4", "fp4"), ("fp4", None), (None, "fp4"), ("int8", "fp4"), ("fp4", "int8")])
def test_generation_in_4_bits(tiny_model_dirs, dtype, kinds):
    """Alone or in a batch, launched or replayed: the same tokens.  (A product's row depends on the row alone, and a row's attention
    on its own sequence.)"""
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 300, (n,), generator=g).tolist() for n in (3, 70, 200, 33, 129)]
    sp = SamplingParams(max_new_tokens=12, ignore_eos=True)

    def engine(**kw):
        return Engine(EngineConfig(model_path=str(tiny_model_dirs["d"]), dtype=dtype, weight_dtype=kinds[0], cache_dtype=kinds[1],
                                   library_products=False, kv_pool_tokens=4096, max_seq_len=512, **kw))

    with_graphs = [o.token_ids for o in engine().generate(prompts, sp)]
    launched = engine(cuda_graphs=False)
    assert [o.token_ids for o in launched.generate(prompts, sp)] == with_graphs
    assert [launched.generate([p], sp)[0].token_ids for p in prompts] == with_graphs
    ops.check_kernel_status()


def test_a_cache_in_4_bits_holds_more(tiny_model_dirs):
    kw = dict(model_path=str(tiny_model_dirs["d"]), kv_pool_tokens=1024, max_seq_len=512)
    wide, narrow = ModelRunner(EngineConfig(**kw)), ModelRunner(EngineConfig(cache_dtype="fp4", **kw))
    assert narrow.cache.bytes_per_page() * 256 == wide.cache.bytes_per_page() * 73      # 64 + 8 + 1 bytes a row for 256


def test_designs_that_do_not_run_in_4_bits():
    from deterministic_inference_b200 import preset
    for name in ("weight_dtype", "cache_dtype"):
        with pytest.raises(ValueError, match=name):
            ModelRunner(EngineConfig(model_config=preset("gamilorn_tiny"), random_seed=0, kv_pool_tokens=256, **{name: "fp4"}))
