"""The engine with its matrices and its cache in 8 bits: the fused norm, rotation and cache write against the kernel that
writes an unquantised cache, the model against a restatement in 64 bits with the same quantisation, and generation that does
not depend on the batch or on graph replay."""

from __future__ import annotations

import pytest
import torch

from deterministic_inference_b200 import Engine, EngineConfig, SamplingParams
from deterministic_inference_b200.engine.batch import SequenceInput
from deterministic_inference_b200.engine.runner import ModelRunner
from deterministic_inference_b200.kernels import ops
from tests import plain_qwen3 as plain
from tests.int8_util import codes_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,hq,hkv,d,rotary,norm", [(1, 16, 8, 128, 128, True), (70, 4, 2, 64, 64, True), (33, 6, 3, 48, 32, True),
                                                    (5, 2, 1, 256, 256, True), (9, 3, 3, 144, 96, False), (200, 8, 1, 128, 0, True)])
def test_norm_rotation_and_write(t, hq, hkv, d, rotary, norm, dtype):
    """Queries as the kernel with an unquantised cache gives them, and the cache the quantisation of what it stores.  (The
    same operations in the same order for heads of 128; another order of the norm's sum for others: 2^-20 of a value in 32
    bits, a step in 16, and then a code next to it.)"""
    g = torch.Generator().manual_seed(t + d)
    qkv = torch.randn(t, (hq + 2 * hkv) * d, generator=g).cuda().to(dtype)
    weights = [(1 + 0.1 * torch.randn(d, generator=g)).cuda() if norm else None for _ in range(2)]
    table = torch.randn(64, rotary, generator=g).cuda() if rotary else None
    pos = torch.randint(0, 64, (t,), generator=g).to(torch.int32).cuda()
    page = 16
    slots = torch.randperm(t + 40, generator=g)[:t].to(torch.int32).cuda()
    if t > 1:
        slots[t // 2] = -1
    pages = (t + 40) // page + 1
    kv = torch.zeros(pages, 2, hkv, page, d, dtype=dtype, device="cuda")
    cache = ops.Int8Cache.zeros(pages, hkv, page, d)
    args = (hq, hkv, d, *weights, 1e-6, table, pos)
    want = ops.qk_norm_rope_cache(qkv, *args, kv, slots, page)
    got = ops.qk_norm_rope_cache(qkv, *args, cache, slots, page)
    codes, scales = codes_of(kv)
    written = torch.zeros(pages * page, dtype=torch.bool, device="cuda")
    written[slots[slots >= 0].long()] = True
    written = written.view(pages, 1, 1, page).expand_as(cache.scales)
    assert not cache.data[~written].any() and not cache.scales[~written].any()
    off = (got.double() - want.double()).abs()
    step = 2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -20
    assert (off <= step * want.double().abs() + 1e-6).all()
    diff = (cache.data[written].int() - codes[written].int()).abs()
    assert diff.max() <= 1 and diff.double().mean() < 0.02
    assert torch.allclose(cache.scales[written], scales[written], rtol=step, atol=0)
    if d == 128:
        assert torch.equal(got, want) and diff.max() == 0


def _quantised(x):
    codes, scales = codes_of(x)
    return codes.double() * scales.double()[..., None]


def _plain_layer(cfg, w, i, x):
    """Layer i on the residual stream x of a whole sequence in 64 bits: what it adds to the stream, its weights, the products'
    inputs, keys and values quantised by rows."""
    d, eps, n = cfg["head_dim"], cfg["rms_norm_eps"], x.shape[0]
    product = lambda x, m: _quantised(x) @ _quantised(m).T
    angles = plain.rope_angles(torch.arange(n), d, cfg["rope_theta"])
    p = f"model.layers.{i}."
    h = plain.rms_norm(x, w[p + "input_layernorm.weight"], eps)
    q, k, v = (product(h, w[p + f"self_attn.{name}_proj.weight"]).view(n, -1, d) for name in "qkv")
    q = plain.apply_rope(plain.rms_norm(q, w[p + "self_attn.q_norm.weight"], eps), angles)
    k = plain.apply_rope(plain.rms_norm(k, w[p + "self_attn.k_norm.weight"], eps), angles)
    o = plain.attention(q, _quantised(k), _quantised(v), d ** -0.5, plain.layer_window(cfg, i))
    o = product(o.reshape(n, -1), w[p + "self_attn.o_proj.weight"])
    h = plain.rms_norm(x + o, w[p + "post_attention_layernorm.weight"], eps)
    gate, up = product(h, w[p + "mlp.gate_proj.weight"]), product(h, w[p + "mlp.up_proj.weight"])
    return o + product(gate * torch.sigmoid(gate) * up, w[p + "mlp.down_proj.weight"])


@pytest.mark.parametrize("name,page", [("a", 16), ("d", 16), ("e", 32)])
def test_layers_in_8_bits(tiny_model_dirs, name, page):
    """A prompt in one step, its tail in small ones; every layer on the stream that the engine gave it.  A value next to the
    edge between two codes may fall to either side, a step of 1 / 254 of its row's largest, and moves others behind it in the
    layer: 4 % of the norm of what the layer adds allowed, and far less as a rule.  (Through several layers such steps add
    up to as much as the quantisation itself, so the layers are looked at one by one.)"""
    cfg, w = plain.read_model_dir(tiny_model_dirs[name], torch.float64)
    ids = torch.randint(0, cfg["vocab_size"], (150,), generator=torch.Generator().manual_seed(4)).tolist()
    runner = ModelRunner(EngineConfig(model_path=str(tiny_model_dirs[name]), dtype="float32", weight_dtype="int8",
                                      cache_dtype="int8", kv_pool_tokens=1024, page_size=page, debug_checks=True,
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
        assert rel.max() < 0.04, (i, rel.max())
        x = torch.cat(stream)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_generation_in_8_bits(tiny_model_dirs, dtype):
    """Alone or in a batch, launched or replayed: the same tokens.  (Every product's sum is exact, and a row's attention
    depends on its own sequence.)"""
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 300, (n,), generator=g).tolist() for n in (3, 70, 200, 33, 129)]
    sp = SamplingParams(max_new_tokens=12, ignore_eos=True)

    def engine(**kw):
        return Engine(EngineConfig(model_path=str(tiny_model_dirs["d"]), dtype=dtype, weight_dtype="int8", cache_dtype="int8",
                                   kv_pool_tokens=4096, max_seq_len=512, **kw))

    with_graphs = [o.token_ids for o in engine().generate(prompts, sp)]
    launched = engine(cuda_graphs=False)
    assert [o.token_ids for o in launched.generate(prompts, sp)] == with_graphs
    assert [launched.generate([p], sp)[0].token_ids for p in prompts] == with_graphs


def test_a_cache_in_8_bits_holds_more(tiny_model_dirs):
    kw = dict(model_path=str(tiny_model_dirs["d"]), kv_pool_tokens=1024, max_seq_len=512)
    wide, narrow = ModelRunner(EngineConfig(**kw)), ModelRunner(EngineConfig(cache_dtype="int8", **kw))
    assert narrow.cache.bytes_per_page() * 256 == wide.cache.bytes_per_page() * 132      # 128 + 4 bytes a row for 256


def test_designs_that_do_not_run_in_8_bits():
    from deterministic_inference_b200 import preset
    for name in ("weight_dtype", "cache_dtype"):
        with pytest.raises(ValueError, match=name):
            ModelRunner(EngineConfig(model_config=preset("gamilorn_tiny"), random_seed=0, kv_pool_tokens=256, **{name: "int8"}))
