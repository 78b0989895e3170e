"""The engine with a 4-bit KV cache on CPU: generation, prefix sharing, speculative commits, capacity, refusals."""
import json

import pytest
import torch

from mlc_llm_b200 import _core, ops
from mlc_llm_b200.serve.config import EngineConfig
from mlc_llm_b200.serve.sync_engine import SyncMLCEngine

MODEL = "random://tiny-llama?quant=q0f32&seed=11"
GREEDY = {"temperature": 0.0, "debug_config": {"ignore_eos": True}}


def _engine(model=MODEL, **over):
    kw = dict(mode="server", max_num_sequence=4, max_total_sequence_length=1024, prefill_chunk_size=64,
              kv_cache_dtype="int4")
    kw.update(over)
    return SyncMLCEngine(model, "cpu", engine_config=EngineConfig(**kw))


def _run(eng, prompts, n=12):
    _, toks = eng.generate([list(p) for p in prompts], dict(GREEDY, max_tokens=n))
    return [t[0] for t in toks]


PROMPTS = [[5, 9, 100, 7], list(range(10, 90)), [3] * 17]


def test_generation_is_attention_over_the_quantised_values(monkeypatch):
    eng = _engine()
    model = eng.runtime.models[0]
    assert model.kv4 and model.kv_pages.shape[-1] == ops.kv4_row(model.d, model.kv_dtype)
    toks = _run(eng, PROMPTS)
    assert [len(t) for t in toks] == [12, 12, 12]
    assert _run(eng, PROMPTS) == toks                                        # shared prefixes
    assert _run(_engine(prefill_chunk_size=16, max_num_sequence=1), PROMPTS) == toks
    # a full cache that is handed the values the packed rows stand for generates the same tokens
    append = ops.rope_append

    def through(qkv, kv_pages, pos, slot, inv_freq, hq, hkv, d, rot_dim, page, attn_factor=1.0):
        t = qkv.shape[0]
        packed, at = ops.kv4_cache(t // page + 1, hkv, d, page, qkv.dtype, "cpu"), torch.arange(t, dtype=torch.int32)
        append(qkv, packed, pos, at, inv_freq, hq, hkv, d, rot_dim, page, attn_factor)
        k, v = ops.kv4_read(packed, at, d)
        live = slot >= 0
        sl = slot[live].long()
        kv_pages[sl // page, 0, :, sl % page], kv_pages[sl // page, 1, :, sl % page] = k[live], v[live]

    monkeypatch.setattr(ops, "rope_append", through)
    full = _engine(kv_cache_dtype="auto")
    assert not full.runtime.models[0].kv4
    assert _run(full, PROMPTS) == toks


def test_speculative_commit_moves_packed_rows():
    plain = _run(_engine(), PROMPTS)
    spec = _engine(speculative_mode="small_draft", spec_draft_length=3,
                   additional_models=["random://tiny-llama?quant=q0f32&seed=12&num_hidden_layers=1"])
    assert _run(spec, PROMPTS) == plain
    tree = _engine(speculative_mode="small_draft", spec_draft_length=3, spec_tree_width=2, additional_models=[MODEL])
    assert _run(tree, PROMPTS) == plain


def test_capacity_counts_packed_rows():
    info = {"params_bytes": 0, "num_layers": 32, "num_qo_heads": 32, "num_kv_heads": 8, "head_dim": 128,
            "vocab_size": 32000, "context_window_size": 1 << 20, "prefill_chunk_size": 2048, "max_batch_size": 64,
            "kv_bytes_per_element": 2}
    cfg = json.dumps({"mode": "server"})
    full = _core.infer_capacity(cfg, [info], 64 << 30)
    packed = _core.infer_capacity(json.dumps({"mode": "server", "kv_cache_dtype": "int4"}), [dict(info, kv_row_bytes=80)], 64 << 30)
    assert abs(full["kv_bytes_per_token"] - (32 * 8 * 2 * 256 + 1.25)) < 1
    assert abs(packed["kv_bytes_per_token"] - (32 * 8 * 2 * 80 + 1.25)) < 1
    assert packed["num_pages"] > 3.1 * full["num_pages"]
    assert json.loads(packed["config_json"])["kv_cache_dtype"] == "int4"
    with pytest.raises(Exception, match="kv_cache_dtype"):
        _core.infer_capacity(json.dumps({"kv_cache_dtype": "fp3"}), [info], 64 << 30)


def test_models_whose_rows_cannot_be_packed_are_refused():
    from mlc_llm_b200.models import presets

    names = [n for n, c in presets.MODEL_PRESETS.items() if c.get("model_type") in ("deepseek_v2", "rwkv5") and "tiny" in n]
    assert len(names) >= 2
    for name in names:
        with pytest.raises(ValueError):
            _engine(f"random://{name}?seed=1&quant=q0f32")
    with pytest.raises(ValueError):
        _engine(kv_cache_dtype="int3")


def test_hybrid_model_packs_its_attention_layers():
    eng = _engine("random://tiny-qwen35?quant=q0f32&seed=3")
    assert eng.runtime.models[0].kv4
    toks = _run(eng, PROMPTS)
    assert [len(t) for t in toks] == [12, 12, 12]
