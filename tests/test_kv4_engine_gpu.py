"""The engine with a 4-bit KV cache on the GPU, against the same engine with a 16-bit cache that is handed the values
the packed rows stand for (so both attend to the same numbers, with different kernels)."""
import numpy as np
import pytest
import torch

from mlc_llm_b200 import ops
from mlc_llm_b200.ops import _lib
from mlc_llm_b200.serve.config import EngineConfig
from mlc_llm_b200.serve.sync_engine import SyncMLCEngine

pytestmark = pytest.mark.gpu


def _through(append):
    def rope_append(qkv, kv_pages, pos, slot, inv_freq, hq, hkv, d, rot_dim, page, attn_factor=1.0):
        t = qkv.shape[0]
        packed = ops.kv4_cache(t // page + 1, hkv, d, page, qkv.dtype, qkv.device)
        at = torch.arange(t, dtype=torch.int32, device=qkv.device)
        append(qkv, packed, pos, at, inv_freq, hq, hkv, d, rot_dim, page, attn_factor)
        # rotated already: write the rows' values into the full cache with the 16-bit kernel
        k, v = ops.kv4_read(packed, at, d)
        rows = torch.cat([k.reshape(t, -1), v.reshape(t, -1)], dim=1)
        append(rows, kv_pages, pos, slot, None, 0, hkv, d, 0, page)

    return rope_append


def _engine(model, dtype, **kw):
    eng = SyncMLCEngine("random://" + model, "cuda",
                        engine_config=EngineConfig(mode="server", max_num_sequence=8, prefill_chunk_size=256,
                                                   max_total_sequence_length=4096, kv_cache_dtype=dtype, **kw))
    assert eng.runtime.models[0].kv4 == (dtype == "int4")
    return eng


def _logged(eng, prompt, n):
    """Tokens of a greedy run and the logits row behind each."""
    model, rows = eng.runtime.models[0], []
    keep = type(model).logits

    def logits(hidden, index, *args, **kw):
        out = keep(model, hidden, index, *args, **kw)
        rows.append(out.reshape(-1, out.shape[-1])[-1].float().cpu())
        return out

    model.logits = logits
    _, toks = eng.generate([prompt], {"max_tokens": n, "temperature": 0.0, "debug_config": {"ignore_eos": True}})
    del model.logits
    _lib.check_status(torch.device("cuda"))
    return toks[0][0], rows


@pytest.mark.parametrize("model,tol", [
    ("tiny-llama-gpu?quant=q0f16&seed=0", 2e-2), ("tiny-llama-gpu?quant=q4f16_1&seed=0", 2e-2),
    ("tiny-llama?quant=q0bf16&seed=1", 6e-2),                    # heads of 64
    ("tiny-gemma2-gpu?quant=q0bf16&seed=2", 6e-2)])              # windows and soft-capped logits
def test_engine_matches_a_full_cache_of_the_same_values(model, tol, monkeypatch):
    """``tol``: what the suite grants the logits of these models between two execution paths (fp16, bf16). Greedy tokens
    may part only where the best two logits are closer than that."""
    rng = np.random.default_rng(2)
    prompts = [rng.integers(0, 32000, int(n)).tolist() for n in (90, 7, 33, 400)]
    eng = _engine(model, "int4")
    _logged(eng, prompts[0], 6)
    packed = [_logged(eng, p, 6) for p in prompts]
    if "gemma" not in model:
        assert eng.runtime.executor.graph_replays > 0
    del eng
    monkeypatch.setattr(ops, "rope_append", _through(ops.rope_append))
    monkeypatch.setenv("MLCB_CUDA_GRAPH", "0")
    eng = _engine(model, "auto")
    for prompt, (toks, rows) in zip(prompts, packed):
        want, base = _logged(eng, prompt, 6)
        assert len(rows) == len(base) and len(toks) == len(want) == 6
        for i, (a, b) in enumerate(zip(rows, base)):
            assert float((a - b).abs().max()) < tol
            if toks[i] != want[i]:
                best = b.topk(2).values
                assert float(best[0] - best[1]) < 2 * tol
                break


def test_engine_speculation_on_packed_rows():
    rng = np.random.default_rng(2)
    prompts = [rng.integers(0, 32000, int(n)).tolist() for n in (90, 7, 33, 400)]
    cfg = {"max_tokens": 12, "temperature": 0.0, "debug_config": {"ignore_eos": True}}
    model, outs = "tiny-llama-gpu?quant=q0f16&seed=0", []
    for kw in ({}, {"speculative_mode": "small_draft", "spec_draft_length": 3, "spec_tree_width": 2,
                    "additional_models": ["random://" + model]}):
        eng = _engine(model, "int4", **kw)
        _, toks = eng.generate(prompts, cfg)
        _lib.check_status(torch.device("cuda"))
        outs.append([t[0] for t in toks])
        del eng
    same = sum(int(a == b) for x, y in zip(*outs) for a, b in zip(x, y))
    assert [x[0] for x in outs[0]] == [y[0] for y in outs[1]] and same >= 0.7 * 48, outs


def test_packed_rows_between_engine_pools():
    """The row copy of the prefill / decode hand-off moves packed rows of any head size."""
    import ctypes

    for d, dtype in ((128, torch.float16), (64, torch.bfloat16), (96, torch.float16)):
        row = ops.kv4_row(d, dtype)
        src = torch.randint(0, 1 << 15, (2, 5, 2, 3, 16, row), dtype=torch.int16, device="cuda")
        dst = torch.zeros(2, 7, 2, 3, 16, row, dtype=torch.int16, device="cuda")
        ss = torch.tensor([3, 79, 17], dtype=torch.int32, device="cuda")
        ds = torch.tensor([100, 5, 64], dtype=torch.int32, device="cuda")
        ll, i, p = ctypes.c_longlong, ctypes.c_int, _lib.ptr
        rc = _lib.lib().mlcb_kv_slot_copy(p(src), p(dst), p(ss), p(ds), i(3), i(2), ll(src.stride(0) * 2), ll(dst.stride(0) * 2),
                                          i(3), i(16), i(row * 2), i(5), i(7), p(_lib.status_word(src.device)), _lib.stream_ptr())
        assert rc == 0
        want = torch.zeros_like(dst)
        s, t = ss.long(), ds.long()
        want[:, t // 16, :, :, t % 16] = src[:, s // 16, :, :, s % 16]
        assert torch.equal(dst, want)
