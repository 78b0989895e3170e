"""What the engine hands to the attention kernels of the 4-bit cache."""
import inspect

import numpy as np
import pytest
import torch

from mlc_llm_b200 import ops
from mlc_llm_b200.ops import _lib
from mlc_llm_b200.serve.config import EngineConfig
from mlc_llm_b200.serve.sync_engine import SyncMLCEngine

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("model", ["tiny-llama-gpu?quant=q0f16&seed=0", "tiny-gemma2-gpu?quant=q0bf16&seed=2"])
def test_engine_plans_name_the_rows_of_their_largest_decode_item(model, monkeypatch):
    """Steps that mix prompts, single tokens and verify chunks: the kernel for 16 rows runs where an item needs it."""
    seen = []
    keep = ops.kv4._decode

    def decode(*args):
        a = inspect.signature(keep).bind(*args).arguments
        plan = a["plan"]
        seen.append((plan.dec_rows, int(a["q"].shape[0]) == plan.num_dec, plan.dec_ntok.clone(), a["hq"] // a["hkv"]))
        keep(*args)

    monkeypatch.setattr(ops.kv4, "_decode", decode)
    monkeypatch.setenv("MLCB_CUDA_GRAPH", "0")
    rng = np.random.default_rng(2)
    prompts = [rng.integers(0, 32000, int(n)).tolist() for n in (90, 7, 33, 400, 1, 2, 3)]
    for kw in ({}, {"speculative_mode": "small_draft", "spec_draft_length": 3, "additional_models": ["random://" + model]}):
        eng = SyncMLCEngine("random://" + model, "cuda",
                            engine_config=EngineConfig(mode="server", max_num_sequence=8, prefill_chunk_size=256,
                                                       max_total_sequence_length=4096, kv_cache_dtype="int4", **kw))
        eng.generate(prompts, {"max_tokens": 8, "temperature": 0.0, "debug_config": {"ignore_eos": True}})
        _lib.check_status(torch.device("cuda"))
        del eng
    mixed = 0
    for rows, single, ntok, group in seen:
        assert rows == int(ntok.max()) * group
        mixed += not single and rows <= 8
    assert mixed > 0 and any(rows > 8 for rows, *_ in seen)
