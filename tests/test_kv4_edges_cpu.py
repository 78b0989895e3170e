"""The 4-bit KV cache: what can be seen of its kernels, plans and engine wiring without a GPU."""
import dataclasses
import re
from pathlib import Path

import numpy as np
import pytest
import torch

import mlc_llm_b200
from mlc_llm_b200 import ops

KERNELS = Path(mlc_llm_b200.__file__).parent / "csrc" / "kernels"


def _code(name):
    """A kernel file without its comments."""
    text = (KERNELS / name).read_text()
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


def test_the_join_of_cut_units_never_reads_a_count_that_was_not_written():
    """The join kernel takes row counts and addresses from ``part_unit``. The producer writes a CTA's entry with the last
    piece of its share, which a wait that ran out can keep it from reaching, and the scratch is not cleared by the caller: so
    every CTA has to write 0 rows before any role starts, and the join must not run after a launch that failed."""
    code = _code("kv4_decode.cu")
    body = code[re.search(r"kv4_decode_kernel\(const [^)]*Kv4DecParams p\) {", code).end():]
    head = body[: body.index("__syncthreads()")]
    at = head.index("p.part_unit[blockIdx.x * 4] = 0;")
    # by thread 0, outside of any other condition
    opened = head[:at].rsplit("if (threadIdx.x == 0) {", 1)
    assert len(opened) == 2 and "}" not in opened[1] and "if" not in opened[1]
    assert "return" not in head[:at]
    launch = code[code.index("kern<<<"): code.index("kv4_decode_merge_kernel<T, D>, part")]
    assert re.search(r"err = cudaGetLastError\(\);\s*if \(err != cudaSuccess\) return", launch)


def test_a_plan_of_other_sequences_or_another_device_is_refused():
    """The kernels read the plan's items from its arrays and two entries of ``page_indptr`` per item."""
    hq, hkv, d = 8, 2, 64
    cache = ops.kv4_cache(8, hkv, d, 16, torch.float16, "cpu")
    lens, new = [20, 30, 5], [1, 12, 1]                # 12 tokens of 4 heads: a prefill tile; the others: decode items
    q = torch.zeros(14, hq * d, dtype=torch.float16)
    seq = torch.tensor(np.repeat([0, 1, 2], new), dtype=torch.int32)
    kvlen = torch.cat([torch.arange(n - m + 1, n + 1) for n, m in zip(lens, new)]).to(torch.int32)
    indptr, indices = torch.tensor([0, 2, 4, 5], dtype=torch.int32), torch.arange(5, dtype=torch.int32)
    plan = ops.kv4_plan([0, 1, 13, 14], kvlen, indptr, indices, hq, hkv, 30)
    assert plan.num_dec == 2 and plan.num_tiles == 1
    call = lambda p, ip: ops.paged_attention(q, cache, seq, kvlen, ip, indices, hq, hkv, d, 16, 0.125, plan=p)
    assert call(plan, indptr).shape == q.shape
    with pytest.raises(ValueError, match="page_indptr"):
        call(plan, indptr[:3])
    for name in ("dec_seq", "tile_seq"):
        other = dataclasses.replace(plan, **{name: getattr(plan, name).to("meta")})
        with pytest.raises(ValueError, match="plan's items"):
            call(other, indptr)


def test_rows_of_the_largest_decode_item(monkeypatch):
    from mlc_llm_b200.ops.attention import build_tiles, decode_rows

    rng = np.random.default_rng(1)
    for group in (1, 3, 4, 8, 16, 20):
        for _ in range(50):
            q_indptr = np.concatenate([[0], np.cumsum(rng.integers(0, 20, rng.integers(0, 6)))])
            items = build_tiles(q_indptr, group)["dec_ntok"]
            assert decode_rows(q_indptr, group) == (int(items.max()) * group if items.size else 16)
    # the kernel that a captured step holds depends on it
    monkeypatch.setattr(ops.kv4, "sm_count", lambda device: 148)
    launch = lambda rows, d=128: ops.kv4.decode_launch(8, 2, d, 100, rows, torch.device("cuda"))
    assert launch(4) == launch(8) != launch(9) == launch(16) and launch(4, 256) != launch(16, 256)
