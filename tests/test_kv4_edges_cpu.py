"""The 4-bit KV cache: what can be seen of its kernels, plans and engine wiring without a GPU."""
import re
from pathlib import Path

import mlc_llm_b200

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
    body = code[code.index("kv4_decode_kernel(const Kv4DecParams p) {"):]
    head = body[: body.index("__syncthreads()")]
    at = head.index("p.part_unit[blockIdx.x * 4] = 0;")
    # by thread 0, outside of any other condition
    opened = head[:at].rsplit("if (threadIdx.x == 0) {", 1)
    assert len(opened) == 2 and "}" not in opened[1] and "if" not in opened[1]
    assert "return" not in head[:at]
    launch = code[code.index("kern<<<"): code.index("kv4_decode_merge_kernel<T, D>, part")]
    assert re.search(r"err = cudaGetLastError\(\);\s*if \(err != cudaSuccess\) return", launch)
