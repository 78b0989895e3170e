"""The 4-bit KV cache kernels where the ordinary cases do not go: strides of a single token, many KV heads, small pages,
more decode items than one launch takes, released pages, negative scales, wide query groups, queries that are not finite,
and cached values of very different sizes that some rows of a tile do not see.

Oracle and tolerance are those of ``test_kv4_gpu`` (``Step``).
"""
import copy
import math

import numpy as np
import pytest
import torch

import test_kv4_gpu as base
from test_kv4_gpu import DEV, TYPES, Step, _kv, _same_bytes
from mlc_llm_b200 import ops

pytestmark = pytest.mark.gpu


def _attend(st, plan=True, q=None, scale=None):
    """``Step.run`` with another scale."""
    on = lambda x: None if x is None else x.to(DEV)
    return ops.paged_attention(st.q if q is None else q, st.cache, on(torch.from_numpy(st.seq.astype(np.int32))), on(st.kvlen),
                               st.indptr, st.indices, st.hq, st.hkv, st.d, st.page, st.d ** -0.5 if scale is None else scale,
                               q_kvstart=on(st.kvstart), sink=st.sink, tree_mask=on(st.tree), softcap=st.cap,
                               return_lse=True, plan=st.plan if plan else None)


def _check_rows(st, out, lse, rows):
    """``Step.check`` of some tokens only."""
    part = copy.copy(st)
    part.q, part.seq, part.kvlen = st.q[rows], st.seq[rows], st.kvlen[rows]
    part.kvstart = None if st.kvstart is None else st.kvstart[rows]
    part.tree = None if st.tree is None else st.tree[rows]
    part.check(out[rows], lse[rows])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,new,hq,hkv,d", [([100, 40], [1, 1], 32, 1, 128), ([300, 40], [5, 1], 71, 1, 64),
                                               ([90, 900], [1, 1], 20, 1, 256), ([60, 30], [2, 1], 300, 1, 64),
                                               ([200, 300, 60], [1, 4, 1], 16, 4, 256), ([200, 300], [4, 1], 16, 4, 128)])
def test_query_groups(dtype, lens, new, hq, hkv, d):
    """More than 16 heads per KV head (single tokens become prefill tiles), more than a tile holds (the generic kernel), and
    items of different row counts in one launch."""
    st = Step(dtype, lens, new, hq, hkv, d, seed=hq)
    out, lse = st.run()
    ops.check_status(out.device)
    st.check(out, lse)
