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


@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (8, 2, 64), (4, 2, 96), (8, 4, 256), (32, 1, 128), (4, 2, 32)])
def test_one_token_of_a_row_of_any_width(hq, hkv, d):
    """A single token's row has no next row: the width of the buffer it lies in does not matter."""
    st = Step(torch.float16, [77], [1], hq, hkv, d)
    for extra in (1, 4, 8):
        wide = torch.zeros(1, hq * d + extra, dtype=torch.float16, device=DEV)
        q = wide[:, : hq * d]
        q.copy_(st.q)
        assert q.stride(0) == hq * d + extra
        for plan in (True, False):
            out, lse = _attend(st, plan, q)
            ops.check_status(out.device)
            st.check(out, lse)


# ------------------------------------------------------------------------------------------------- append
@pytest.mark.parametrize("t,hkv,d,rot", [(300, 90, 256, 256), (300, 185, 128, 128), (300, 92, 256, 64), (4, 190, 256, 256),
                                         (300, 94, 256, 256), (300, 500, 64, 64)])
def test_append_of_many_heads(t, hkv, d, rot):
    """Heads beyond what the shared memory of a block holds, at enough tokens that a block takes all heads of its token."""
    g = torch.Generator().manual_seed(hkv)
    x = _kv(g, t, hkv, d, torch.float16).contiguous()
    pos = torch.randint(0, 4096, (t,), generator=g).to(torch.int32)
    slot, inv = torch.arange(t, dtype=torch.int32), base.ref.rope_inv_freq(rot, 10000.0)
    pages = (t + 15) // 16
    cache, want_cache = (ops.kv4_cache(pages, hkv, d, 16, torch.float16, dev) for dev in (DEV, "cpu"))
    mine, want = x.to(DEV), x.clone()
    ops.rope_append(mine, cache, pos.to(DEV), slot.to(DEV), inv.to(DEV), 0, hkv, d, rot, 16)
    ops.rope_append(want, want_cache, pos, slot, inv, 0, hkv, d, rot, 16)
    ops.check_status(cache.device)
    assert _same_bytes(mine, want) and _same_bytes(cache, want_cache)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,rot", [(128, 128), (64, 64), (256, 256), (128, 64), (192, 192)])
def test_append_scales_angles_in_64_bits(dtype, d, rot):
    """The factor on sines and cosines (YaRN: 0.1 ln s + 1) keeps its 64 bits: rounded to 32 it moves keys across borders."""
    t, hkv = 2000, 4
    g = torch.Generator().manual_seed(d + rot)
    x = _kv(g, t, hkv, d, dtype).contiguous()
    pos = torch.randint(0, 131072, (t,), generator=g).to(torch.int32)
    slot, inv = torch.arange(t, dtype=torch.int32), base.ref.rope_inv_freq(rot, 500000.0)
    factor = 0.1 * math.log(40.0) + 1.0
    cache, want_cache = (ops.kv4_cache(t // 16, hkv, d, 16, dtype, dev) for dev in (DEV, "cpu"))
    mine, want = x.to(DEV), x.clone()
    ops.rope_append(mine, cache, pos.to(DEV), slot.to(DEV), inv.to(DEV), 0, hkv, d, rot, 16, factor)
    ops.rope_append(want, want_cache, pos, slot, inv, 0, hkv, d, rot, 16, factor)
    ops.check_status(cache.device)
    assert _same_bytes(mine, want) and _same_bytes(cache, want_cache)


@pytest.mark.parametrize("d,page,pages", [(32, 1, 3), (32, 3, 1), (96, 1, 1), (160, 1, 3)])
def test_layers_of_small_pages(d, page, pages):
    """Layers that do not begin on 16 bytes: rows are whole 32-bit words, which is all that the kernels ask of them."""
    dtype, hq, hkv, n = torch.float16, 2, 1, pages * page
    cache = ops.kv4_cache(pages, hkv, d, page, dtype, DEV, layers=3)
    want = ops.kv4_cache(pages, hkv, d, page, dtype, "cpu", layers=3)
    assert any(c.data_ptr() % 16 for c in cache)
    g = torch.Generator().manual_seed(d)
    at = torch.arange(n, dtype=torch.int32)
    indptr, indices = torch.tensor([0, pages], dtype=torch.int32), torch.arange(pages, dtype=torch.int32)
    one, length = torch.zeros(1, dtype=torch.int32), torch.tensor([n], dtype=torch.int32)
    for li in range(3):
        x = _kv(g, n, hkv, d, dtype)
        q = torch.randn(1, hq * d, generator=g).to(dtype)
        res = []
        for c, dev in ((cache[li], DEV), (want[li], "cpu")):
            ops.rope_append(x.to(dev), c, at.to(dev), at.to(dev), None, 0, hkv, d, 0, page)
            k, _ = ops.kv4_read(c, at.to(dev), d)
            res.append((k.cpu(), ops.paged_attention(q.to(dev), c, one.to(dev), length.to(dev), indptr.to(dev),
                                                     indices.to(dev), hq, hkv, d, page, d ** -0.5).cpu()))
        # lo + s c rounded once against twice, in fp16; the weighted mean of at most three values rounded once more
        assert bool(((res[0][0].double() - res[1][0].double()).abs() <= 2.0 ** -10 * res[1][0].double().abs() + 1e-6).all())
        assert bool(((res[0][1].double() - res[1][1].double()).abs() <= 2.0 ** -8 * res[1][1].double().abs().max()).all())
    ops.check_status(cache.device)
    assert _same_bytes(cache, want)


@pytest.mark.parametrize("d", [64, 128])
def test_a_cache_that_begins_on_any_word(d):
    """A cache that is a part of a larger buffer, 4 bytes behind a 16-byte boundary."""
    st = Step(torch.float16, [300, 40, 33], [1, 30, 33], 8, 2, d, seed=2)
    flat = torch.zeros(st.cache.numel() + 8, dtype=torch.float16, device=DEV)
    moved = flat[2: 2 + st.cache.numel()].view(st.cache.shape)
    moved.copy_(st.cache)
    assert moved.is_contiguous() and moved.data_ptr() % 16 == 4
    k, v = ops.kv4_read(st.cache, (st.indices[:3] * 16).contiguous(), d)
    mk, mv = ops.kv4_read(moved, (st.indices[:3] * 16).contiguous(), d)
    assert torch.equal(k, mk) and torch.equal(v, mv)
    st.cache = moved
    out, lse = st.run()
    ops.check_status(out.device)
    st.check(out, lse)


def test_bf16_numbers_below_the_normal_ones_count_as_zero():
    row = torch.tensor([2.0 ** -130, -2.0 ** -128, 2.0 ** -133, 0.0] * 8 + [2.0 ** -100, 2.0 ** -130, 0.0, -2.0 ** -101] * 8
                       + [2.0 ** -126] * 32 + [1.0] * 32).to(torch.bfloat16).view(1, 128).repeat(1, 2)
    cache = ops.kv4_cache(1, 1, 128, 16, torch.bfloat16, DEV)
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.rope_append(row.to(DEV), cache, zero, zero, None, 0, 1, 128, 0, 16)
    k, v = ops.kv4_read(cache, zero, 128)
    ops.check_status(cache.device)
    assert torch.equal(k, v)
    k = k.view(4, 32).cpu().double()
    # the group's whole range is below the smallest normal number; in the second, half a step of 1.5 * 2^-100 / 15 each way
    assert bool((k[0].abs() < 2.0 ** -126).all())
    assert bool(((k[1] - row[0, 32:64].double()).abs() <= 2.0 ** -100 * 1.5 / 15 * (0.5 + 15 * 2.0 ** -9)).all())
    assert bool((k[2] == 2.0 ** -126).all()) and bool((k[3] == 1).all())


# ------------------------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lens,new", [([0], [1]), ([1], [1]), ([33], [1]), ([100], [3]), ([3000, 40, 5000] * 30, [1] * 90),
                                      ([1, 2, 500], [1, 2, 4]), ([40], [40]), ([129], [129]), ([3000], [40]), ([900, 260], [300, 129])])
def test_waiting_for_copies_in_flight_takes_no_time(lens, new, d):
    """Before a CTA ends it waits for its last copies and products. They are over then: a wait on a wrong phase would
    take its limit, some 50 ms each."""
    st = Step(torch.float16, [max(n, 1) for n in lens], new, 8, 2, d, kvlen=[0] if lens == [0] else None)
    st.run()
    torch.cuda.synchronize()
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    out, lse = st.run()
    b.record()
    torch.cuda.synchronize()
    assert a.elapsed_time(b) < 20.0
    ops.check_status(out.device)
    st.check(out, lse)


@pytest.mark.parametrize("dtype", TYPES)
def test_more_decode_items_than_one_launch_takes(dtype):
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(1, 41, (1100,), generator=g).tolist()
    lens[5], lens[1060] = 900, 5000      # one unit cut between CTAs in either batch of items
    st = Step(dtype, lens, [1] * 1100, 8, 2, 64, seed=9)
    assert st.plan.num_dec == 1100
    out, lse = st.run()
    ops.check_status(out.device)
    st.check(out, lse)
    assert _same_bytes(out, st.run(lse=False))


@pytest.mark.parametrize("lens,new,hq,hkv,d", [([1000, 300], [1, 1], 8, 2, 128), ([1000, 300], [3, 4], 8, 2, 64),
                                               ([1000, 300], [40, 70], 8, 2, 128), ([1000, 300], [30, 50], 8, 4, 256),
                                               ([500, 300], [1, 2], 4, 2, 32)])
def test_pages_that_a_window_released(lens, new, hq, hkv, d):
    """Pages between the sinks and the window of a sequence's first query row are given back: their numbers are -1."""
    for dtype in TYPES:
        st = Step(dtype, lens, new, hq, hkv, d, window=70, sink=4, seed=d)
        kept = [st.run(plan=plan) for plan in (True, False)]
        gone = 0
        for i in range(len(lens)):
            first = int(st.kvstart[int(st.q_indptr[i])])
            for pg in range(1, first // 16):  # page 0 holds the sinks
                st.indices[int(st.indptr[i]) + pg] = -1
                gone += 1
        assert gone > 20
        for plan, want in zip((True, False), kept):
            out, lse = st.run(plan=plan)
            ops.check_status(out.device)
            st.check(out, lse)
            assert _same_bytes(out, want[0]) and _same_bytes(lse, want[1])


@pytest.mark.parametrize("lens,new,d", [([900, 33], [1, 3], 128), ([900, 90], [60, 33], 128), ([900, 90], [60, 33], 256), ([90, 9], [2, 1], 32)])
def test_sinks_beyond_every_length(lens, new, d):
    """A window with more sinks than there are positions hides nothing."""
    for sink in (2 ** 31 - 1, 2 ** 31 - 20, 1000):
        st = Step(torch.float16, lens, new, 8, 2, d, seed=3, window=20, sink=sink)
        out, lse = st.run()
        ops.check_status(out.device)
        st.check(out, lse)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,new,d,extra", [([200, 33], [1, 3], 128, {}), ([200, 90], [60, 33], 128, {}),
                                              ([200, 90], [60, 33], 256, {"cap": 30.0}), ([200, 33], [1, 3], 64, {"cap": 30.0})])
def test_negative_scale(dtype, lens, new, d, extra):
    st = Step(dtype, lens, new, 8, 2, d, seed=4, **extra)
    flipped = torch.empty_like(st.qkv).copy_(st.qkv).neg_()[:, : 8 * d]
    for plan in (True, False):
        out, lse = _attend(st, plan, flipped, -(d ** -0.5))
        ops.check_status(out.device)
        st.check(out, lse)


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


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,new,d", [([200, 33], [1, 3], 128), ([200, 90], [60, 33], 128), ([200, 90], [60, 33], 256),
                                        ([200, 33], [1, 3], 64), ([50, 20], [4, 1], 32)])
def test_queries_that_are_not_finite(dtype, lens, new, d):
    st = Step(dtype, lens, new, 8, 2, d, seed=7)
    clean = st.run()
    st.check(*clean)
    bad = sum(new) - 2
    others = [t for t in range(sum(new)) if t != bad]
    for value in (math.nan, math.inf, -math.inf):
        q = st.qkv.clone()
        q[bad, 3: 8 * d: d] = value  # one channel of every head
        for plan in (True, False):
            out, lse = st.run(plan=plan, q=q[:, : 8 * d])
            ops.check_status(out.device)
            _check_rows(st, out, lse, others)
            if value != value:
                assert bool(torch.isnan(out[bad]).all()) and bool(torch.isnan(lse[bad]).all())


@pytest.mark.parametrize("by", [2.0 ** 30, math.inf])
@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("lens,new,at,extra", [
    ([200, 50], [4, 3], 199, {}), ([200, 50], [4, 4], 249, {}), ([120, 70], [4, 4], 119, {"tree": True}),
    ([100], [4], 81, {"window": 16}), ([2000], [2], 1999, {}), ([4], [4], 2, {}),
    ([300], [300], 150, {}), ([700, 90], [200, 40], 600, {}), ([3000], [40], 2985, {}), ([400], [60], 380, {"tree": True}),
    ([300], [300], 100, {"window": 64}), ([300], [300], 3, {"window": 64, "sink": 2}), ([500], [130], 499, {"cap": 30.0})])
def test_a_huge_value_that_a_row_does_not_see(lens, new, at, extra, d, what, by, monkeypatch):
    """bf16: what later tokens, other branches of a draft tree or tokens below a row's window hold does not touch that row,
    however large it is (infinity is cached as 2^126)."""
    plain = base._kv

    def planted(g, n, hkv, d, dtype):
        rows = plain(g, n, hkv, d, dtype)
        col = hkv * d if what == "v" else 0
        rows[at, col + 5: col + hkv * d: 32] = by
        return rows

    monkeypatch.setattr(base, "_kv", planted)
    st = Step(torch.bfloat16, lens, new, 8, 2, d, seed=d + len(lens), **extra)
    # which sequence and position the planted row is
    seq, pos = (0, at) if at < lens[0] else (1, at - lens[0])
    blind = []
    for t in range(sum(new)):
        n, start = int(st.kvlen[t]), int(st.kvstart[t]) if st.kvstart is not None else 0
        sees = st.seq[t] == seq and (start <= pos < n or (pos < min(n, st.sink) and st.kvstart is not None))
        if st.tree is not None and st.seq[t] == seq and 0 <= pos - n < 63:
            sees = bool((int(st.tree[t]) >> (pos - n)) & 1)
        if not sees:
            blind.append(t)
    assert 0 < len(blind) < sum(new)
    out, lse = st.run()
    ops.check_status(out.device)
    _check_rows(st, out, lse, blind)
    assert what == "k" or bool(torch.isfinite(out).all())
    assert _same_bytes(out, st.run(lse=False))
