"""The 4-bit KV cache on CPU: the format against a scalar restatement, the operators' CPU path, their refusals."""
import math
import struct

import numpy as np
import pytest
import torch

from mlc_llm_b200 import ops
from mlc_llm_b200.ops import reference as ref

TYPES = [torch.float16, torch.bfloat16, torch.float32]


def _round_to(x: float, dtype) -> float:
    return float(torch.tensor(x, dtype=torch.float32).to(dtype))


def _scalar_row(row, dtype):
    """The format, value by value: (codes, lo per group, s per group, values)."""
    bound = {torch.float16: 65440.0}.get(dtype, 2.0 ** 126)
    codes, los, steps, values = [], [], [], []
    for a in range(0, len(row), 32):
        part = [0.0 if math.isnan(x) else min(max(x, -bound), bound) for x in row[a:a + 32]]
        lo, hi = min(part), max(part)
        s = _round_to(float(np.float32(np.float32(hi) - np.float32(lo)) * np.float32(1.0 / 15.0)), dtype)
        for x in part:
            c = 0 if s == 0 else int(np.clip(np.rint(np.float32(np.float32(x) - np.float32(lo)) / np.float32(s)), 0, 15))
            codes.append(c)
            values.append(lo + s * c)
        los.append(lo)
        steps.append(s)
    return codes, los, steps, values


def _bytes_of(packed):
    return packed.contiguous().view(torch.uint8).numpy().tobytes()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [32, 64, 96, 128, 256])
def test_packed_row_layout(dtype, d):
    g = torch.Generator().manual_seed(d)
    x = (torch.randn(5, d, generator=g) * torch.tensor([1.0, 1e-3, 30.0, 0.0, 2.0]).view(5, 1)).to(dtype)
    x[4, 3] = 40.0  # an outlier channel
    packed = ref.kv4_pack(x)
    assert packed.shape == (5, ops.kv4_row(d, dtype)) and packed.dtype == dtype
    back = ref.kv4_unpack(packed, d)
    for i in range(5):
        codes, los, steps, values = _scalar_row(x[i].float().tolist(), dtype)
        raw = _bytes_of(packed[i])
        for ch in range(d):
            (word,) = struct.unpack_from("<I", raw, ch // 8 * 4)
            j = ch % 8
            assert (word >> ((j & 1) * 16 + (j >> 1) * 4)) & 15 == codes[ch]
        meta = packed[i, d // 2 // dtype.itemsize:].float().view(-1, 2)
        assert meta[:, 0].tolist() == los and meta[:, 1].tolist() == steps
        # lo + s c in fp32 against 64 bits: one product and one sum, each off by half a step of 2^-23 at most
        want = torch.tensor(values, dtype=torch.float64)
        room = 2.0 ** -23 * (want.abs() + torch.tensor([abs(v) for v in los], dtype=torch.float64).repeat_interleave(32))
        assert bool(((back[i].double() - want).abs() <= room).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_quantisation_error_is_half_a_step(dtype):
    x = torch.randn(200, 128, generator=torch.Generator().manual_seed(1)).to(dtype)
    packed = ref.kv4_pack(x)
    back = ref.kv4_unpack(packed, 128)
    s = packed[:, 64 // dtype.itemsize:].float().view(200, 4, 2)[..., 1].repeat_interleave(32, dim=1)
    # half a step, plus what rounding the step to T moves the upper end: 15 s eps / 2
    assert bool(((back - x.float()).abs() <= s * (0.5 + 15 * torch.finfo(dtype).eps / 2) + 1e-6).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_not_finite_and_huge_values_stay_finite(dtype):
    big = torch.finfo(dtype).max
    x = torch.tensor([math.nan, math.inf, -math.inf, big, -big, 0.0, 1.0, -1.0] * 8).to(dtype).view(1, 64)
    back = ref.kv4_unpack(ref.kv4_pack(x), 64).to(dtype)
    assert bool(torch.isfinite(back).all())
    assert back[0, 1] > 0.99 * min(big, ref.KV4_BOUND[dtype]) and back[0, 2] == -ref.KV4_BOUND[dtype]
    same = torch.full((1, 32), 3.0).to(dtype)
    assert torch.equal(ref.kv4_unpack(ref.kv4_pack(same), 32).to(dtype), same)   # s = 0: the value itself
    assert bool((ref.kv4_unpack(torch.zeros(1, ops.kv4_row(32, dtype), dtype=dtype), 32) == 0).all())


def _step(dtype, lens, new, hq, hkv, d, page=16, seed=0):
    """A cache filled by appending, and the arrays of one step over it."""
    g = torch.Generator().manual_seed(seed)
    held = [(n + page - 1) // page for n in lens]
    pages = sum(held) + 2
    perm = torch.randperm(pages, generator=g)[: sum(held)].to(torch.int32)
    indptr = np.concatenate([[0], np.cumsum(held)]).astype(np.int32)
    cache = ops.kv4_cache(pages, hkv, d, page, dtype, "cpu")
    rows, slots = [], []
    for i, n in enumerate(lens):
        for j in range(n):
            slots.append(int(perm[indptr[i] + j // page]) * page + j % page)
    kv = torch.randn(len(slots), 2 * hkv * d, generator=g).to(dtype)
    pos = torch.zeros(len(slots), dtype=torch.int32)
    ops.rope_append(kv.clone(), cache, pos, torch.tensor(slots, dtype=torch.int32), None, 0, hkv, d, 0, page)
    t = sum(new)
    q = torch.randn(t, hq * d, generator=g).to(dtype)
    q_seq = torch.from_numpy(np.repeat(np.arange(len(new)), new).astype(np.int32))
    kvlen = torch.cat([torch.arange(n - m + 1, n + 1) for n, m in zip(lens, new)]).to(torch.int32)
    return cache, kv, torch.tensor(slots, dtype=torch.int32), q, q_seq, kvlen, torch.from_numpy(indptr), perm


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [16, 4])
def test_cpu_append_read_attend(dtype, page):
    hq, hkv, d = 6, 2, 64
    lens, new = [1, 17, 40], [1, 3, 2]
    cache, kv, slots, q, q_seq, kvlen, indptr, perm = _step(dtype, lens, new, hq, hkv, d, page)
    k, v = ops.kv4_read(cache, slots, d)
    want = ref.kv4_unpack(ref.kv4_pack(kv.view(-1, 2, hkv, d)), d).to(dtype)
    assert torch.equal(k, want[:, 0]) and torch.equal(v, want[:, 1])
    # attention over the packed cache is attention over the values it stands for, in a 32-bit cache
    plain = ref.kv4_unpack(cache, d)
    got, lse = ops.paged_attention(q, cache, q_seq, kvlen, indptr, perm, hq, hkv, d, page, d ** -0.5, return_lse=True)
    base, blse = ref.paged_attention(q.view(-1, hq, d), plain, q_seq, kvlen, indptr, perm, hq, hkv, d, page, d ** -0.5,
                                     return_lse=True)
    assert torch.equal(got, base.reshape(-1, hq * d)) and torch.equal(lse, blse)


def test_cpu_append_rotates_in_64_bits_and_skips_negative_slots():
    hq, hkv, d, rot = 2, 1, 64, 32
    cache = ops.kv4_cache(3, hkv, d, 16, torch.float32, "cpu")
    before = cache.clone()
    inv = ref.rope_inv_freq(rot, 500000.0)
    x = torch.randn(2, (hq + 2) * d, generator=torch.Generator().manual_seed(3))
    row = x.clone()
    pos = torch.tensor([131071, 5], dtype=torch.int32)
    ops.rope_append(row, cache, pos, torch.tensor([-1, -1], dtype=torch.int32), inv, hq, hkv, d, rot, 16)
    assert torch.equal(cache.view(torch.int32), before.view(torch.int32))
    for t in range(2):
        for h in range(hq + hkv):
            for j in range(rot // 2):
                a = float(pos[t]) * float(inv[j])
                u, w = float(x[t, h * d + j]), float(x[t, h * d + j + rot // 2])
                assert row[t, h * d + j].item() == np.float32(u * math.cos(a) - w * math.sin(a))
                assert row[t, h * d + j + rot // 2].item() == np.float32(w * math.cos(a) + u * math.sin(a))
    assert torch.equal(row[:, 3 * d:], x[:, 3 * d:])


def test_refusals():
    cache = ops.kv4_cache(4, 2, 64, 16, torch.float16, "cpu")
    qkv = torch.zeros(3, (4 + 4) * 64, dtype=torch.float16)
    pos, slot = torch.zeros(3, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    inv = torch.ones(32)

    def append(qkv=qkv, cache=cache, pos=pos, slot=slot, inv=inv, hq=4, hkv=2, d=64, rot=64, page=16):
        ops.rope_append(qkv, cache, pos, slot, inv, hq, hkv, d, rot, page)

    append()
    for bad in (dict(qkv=qkv.bfloat16()), dict(qkv=qkv[:, :-64]), dict(qkv=qkv.t().contiguous().t()), dict(hkv=1),
                dict(page=8), dict(slot=slot.long()), dict(slot=slot[:2]), dict(pos=pos.long()), dict(inv=inv.double()),
                dict(inv=inv[:8]), dict(rot=33), dict(rot=128), dict(cache=cache[:, :, :, ::2]),
                dict(cache=cache.unsqueeze(0))):
        with pytest.raises(ValueError):
            append(**bad)
    for bad in ((cache, slot.long(), 64), (cache, slot, 128), (cache.float(), slot, 64), (cache, slot.view(1, 3), 64)):
        with pytest.raises(ValueError):
            ops.kv4_read(*bad)
    q = torch.zeros(3, 4 * 64, dtype=torch.float16)
    one = torch.ones(3, dtype=torch.int32)
    indptr, indices = torch.tensor([0, 1], dtype=torch.int32), torch.zeros(1, dtype=torch.int32)

    def attend(q=q, cache=cache, q_seq=slot, kvlen=one, indptr=indptr, indices=indices, hq=4, hkv=2, page=16, **kw):
        return ops.paged_attention(q, cache, q_seq, kvlen, indptr, indices, hq, hkv, 64, page, 0.125, **kw)

    assert attend().shape == (3, 256)
    for bad in (dict(q=q.bfloat16()), dict(q=q[:, ::2]), dict(q=q[:, :192]), dict(hq=3, q=q[:, :192]), dict(hkv=4),
                dict(page=8), dict(kvlen=one.long()), dict(q_seq=slot[:2]), dict(indices=indices.long()),
                dict(q_kvstart=one.float()), dict(tree_mask=one)):
        with pytest.raises(ValueError):
            attend(**bad)
    with pytest.raises(ValueError):
        ops.kv4_cache(4, 2, 80, 16, torch.float16, "cpu")
    with pytest.raises(ValueError):
        ops.kv4_cache(4, 2, 64, 16, torch.int8, "cpu")


def test_a_plan_serves_only_the_step_and_cache_it_was_made_for():
    d, hq, hkv = 64, 8, 2
    cache = ops.kv4_cache(40, hkv, d, 16, torch.float16, "cpu")
    q = torch.zeros(30, hq * d, dtype=torch.float16)
    seq, kvlen = torch.zeros(30, dtype=torch.int32), torch.arange(1, 31, dtype=torch.int32)
    indptr, indices = torch.tensor([0, 2], dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32)
    plan = ops.kv4_plan([0, 30], kvlen, indptr, indices, hq, hkv, 30)
    call = lambda x, kv, heads, p: ops.paged_attention(x, kv, seq, kvlen, indptr, indices, heads, hkv, d, 16, 0.125, plan=p)
    assert call(q, cache, hq, plan).shape == q.shape
    with pytest.raises(ValueError, match="the plan is for 30 tokens"):
        call(q[:29], cache, hq, plan)
    with pytest.raises(ValueError, match="4 query heads per KV head"):
        call(q[:, : 4 * d].contiguous(), cache, 4, plan)
    with pytest.raises(ValueError, match="for a 4-bit cache"):  # tiles of 256 rows
        call(q, torch.zeros(40, 2, hkv, 16, d, dtype=torch.float16), hq, plan)


def test_tiles_in_rising_order_of_the_positions_they_visit():
    from mlc_llm_b200.ops.attention import build_tiles

    q_indptr = np.array([0, 300, 301, 420])                       # 4 heads per KV head: tiles of 64 tokens, one decode item
    kvlen = np.concatenate([np.arange(2001, 2301), [900], np.arange(1, 120)])
    plain = build_tiles(q_indptr, 4, tile_rows=256)
    tiles = build_tiles(q_indptr, 4, tile_rows=256, q_kvlen=kvlen)
    as_set = lambda t: {tuple(map(int, x)) for x in zip(t["tile_seq"], t["tile_qstart"], t["tile_ntok"])}
    assert as_set(tiles) == as_set(plain) and len(tiles["tile_seq"]) == 7
    reach = kvlen[tiles["tile_qstart"] + tiles["tile_ntok"] - 1]
    assert (np.diff(reach) >= 0).all() and reach[-1] == 2300 and reach[0] == 64
    assert all(np.array_equal(tiles[k], plain[k]) for k in ("dec_seq", "dec_qstart", "dec_ntok"))


def test_plan_refusals():
    lens, indptr, indices = torch.ones(4, dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="do not divide"):
        ops.kv4_plan([0, 4], lens, indptr, indices, 6, 4, 4)
    for bad in ([1, 4], [0, 3, 2], [[0, 4]], []):
        with pytest.raises(ValueError, match="rise from 0"):
            ops.kv4_plan(bad, lens, indptr, indices, 8, 4, 4)
    with pytest.raises(ValueError, match="5 tokens"):
        ops.kv4_plan([0, 5], lens, indptr, indices, 8, 4, 5)
    assert ops.kv4_plan([0], lens[:0], indptr, indices, 8, 4, 0).num_tiles == 0
