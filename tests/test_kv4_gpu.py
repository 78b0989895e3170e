"""The 4-bit KV cache kernels against 64-bit restatements: append, read-back, attention for decode, verify and prefill.

Attention tolerance (``_bound``). With u = eps / 2 of the rows' type: expanded keys are off by u each, so a score by
at most u * scale * sum|q k| (and 1e-5 * that in fp32 accumulation), a soft cap does not enlarge that; every weight is
then off by the factor e^(2 ds), with ds the largest such error of the row; P and V are rounded once each. The row's
output is a weighted mean of v, so it is off by at most (2 ds + 2 u + 1e-5) * mean|v| (first order; ds <= 1/4 is
asserted, second order adds a factor e^(2 ds) <= 1.65) plus u |out| for the final rounding.
"""
import math

import numpy as np
import pytest
import torch

from mlc_llm_b200 import ops
from mlc_llm_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float16, torch.bfloat16]


def _kv(g, n, hkv, d, dtype):
    k = torch.randn(n, hkv, d, generator=g)
    k[..., 5::37] *= 6.0
    v = torch.randn(n, hkv, d, generator=g) * 0.5
    return torch.cat([k.view(n, -1), v.view(n, -1)], dim=1).to(dtype)


def _same_bytes(a, b):
    return torch.equal(a.cpu().contiguous().view(torch.uint8), b.cpu().contiguous().view(torch.uint8))


# ------------------------------------------------------------------------------------------------- append, read
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,hq,hkv,d,rot,page", [(1, 32, 8, 128, 128, 16), (7, 14, 2, 64, 64, 16), (300, 8, 4, 256, 256, 16),
                                                 (33, 16, 16, 96, 48, 16), (5, 3, 1, 32, 10, 4), (601, 6, 3, 128, 32, 16),
                                                 (2, 0, 5, 64, 0, 1), (9, 2, 128, 256, 256, 16)])
def test_append_matches_the_format(dtype, t, hq, hkv, d, rot, page):
    g = torch.Generator().manual_seed(t + d)
    x = torch.cat([torch.randn(t, hq * d, generator=g).to(dtype), _kv(g, t, hkv, d, dtype)], dim=1).contiguous()
    pos = torch.randint(0, 131072, (t,), generator=g).to(torch.int32)
    pages = t // page + 4
    slot = torch.randperm(pages * page, generator=g)[:t].to(torch.int32)
    slot[t // 2] = -1 if t > 2 else slot[t // 2]
    inv = ref.rope_inv_freq(rot, 500000.0) if rot else None
    cache = ops.kv4_cache(pages, hkv, d, page, dtype, DEV)
    mine = x.to(DEV)
    ops.rope_append(mine, cache, pos.to(DEV), slot.to(DEV), None if inv is None else inv.to(DEV), hq, hkv, d, rot, page)
    ops.check_status(cache.device)
    want_cache, want = ops.kv4_cache(pages, hkv, d, page, dtype, "cpu"), x.clone()
    ops.rope_append(want, want_cache, pos, slot, inv, hq, hkv, d, rot, page)
    assert _same_bytes(cache, want_cache)
    assert _same_bytes(mine[:, hq * d:], want[:, hq * d:])
    # q: one rounding to the type, and 32-bit products: 4 roundings of 2^-24 of |a| + |b|
    u = torch.finfo(dtype).eps / 2
    a = x[:, : hq * d].double().view(t, hq, d)
    room = 2 * u * want[:, : hq * d].double().abs() + 2.0 ** -22 * a.abs().amax(-1, keepdim=True).expand(t, hq, d).reshape(t, hq * d) * 2
    err = (mine[:, : hq * d].double().cpu() - want[:, : hq * d].double()).abs()
    assert bool((err <= room).all()) if hq else True
    k, v = ops.kv4_read(cache, slot.to(DEV), d)
    rk, rv = ops.kv4_read(want_cache, slot, d)
    # lo + s c is rounded once by the kernel, twice by the fp32 restatement: equal up to a double rounding
    for got, exp in ((k, rk), (v, rv)):
        e = exp.double()
        room = 2.0 ** -23 * 4 * e.abs().amax().item() + u * 2 * e.abs()
        assert bool(((got.cpu().double() - e).abs() <= room).all())
        full = ref.kv4_unpack(want_cache[slot.clamp(min=0).long() // page, :, :, slot.clamp(min=0).long() % page, :], d)
    assert full.shape == (t, 2, hkv, d)


@pytest.mark.parametrize("rot", [128, 64])
def test_append_at_positions_far_beyond_a_million(rot):
    """Angles keep their 64 bits: the rotated keys and codes are those of 64-bit sines of pos * inv_freq."""
    g = torch.Generator().manual_seed(rot)
    t, hkv, d = 1024, 8, 128
    x = _kv(g, t, hkv, d, torch.float16).contiguous()
    pos = torch.randint(2 ** 29, 2 ** 30, (t,), generator=g).to(torch.int32)
    slot, inv = torch.arange(t, dtype=torch.int32), ref.rope_inv_freq(rot, 500000.0)
    cache, want_cache = (ops.kv4_cache(t // 16, hkv, d, 16, torch.float16, dev) for dev in (DEV, "cpu"))
    mine, want = x.to(DEV), x.clone()
    ops.rope_append(mine, cache, pos.to(DEV), slot.to(DEV), inv.to(DEV), 0, hkv, d, rot, 16)
    ops.rope_append(want, want_cache, pos, slot, inv, 0, hkv, d, rot, 16)
    ops.check_status(cache.device)
    assert _same_bytes(mine, want) and _same_bytes(cache, want_cache)


@pytest.mark.parametrize("dtype", TYPES)
def test_append_of_values_that_are_not_finite(dtype):
    big = torch.finfo(dtype).max
    row = torch.tensor([math.nan, math.inf, -math.inf, big, -big, 0.0, 1.0, -1.0] * 16 + [math.nan] * 32 + [2.5] * 32
                       + [1e-7, -1e-7] * 32).to(dtype).view(1, 256)
    x = row.repeat(1, 1).to(DEV)
    cache = ops.kv4_cache(1, 1, 128, 16, dtype, DEV)
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.rope_append(x, cache, zero, zero, None, 0, 1, 128, 0, 16)
    want = ops.kv4_cache(1, 1, 128, 16, dtype, "cpu")
    ops.rope_append(row.clone(), want, zero.cpu(), zero.cpu(), None, 0, 1, 128, 0, 16)
    assert _same_bytes(cache, want)
    k, v = ops.kv4_read(cache, zero, 128)
    assert bool(torch.isfinite(k).all()) and bool(torch.isfinite(v).all())


def test_append_and_read_report_bad_slots():
    cache = ops.kv4_cache(2, 1, 64, 16, torch.float16, DEV)
    x = torch.ones(2, 128, dtype=torch.float16, device=DEV)
    bad = torch.tensor([3, 32], dtype=torch.int32, device=DEV)  # the pool has 32 slots
    ops.rope_append(x, cache, bad, bad, None, 0, 1, 64, 0, 16)
    with pytest.raises(ops.KernelError):
        ops.check_status(cache.device)
    k, _ = ops.kv4_read(cache, bad, 64)
    with pytest.raises(ops.KernelError):
        ops.check_status(cache.device)
    assert bool((k[0] == 1).all()) and bool((k[1] == 0).all())


@pytest.mark.parametrize("t", [0, 1, 4097])
def test_read_lengths(t):
    cache = ops.kv4_cache(300, 3, 96, 16, torch.bfloat16, DEV)
    g = torch.Generator().manual_seed(0)
    kv = _kv(g, 4800, 3, 96, torch.bfloat16)
    slots = torch.arange(4800, dtype=torch.int32, device=DEV)
    ops.rope_append(kv.to(DEV), cache, slots, slots, None, 0, 3, 96, 0, 16)
    pick = torch.randint(0, 4800, (t,), generator=g).to(torch.int32)
    k, v = ops.kv4_read(cache, pick.to(DEV), 96)
    want = ref.kv4_unpack(ref.kv4_pack(kv.view(4800, 2, 3, 96)), 96)[pick.long()]
    assert k.shape == (t, 3, 96) and v.shape == (t, 3, 96)
    u = torch.finfo(torch.bfloat16).eps / 2
    for got, exp in ((k, want[:, 0]), (v, want[:, 1])):
        assert bool(((got.cpu().float() - exp).abs() <= u * exp.abs() * 1.01 + 1e-5).all())


# ------------------------------------------------------------------------------------------------- attention
class Step:
    """A filled cache, one step's queries over it, and the oracle. Everything the step may not look at (rows of the
    last pages behind the sequence, pages of nobody) holds NaN."""

    def __init__(self, dtype, lens, new, hq, hkv, d, page=16, window=0, sink=0, cap=0.0, tree=False, seed=0,
                 first_page=0, kvlen=None, q_by=1.0, k_by=1.0):
        g = torch.Generator().manual_seed(seed)
        self.hq, self.hkv, self.d, self.page, self.sink, self.cap, self.dtype = hq, hkv, d, page, sink, cap, dtype
        held = [(n + page - 1) // page for n in lens]
        pages = sum(held) + 3
        perm = torch.randperm(pages, generator=g)[: sum(held)]
        indptr = np.concatenate([[0], np.cumsum(held)]).astype(np.int32)
        slots = torch.tensor([int(perm[indptr[i] + j // page]) * page + j % page for i, n in enumerate(lens) for j in range(n)],
                             dtype=torch.int64)
        kv = _kv(g, len(slots), hkv, d, dtype)
        kv[:, : hkv * d] *= k_by
        self.cache = torch.full((pages + first_page, 2, hkv, page, ops.kv4_row(d, dtype)), math.nan, dtype=dtype, device=DEV)
        if len(slots):
            at = (slots + first_page * page).to(torch.int32).to(DEV)
            ops.rope_append(kv.to(DEV), self.cache, at, at, None, 0, hkv, d, 0, page)
        vals = ref.kv4_unpack(ref.kv4_pack(kv.view(-1, 2, hkv, d)), d).double()
        cut = np.concatenate([[0], np.cumsum(lens)])
        self.vals = [vals[cut[i]:cut[i + 1]] for i in range(len(lens))]
        t = sum(new)
        qkv = (torch.randn(t, (hq + 2 * hkv) * d, generator=g) * q_by).to(dtype)
        self.qkv = qkv.to(DEV)
        self.q = self.qkv[:, : hq * d]
        self.q_indptr = np.concatenate([[0], np.cumsum(new)]).astype(np.int64)
        self.seq = np.repeat(np.arange(len(new)), new)
        self.tree = None
        if tree:
            masks = []
            for n in new:
                seen = []
                for j in range(n):
                    up = seen[int(torch.randint(0, j, (1,), generator=g))] if j else 0
                    seen.append(up | (1 << j))
                masks += seen
            self.tree = torch.tensor(masks, dtype=torch.int64)
            self.kvlen = torch.tensor(np.repeat([n - m for n, m in zip(lens, new)], new), dtype=torch.int32)
        else:
            self.kvlen = torch.cat([torch.arange(n - m + 1, n + 1) for n, m in zip(lens, new)]).to(torch.int32)
        if kvlen is not None:
            self.kvlen = torch.tensor(kvlen, dtype=torch.int32)
        self.kvstart = torch.clamp(self.kvlen - window, min=0).to(torch.int32) if window else None
        self.indptr = torch.from_numpy(indptr).to(DEV)
        self.indices = (perm + first_page).to(torch.int32).to(DEV)
        self.max_len = max(lens)
        self.plan = ops.kv4_plan(self.q_indptr, self.kvlen.to(DEV), self.indptr, self.indices, hq, hkv, self.max_len)

    def run(self, plan=True, lse=True, q=None):
        on = lambda x: None if x is None else x.to(DEV)
        return ops.paged_attention(self.q if q is None else q, self.cache, on(torch.from_numpy(self.seq.astype(np.int32))), on(self.kvlen), self.indptr,
                                   self.indices, self.hq, self.hkv, self.d, self.page, self.d ** -0.5, q_kvstart=on(self.kvstart),
                                   sink=self.sink, tree_mask=on(self.tree), softcap=self.cap, return_lse=lse,
                                   plan=self.plan if plan else None)

    def check(self, out, lse=None):
        hq, hkv, d, g = self.hq, self.hkv, self.d, self.hq // self.hkv
        u, scale = torch.finfo(self.dtype).eps / 2, d ** -0.5
        q = self.q.cpu().double().view(-1, hkv, g, d)
        assert out.shape == (q.shape[0], hq * d)
        got = out.cpu().double().view(-1, hkv, g, d)
        for t in range(q.shape[0]):
            n = int(self.kvlen[t])
            kv = self.vals[self.seq[t]]
            see = torch.zeros(kv.shape[0], dtype=torch.bool)
            first = int(self.kvstart[t]) if self.kvstart is not None else 0
            see[first:n] = True
            if self.kvstart is not None:
                see[: min(n, self.sink)] = True
            if self.tree is not None:
                for b in range(63):
                    if (int(self.tree[t]) >> b) & 1:
                        see[n + b] = True
            if not bool(see.any()):
                assert bool((got[t] == 0).all())
                if lse is not None:
                    assert bool((lse[t] == -math.inf).all())
                continue
            k, v = kv[see, 0], kv[see, 1]                      # [n, hkv, d]
            s = torch.einsum("hgd,nhd->hgn", q[t], k) * scale
            ds = (u + 1e-5) * scale * torch.einsum("hgd,nhd->hgn", q[t].abs(), k.abs()).amax(-1, keepdim=True)
            if self.cap:
                s = self.cap * torch.tanh(s / self.cap)
                ds = ds + 1e-6 * self.cap
            assert float(ds.max()) <= 0.25
            z = torch.logsumexp(s, -1, keepdim=True)
            p = torch.exp(s - z)
            want = torch.einsum("hgn,nhd->hgd", p, v)
            mean = torch.einsum("hgn,nhd->hgd", p, v.abs())
            room = (2 * ds + 2 * u + 1e-5) * torch.exp(2 * ds) * mean + u * want.abs() + torch.finfo(self.dtype).tiny
            err = (got[t] - want).abs()
            assert bool((err <= room).all()), (t, float((err / room).max()))
            if lse is not None:
                # ln sum p: off by the scores' error, and 2^-23 of itself and of log2's argument scale
                off = (lse[t].cpu().double().view(hkv, g, 1) - z).abs()
                assert bool((off <= ds + 1e-5 + 1e-6 * z.abs()).all()), (t, float(off.max()))


DECODE = [
    # lens, new, hq, hkv, d, extras
    ([1], [1], 4, 2, 128, {}),
    ([15, 16, 17, 31, 32, 33, 48, 1], [1] * 8, 32, 8, 128, {}),
    ([5000], [1], 8, 2, 128, {}),                                  # split over the KV range and joined
    ([700, 3, 2500], [1, 1, 1], 14, 2, 64, {}),                    # seven heads per KV head
    ([333, 64, 100], [1, 1, 1], 8, 4, 256, {}),
    ([90, 40], [1, 1], 16, 1, 256, {}),                            # 16 rows of 256: two row blocks
    ([200, 65], [1, 1], 8, 8, 64, {}),                             # one head per KV head
    ([200, 65, 30], [1, 1, 1], 16, 1, 128, {}),
    ([50, 300, 7], [4, 2, 3], 8, 2, 128, {}),                      # short verify chunks, causal
    ([50, 300, 8], [4, 2, 5], 6, 2, 64, {"tree": True}),
    ([120, 700], [4, 4], 8, 2, 128, {"tree": True}),
    ([120, 70], [4, 3], 8, 4, 256, {"tree": True}),
    ([1000, 20, 129, 600], [1, 1, 1, 1], 8, 2, 128, {"window": 128, "sink": 4}),
    ([1000, 20, 129], [2, 1, 3], 8, 2, 64, {"window": 100, "sink": 20}),
    ([1000, 77], [1, 1], 8, 4, 256, {"window": 500, "cap": 50.0}),
    ([400, 77], [1, 1], 32, 8, 128, {"cap": 30.0}),
    ([300, 77], [1, 2], 8, 2, 128, {"q_by": 3000.0, "k_by": 2.0 ** -11}),  # sums of q beyond fp16
    ([300, 77], [1, 2], 8, 2, 128, {"q_by": 1e-3, "k_by": 500.0}),
    ([2000] * 40, [1] * 40, 32, 8, 128, {}),                       # more units than CTAs
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(DECODE)))
def test_decode(dtype, case):
    lens, new, hq, hkv, d, extra = DECODE[case]
    st = Step(dtype, lens, new, hq, hkv, d, seed=case, **extra)
    assert st.plan.num_tiles == 0
    out, lse = st.run()
    ops.check_status(out.device)
    st.check(out, lse)
    again = st.run(lse=False)
    assert _same_bytes(out, again)   # no atomics: the same call gives the same bits


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_decode_ignores_what_ran_before(dtype, d):
    """Four live rows use half of a column block. What earlier launches left in shared memory for the other half, here
    rows of very small and very large queries, changes no bit of theirs."""
    st = Step(dtype, [2000] * 24, [1] * 24, 8, 2, d, seed=1)
    small = Step(dtype, [2000] * 24, [1] * 24, 16, 2, d, seed=2, q_by=1e-4)
    large = Step(dtype, [2000] * 24, [1] * 24, 16, 2, d, seed=2, q_by=200.0)
    outs = []
    for other in (small, large, small):
        other.run()
        outs.append(st.run())
    ops.check_status(st.cache.device)
    for out, lse in outs[1:]:
        assert _same_bytes(out, outs[0][0]) and _same_bytes(lse, outs[0][1])


PREFILL = [
    ([100], [100], 8, 2, 128, {}),
    ([300, 17, 64, 1], [300, 17, 64, 1], 8, 2, 128, {}),           # two query tiles, one, and decode items next to them
    ([700, 260], [200, 129], 32, 8, 128, {}),                      # chunks behind a cached prefix
    ([3000], [40], 8, 2, 128, {}),                                 # few rows, long prefix: split and joined
    ([2500, 700], [33, 70], 14, 2, 64, {}),                        # 7 heads: rows of a token straddle the tiles
    ([150, 129], [150, 64], 4, 4, 64, {}),
    ([400, 90], [300, 90], 8, 4, 256, {}),
    ([1500], [45], 16, 1, 256, {}),                                # more than 128 rows per tile at d = 256, split
    ([200, 500, 31], [130, 60, 1], 4, 4, 96, {}),
    ([70, 129], [1, 1], 6, 2, 96, {}),                             # d = 96 decodes through this kernel too
    ([600, 300], [300, 100], 8, 2, 128, {"window": 100, "sink": 20}),
    ([2000], [60], 8, 2, 128, {"window": 300, "sink": 4}),
    ([300, 140], [300, 40], 8, 2, 64, {"window": 64}),
    ([300, 150], [150, 150], 8, 4, 256, {"window": 128, "sink": 4, "cap": 50.0}),
    ([200, 90], [200, 30], 8, 2, 128, {"cap": 30.0}),
    ([400, 1000, 60], [60, 31, 25], 8, 2, 128, {"tree": True}),
    ([400, 100], [20, 50], 8, 4, 256, {"tree": True}),
    ([300, 77], [200, 20], 8, 2, 128, {"q_by": 3000.0, "k_by": 2.0 ** -11}),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(PREFILL)))
def test_prefill(dtype, case):
    lens, new, hq, hkv, d, extra = PREFILL[case]
    st = Step(dtype, lens, new, hq, hkv, d, seed=case, **extra)
    out, lse = st.run()
    ops.check_status(out.device)
    st.check(out, lse)
    assert _same_bytes(out, st.run(lse=False))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,new,hq,hkv,d,page,extra", [
    ([60, 5], [3, 5], 4, 4, 96, 16, {}), ([60, 5], [1, 2], 4, 2, 32, 16, {"cap": 20.0}),
    ([60, 9], [20, 9], 4, 2, 64, 4, {"window": 30, "sink": 2}), ([100], [4], 4, 1, 160, 16, {"tree": True}),
    ([30, 20], [1, 1], 4, 2, 128, 1, {})])
def test_generic_shapes(dtype, lens, new, hq, hkv, d, page, extra):
    st = Step(dtype, lens, new, hq, hkv, d, page=page, **extra)
    for plan in (True, False):
        out, lse = st.run(plan=plan)
        ops.check_status(out.device)
        st.check(out, lse)


@pytest.mark.parametrize("dtype,d,q_by", [(torch.float16, 64, 6.0), (torch.float16, 128, 6.0), (torch.float16, 256, 6.0),
                                          (torch.bfloat16, 64, 3.0), (torch.bfloat16, 128, 3.0), (torch.bfloat16, 256, 2.5)])
def test_maxima_that_rise_along_the_sequence(dtype, d, q_by):
    """Scores of a standard deviation of 6 (bf16: what the oracle's bound on their error allows): later blocks exceed the
    running reference by more than its slack of 2^8, so sums and accumulators are rescaled."""
    st = Step(dtype, [1700, 400], [300, 150], 8, 2, d, seed=d, q_by=q_by)
    assert st.plan.num_tiles
    out, lse = st.run()
    ops.check_status(out.device)
    st.check(out, lse)
    st = Step(dtype, [3000, 400, 90], [1, 2, 1], 8, 2, d, seed=d + 1, q_by=q_by)
    assert st.plan.num_tiles == 0
    out, lse = st.run()
    ops.check_status(out.device)
    st.check(out, lse)


@pytest.mark.parametrize("span", [-32, 16, 32])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_values_of_very_different_sizes_along_the_sequence(d, span, monkeypatch):
    """bf16 values that shrink or grow, by up to 2^10 within a block of 128: a row that sees only the small ones keeps its
    precision, although it shares a tile, and larger values beside it, with rows that see them."""
    plain = _kv

    def scaled(g, n, hkv, d, dtype):
        rows = plain(g, n, hkv, d, dtype)
        by = torch.exp2(torch.linspace(-span / 2, span / 2, n).round())
        rows[:, hkv * d:] = (rows[:, hkv * d:].float() * by[:, None]).to(dtype)
        return rows

    monkeypatch.setitem(globals(), "_kv", scaled)
    for lens, new in (([400], [400]), ([150], [150]), ([400], [1])):
        st = Step(torch.bfloat16, lens, new, 8, 2, d, seed=d)
        out, lse = st.run()
        ops.check_status(out.device)
        st.check(out, lse)


@pytest.mark.parametrize("dtype", TYPES)
def test_more_tiles_than_the_gpu_holds_at_once(dtype):
    st = Step(dtype, [500, 1100, 900, 3], [500, 650, 130, 1], 32, 8, 64, seed=5)
    assert st.plan.num_tiles * 8 > torch.cuda.get_device_properties(0).multi_processor_count and st.plan.num_dec == 1
    ends = st.kvlen[(st.plan.tile_qstart + st.plan.tile_ntok - 1).long().cpu()]
    assert bool((ends.diff() >= 0).all())  # the longest last, where the kernel begins
    out, lse = st.run()
    ops.check_status(out.device)
    st.check(out, lse)


@pytest.mark.parametrize("d", [128, 64])
def test_rows_that_see_nothing(d):
    # a padded batch entry (length 0), and a row whose window starts behind it
    st = Step(torch.float16, [40, 40, 40], [1, 1, 1], 8, 2, d, kvlen=[40, 0, 17])
    out, lse = st.run()
    ops.check_status(out.device)
    st.check(out, lse)
    st = Step(torch.bfloat16, [40, 40], [1, 1], 8, 2, d, window=16, kvlen=[40, 20])
    st.kvstart = torch.tensor([40, 4], dtype=torch.int32)
    for plan in (True, False):
        out, lse = st.run(plan=plan)
        ops.check_status(out.device)
        st.check(out, lse)
    # the same among the rows of a prefill tile
    st = Step(torch.float16, [200, 60], [150, 50], 8, 2, d, window=64, sink=2)
    st.kvlen[10], st.kvlen[151], st.kvstart[20], st.kvstart[160] = 0, 0, 5000, 200
    for plan in (True, False):
        out, lse = st.run(plan=plan)
        ops.check_status(out.device)
        st.check(out, lse)


def test_page_numbers_outside_the_cache_are_reported():
    for plan in (True, False):
        for new in ([1, 1], [20, 20]):
            st = Step(torch.float16, [40, 40], new, 8, 2, 128)
            st.indices[1] = st.cache.shape[0]
            st.run(plan=plan)
            with pytest.raises(ops.KernelError):
                ops.check_status(st.cache.device)
            st = Step(torch.float16, [40, 40], new, 8, 2, 128)
            st.kvlen[-1] = 60  # three pages hold 48 tokens
            st.run(plan=plan)
            with pytest.raises(ops.KernelError):
                ops.check_status(st.cache.device)


def test_offsets_beyond_32_bits():
    # 2 * 8 * 16 * 80 bytes per page: the last pages start behind 4 GiB
    st = Step(torch.float16, [100, 37], [1, 1], 16, 8, 128, first_page=212000)
    assert st.cache.numel() * 2 > 1 << 32
    out, lse = st.run()
    ops.check_status(out.device)
    st.check(out, lse)
    out, lse = st.run(plan=False)
    st.check(out, lse)
    k, v = ops.kv4_read(st.cache, (st.indices[:1] * 16).contiguous(), 128)
    want = st.vals[0][0].to(k.device)
    assert bool(((k[0].double() - want[0]).abs() <= 2.0 ** -11 * want[0].abs() + 1e-6).all())


def test_graph_replay_and_other_stream():
    st = Step(torch.bfloat16, [900, 33, 5000], [1, 1, 1], 8, 2, 128)
    want = st.run(lse=False).clone()
    seq, kvlen = torch.from_numpy(st.seq.astype(np.int32)).to(DEV), st.kvlen.to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def call():
        return ops.paged_attention(st.q, st.cache, seq, kvlen, st.indptr, st.indices, 8, 2, 128, 16, 128 ** -0.5, plan=st.plan)

    with torch.cuda.stream(side):
        got = call()
    torch.cuda.current_stream().wait_stream(side)
    assert _same_bytes(got, want)
    graphs, outs = [], []
    for _ in range(2):  # two captured graphs in one pool, replayed one after the other
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            outs.append(call())
        graphs.append(g)
    for g, o in zip(graphs, outs):
        g.replay()
        torch.cuda.synchronize()
        assert _same_bytes(o, want)
    # new queries in the captured buffers
    st.qkv.neg_()
    graphs[0].replay()
    torch.cuda.synchronize()
    assert _same_bytes(outs[0], st.run(lse=False))


def test_append_then_attend_over_a_generation():
    """As a model uses them: a prompt, then tokens one by one, each step appending and attending, with rotation."""
    dtype, hq, hkv, d, page = torch.float16, 8, 2, 128, 16
    g = torch.Generator().manual_seed(11)
    prompt, steps = 37, 20
    inv = ref.rope_inv_freq(d, 10000.0)
    cache, host = ops.kv4_cache(8, hkv, d, page, dtype, DEV), ops.kv4_cache(8, hkv, d, page, dtype, "cpu")
    table = torch.tensor([5, 2, 7, 1], dtype=torch.int32)
    indptr = torch.tensor([0, 4], dtype=torch.int32)
    done = 0
    for n in [prompt] + [1] * steps:
        x = torch.randn(n, (hq + 2 * hkv) * d, generator=g).to(dtype)
        pos = torch.arange(done, done + n, dtype=torch.int32)
        slot = (table[(pos // page).long()] * page + pos % page).to(torch.int32)
        kvlen, seq = pos + 1, torch.zeros(n, dtype=torch.int32)
        done += n
        res = []
        for dev, c in ((DEV, cache), ("cpu", host)):
            y = x.to(dev)
            ops.rope_append(y, c, pos.to(dev), slot.to(dev), inv.to(dev), hq, hkv, d, d, page)
            plan = ops.kv4_plan([0, n], kvlen.to(dev), indptr.to(dev), table.to(dev), hq, hkv, done)
            res.append(ops.paged_attention(y[:, : hq * d], c, seq.to(dev), kvlen.to(dev), indptr.to(dev), table.to(dev), hq,
                                           hkv, d, page, d ** -0.5, plan=plan).float().cpu())
        ops.check_status(cache.device)
        assert _same_bytes(cache, host)
        # both sides round q and the output once; the bound of _Step with scores of |q||k| / sqrt(d) around 10
        assert float((res[0] - res[1]).abs().max()) <= 2 * 2.0 ** -11 * (2 * 10 + 3) * float(res[1].abs().max() + 1)
