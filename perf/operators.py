"""Cases of the operators on a paged KV cache held in 4 bits: writing it (rotary embedding + quantisation), reading it
back, and attention over it for single tokens, short verification chunks and prefill chunks.

``own = False`` computes every operator from elementary torch operations, ``own = True`` calls the package.

A cache row is the ``d`` values of one (token, K or V, KV head). It is cut into groups of 32 channels; a group keeps its
minimum ``lo`` and a step ``s = (max - lo) / 15``, both in the type of the rows, and a code ``c`` of 4 bits per value, the
nearest to ``(x - lo) / s``. The group stands for ``lo + s * c``. Before that, NaN becomes 0 and values are clamped to a
finite bound (65440 in fp16, 2^126 in bf16). Keys are rounded to the type of the rows between rotation and quantisation.
"""

import math
import random

import numpy as np
import torch

own = False

PAGE = 16
GROUP = 32
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
BOUND = {torch.float16: 65440.0, torch.bfloat16: 2.0 ** 126}


# ------------------------------------------------------------------------------------------------- cases
def _append(name, dtype, tokens, hq, hkv, d, rot, far):
    return {"name": name, "op": "append", "dtype": dtype, "tokens": tokens, "hq": hq, "hkv": hkv, "d": d, "rot": rot,
            "far": far}


def _read(name, dtype, tokens, hkv, d):
    return {"name": name, "op": "read", "dtype": dtype, "tokens": tokens, "hkv": hkv, "d": d}


def _attend(name, dtype, batch, ctx_lo, ctx_hi, new_lo, new_hi, hq, hkv, d, window=0, sink=0, cap=0.0, tree=False):
    return {"name": name, "op": "attend", "dtype": dtype, "batch": batch, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi,
            "new_lo": new_lo, "new_hi": new_hi, "hq": hq, "hkv": hkv, "d": d, "window": window, "sink": sink,
            "cap": cap, "tree": tree}


def listed():
    return [
        # one decode step of one conversation: launch latency
        _append("append_one_token", "f16", 1, 32, 8, 128, 128, 8191),
        # one decode step of a full server batch at far positions
        _append("append_decode_batch", "bf16", 256, 32, 8, 128, 128, 131071),
        # an uneven prefill chunk of a small model with seven query heads per KV head
        _append("append_small_heads", "f16", 777, 14, 2, 64, 64, 32767),
        # a full prefill chunk
        _append("append_prefill_chunk", "bf16", 2048, 32, 8, 128, 128, 131071),
        # a few rows read back, as a debugging or migration tool does
        _read("read_few_rows", "bf16", 77, 8, 128),
        # a whole long sequence read back
        _read("read_long_sequence", "f16", 65536, 8, 128),
        # one conversation's next token
        _attend("decode_one", "f16", 1, 1000, 1000, 1, 1, 32, 8, 128),
        # the serving benchmark's decode step: a full batch, ragged lengths
        _attend("decode_batch", "f16", 256, 512, 2048, 1, 1, 32, 8, 128),
        # few long conversations
        _attend("decode_long", "bf16", 8, 16000, 16384, 1, 1, 32, 8, 128),
        # wide heads, soft-capped logits, a sliding window with attention sinks
        _attend("decode_window_wide", "bf16", 32, 3, 6000, 1, 1, 8, 4, 256, window=4096, sink=4, cap=50.0),
        # a draft tree of four tokens per sequence under verification
        _attend("verify_tree", "f16", 64, 100, 4000, 4, 4, 32, 8, 128, tree=True),
        # a prefill chunk behind a long cached prefix, next to shorter prompts
        _attend("prefill_chunk", "bf16", 4, 0, 8192, 512, 2048, 32, 8, 128),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    heads = rng.choice([(32, 8, 128), (32, 32, 128), (64, 8, 128), (28, 4, 128), (8, 2, 128), (8, 1, 128), (14, 2, 64),
                        (32, 8, 64), (4, 2, 64), (8, 4, 256), (16, 16, 96)])
    hq, hkv, d = heads
    dtype = rng.choice(["f16", "bf16"])
    kind = rng.choice(["append", "read", "decode", "decode", "verify", "prefill", "prefill"])
    heavy = hkv * d / 1024.0
    if kind == "append":
        rot = rng.choice([d, d, d // 2])
        c = _append("", dtype, _spread(rng, 1, 1900 if hq < 64 else 900), hq, hkv, d, rot, _spread(rng, 100, 131071))
    elif kind == "read":
        c = _read("", dtype, _spread(rng, 1, int(60000 / max(1.0, heavy))), hkv, d)
    else:
        window, sink, cap = 0, 0, 0.0
        if rng.random() < 0.25:
            window, sink = rng.choice([128, 500, 4096]), rng.choice([0, 4, 20])
        if rng.random() < 0.2:
            cap = rng.choice([30.0, 50.0])
        if kind == "prefill":
            new_hi = _spread(rng, 17, 2000)
            batch = rng.randint(1, 3 if hq < 64 else 1)
            ctx_hi = rng.choice([0, _spread(rng, 1, 8000)])
            c = _attend("", dtype, batch, ctx_hi // 3, ctx_hi, max(2, new_hi // 3), new_hi, hq, hkv, d, window, sink, cap)
        else:
            batch = _spread(rng, 1, 200)
            most = int(min(16000, 260000 / batch / max(1.0, heavy)))
            ctx_hi = _spread(rng, 1, max(2, most))
            new = 1 if kind == "decode" else rng.randint(2, 6)
            c = _attend("", dtype, batch, ctx_hi // 4, ctx_hi, new, new, hq, hkv, d, window, sink, cap,
                        tree=kind == "verify" and window == 0 and rng.random() < 0.6)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------- inputs
def _lengths(case):
    """Context and appended tokens of every sequence: a function of the case alone."""
    rng = random.Random("%(batch)d %(ctx_lo)d %(ctx_hi)d %(new_lo)d %(new_hi)d" % case)
    ctx = [rng.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["batch"])]
    new = [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["batch"])]
    ctx[-1], new[0] = case["ctx_hi"], case["new_hi"]
    return ctx, new


def _inv_freq(rot):
    inv = 1.0 / (500000.0 ** (torch.arange(0, rot, 2, dtype=torch.float64) / rot))
    return inv.to(torch.float32).cuda()


def _kv_rows(gen, n, hkv, d, dtype):
    """Keys with a few channels far larger than the rest, as trained models have, and plain values: [n, 2, hkv, d]."""
    big = torch.ones(hkv, d, device="cuda")
    big[:, 5::37] = 6.0
    shift = torch.zeros(hkv, d, device="cuda")
    shift[:, 7::53] = 3.0
    out = torch.empty(n, 2, hkv, d, dtype=dtype, device="cuda")
    step = max(1, (1 << 26) // (hkv * d))
    for a in range(0, n, step):
        b = min(n, a + step)
        out[a:b, 0] = (torch.randn(b - a, hkv, d, generator=gen, device="cuda") * big + shift).to(dtype)
        out[a:b, 1] = (torch.randn(b - a, hkv, d, generator=gen, device="cuda") * 0.5).to(dtype)
    return out


def _inputs(case, seed):
    """The tensors of a case, before any cache is laid out."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = TYPES[case["dtype"]]
    hkv, d = case["hkv"], case["d"]
    st = {"dtype": dtype}
    if case["op"] == "append":
        n, hq = case["tokens"], case["hq"]
        kv = _kv_rows(gen, n, hkv, d, dtype)
        q = torch.randn(n, hq * d, generator=gen, device="cuda").to(dtype)
        st["fresh"] = torch.cat([q, kv[:, 0].reshape(n, -1), kv[:, 1].reshape(n, -1)], dim=1).contiguous()
        st["pos"] = torch.randint(0, case["far"] + 1, (n,), generator=gen, device="cuda").to(torch.int32)
        pages = n // PAGE + 9
        st["slot"] = torch.randperm(pages * PAGE, generator=gen, device="cuda")[:n].to(torch.int32)
        st["pages"] = pages
        st["inv_freq"] = _inv_freq(case["rot"])
        return st
    if case["op"] == "read":
        n = case["tokens"]
        pages = n // PAGE + 3
        st["pages"] = pages
        st["rows"] = _kv_rows(gen, pages * PAGE, hkv, d, dtype)
        st["slot"] = torch.randperm(pages * PAGE, generator=gen, device="cuda")[:n].to(torch.int32)
        return st
    ctx, new = _lengths(case)
    total = [c + n for c, n in zip(ctx, new)]
    held = [(t + PAGE - 1) // PAGE for t in total]
    pages = sum(held) + 3
    st["pages"] = pages
    st["rows"] = _kv_rows(gen, pages * PAGE, hkv, d, dtype)
    st["page_indices"] = torch.randperm(pages, generator=gen, device="cuda")[:sum(held)].to(torch.int32)
    st["page_indptr_host"] = np.concatenate([[0], np.cumsum(held)]).astype(np.int32)
    st["q_indptr_host"] = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    t = sum(new)
    # rows of a fused projection: q is a view with a row stride wider than its columns
    qkv = torch.randn(t, (case["hq"] + 2 * hkv) * d, generator=gen, device="cuda").to(dtype)
    st["q"] = qkv[:, : case["hq"] * d]
    st["q_seq"] = torch.from_numpy(np.repeat(np.arange(len(new)), new).astype(np.int32)).cuda()
    st["tree_mask"] = st["kvstart"] = None
    if case["tree"]:
        # a root, then every node under a drawn earlier one; a node sees its ancestors and itself
        rng = random.Random(seed)
        masks = []
        for n in new:
            seen = []
            for j in range(n):
                up = seen[rng.randint(0, j - 1)] if j else 0
                seen.append(up | (1 << j))
            masks += seen
        st["tree_mask"] = torch.tensor(masks, dtype=torch.int64, device="cuda")
        kvlen = np.repeat(np.asarray(ctx), new)
    else:
        kvlen = np.concatenate([np.arange(c + 1, c + n + 1) for c, n in zip(ctx, new)])
    st["kvlen"] = torch.from_numpy(kvlen.astype(np.int32)).cuda()
    if case["window"]:
        st["kvstart"] = torch.clamp(st["kvlen"] - case["window"], min=0).to(torch.int32)
    st["total"], st["new"] = total, new
    return st


def _own_cache(st, hkv, d):
    """The packed cache of `rows` (slot i holds row i), written through the package."""
    from mlc_llm_b200 import ops

    cache = ops.kv4_cache(st["pages"], hkv, d, PAGE, st["dtype"], torch.device("cuda"))
    rows = st["rows"]
    zero = torch.zeros(1 << 16, dtype=torch.int32, device="cuda")
    for a in range(0, rows.shape[0], 1 << 16):
        part = rows[a:a + (1 << 16)].reshape(-1, 2 * hkv * d)
        slot = torch.arange(a, a + part.shape[0], dtype=torch.int32, device="cuda")
        ops.rope_append(part, cache, zero[: part.shape[0]], slot, None, 0, hkv, d, 0, PAGE)
    return cache


def _pack(x):
    """Rows [..., d] -> (codes of two channels per byte [..., d / 2], lo, s [..., d / 32])."""
    b = BOUND[x.dtype]
    g = torch.nan_to_num(x.float(), nan=0.0, posinf=b, neginf=-b).clamp(-b, b)
    g = g.reshape(*x.shape[:-1], -1, GROUP)
    lo, hi = g.amin(-1), g.amax(-1)
    s = ((hi - lo) / 15.0).to(x.dtype).float()
    one = torch.where(s > 0, s, torch.ones_like(s)).unsqueeze(-1)
    c = torch.round((g - lo.unsqueeze(-1)) / one).clamp(0, 15)
    c = torch.where(s.unsqueeze(-1) > 0, c, torch.zeros_like(c)).to(torch.uint8).reshape(x.shape)
    return c[..., 0::2] | (c[..., 1::2] << 4), lo.to(x.dtype), s.to(x.dtype)


def _unpack(codes, lo, s):
    """The values, in fp32."""
    c = torch.stack([codes & 15, codes >> 4], dim=-1).reshape(*lo.shape, GROUP).float()
    return (lo.float().unsqueeze(-1) + s.float().unsqueeze(-1) * c).reshape(*lo.shape[:-1], -1)


def _plain_cache(st):
    parts = [_pack(p) for p in st["rows"].split(1 << 15)]
    return tuple(torch.cat([p[i] for p in parts]) for i in range(3))


def prepare(case, seed):
    st = _inputs(case, seed)
    hkv, d = case["hkv"], case["d"]
    st["case"] = case
    if case["op"] == "append":
        st["qkv"] = torch.empty_like(st["fresh"])
        if own:
            from mlc_llm_b200 import ops

            st["cache"] = ops.kv4_cache(st["pages"], hkv, d, PAGE, st["dtype"], torch.device("cuda"))
        else:
            n = st["pages"] * PAGE
            st["cache"] = (torch.zeros(n, 2, hkv, d // 2, dtype=torch.uint8, device="cuda"),
                           torch.zeros(n, 2, hkv, d // GROUP, dtype=st["dtype"], device="cuda"),
                           torch.zeros(n, 2, hkv, d // GROUP, dtype=st["dtype"], device="cuda"))
        return st
    st["cache"] = _own_cache(st, hkv, d) if own else _plain_cache(st)
    del st["rows"]
    if case["op"] == "attend":
        st["page_indptr"] = torch.from_numpy(st["page_indptr_host"]).cuda()
        if own:
            from mlc_llm_b200 import ops

            # the tiling of the step, made once for all layers of a forward
            st["plan"] = ops.kv4_plan(st["q_indptr_host"], st["kvlen"], st["page_indptr"], st["page_indices"],
                                      case["hq"], hkv, max(st["total"]))
    return st


# ------------------------------------------------------------------------------------------------- plain forms
def _rotate(qkv, pos, inv_freq, heads, d, attn_factor=1.0):
    """Rotary embedding of the first `heads` heads, in place. Angles and products in 64 bits: a key next to a rounding
    border would otherwise land in another code."""
    rot = 2 * inv_freq.numel()
    ang = pos.double().unsqueeze(-1) * inv_freq.double()
    cos, sin = torch.cos(ang).unsqueeze(1) * attn_factor, torch.sin(ang).unsqueeze(1) * attn_factor
    x = qkv.view(qkv.shape[0], -1, d)[:, :heads, :rot]
    a, b = x[..., : rot // 2].double(), x[..., rot // 2:].double()
    lo, hi = a * cos - b * sin, b * cos + a * sin
    x[..., : rot // 2] = lo.float().to(qkv.dtype)
    x[..., rot // 2:] = hi.float().to(qkv.dtype)


def _plain_append(st, case):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    qkv = st["qkv"]
    qkv.copy_(st["fresh"])
    _rotate(qkv, st["pos"], st["inv_freq"], hq + hkv, d)
    kv = qkv.view(qkv.shape[0], -1, d)[:, hq:].reshape(-1, 2, hkv, d)
    slot = st["slot"].long()
    for dst, src in zip(st["cache"], _pack(kv)):
        dst[slot] = src
    got = _unpack(*(c[slot] for c in st["cache"])).to(st["dtype"])
    return [qkv[:, : hq * d], got[:, 0], got[:, 1]]


def _plain_read(st):
    slot = st["slot"].long()
    got = _unpack(*(c[slot] for c in st["cache"])).to(st["dtype"])
    return [got[:, 0], got[:, 1]]


def _visible(st, case, a, b, total):
    """[tokens of the sequence, total]: which cached positions each appended token sees."""
    at = torch.arange(total, device="cuda").unsqueeze(0)
    n = st["kvlen"][a:b].unsqueeze(1)
    see = at < n
    if st["kvstart"] is not None:
        see = see & ((at >= st["kvstart"][a:b].unsqueeze(1)) | (at < case["sink"]))
    if st["tree_mask"] is not None:
        bit = (at - n).clamp(0, 62)
        see = see | ((at >= n) & (at - n < 63) & (((st["tree_mask"][a:b].unsqueeze(1) >> bit) & 1) == 1))
    return see


def _plain_attend(st, case):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    q, g = st["q"], case["hq"] // case["hkv"]
    scale = d ** -0.5
    out = torch.empty(q.shape[0], hq * d, dtype=q.dtype, device="cuda")
    paged = [c.view(-1, PAGE, *c.shape[1:]) for c in st["cache"]]
    ip, qp = st["page_indptr_host"], st["q_indptr_host"]
    for i, total in enumerate(st["total"]):
        a, b = int(qp[i]), int(qp[i + 1])
        pages = st["page_indices"][int(ip[i]): int(ip[i + 1])].long()
        kv = _unpack(*(c[pages].flatten(0, 1)[:total] for c in paged))           # [total, 2, hkv, d]
        k, v = kv[:, 0].permute(1, 2, 0), kv[:, 1].transpose(0, 1)               # [hkv, d, total], [hkv, total, d]
        qs = q[a:b].view(b - a, hkv, g, d).permute(1, 2, 0, 3).reshape(hkv, g * (b - a), d).float()
        s = torch.bmm(qs, k).mul_(scale)
        if case["cap"]:
            s = case["cap"] * torch.tanh(s / case["cap"])
        hidden = ~_visible(st, case, a, b, total)
        s = s.view(hkv, g, b - a, total).masked_fill_(hidden, -math.inf)
        top = s.amax(-1, keepdim=True)
        top = torch.where(top == -math.inf, torch.zeros_like(top), top)
        p = s.sub_(top).exp_()
        norm = p.sum(-1, keepdim=True)
        o = torch.bmm(p.view(hkv, -1, total), v).view(hkv, g, b - a, d) / torch.where(norm > 0, norm, torch.ones_like(norm))
        out[a:b] = o.permute(2, 0, 1, 3).reshape(b - a, hq * d).to(q.dtype)
    return [out]


def run(state):
    case = state["case"]
    hkv, d = case["hkv"], case["d"]
    if not own:
        if case["op"] == "append":
            return _plain_append(state, case)
        return _plain_read(state) if case["op"] == "read" else _plain_attend(state, case)
    from mlc_llm_b200 import ops

    if case["op"] == "append":
        # the projection's rows, rotated in place by the call, and what the written slots now stand for
        qkv = state["qkv"]
        qkv.copy_(state["fresh"])
        ops.rope_append(qkv, state["cache"], state["pos"], state["slot"], state["inv_freq"], case["hq"], hkv, d,
                        case["rot"], PAGE)
        k, v = ops.kv4_read(state["cache"], state["slot"], d)
        return [qkv[:, : case["hq"] * d], k, v]
    if case["op"] == "read":
        return list(ops.kv4_read(state["cache"], state["slot"], d))
    return [ops.paged_attention(state["q"], state["cache"], state["q_seq"], state["kvlen"], state["page_indptr"],
                                state["page_indices"], case["hq"], hkv, d, PAGE, d ** -0.5,
                                q_kvstart=state["kvstart"], sink=case["sink"], tree_mask=state["tree_mask"],
                                softcap=case["cap"], plan=state["plan"])]


# ------------------------------------------------------------------------------------------------- what has to be done
def _row_bytes(d):
    return d // 2 + d // GROUP * 4


def work(case):
    hkv, d = case["hkv"], case["d"]
    row = _row_bytes(d)
    if case["op"] == "append":
        n, hq = case["tokens"], case["hq"]
        groups = 2 * hkv * d
        return {"bytes": n * ((hq + 2 * hkv) * d * 2 + hq * d * 2 + 2 * hkv * row + 2 * hkv * d * 2 + 8),
                "flops": n * ((hq + hkv) * case["rot"] * 3 + groups * 8)}
    if case["op"] == "read":
        n = case["tokens"]
        return {"bytes": n * 2 * hkv * (row + 2 * d) + 4 * n, "flops": n * 2 * hkv * d * 2}
    ctx, new = _lengths(case)
    hq = case["hq"]
    pairs = rows = 0
    for c, n in zip(ctx, new):
        touched = 0
        for j in range(n):
            upto = c + (n + 1) // 2 if case["tree"] else c + j + 1  # a drawn tree shows about half of its nodes
            seen = upto
            if case["window"] and upto > case["window"]:
                seen = min(upto, case["window"] + min(case["sink"], upto - case["window"]))
            pairs += seen
            touched = max(touched, seen)
        rows += max(touched, min(c + n, touched + n - 1))
    return {"bytes": rows * 2 * hkv * row + sum(new) * hq * 4 * d, "flops": 4 * pairs * hq * d}


# ------------------------------------------------------------------------------------------------- in 64 bits
def _exact_values(x):
    """The values that a quantised row stands for, from the definition. The step is the fp32 quotient rounded to the
    rows' type, as the format stores it; everything else is in 64 bits."""
    bound = BOUND[x.dtype]
    v = x.double()
    v = torch.where(torch.isnan(v), torch.zeros_like(v), v).clamp(min=-bound, max=bound)
    out = torch.empty_like(v)
    for a in range(0, x.shape[-1], GROUP):
        part = v[..., a:a + GROUP]
        low, high = part.min(dim=-1, keepdim=True).values, part.max(dim=-1, keepdim=True).values
        step = ((high.float() - low.float()) / 15.0).to(x.dtype).double()
        code = torch.where(step > 0, ((part - low) / torch.where(step > 0, step, 1.0)).round().clamp(0, 15), 0.0)
        out[..., a:a + GROUP] = low + step * code
    return out


def _exact_append(st, case):
    hq, hkv, d, rot = case["hq"], case["hkv"], case["d"], case["rot"]
    n = case["tokens"]
    x = st["fresh"].view(n, hq + 2 * hkv, d)
    half = rot // 2
    turned = x[:, : hq + hkv].double()
    for j in range(half):
        ang = st["pos"].double() * float(st["inv_freq"][j])
        c, s = torch.cos(ang).view(n, 1), torch.sin(ang).view(n, 1)
        u, w = x[:, : hq + hkv, j].double(), x[:, : hq + hkv, j + half].double()
        turned[:, :, j] = u * c - w * s
        turned[:, :, j + half] = u * s + w * c
    k = turned[:, hq:].float().to(st["dtype"])
    return [turned[:, :hq].reshape(n, hq * d), _exact_values(k), _exact_values(x[:, hq + hkv:])]


def _exact_attend(st, case):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    g, scale = hq // hkv, 1.0 / math.sqrt(d)
    t = st["q"].shape[0]
    out = torch.zeros(t, hq, d, dtype=torch.float64, device="cuda")
    for i, total in enumerate(st["total"]):
        a, b = int(st["q_indptr_host"][i]), int(st["q_indptr_host"][i + 1])
        table = st["page_indices"][int(st["page_indptr_host"][i]): int(st["page_indptr_host"][i + 1])].long()
        where = torch.arange(total, device="cuda")
        kv = _exact_values(st["rows"][table[where // PAGE] * PAGE + where % PAGE])   # [total, 2, hkv, d]
        for lo in range(a, b, 256):
            hi = min(b, lo + 256)
            see = torch.zeros(hi - lo, total, dtype=torch.bool, device="cuda")
            for r in range(lo, hi):
                n = int(st["kvlen"][r])
                first = int(st["kvstart"][r]) if st["kvstart"] is not None else 0
                see[r - lo, first:n] = True
                see[r - lo, : min(n, case["sink"] if st["kvstart"] is not None else 0)] = True
                if st["tree_mask"] is not None:
                    m = int(st["tree_mask"][r])
                    for bit in range(m.bit_length()):
                        if (m >> bit) & 1:
                            see[r - lo, n + bit] = True
            for h in range(hkv):
                heads = slice(h * g, (h + 1) * g)
                x = st["q"][lo:hi].reshape(hi - lo, hq, d)[:, heads].double()
                s = torch.einsum("tgd,nd->gtn", x, kv[:, 0, h]) * scale
                if case["cap"]:
                    s = case["cap"] * torch.tanh(s / case["cap"])
                s = torch.where(see.unsqueeze(0), s, -math.inf)
                z = torch.logsumexp(s, dim=-1)                                       # [g, rows]
                p = torch.where(z.unsqueeze(-1) > -math.inf, torch.exp(s - z.unsqueeze(-1)), 0.0)
                out[lo:hi, heads] = torch.einsum("gtn,nd->tgd", p, kv[:, 1, h])
    return [out.reshape(t, hq * d)]


def exact(case, seed):
    st = _inputs(case, seed)
    if case["op"] == "append":
        return _exact_append(st, case)
    if case["op"] == "read":
        got = _exact_values(st["rows"][st["slot"].long()])
        return [got[:, 0], got[:, 1]]
    ctx, new = _lengths(case)
    # 64-bit products run at a few TFLOP/s: leave out what would take long
    if 4.0 * sum((c + n) * n for c, n in zip(ctx, new)) * case["hq"] * case["d"] > 1.5e12:
        return None
    return _exact_attend(st, case)
