"""Paged KV cache held in 4 bits: the cache itself, writing it, reading it back, attention over it.

A row is the ``d`` values of one (token, K or V, KV head), cut into groups of 32 channels. A group keeps its minimum
``lo`` and a step ``s = T((max - lo) / 15)``, both in the cache's type ``T``, and per value the code
``c = clamp(rint((x - lo) / s), 0, 15)``; it stands for ``lo + s * c`` (``s == 0``: for ``lo``). Before that NaN becomes 0
and values are clamped to a finite bound (``KV4_BOUND``), so a cache never holds anything but finite numbers and a
token's NaN cannot reach the tokens after it. That is 5 bits per value with 16-bit steps: 80 bytes for ``d = 128``.

A packed cache has the shape of the 16-bit one, ``[num_pages, 2, hkv, page, row]`` and its type, with
``row = kv4_row(d, dtype)`` elements of raw bytes in place of ``d`` values: ``d / 2`` code bytes, then ``d / 32`` pairs
``(lo, s)``. A code byte order: 32-bit words of 8 channels, nibble ``i`` of the low half is channel ``2 i``, of the high
half channel ``2 i + 1``. Rows of a token can be copied and moved like those of the 16-bit cache.
``ops.rope_append`` and ``ops.paged_attention`` recognise a packed cache by its row length.

On a GPU the rows are fp16 or bf16 and ``d`` a multiple of 32 up to 256; on CPU fp32 rows work as well.
"""

from __future__ import annotations

import contextlib
import ctypes
from typing import Optional, Tuple

import numpy as np
import torch

from . import reference as ref
from ._lib import DTYPE_CODE, check, lib, ptr, status_word, stream_ptr
from .attention import AttentionPlan, build_tiles, sm_count
from .reference import KV4_BOUND, KV4_GROUP, is_kv4, kv4_row

c_int = ctypes.c_int
c_ll = ctypes.c_longlong
c_float = ctypes.c_float


def kv4_cache(num_pages: int, hkv: int, d: int, page: int = 16, dtype: torch.dtype = torch.float16,
              device="cuda", layers: Optional[int] = None) -> torch.Tensor:
    """A zeroed packed cache ``[num_pages, 2, hkv, page, kv4_row(d, dtype)]`` (with ``layers``: one more leading
    dimension). Every row reads back as zeros."""
    shape = (num_pages, 2, hkv, page, kv4_row(d, dtype))
    return torch.zeros(shape if layers is None else (layers, *shape), dtype=dtype, device=device)


def _guard(device: torch.device):
    """Launches go to the tensors' device, whichever is current."""
    if device.index is None or device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _check_cache(kv_pages: torch.Tensor, d: int, what: str) -> None:
    if kv_pages.dim() != 5 or kv_pages.shape[1] != 2 or not is_kv4(kv_pages, d):
        raise ValueError(f"{what}: not a 4-bit cache of head size {d}: {tuple(kv_pages.shape)} {kv_pages.dtype}")
    if not kv_pages.is_contiguous():
        raise ValueError(f"{what}: the cache must be contiguous")
    if kv_pages.is_cuda and (kv_pages.dtype not in (torch.float16, torch.bfloat16) or d > 256):
        raise ValueError(f"{what}: on a GPU a 4-bit cache holds fp16 or bf16 rows of at most 256 channels, got "
                         f"{kv_pages.dtype} and {d}")


def _check_index(t: Optional[torch.Tensor], n: Optional[int], like: torch.Tensor, what: str,
                 dtype: torch.dtype = torch.int32) -> None:
    if t is None:
        return
    if t.dtype != dtype or t.dim() != 1 or t.device != like.device or not t.is_contiguous() \
            or (n is not None and t.shape[0] < n):
        raise ValueError(f"{what} must be a contiguous {dtype} vector on {like.device}"
                         + (f" of at least {n} entries" if n is not None else "") + f", got {t.dtype} {tuple(t.shape)}")


def append(qkv: torch.Tensor, kv_pages: torch.Tensor, pos: torch.Tensor, slot: torch.Tensor,
           inv_freq: Optional[torch.Tensor], hq: int, hkv: int, d: int, rot_dim: int, page: int,
           attn_factor: float = 1.0) -> None:
    """``ops.rope_append`` for a packed cache: rotate the q and k heads of ``qkv [T, (hq + 2 hkv) d]`` in place and
    write k and v, quantised, to ``slot`` (negative: rotate only). Angles are computed in 64 bits, so that keys at
    far positions do not change codes."""
    _check_cache(kv_pages, d, "rope_append")
    t = qkv.shape[0]
    if kv_pages.shape[2] != hkv or kv_pages.shape[3] != page:
        raise ValueError(f"rope_append: the cache has {kv_pages.shape[2]} heads and pages of {kv_pages.shape[3]} tokens, "
                         f"the call {hkv} and {page}")
    if qkv.dtype != kv_pages.dtype or qkv.device != kv_pages.device:
        raise ValueError(f"rope_append: rows are {qkv.dtype} on {qkv.device}, the cache {kv_pages.dtype} on {kv_pages.device}")
    if qkv.dim() != 2 or qkv.shape[1] != (hq + 2 * hkv) * d or not qkv.is_contiguous():
        raise ValueError(f"rope_append: rows of {(hq + 2 * hkv) * d} contiguous values expected, got {tuple(qkv.shape)}")
    if inv_freq is None:
        rot_dim = 0
    if rot_dim % 2 or not 0 <= rot_dim <= d:
        raise ValueError(f"rope_append: rotary size {rot_dim} does not fit heads of {d}")
    if rot_dim and (inv_freq.dtype != torch.float32 or inv_freq.numel() < rot_dim // 2 or not inv_freq.is_contiguous()
                    or inv_freq.device != qkv.device):
        raise ValueError(f"rope_append: {rot_dim // 2} fp32 frequencies on {qkv.device} expected")
    _check_index(pos if rot_dim else None, t, qkv, "rope_append: positions")
    _check_index(slot, t, qkv, "rope_append: slots")
    if not qkv.is_cuda:
        ref.rope_append(qkv, kv_pages, pos, slot, inv_freq, hq, hkv, d, rot_dim, page, attn_factor)
        return
    with _guard(qkv.device):
        rc = lib().mlcb_kv4_append(ptr(qkv), ptr(kv_pages), ptr(pos), ptr(slot), ptr(inv_freq), c_int(t), c_int(hq),
                                   c_int(hkv), c_int(d), c_int(rot_dim), c_int(page), c_float(attn_factor),
                                   c_ll(kv_pages.shape[0] * page), c_int(DTYPE_CODE[qkv.dtype]),
                                   ptr(status_word(qkv.device)), stream_ptr())
        check(rc, "mlcb_kv4_append")


def kv4_read(kv_pages: torch.Tensor, slot: torch.Tensor, d: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """The values that the rows at ``slot`` (int32 ``[T]``) of one layer's packed cache stand for: ``k, v [T, hkv, d]``
    in the cache's type. A negative slot reads as zeros."""
    _check_cache(kv_pages, d, "kv4_read")
    _check_index(slot, None, kv_pages, "kv4_read: slots")
    pages, _, hkv, page, _ = kv_pages.shape
    t = slot.shape[0]
    if not kv_pages.is_cuda:
        return ref.kv4_read(kv_pages, slot, d)
    k = torch.empty(t, hkv, d, dtype=kv_pages.dtype, device=kv_pages.device)
    v = torch.empty_like(k)
    with _guard(kv_pages.device):
        rc = lib().mlcb_kv4_read(ptr(kv_pages), ptr(slot), ptr(k), ptr(v), c_int(t), c_int(hkv), c_int(d), c_int(page),
                                 c_ll(pages * page), c_int(DTYPE_CODE[k.dtype]), ptr(status_word(k.device)), stream_ptr())
        check(rc, "mlcb_kv4_read")
    return k, v


# --------------------------------------------------------------------------- attention
KV4_TILE_ROWS = 256  # query rows that share one expansion of the cached blocks


def kv4_plan(q_indptr, q_kvlen: torch.Tensor, page_indptr: torch.Tensor, page_indices: torch.Tensor, hq: int, hkv: int,
             max_len: int) -> AttentionPlan:
    """The tiling of one step for ``ops.paged_attention`` over a packed cache (shared by all layers). ``q_indptr``:
    host array, first token of every sequence's chunk; ``max_len``: the longest sequence, appended tokens included."""
    q_indptr = np.asarray(q_indptr, dtype=np.int64)
    tiles = build_tiles(q_indptr, hq // hkv, tile_rows=KV4_TILE_ROWS)
    dev = q_kvlen.device
    on = {k: torch.from_numpy(a).to(dev) for k, a in tiles.items()}
    num_dec = len(tiles["dec_seq"])
    return AttentionPlan(on["tile_seq"], on["tile_qstart"], on["tile_ntok"], q_kvlen, page_indptr, page_indices,
                         len(tiles["tile_seq"]), dec_seq=on["dec_seq"], dec_qstart=on["dec_qstart"], dec_ntok=on["dec_ntok"],
                         num_dec=num_dec, dec_splits=1, max_pages=(int(max_len) + 15) // 16, tile_rows=KV4_TILE_ROWS,
                         dec_rows=int(tiles["dec_ntok"].max()) * (hq // hkv) if num_dec else 16)


def _decode_ctas(num_items: int, rows: int, hkv: int, max_pages: int, device: torch.device) -> int:
    """CTAs of the decode kernel: as many as stay resident, but no more than one per four 32-token slots."""
    slots = num_items * hkv * ((rows + 7) // 8) * max(1, (max_pages + 1) // 2)
    return max(1, min(4 * sm_count(device), (slots + 3) // 4))


def attend(q: torch.Tensor, kv_pages: torch.Tensor, q_seq: torch.Tensor, q_kvlen: torch.Tensor, page_indptr: torch.Tensor,
           page_indices: torch.Tensor, hq: int, hkv: int, d: int, page: int, sm_scale: float,
           q_kvstart: Optional[torch.Tensor], sink: int, tree_mask: Optional[torch.Tensor], softcap: float,
           return_lse: bool, plan: Optional[AttentionPlan]):
    """``ops.paged_attention`` for a packed cache."""
    _check_cache(kv_pages, d, "paged_attention")
    t = q.shape[0]
    if hkv <= 0 or hq <= 0 or hq % hkv or kv_pages.shape[2] != hkv or kv_pages.shape[3] != page:
        raise ValueError(f"paged_attention: {hq} query and {hkv} KV heads, pages of {page} tokens do not fit a cache of "
                         f"{kv_pages.shape[2]} heads and pages of {kv_pages.shape[3]} tokens")
    if q.dtype != kv_pages.dtype or q.device != kv_pages.device:
        raise ValueError(f"paged_attention: q is {q.dtype} on {q.device}, the cache {kv_pages.dtype} on {kv_pages.device}")
    if q.dim() != 2 or q.shape[1] != hq * d or (t and (q.stride(1) != 1 or (t > 1 and q.stride(0) < hq * d))):
        raise ValueError(f"paged_attention: q must be [T, {hq * d}] with contiguous rows, got {tuple(q.shape)} {q.stride()}")
    _check_index(q_seq, t, q, "paged_attention: q_seq")
    _check_index(q_kvlen, t, q, "paged_attention: q_kvlen")
    _check_index(q_kvstart, t, q, "paged_attention: q_kvstart")
    _check_index(page_indptr, None, q, "paged_attention: page_indptr")
    _check_index(page_indices, None, q, "paged_attention: page_indices")
    _check_index(tree_mask, t, q, "paged_attention: tree_mask", torch.int64)
    if not q.is_cuda:
        res = ref.paged_attention(q.reshape(t, hq, d), kv_pages, q_seq, q_kvlen, page_indptr, page_indices, hq, hkv, d,
                                  page, sm_scale, q_kvstart, sink, tree_mask, softcap, return_lse)
        return (res[0].reshape(t, hq * d), res[1]) if return_lse else res.reshape(t, hq * d)
    out = torch.empty(t, hq * d, dtype=q.dtype, device=q.device)
    lse = torch.empty(t, hq, dtype=torch.float32, device=q.device) if return_lse else None
    with _guard(q.device):
        _launch(q, kv_pages, out, lse, q_seq, q_kvlen, page_indptr, page_indices, hq, hkv, d, page, sm_scale, q_kvstart,
                int(sink), tree_mask, float(softcap), plan)
    return (out, lse) if return_lse else out


def _decode(q, kv_pages, out, lse, q_kvlen, page_indptr, page_indices, hq, hkv, d, sm_scale, q_kvstart, sink, tree_mask,
            softcap, plan) -> None:
    # with one token per item the rows are the group's heads, whatever the plan was made for
    rows = hq // hkv if q.shape[0] == plan.num_dec else min(16, plan.dec_rows)
    ctas = _decode_ctas(plan.num_dec, rows, hkv, plan.max_pages, q.device)
    part = torch.empty(ctas * (2 * 16 * (d + 2) + 4), dtype=torch.float32, device=q.device)
    part_unit, part_ml, part_o = part[: 4 * ctas], part[4 * ctas: 68 * ctas], part[68 * ctas:]
    rc = lib().mlcb_kv4_decode(ptr(q), ptr(kv_pages), ptr(out), ptr(lse), ptr(plan.dec_seq), ptr(plan.dec_qstart),
                               ptr(plan.dec_ntok), ptr(q_kvlen), ptr(page_indptr), ptr(page_indices), c_int(plan.num_dec),
                               c_int(rows), c_ll(q.stride(0)), c_int(hq), c_int(hkv), c_int(d), c_ll(kv_pages.shape[0]),
                               c_float(sm_scale), c_int(DTYPE_CODE[q.dtype]), c_int(ctas), ptr(part_o), ptr(part_ml),
                               ptr(part_unit), ptr(status_word(q.device)), stream_ptr(), ptr(q_kvstart), ptr(tree_mask),
                               c_int(sink), c_float(softcap))
    check(rc, "mlcb_kv4_decode")


def _prefill_splits(ctas: int, blocks: int, device: torch.device) -> int:
    """KV splits of the prefill kernel (one CTA per SM): few tiles are cut so that they cover the SMs, two blocks of
    cached positions per split at least."""
    return max(1, min(sm_count(device) // max(1, ctas), blocks // 2, 64))


def _prefill(q, kv_pages, out, lse, q_kvlen, page_indptr, page_indices, hq, hkv, d, sm_scale, q_kvstart, sink, tree_mask,
             softcap, plan, decode_items: bool) -> None:
    if decode_items:
        seq, qstart, ntok, num, rows = plan.dec_seq, plan.dec_qstart, plan.dec_ntok, plan.num_dec, min(16, plan.dec_rows)
    else:
        seq, qstart, ntok, num, rows = plan.tile_seq, plan.tile_qstart, plan.tile_ntok, plan.num_tiles, plan.tile_rows
    ctas = num * hkv * (2 if d == 256 and rows > 128 else 1)
    splits = _prefill_splits(ctas, plan.max_pages // (4 if d == 256 else 8), q.device)
    part_o = part_ml = None
    if splits > 1:
        part = torch.empty(num * hkv * splits * 256 * (d + 2), dtype=torch.float32, device=q.device)
        part_ml, part_o = part[: num * hkv * splits * 512], part[num * hkv * splits * 512:]
    rc = lib().mlcb_kv4_prefill(ptr(q), ptr(kv_pages), ptr(out), ptr(lse), ptr(seq), ptr(qstart), ptr(ntok), ptr(q_kvlen),
                                ptr(page_indptr), ptr(page_indices), c_int(num), c_int(rows), c_ll(q.stride(0)), c_int(hq),
                                c_int(hkv), c_int(d), c_ll(kv_pages.shape[0]), c_float(sm_scale),
                                c_int(DTYPE_CODE[q.dtype]), c_int(splits), ptr(part_o), ptr(part_ml),
                                ptr(status_word(q.device)), stream_ptr(), ptr(q_kvstart), ptr(tree_mask), c_int(sink),
                                c_float(softcap))
    check(rc, "mlcb_kv4_prefill")


def _launch(q, kv_pages, out, lse, q_seq, q_kvlen, page_indptr, page_indices, hq, hkv, d, page, sm_scale, q_kvstart, sink,
            tree_mask, softcap, plan) -> None:
    t = q.shape[0]
    aligned = q.data_ptr() % 16 == 0 and (q.stride(0) % 8 == 0 or t == 1)
    if plan is not None and plan.use_tensor_core and page == 16 and d in (64, 96, 128, 256) and aligned \
            and hq // hkv <= plan.tile_rows:
        args = (q, kv_pages, out, lse, q_kvlen, page_indptr, page_indices, hq, hkv, d, sm_scale, q_kvstart, sink, tree_mask,
                softcap, plan)
        if plan.num_dec:
            if d == 96:  # no decode kernel: its lanes own powers of two of channels
                _prefill(*args, decode_items=True)
            else:
                _decode(*args)
        if plan.num_tiles:
            _prefill(*args, decode_items=False)
        return
    rc = lib().mlcb_kv4_attn_simt(ptr(q), ptr(kv_pages), ptr(out), ptr(lse), ptr(q_seq), ptr(q_kvlen), ptr(q_kvstart),
                                  ptr(tree_mask), ptr(page_indptr), ptr(page_indices), c_int(t), c_ll(q.stride(0)),
                                  c_int(hq), c_int(hkv), c_int(d), c_int(page), c_ll(kv_pages.shape[0]), c_int(sink),
                                  c_float(sm_scale), c_float(softcap), c_int(DTYPE_CODE[q.dtype]),
                                  ptr(status_word(q.device)), stream_ptr())
    check(rc, "mlcb_kv4_attn_simt")


__all__ = ["KV4_BOUND", "KV4_GROUP", "is_kv4", "kv4_cache", "kv4_plan", "kv4_read", "kv4_row"]
