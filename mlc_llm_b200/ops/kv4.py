"""Paged KV cache held in 4 bits: the cache itself, writing it, reading it back, attention over it.

A row is the ``d`` values of one (token, K or V, KV head), cut into groups of 32 channels. A group keeps its minimum
``lo`` and a step ``s = T((max - lo) * r)``, both in the cache's type ``T`` (``r`` is 1 / 15 in fp32), and per value the code
``c = clamp(rint((x - lo) / s), 0, 15)``; it stands for ``lo + s * c`` (``s == 0``: for ``lo``). Before that NaN becomes 0
and values are clamped to a finite bound (``KV4_BOUND``), so a cache never holds anything but finite numbers and a
token's NaN cannot reach the tokens after it. (On a GPU bf16 numbers below 2^-126 count as 0.) That is 5 bits per value with 16-bit steps: 80 bytes for ``d = 128``.

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
from ._lib import DTYPE_CODE, check, lib, status_word
from .attention import AttentionPlan, build_tiles, decode_rows, sm_count
from .reference import KV4_BOUND, KV4_GROUP, is_kv4, kv4_row

_P, _I, _L, _F, _D = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float, ctypes.c_double
_ARGS = {
    "mlcb_kv4_append": [_P] * 5 + [_I] * 6 + [_D, _L, _I, _P, _P],
    "mlcb_kv4_read": [_P] * 4 + [_I] * 4 + [_L, _I, _P, _P],
    "mlcb_kv4_decode": [_P] * 10 + [_I, _I, _L, _I, _I, _I, _L, _F, _I, _I] + [_P] * 7 + [_I, _F],
    "mlcb_kv4_prefill": [_P] * 10 + [_I, _I, _L, _I, _I, _I, _L, _F, _I, _I] + [_P] * 6 + [_I, _F],
    "mlcb_kv4_attn_simt": [_P] * 10 + [_I, _L, _I, _I, _I, _I, _L, _I, _F, _F, _I, _P, _P],
}
_FN = {}
_HERE = contextlib.nullcontext()


def _call(name: str, *args) -> None:
    """A kernel entry point with declared argument types: plain numbers and addresses (``None``: null) go in unwrapped,
    which takes a fifth of the time of a wrapper object per argument."""
    fn = _FN.get(name)
    if fn is None:
        fn = getattr(lib(), name)
        fn.argtypes = _ARGS[name]
        _FN[name] = fn
    check(fn(*args), name)


def _at(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _env(device: torch.device):
    """Status word and current stream of a device."""
    return status_word(device).data_ptr(), torch._C._cuda_getCurrentRawStream(device.index)  # pylint: disable=protected-access


def kv4_cache(num_pages: int, hkv: int, d: int, page: int = 16, dtype: torch.dtype = torch.float16,
              device="cuda", layers: Optional[int] = None) -> torch.Tensor:
    """A zeroed packed cache ``[num_pages, 2, hkv, page, kv4_row(d, dtype)]`` (with ``layers``: one more leading
    dimension). Every row reads back as zeros."""
    shape = (num_pages, 2, hkv, page, kv4_row(d, dtype))
    return torch.zeros(shape if layers is None else (layers, *shape), dtype=dtype, device=device)


def _guard(device: torch.device):
    """Launches go to the tensors' device, whichever is current."""
    return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _check_cache(kv_pages: torch.Tensor, d: int, what: str) -> None:
    shape = kv_pages.shape
    if len(shape) != 5 or shape[1] != 2 or not is_kv4(kv_pages, d):
        raise ValueError(f"{what}: not a 4-bit cache of head size {d}: {tuple(shape)} {kv_pages.dtype}")
    if not kv_pages.is_contiguous():
        raise ValueError(f"{what}: the cache must be contiguous")
    if kv_pages.is_cuda and (kv_pages.dtype == torch.float32 or d > 256):
        raise ValueError(f"{what}: on a GPU a 4-bit cache holds fp16 or bf16 rows of at most 256 channels, got "
                         f"{kv_pages.dtype} and {d}")


def _check_index(t: Optional[torch.Tensor], n: int, where: int, what: str, dtype: torch.dtype = torch.int32) -> None:
    if t is not None and (t.dtype != dtype or t.get_device() != where or t.dim() != 1 or t.numel() < n
                          or not t.is_contiguous()):
        raise ValueError(f"{what} must be a contiguous {dtype} vector of at least {n} entries on the cache's device, got "
                         f"{t.dtype} {tuple(t.shape)} on {t.device}")


def append(qkv: torch.Tensor, kv_pages: torch.Tensor, pos: torch.Tensor, slot: torch.Tensor,
           inv_freq: Optional[torch.Tensor], hq: int, hkv: int, d: int, rot_dim: int, page: int,
           attn_factor: float = 1.0) -> None:
    """``ops.rope_append`` for a packed cache: rotate the q and k heads of ``qkv [T, (hq + 2 hkv) d]`` in place and
    write k and v, quantised, to ``slot`` (negative: rotate only; the others differ from each other). Angles are computed
    in 64 bits, so that keys at far positions do not change codes."""
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
    where = qkv.get_device()
    if rot_dim:
        _check_index(pos, t, where, "rope_append: positions")
    _check_index(slot, t, where, "rope_append: slots")
    if not qkv.is_cuda:
        ref.rope_append(qkv, kv_pages, pos, slot, inv_freq, hq, hkv, d, rot_dim, page, attn_factor)
        return
    with _guard(qkv.device):
        _call("mlcb_kv4_append", qkv.data_ptr(), kv_pages.data_ptr(), _at(pos), slot.data_ptr(), _at(inv_freq), t, hq, hkv, d,
              rot_dim, page, attn_factor, kv_pages.shape[0] * page, DTYPE_CODE[qkv.dtype], *_env(qkv.device))


def kv4_read(kv_pages: torch.Tensor, slot: torch.Tensor, d: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """The values that the rows at ``slot`` (int32 ``[T]``) of one layer's packed cache stand for: ``k, v [T, hkv, d]``
    in the cache's type. A negative slot reads as zeros."""
    _check_cache(kv_pages, d, "kv4_read")
    _check_index(slot, 0, kv_pages.get_device(), "kv4_read: slots")
    pages, _, hkv, page, _ = kv_pages.shape
    t = slot.shape[0]
    if not kv_pages.is_cuda:
        return ref.kv4_read(kv_pages, slot, d)
    k = torch.empty(t, hkv, d, dtype=kv_pages.dtype, device=kv_pages.device)
    v = torch.empty_like(k)
    with _guard(kv_pages.device):
        _call("mlcb_kv4_read", kv_pages.data_ptr(), slot.data_ptr(), k.data_ptr(), v.data_ptr(), t, hkv, d, page,
              pages * page, DTYPE_CODE[k.dtype], *_env(k.device))
    return k, v


# --------------------------------------------------------------------------- attention
KV4_TILE_ROWS = 256  # query rows that share one expansion of the cached blocks
KV4_HEAD_DIMS = (64, 96, 128, 256)  # of the tensor-core kernels; other multiples of 32 take the generic one


def kv4_plan(q_indptr, q_kvlen: torch.Tensor, page_indptr: torch.Tensor, page_indices: torch.Tensor, hq: int, hkv: int,
             max_len: int) -> AttentionPlan:
    """The tiling of one step for ``ops.paged_attention`` over a packed cache (shared by all layers). ``q_indptr``:
    host array, first token of every sequence's chunk; ``max_len``: the longest sequence, appended tokens included."""
    q_indptr = np.asarray(q_indptr, dtype=np.int64)
    if hkv <= 0 or hq <= 0 or hq % hkv:
        raise ValueError(f"kv4_plan: {hq} query heads do not divide over {hkv} KV heads")
    if q_indptr.ndim != 1 or len(q_indptr) < 1 or q_indptr[0] != 0 or (np.diff(q_indptr) < 0).any():
        raise ValueError("kv4_plan: q_indptr must rise from 0")
    if q_kvlen.dim() != 1 or q_kvlen.shape[0] < q_indptr[-1]:
        raise ValueError(f"kv4_plan: {int(q_indptr[-1])} tokens, but lengths of {tuple(q_kvlen.shape)}")
    tiles = build_tiles(q_indptr, hq // hkv, tile_rows=KV4_TILE_ROWS)
    dev = q_kvlen.device
    on = {k: torch.from_numpy(a).to(dev) for k, a in tiles.items()}
    num_dec, num_tiles = len(tiles["dec_seq"]), len(tiles["tile_seq"])
    if dev.type == "cuda" and num_tiles * hkv > sm_count(dev):
        # more CTAs than SMs: the longest tiles start first, which is from the end (sequences of 512 to 2048 new tokens
        # behind 0 to 8192 cached ones: 527 us in the order of the batch, 483 us like this)
        order = torch.argsort(q_kvlen[(on["tile_qstart"] + on["tile_ntok"] - 1).long()], stable=True)
        for k in ("tile_seq", "tile_qstart", "tile_ntok"):
            on[k] = on[k][order]
    return AttentionPlan(on["tile_seq"], on["tile_qstart"], on["tile_ntok"], q_kvlen, page_indptr, page_indices,
                         num_tiles, dec_seq=on["dec_seq"], dec_qstart=on["dec_qstart"], dec_ntok=on["dec_ntok"],
                         num_dec=num_dec, dec_splits=1, max_pages=(int(max_len) + 15) // 16, tile_rows=KV4_TILE_ROWS,
                         dec_rows=decode_rows(q_indptr, hq // hkv), tokens=int(q_indptr[-1]), group=hq // hkv,
                         seqs=len(q_indptr) - 1)


def _decode_ctas(num_items: int, hkv: int, max_pages: int, device: torch.device) -> int:
    """CTAs of the decode kernel: no more than one per four 32-token slots, rounded up to a power of two (a captured
    launch serves every length up to the next one), and no more than can be resident."""
    slots = num_items * hkv * max(1, (max_pages + 1) // 2)
    return min(4 * sm_count(device), 1 << max(0, (slots + 3) // 4 - 1).bit_length())


def decode_launch(num_dec: int, hkv: int, d: int, max_pages: int, rows: int, device: torch.device) -> int:
    """What the launch of ``num_dec`` decode items of at most ``rows`` query rows depends on besides array shapes: a
    captured graph holds for equal values of this number."""
    if d not in KV4_HEAD_DIMS:
        return 0
    if d == 96:
        return _prefill_splits(num_dec * hkv, max_pages // 8, device)
    return _decode_ctas(num_dec, hkv, max_pages, device) * 2 + (rows > 8)  # more than 8 rows: another kernel, or two units


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
    if plan is not None and plan.group and (plan.tokens != t or plan.group != hq // hkv):
        raise ValueError(f"paged_attention: the plan is for {plan.tokens} tokens and {plan.group} query heads per KV head, "
                         f"the call has {t} and {hq // hkv}")
    where = q.get_device()
    if plan is not None and ((plan.num_dec and plan.dec_seq.device != q.device)
                             or (plan.num_tiles and plan.tile_seq.device != q.device)):
        raise ValueError(f"paged_attention: q is on {q.device}, the plan's items are not")
    _check_index(q_seq, t, where, "paged_attention: q_seq")
    _check_index(q_kvlen, t, where, "paged_attention: q_kvlen")
    _check_index(q_kvstart, t, where, "paged_attention: q_kvstart")
    seqs = plan.seqs if plan is not None else 0
    _check_index(page_indptr, max(seqs, 1) + 1 if t else 0, where, "paged_attention: page_indptr")
    _check_index(page_indices, 0, where, "paged_attention: page_indices")
    _check_index(tree_mask, t, where, "paged_attention: tree_mask", torch.int64)
    if not q.is_cuda:
        res = ref.paged_attention(q.reshape(t, hq, d), kv_pages, q_seq, q_kvlen, page_indptr, page_indices, hq, hkv, d,
                                  page, sm_scale, q_kvstart, sink, tree_mask, softcap, return_lse)
        return (res[0].reshape(t, hq * d), res[1]) if return_lse else res.reshape(t, hq * d)
    out = torch.empty(t, hq * d, dtype=q.dtype, device=q.device)
    lse = torch.empty(t, hq, dtype=torch.float32, device=q.device) if return_lse else None
    with _guard(q.device):
        _launch(q, kv_pages, out, lse, q_seq, q_kvlen, page_indptr, page_indices, hq, hkv, d, page, sm_scale, q_kvstart,
                max(0, min(int(sink), 1 << 30)), tree_mask, float(softcap), plan)  # room for rounding up to whole blocks
    return (out, lse) if return_lse else out


def _decode(q, q_stride, kv_pages, out, lse, q_kvlen, page_indptr, page_indices, hq, hkv, d, sm_scale, q_kvstart, sink, tree_mask,
            softcap, plan) -> None:
    # with one token per item the rows are the group's heads, whatever the plan was made for
    rows = hq // hkv if q.shape[0] == plan.num_dec else min(16, plan.dec_rows)
    ctas = _decode_ctas(plan.num_dec, hkv, plan.max_pages, q.device)
    # per CTA: a unit descriptor, (max, sum) of two pieces of 16 rows, and their rows
    scratch = torch.empty(ctas * (2 * 16 * (d + 2) + 4), dtype=torch.float32, device=q.device)
    part = scratch.data_ptr()
    _call("mlcb_kv4_decode", q.data_ptr(), kv_pages.data_ptr(), out.data_ptr(), _at(lse), plan.dec_seq.data_ptr(),
          plan.dec_qstart.data_ptr(), plan.dec_ntok.data_ptr(), q_kvlen.data_ptr(), page_indptr.data_ptr(),
          page_indices.data_ptr(), plan.num_dec, rows, q_stride, hq, hkv, d, kv_pages.shape[0], sm_scale,
          DTYPE_CODE[q.dtype], ctas, part + ctas * 272, part + ctas * 16, part, *_env(q.device), _at(q_kvstart),
          _at(tree_mask), sink, softcap)


def _prefill_splits(ctas: int, blocks: int, device: torch.device) -> int:
    """KV splits of the prefill kernel (one CTA per SM): few tiles are cut so that they cover the SMs, two blocks of
    cached positions per split at least; a power of two, as in :func:`_decode_ctas`."""
    most = max(1, min(sm_count(device) // max(1, ctas), blocks // 2, 64))
    return 1 << (most.bit_length() - 1)


def _prefill(q, q_stride, kv_pages, out, lse, q_kvlen, page_indptr, page_indices, hq, hkv, d, sm_scale, q_kvstart, sink, tree_mask,
             softcap, plan, decode_items: bool) -> None:
    if decode_items:
        seq, qstart, ntok, num, rows = plan.dec_seq, plan.dec_qstart, plan.dec_ntok, plan.num_dec, min(16, plan.dec_rows)
    else:
        seq, qstart, ntok, num, rows = plan.tile_seq, plan.tile_qstart, plan.tile_ntok, plan.num_tiles, plan.tile_rows
    ctas = num * hkv * (2 if d == 256 and rows > 128 else 1)
    splits = _prefill_splits(ctas, plan.max_pages // (4 if d == 256 else 8), q.device)
    part_o = part_ml = None
    if splits > 1:  # 256 rows and their (max, sum) per (tile, kv head, split)
        blocks = num * hkv * splits
        scratch = torch.empty(blocks * 256 * (d + 2), dtype=torch.float32, device=q.device)
        part_ml = scratch.data_ptr()
        part_o = part_ml + blocks * 2048
    _call("mlcb_kv4_prefill", q.data_ptr(), kv_pages.data_ptr(), out.data_ptr(), _at(lse), seq.data_ptr(), qstart.data_ptr(),
          ntok.data_ptr(), q_kvlen.data_ptr(), page_indptr.data_ptr(), page_indices.data_ptr(), num, rows, q_stride, hq,
          hkv, d, kv_pages.shape[0], sm_scale, DTYPE_CODE[q.dtype], splits, part_o, part_ml, *_env(q.device),
          _at(q_kvstart), _at(tree_mask), sink, softcap)


def _launch(q, kv_pages, out, lse, q_seq, q_kvlen, page_indptr, page_indices, hq, hkv, d, page, sm_scale, q_kvstart, sink,
            tree_mask, softcap, plan) -> None:
    t = q.shape[0]
    q_stride = q.stride(0) if t > 1 else hq * d  # of a single row nothing is read behind it, however wide its buffer
    aligned = (q.data_ptr() | kv_pages.data_ptr()) % 16 == 0 and q_stride % 8 == 0
    if plan is not None and plan.use_tensor_core and page == 16 and d in KV4_HEAD_DIMS and aligned \
            and hq // hkv <= plan.tile_rows:
        args = (q, q_stride, kv_pages, out, lse, q_kvlen, page_indptr, page_indices, hq, hkv, d, sm_scale, q_kvstart, sink,
                tree_mask, softcap, plan)
        if plan.num_dec:
            if d == 96:  # no decode kernel: its lanes own powers of two of channels
                _prefill(*args, decode_items=True)
            else:
                _decode(*args)
        if plan.num_tiles:
            _prefill(*args, decode_items=False)
        return
    _call("mlcb_kv4_attn_simt", q.data_ptr(), kv_pages.data_ptr(), out.data_ptr(), _at(lse), q_seq.data_ptr(),
          q_kvlen.data_ptr(), _at(q_kvstart), _at(tree_mask), page_indptr.data_ptr(), page_indices.data_ptr(), t, q_stride,
          hq, hkv, d, page, kv_pages.shape[0], sink, sm_scale, softcap, DTYPE_CODE[q.dtype], *_env(q.device))


__all__ = ["KV4_BOUND", "KV4_GROUP", "is_kv4", "kv4_cache", "kv4_plan", "kv4_read", "kv4_row"]
