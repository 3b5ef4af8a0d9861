"""The KV cache in pages: storing rows, attention over it, forks, room, compaction (libgguf_hip).

The reference attends over one cache per sequence (attention.wgsl:60-234).  Here the caches of a
batch are pages of 16 to 256 slots, in f16 or bf16, that a table per sequence names, so that
sequences may share the pages of a common beginning and a pool holds what its sequences use.

One layer's pool is a tensor ``[n_pages, 2, n_kv_heads, page, head_dim]`` (``empty``; the order of
V's values is in include/gguf_hip_paged.h), all layers' ``[n_layers, ...]``; a page number means
that page of every layer.  Sequence ``s`` has ``lengths[s]`` slots in use (device int64), slot t in
page ``tables[s, t // page]`` (device int32, -1: none) at RoPE position t.  ``refs`` (device int32
``[n_pages]``) counts the table entries that hold a page; 0 is a free page.

    fork     sequences become forks of others, or are freed
    grow     pages for new rows: free ones, and copies where others hold the page too
    append   rows of prompts into their pages
    attention  one new row per sequence stored, and its attention
    load     cached rows in f32
    compact  the pages in use moved to the front of the pool

As in ``glue``, every buffer is checked against the launch before the C ABI sees it, calls run on
the current HIP stream, and none allocates or synchronises, so all can be captured in a graph.  A
workspace serves calls of its own shape that do not overlap.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _native

BLOCK = 16
PAGES = (16, 32, 64, 128, 256)
_DTYPES = {torch.float16: _native.PAGED_F16, torch.bfloat16: _native.PAGED_BF16}
_call, _direct = _native.call, _native.direct


def pool_bytes(n_pages: int, n_kv_heads: int, head_dim: int, page: int = 16) -> int:
    """Bytes of one layer's pool; ValueError for a shape that there is no pool of."""
    lib = _native.load_library()
    return _native.check(lib.gguf_hip_paged_bytes(n_pages, page, n_kv_heads, head_dim), lib)


def empty(n_pages: int, n_kv_heads: int, head_dim: int, page: int = 16, dtype=torch.float16,
          device="cuda", n_layers: Optional[int] = None) -> torch.Tensor:
    """A pool of one layer, or ``[n_layers, ...]`` of several, every value zero."""
    pool_bytes(n_pages, n_kv_heads, head_dim, page)
    if dtype not in _DTYPES:
        raise ValueError(f"paged: pages are float16 or bfloat16, not {dtype}")
    shape = (n_pages, 2, n_kv_heads, page, head_dim)
    return torch.zeros(shape if n_layers is None else (n_layers, *shape), dtype=dtype, device=device)


def empty_tables(n_seq: int, columns: int, n_pages: int, device="cuda"):
    """``tables``, ``lengths`` and ``refs`` of ``n_seq`` sequences without pages."""
    return (torch.full((n_seq, columns), -1, dtype=torch.int32, device=device),
            torch.zeros(n_seq, dtype=torch.int64, device=device),
            torch.zeros(n_pages, dtype=torch.int32, device=device))


def _pool(kv: torch.Tensor, layers: bool = False):
    """(device index, layers, pages, KV heads, page, head_dim) of a pool."""
    shape = kv.shape
    n_layers = 1
    if layers and len(shape) == 6:
        n_layers, *shape = shape
    device = kv.get_device()
    if len(shape) != 5 or device < 0 or kv.dtype not in _DTYPES or not kv.is_contiguous():
        raise ValueError(f"paged: pool {kv.dtype} {tuple(kv.shape)} on {kv.device}, need a contiguous "
                         f"float16 or bfloat16 device tensor [{'layers, ' if layers else ''}n_pages, "
                         "2, n_kv_heads, page, head_dim]")
    n_pages, two, n_kv, page, hd = shape
    if two != 2 or not (n_layers and n_pages and n_kv and page and hd):
        raise ValueError(f"paged: pool of shape {tuple(kv.shape)} is not [.., n_pages, 2, ..]")
    return device, n_layers, n_pages, n_kv, page, hd


# The calls below are made straight from the tensors where these fit (``_native.direct``, which raises
# if a call fails); what follows there says what does not fit, and makes those calls whose device is
# not the current one.
def _array(name: str, t: torch.Tensor, dtype, shape, device: int) -> int:
    if (t.dtype is dtype and t.shape == shape and t.is_contiguous() and t.get_device() == device):
        return t.data_ptr()
    raise ValueError(f"paged: {name} must be a contiguous {dtype} tensor {tuple(shape)} on device "
                     f"{device}, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _tables(tables: torch.Tensor, device: int):
    if tables.dim() != 2:
        raise ValueError("paged: tables must be [n_seq, columns]")
    shape = tables.shape
    return *shape, _array("tables", tables, torch.int32, shape, device)


def _row_matrix(name: str, t: torch.Tensor, rows: int, width: int, device: int):
    """The address and row stride of ``rows`` f32 rows of at least ``width`` values (any number of
    them: -1)."""
    if t.dtype is torch.float32 and t.dim() == 2 and t.get_device() == device:
        n, columns = t.shape
        ld, step = t.stride()
        if n <= 1:
            ld = columns
        if columns >= width and step == 1 and ld >= columns and (n == rows or rows < 0):
            return t.data_ptr(), ld
    raise ValueError(f"paged: {name} must be {rows if rows >= 0 else ''} float32 rows of at least "
                     f"{width} values with unit column stride on device {device}, got {t.dtype} "
                     f"{tuple(t.shape)} with strides {t.stride()} on {t.device}")


def _rope(cos: torch.Tensor, sin: torch.Tensor, hd: int, device: int):
    if cos.dim() != 2:
        raise ValueError("paged: cos and sin must be [positions, head_dim / 2]")
    shape = (len(cos), hd // 2)
    return (_array("cos", cos, torch.float32, shape, device),
            _array("sin", sin, torch.float32, shape, device), shape[0])


def _work(work: torch.Tensor, device: int):
    if work.get_device() != device or not work.is_contiguous():
        raise ValueError("paged: the workspace must be a contiguous tensor on the pool's device")
    return work.data_ptr(), work.nbytes


def append(qkv: torch.Tensor, lengths: torch.Tensor, tables: torch.Tensor, cos: torch.Tensor,
           sin: torch.Tensor, kv: torch.Tensor, n_heads: int,
           starts: Optional[torch.Tensor] = None,
           room: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Store the K (after RoPE) and V of rows ``[q | k | v]`` behind what the sequences hold.

    Sequence ``s`` owns rows ``starts[s] .. starts[s + 1] - 1`` of ``qkv`` (device int64
    ``[n_seq + 1]``; without it every sequence has the same number of rows, in order).  Its row i
    goes to slot ``lengths[s] + i``; rows outside every sequence, without a page, past the tables
    or ``room[s]`` (``grow``) are not stored, nor those of a sequence of negative length.
    ``lengths`` is the caller's to advance.  One launch."""
    if _direct().append(qkv, lengths, tables, cos, sin, kv, n_heads, starts, room):
        return kv
    dev, _, n_pages, n_kv, page, hd = _pool(kv)
    qp, ld = _row_matrix("qkv", qkv, -1, (n_heads + 2 * n_kv) * hd, dev)
    n_seq, columns, tp = _tables(tables, dev)
    lp = _array("lengths", lengths, torch.int64, (n_seq,), dev)
    mp = 0 if room is None else _array("room", room, torch.int64, (n_seq,), dev)
    st = 0 if starts is None else _array("starts", starts, torch.int64, (n_seq + 1,), dev)
    _call(_native.PAGED_APPEND, dev, qp, ld, len(qkv), st, lp, mp, tp, *_rope(cos, sin, hd, dev),
          kv.data_ptr(), _DTYPES[kv.dtype], n_pages, page, columns, n_seq, n_heads, n_kv, hd)
    return kv


def attention_workspace(kv: torch.Tensor, tables: torch.Tensor, n_heads: int) -> torch.Tensor:
    """Device workspace of ``attention`` calls over such tables."""
    dev, _, _, n_kv, page, hd = _pool(kv)
    n_seq, columns, _ = _tables(tables, dev)
    lib = _native.load_library()
    n = _native.check(lib.gguf_hip_paged_attention_workspace(page, columns, n_seq, n_heads, n_kv, hd),
                      lib)
    return torch.empty(n, dtype=torch.uint8, device=kv.device)


def attention(qkv: torch.Tensor, lengths: torch.Tensor, tables: torch.Tensor, cos: torch.Tensor,
              sin: torch.Tensor, kv: torch.Tensor, out: torch.Tensor, n_heads: int,
              work: torch.Tensor, room: Optional[torch.Tensor] = None) -> torch.Tensor:
    """RoPE, storing and GQA attention of one new row ``[q | k | v]`` of every sequence.

    Row s is stored in slot ``lengths[s]`` and attends to slots ``0 .. lengths[s]``, of which those
    without a page are not seen.  A sequence whose row cannot be stored (negative length, no page,
    past the tables or ``room[s]``) takes no part: nothing of it is written."""
    if _direct().attention(qkv, lengths, tables, cos, sin, kv, out, n_heads, work, room):
        return out
    dev, _, n_pages, n_kv, page, hd = _pool(kv)
    n_seq, columns, tp = _tables(tables, dev)
    qp, ld = _row_matrix("qkv", qkv, n_seq, (n_heads + 2 * n_kv) * hd, dev)
    op, ldo = _row_matrix("out", out, n_seq, n_heads * hd, dev)
    lp = _array("lengths", lengths, torch.int64, (n_seq,), dev)
    mp = 0 if room is None else _array("room", room, torch.int64, (n_seq,), dev)
    _call(_native.PAGED_ATTENTION, dev, qp, ld, lp, mp, tp, *_rope(cos, sin, hd, dev), kv.data_ptr(),
          _DTYPES[kv.dtype], op, ldo, n_pages, page, columns, n_seq, n_heads, n_kv, hd,
          *_work(work, dev))
    return out


def load(kv: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor, k_out: torch.Tensor,
         v_out: torch.Tensor) -> None:
    """One layer's cached rows in f32: slots ``0 .. lengths[s] - 1`` (at most ``out_slots``) into
    ``k_out`` / ``v_out`` ``[n_seq, n_kv_heads, out_slots, head_dim]``.  Rows from ``lengths[s]`` on,
    and of slots without a page, are not written.  For one sequence this is the layout of
    ``glue.attention_prefill``'s caches.  One launch."""
    if _direct().load(kv, tables, lengths, k_out, v_out):
        return
    dev, _, n_pages, n_kv, page, hd = _pool(kv)
    n_seq, columns, tp = _tables(tables, dev)
    shape = (n_seq, n_kv, k_out.shape[-2] if k_out.dim() > 1 else 0, hd)
    kp = _array("k_out", k_out, torch.float32, shape, dev)
    vp = _array("v_out", v_out, torch.float32, shape, dev)
    lp = _array("lengths", lengths, torch.int64, (n_seq,), dev)
    _call(_native.PAGED_LOAD, dev, kv.data_ptr(), _DTYPES[kv.dtype], tp, lp, kp, vp, shape[2],
          n_pages, page, columns, n_seq, n_kv, hd)


def fork(tables: torch.Tensor, lengths: torch.Tensor, refs: torch.Tensor, parents: torch.Tensor,
         tables_out: Optional[torch.Tensor] = None, lengths_out: Optional[torch.Tensor] = None,
         refs_out: Optional[torch.Tensor] = None) -> None:
    """Sequence ``s`` becomes a fork of sequence ``parents[s]`` (device int64) as that was before
    the call: it gets the parent's length and shares its pages.  ``parents[s] == s`` leaves it as
    it is, a parent outside the sequences (-1) frees it.  In place, or into the ``*_out`` tensors,
    which must not overlap the inputs.  No page is copied: ``grow`` does that before a shared one
    is written.  One launch, or two where ``refs_out`` is another tensor and large."""
    if _direct().fork(tables, lengths, refs, parents, tables_out, lengths_out, refs_out):
        return
    dev = tables.get_device()
    if dev < 0 or refs.dim() != 1:
        raise ValueError("paged: tables must be a device tensor, refs [n_pages]")
    n_seq, columns, tp = _tables(tables, dev)
    n, pages = (n_seq,), refs.shape
    lp = _array("lengths", lengths, torch.int64, n, dev)
    rp = _array("refs", refs, torch.int32, pages, dev)
    pp = _array("parents", parents, torch.int64, n, dev)
    to = tp if tables_out is None else _array("tables_out", tables_out, torch.int32, tables.shape, dev)
    lo = lp if lengths_out is None else _array("lengths_out", lengths_out, torch.int64, n, dev)
    ro = rp if refs_out is None else _array("refs_out", refs_out, torch.int32, pages, dev)
    _call(_native.PAGED_FORK, dev, tp, lp, rp, pp, to, lo, ro, pages[0], columns, n_seq)


def grow_workspace(kv: torch.Tensor, tables: torch.Tensor) -> torch.Tensor:
    """Device workspace of ``grow`` calls over such a pool and tables."""
    dev, _, n_pages, _, page, _ = _pool(kv, layers=True)
    n_seq, columns, _ = _tables(tables, dev)
    lib = _native.load_library()
    n = _native.check(lib.gguf_hip_paged_grow_workspace(n_pages, page, columns, n_seq), lib)
    return torch.empty(n, dtype=torch.uint8, device=kv.device)


def grow(kv: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor, refs: torch.Tensor,
         rows: torch.Tensor, room: torch.Tensor, work: torch.Tensor) -> None:
    """Pages for ``rows[s]`` (device int64) more rows of each sequence, in all layers of ``kv``.

    The columns of slots ``lengths[s] .. lengths[s] + rows[s] - 1`` (as far as the table goes) get
    the lowest free pages, sequences in order: those that have none, and those whose page other
    entries hold too, into whose new page the blocks of 16 slots in use are copied.  ``room[s]``
    becomes the end of the slots that the sequence may write, ``lengths[s]`` at least: less than
    was asked for where the pool has no free page left.  Two launches."""
    if _direct().grow(kv, tables, lengths, refs, rows, room, work):
        return
    dev, n_layers, n_pages, n_kv, page, hd = _pool(kv, layers=True)
    n_seq, columns, tp = _tables(tables, dev)
    n = (n_seq,)
    lp = _array("lengths", lengths, torch.int64, n, dev)
    rp = _array("refs", refs, torch.int32, (n_pages,), dev)
    np_ = _array("rows", rows, torch.int64, n, dev)
    mp = _array("room", room, torch.int64, n, dev)
    _call(_native.PAGED_GROW, dev, kv.data_ptr(), tp, lp, rp, np_, mp, n_layers, n_pages, page,
          columns, n_seq, n_kv, hd, *_work(work, dev))


def compact_workspace(kv: torch.Tensor, tables: torch.Tensor) -> torch.Tensor:
    """Device workspace of ``compact`` calls over such a pool and tables."""
    dev, _, n_pages, _, _, _ = _pool(kv, layers=True)
    n_seq, columns, _ = _tables(tables, dev)
    lib = _native.load_library()
    n = _native.check(lib.gguf_hip_paged_compact_workspace(n_pages, columns, n_seq), lib)
    return torch.empty(n, dtype=torch.uint8, device=kv.device)


def compact(kv: torch.Tensor, tables: torch.Tensor, refs: torch.Tensor, live: torch.Tensor,
            work: torch.Tensor, tables_out: Optional[torch.Tensor] = None,
            refs_out: Optional[torch.Tensor] = None) -> None:
    """Move the pages in use of all layers into the first ``live[0]`` (device int64 ``[1]``, set
    here) of the pool: those behind them, in order, into the free ones among them, in order.
    ``tables`` and ``refs`` follow, in place or into the ``*_out`` tensors, which must not overlap
    the inputs.  Two launches."""
    if _direct().compact(kv, tables, refs, live, work, tables_out, refs_out):
        return
    dev, n_layers, n_pages, n_kv, page, hd = _pool(kv, layers=True)
    n_seq, columns, tp = _tables(tables, dev)
    pages = (n_pages,)
    rp = _array("refs", refs, torch.int32, pages, dev)
    lp = _array("live", live, torch.int64, (1,), dev)
    to = tp if tables_out is None else _array("tables_out", tables_out, torch.int32, tables.shape, dev)
    ro = rp if refs_out is None else _array("refs_out", refs_out, torch.int32, pages, dev)
    _call(_native.PAGED_COMPACT, dev, kv.data_ptr(), tp, rp, to, ro, lp, n_layers, n_pages, page,
          columns, n_seq, n_kv, hd, *_work(work, dev))
