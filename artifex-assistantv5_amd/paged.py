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
from .kv4 import _launch

BLOCK = 16
PAGES = (16, 32, 64, 128, 256)
_DTYPES = {torch.float16: _native.PAGED_F16, torch.bfloat16: _native.PAGED_BF16}


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


def _shape(kv: torch.Tensor, layers: bool = False):
    """(layers, pages, KV heads, page, head_dim) of a pool."""
    if kv.dtype not in _DTYPES or not kv.is_cuda or not kv.is_contiguous():
        raise ValueError("paged: the pool must be a contiguous float16 or bfloat16 device tensor")
    s = kv.shape
    if len(s) == 6 and layers:
        n_layers, s = s[0], s[1:]
    elif len(s) == 5:
        n_layers = 1
    else:
        raise ValueError(f"paged: pool of shape {tuple(kv.shape)}, need [{'layers, ' if layers else ''}"
                         "n_pages, 2, n_kv_heads, page, head_dim]")
    if s[1] != 2 or 0 in kv.shape:
        raise ValueError(f"paged: pool of shape {tuple(kv.shape)} is not [.., n_pages, 2, ..]")
    return n_layers, s[0], s[2], s[3], s[4]


def _tensor(name: str, t: torch.Tensor, dtype, shape, device) -> int:
    if t.dtype != dtype or t.device != device or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"paged: {name} must be a contiguous {dtype} tensor {tuple(shape)} on "
                         f"{device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _tables(tables: torch.Tensor, device):
    if tables.dim() != 2:
        raise ValueError("paged: tables must be [n_seq, columns]")
    n_seq, columns = tables.shape
    return n_seq, columns, _tensor("tables", tables, torch.int32, (n_seq, columns), device)


def _row_matrix(name: str, t: torch.Tensor, width: int, device) -> int:
    """The row stride of f32 rows of at least ``width`` values (unit column stride)."""
    if t.dtype != torch.float32 or t.device != device or t.dim() != 2 or t.shape[1] < width:
        raise ValueError(f"paged: {name} must be float32 rows of at least {width} values on {device}")
    n, columns = t.shape
    ld, step = t.stride()
    if n <= 1:
        ld = columns
    if step != 1 or ld < columns:
        raise ValueError(f"paged: {name} must be rows with unit column stride")
    return ld


def _rows(qkv, lengths, tables, cos, sin, kv, n_heads, room):
    """The checks that append and attention share, and their arguments."""
    _, n_pages, n_kv, page, hd = _shape(kv)
    dev = kv.device
    ld = _row_matrix("qkv", qkv, (n_heads + 2 * n_kv) * hd, dev)
    n_seq, columns, tp = _tables(tables, dev)
    if cos.dim() != 2:
        raise ValueError("paged: cos and sin must be [positions, head_dim / 2]")
    rope = (cos.shape[0], hd // 2)
    return (n_seq, columns, n_pages, n_kv, page, hd, ld, tp,
            _tensor("lengths", lengths, torch.int64, (n_seq,), dev),
            None if room is None else _tensor("room", room, torch.int64, (n_seq,), dev),
            _tensor("cos", cos, torch.float32, rope, dev),
            _tensor("sin", sin, torch.float32, rope, dev))


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
    n_seq, columns, n_pages, n_kv, page, hd, ld, tp, lp, mp, cp, sp = _rows(
        qkv, lengths, tables, cos, sin, kv, n_heads, room)
    st = None if starts is None else _tensor("starts", starts, torch.int64, (n_seq + 1,), kv.device)
    _launch(_native.load_library().gguf_hip_paged_append, kv.device, qkv.data_ptr(), ld,
            qkv.shape[0], st, lp, mp, tp, cp, sp, cos.shape[0], kv.data_ptr(), _DTYPES[kv.dtype],
            n_pages, page, columns, n_seq, n_heads, n_kv, hd)
    return kv


def attention_workspace(kv: torch.Tensor, tables: torch.Tensor, n_heads: int) -> torch.Tensor:
    """Device workspace of ``attention`` calls over such tables."""
    _, _, n_kv, page, hd = _shape(kv)
    n_seq, columns, _ = _tables(tables, kv.device)
    lib = _native.load_library()
    n = _native.check(lib.gguf_hip_paged_attention_workspace(page, columns, n_seq, n_heads, n_kv, hd),
                      lib)
    return torch.empty(n, dtype=torch.uint8, device=kv.device)


def _work(work: torch.Tensor, device):
    if work.device != device or not work.is_contiguous():
        raise ValueError("paged: the workspace must be a contiguous tensor on the pool's device")
    return work.data_ptr(), work.numel() * work.element_size()


def attention(qkv: torch.Tensor, lengths: torch.Tensor, tables: torch.Tensor, cos: torch.Tensor,
              sin: torch.Tensor, kv: torch.Tensor, out: torch.Tensor, n_heads: int,
              work: torch.Tensor, room: Optional[torch.Tensor] = None) -> torch.Tensor:
    """RoPE, storing and GQA attention of one new row ``[q | k | v]`` of every sequence.

    Row s is stored in slot ``lengths[s]`` and attends to slots ``0 .. lengths[s]``, of which those
    without a page are not seen.  A sequence whose row cannot be stored (negative length, no page,
    past the tables or ``room[s]``) takes no part: nothing of it is written."""
    n_seq, columns, n_pages, n_kv, page, hd, ld, tp, lp, mp, cp, sp = _rows(
        qkv, lengths, tables, cos, sin, kv, n_heads, room)
    ldo = _row_matrix("out", out, n_heads * hd, kv.device)
    if qkv.shape[0] != n_seq or out.shape[0] != n_seq:
        raise ValueError(f"paged: qkv has {qkv.shape[0]} rows and out {out.shape[0]} for {n_seq} "
                         "sequences")
    wp, wb = _work(work, kv.device)
    _launch(_native.load_library().gguf_hip_paged_attention, kv.device, qkv.data_ptr(), ld, lp, mp,
            tp, cp, sp, cos.shape[0], kv.data_ptr(), _DTYPES[kv.dtype], out.data_ptr(), ldo, n_pages,
            page, columns, n_seq, n_heads, n_kv, hd, wp, wb)
    return out


def load(kv: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor, k_out: torch.Tensor,
         v_out: torch.Tensor) -> None:
    """One layer's cached rows in f32: slots ``0 .. lengths[s] - 1`` (at most ``out_slots``) into
    ``k_out`` / ``v_out`` ``[n_seq, n_kv_heads, out_slots, head_dim]``.  Rows from ``lengths[s]`` on,
    and of slots without a page, are not written.  For one sequence this is the layout of
    ``glue.attention_prefill``'s caches.  One launch."""
    _, n_pages, n_kv, page, hd = _shape(kv)
    n_seq, columns, tp = _tables(tables, kv.device)
    shape = (n_seq, n_kv, k_out.shape[-2] if k_out.dim() > 1 else 0, hd)
    kp = _tensor("k_out", k_out, torch.float32, shape, kv.device)
    vp = _tensor("v_out", v_out, torch.float32, shape, kv.device)
    lp = _tensor("lengths", lengths, torch.int64, (n_seq,), kv.device)
    _launch(_native.load_library().gguf_hip_paged_load, kv.device, kv.data_ptr(), _DTYPES[kv.dtype],
            tp, lp, kp, vp, shape[2], n_pages, page, columns, n_seq, n_kv, hd)


def _refs(refs: torch.Tensor, device) -> int:
    if refs.dim() != 1:
        raise ValueError("paged: refs must be [n_pages]")
    return _tensor("refs", refs, torch.int32, refs.shape, device)


def fork(tables: torch.Tensor, lengths: torch.Tensor, refs: torch.Tensor, parents: torch.Tensor,
         tables_out: Optional[torch.Tensor] = None, lengths_out: Optional[torch.Tensor] = None,
         refs_out: Optional[torch.Tensor] = None) -> None:
    """Sequence ``s`` becomes a fork of sequence ``parents[s]`` (device int64) as that was before
    the call: it gets the parent's length and shares its pages.  ``parents[s] == s`` leaves it as
    it is, a parent outside the sequences (-1) frees it.  In place, or into the ``*_out`` tensors,
    which must not overlap the inputs.  No page is copied: ``grow`` does that before a shared one
    is written.  One launch, or two where ``refs_out`` is another tensor and large."""
    dev = tables.device
    tables_out = tables if tables_out is None else tables_out
    lengths_out = lengths if lengths_out is None else lengths_out
    refs_out = refs if refs_out is None else refs_out
    if not tables.is_cuda:
        raise ValueError("paged: tables must be a device tensor")
    n_seq, columns, tp = _tables(tables, dev)
    lp = _tensor("lengths", lengths, torch.int64, (n_seq,), dev)
    rp = _refs(refs, dev)
    pp = _tensor("parents", parents, torch.int64, (n_seq,), dev)
    to = _tensor("tables_out", tables_out, torch.int32, tables.shape, dev)
    lo = _tensor("lengths_out", lengths_out, torch.int64, (n_seq,), dev)
    ro = _tensor("refs_out", refs_out, torch.int32, refs.shape, dev)
    _launch(_native.load_library().gguf_hip_paged_fork, dev, tp, lp, rp, pp, to, lo, ro,
            refs.shape[0], columns, n_seq)


def grow_workspace(kv: torch.Tensor, tables: torch.Tensor) -> torch.Tensor:
    """Device workspace of ``grow`` calls over such a pool and tables."""
    _, n_pages, _, page, _ = _shape(kv, layers=True)
    n_seq, columns, _ = _tables(tables, kv.device)
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
    n_layers, n_pages, n_kv, page, hd = _shape(kv, layers=True)
    dev = kv.device
    n_seq, columns, tp = _tables(tables, dev)
    lp = _tensor("lengths", lengths, torch.int64, (n_seq,), dev)
    rp = _tensor("refs", refs, torch.int32, (n_pages,), dev)
    np_ = _tensor("rows", rows, torch.int64, (n_seq,), dev)
    mp = _tensor("room", room, torch.int64, (n_seq,), dev)
    wp, wb = _work(work, dev)
    _launch(_native.load_library().gguf_hip_paged_grow, dev, kv.data_ptr(), tp, lp, rp, np_, mp,
            n_layers, n_pages, page, columns, n_seq, n_kv, hd, wp, wb)


def compact_workspace(kv: torch.Tensor, tables: torch.Tensor) -> torch.Tensor:
    """Device workspace of ``compact`` calls over such a pool and tables."""
    _, n_pages, _, _, _ = _shape(kv, layers=True)
    n_seq, columns, _ = _tables(tables, kv.device)
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
    n_layers, n_pages, n_kv, page, hd = _shape(kv, layers=True)
    dev = kv.device
    tables_out = tables if tables_out is None else tables_out
    refs_out = refs if refs_out is None else refs_out
    n_seq, columns, tp = _tables(tables, dev)
    rp = _tensor("refs", refs, torch.int32, (n_pages,), dev)
    lp = _tensor("live", live, torch.int64, (1,), dev)
    to = _tensor("tables_out", tables_out, torch.int32, tables.shape, dev)
    ro = _tensor("refs_out", refs_out, torch.int32, refs.shape, dev)
    wp, wb = _work(work, dev)
    _launch(_native.load_library().gguf_hip_paged_compact, dev, kv.data_ptr(), tp, rp, to, ro, lp,
            n_layers, n_pages, page, columns, n_seq, n_kv, hd, wp, wb)
