"""The KV cache held in 4 bits: storing rows, attention over it, eviction (libgguf_hip).

The reference attends over f32 caches (attention.wgsl:60-234) and compresses its cache by
other codes (webgpu/src/engine/turboquant-pipeline.ts).  This cache holds Q4_0 blocks of 32
channels, the values of this package's own Q4_0 quantizer: 4.5 bits a value, so a token
costs 9/64 of the bytes that it costs in f32.

One layer's cache is a uint8 tensor ``[n_seq, n_kv_heads, slots / 32, 36 * head_dim]``
(``empty``; the byte order is in include/gguf_hip_kv4.h).  Sequence ``s`` uses its first
``lengths[s]`` slots, and its next token stands at RoPE position ``pos[s]`` (device int64
``[n_seq]`` both; no call but ``evict`` changes them).  ``positions`` (int32) and ``weights``
(f32), ``[n_seq, n_kv_heads, slots]``, hold each slot's position and attention weight.

As in ``glue``, every buffer is checked against the launch before the C ABI sees it, calls
run on the current HIP stream, and none allocates or synchronises, so all can be captured in
a graph.  A workspace serves calls of its own shape that do not overlap.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _native
from .linear import _stream

TILE = _native.KV4_TILE
MAX_ROWS = _native.KV4_MAX_ROWS


def cache_bytes(n_seq: int, n_kv_heads: int, head_dim: int, slots: int) -> int:
    """Bytes of one layer's cache; ValueError for a shape that there is no cache of."""
    lib = _native.load_library()
    return _native.check(lib.gguf_hip_kv4_bytes(n_seq, n_kv_heads, head_dim, slots), lib)


def empty(n_seq: int, n_kv_heads: int, head_dim: int, slots: int, device="cuda",
          n_layers: Optional[int] = None) -> torch.Tensor:
    """A cache of one layer, or ``[n_layers, ...]`` of several, every value zero."""
    cache_bytes(n_seq, n_kv_heads, head_dim, slots)
    shape = (n_seq, n_kv_heads, slots // TILE, 36 * head_dim)
    return torch.zeros(shape if n_layers is None else (n_layers, *shape), dtype=torch.uint8,
                       device=device)


def _shape(kv: torch.Tensor, layers: bool = False):
    """(layers, sequences, KV heads, head_dim, slots) of a cache."""
    if kv.dtype != torch.uint8 or not kv.is_cuda or not kv.is_contiguous():
        raise ValueError("kv4: the cache must be a contiguous uint8 device tensor")
    s = kv.shape
    if len(s) == 5 and layers:
        n_layers, s = s[0], s[1:]
    elif len(s) == 4:
        n_layers = 1
    else:
        raise ValueError(f"kv4: cache of shape {tuple(kv.shape)}, need [{'layers, ' if layers else ''}"
                         "n_seq, n_kv_heads, slots / 32, 36 * head_dim]")
    if 0 in s or s[3] % 36:
        raise ValueError(f"kv4: cache tiles of {s[3]} bytes are not 36 * head_dim")
    return n_layers, s[0], s[1], s[3] // 36, s[2] * TILE


def _tensor(name: str, t: torch.Tensor, dtype, shape, device) -> int:
    if t.dtype != dtype or t.device != device or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"kv4: {name} must be a contiguous {dtype} tensor {tuple(shape)} on "
                         f"{device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _row_matrix(name: str, t: torch.Tensor, width: int, device) -> int:
    """The row stride of f32 rows of at least ``width`` values (unit column stride)."""
    if t.dtype != torch.float32 or t.device != device or t.dim() != 2:
        raise ValueError(f"kv4: {name} must be float32 rows of at least {width} values on {device}")
    n, columns = t.shape
    if columns < width:
        raise ValueError(f"kv4: {name} must be float32 rows of at least {width} values on {device}")
    ld, step = t.stride()
    if n <= 1:
        ld = columns
    if step != 1 or ld < columns:
        raise ValueError(f"kv4: {name} must be rows with unit column stride")
    return ld


def _common(qkv, lengths, pos, cos, sin, kv, n_heads, positions, weights):
    """The checks that append and attention share, and their leading arguments."""
    _, n_seq, n_kv, hd, slots = _shape(kv)
    dev = kv.device
    ld = _row_matrix("qkv", qkv, (n_heads + 2 * n_kv) * hd, dev)
    if cos.dim() != 2:
        raise ValueError("kv4: cos and sin must be [positions, head_dim / 2]")
    table = (cos.shape[0], hd // 2)
    slot = (n_seq, n_kv, slots)
    return (n_seq, n_kv, hd, slots, ld,
            _tensor("lengths", lengths, torch.int64, (n_seq,), dev),
            _tensor("pos", pos, torch.int64, (n_seq,), dev),
            _tensor("cos", cos, torch.float32, table, dev),
            _tensor("sin", sin, torch.float32, table, dev),
            None if positions is None else _tensor("positions", positions, torch.int32, slot, dev),
            None if weights is None else _tensor("weights", weights, torch.float32, slot, dev))


def _launch(fn, dev: torch.device, *args) -> None:
    """``fn`` on the current stream of ``dev``, which need not be the current device."""
    stream = _stream(dev)
    if torch._C._cuda_getDevice() == dev.index:  # current_device(), in less time
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, stream)
    if rc:
        _native.check(rc)


def append(qkv: torch.Tensor, lengths: torch.Tensor, pos: torch.Tensor, cos: torch.Tensor,
           sin: torch.Tensor, kv: torch.Tensor, n_heads: int,
           starts: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
           weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Store the K (after RoPE) and V of rows ``[q | k | v]`` behind what the caches hold.

    Sequence ``s`` owns rows ``starts[s] .. starts[s + 1] - 1`` of ``qkv`` (device int64
    ``[n_seq + 1]``; without it every sequence has the same number of rows, in order).  Its
    row i goes to slot ``lengths[s] + i`` with position ``pos[s] + i``; rows outside every
    sequence, the cache or the tables are not stored, nor those of a sequence of negative
    length or position.  ``lengths`` and ``pos`` are the
    caller's to advance.  The stored slots' ``positions`` are set and their ``weights``
    cleared.  One launch."""
    n_seq, n_kv, hd, slots, ld, lp, pp, cp, sp, posp, wp = _common(
        qkv, lengths, pos, cos, sin, kv, n_heads, positions, weights)
    st = None if starts is None else _tensor("starts", starts, torch.int64, (n_seq + 1,), kv.device)
    _launch(_native.load_library().gguf_hip_kv4_append, kv.device, qkv.data_ptr(), ld,
            qkv.shape[0], st, lp, pp, cp, sp, cos.shape[0], kv.data_ptr(), posp, wp, n_seq, n_heads,
            n_kv, hd, slots)
    return kv


def attention_workspace(kv: torch.Tensor, n_heads: int, rows: int = 1,
                        weights: bool = False) -> torch.Tensor:
    """Device workspace of ``attention`` calls of up to ``rows`` rows per sequence (with
    ``weights`` if any of them has)."""
    _, n_seq, n_kv, hd, slots = _shape(kv)
    lib = _native.load_library()

    def size(m, mode):
        return _native.check(lib.gguf_hip_kv4_attention_workspace(m, mode, n_seq, n_heads, n_kv, hd,
                                                                  slots), lib)

    # not always more for more rows: they are split over fewer workgroups
    n = max([size(rows, int(weights))] + [size(m, int(weights)) for m in range(1, rows)])
    return torch.empty(n, dtype=torch.uint8, device=kv.device)


def attention(qkv: torch.Tensor, lengths: torch.Tensor, pos: torch.Tensor, cos: torch.Tensor,
              sin: torch.Tensor, kv: torch.Tensor, out: torch.Tensor, n_heads: int,
              work: torch.Tensor, store: bool = True, positions: Optional[torch.Tensor] = None,
              weights: Optional[torch.Tensor] = None, accumulate: bool = False) -> torch.Tensor:
    """RoPE, storing and causal GQA attention of new rows ``[q | k | v]`` of every sequence.

    ``qkv`` holds the same number of rows (up to ``MAX_ROWS``) for each sequence, in order.
    Row i of sequence ``s`` is stored in slot ``lengths[s] + i`` at position ``pos[s] + i``
    and attends to slots ``0 .. lengths[s] + i``.  ``store=False``: the slots hold the rows
    already (``append``), as where the last rows of a prompt are asked for their weights.
    ``weights``: each seen slot's softmax weight, summed over the call's rows and the query
    heads of its KV head, is written there (added with ``accumulate``).  A sequence with
    negative length, or without room in the cache or the tables, takes no part and nothing
    of it is written."""
    n_seq, n_kv, hd, slots, ld, lp, pp, cp, sp, posp, wp = _common(
        qkv, lengths, pos, cos, sin, kv, n_heads, positions, weights)
    rows, rest = divmod(qkv.shape[0], n_seq)
    if rest or rows < 1:
        raise ValueError(f"kv4: {qkv.shape[0]} rows for {n_seq} sequences")
    ldo = _row_matrix("out", out, n_heads * hd, kv.device)
    if out.shape[0] != qkv.shape[0]:
        raise ValueError(f"kv4: out has {out.shape[0]} rows, qkv {qkv.shape[0]}")
    if work.device != kv.device or not work.is_contiguous():
        raise ValueError("kv4: the workspace must be a contiguous tensor on the cache's device")
    mode = 0 if weights is None else (_native.KV4_WEIGHTS_ADD if accumulate
                                      else _native.KV4_WEIGHTS_STORE)
    _launch(_native.load_library().gguf_hip_kv4_attention, kv.device, qkv.data_ptr(), ld, rows,
            lp, pp, cp, sp, cos.shape[0], kv.data_ptr(), int(store), posp, wp, mode, out.data_ptr(),
            ldo, n_seq, n_heads, n_kv, hd, slots, work.data_ptr(),
            work.numel() * work.element_size())
    return out


def load(kv: torch.Tensor, lengths: torch.Tensor, k_out: torch.Tensor,
         v_out: torch.Tensor) -> None:
    """The cached rows in f32: slots ``0 .. lengths[s] - 1`` (at most ``out_slots``) into
    ``k_out`` / ``v_out`` ``[..., n_seq, n_kv_heads, out_slots, head_dim]``, with a leading
    dimension of layers if the cache has one.  Rows from ``lengths[s]`` on are not written.
    For one sequence this is the layout of ``glue.attention_prefill``'s caches."""
    n_layers, n_seq, n_kv, hd, slots = _shape(kv, layers=True)
    shape = (*kv.shape[:-2], k_out.shape[-2] if k_out.dim() else 0, hd)
    kp = _tensor("k_out", k_out, torch.float32, shape, kv.device)
    vp = _tensor("v_out", v_out, torch.float32, shape, kv.device)
    lp = _tensor("lengths", lengths, torch.int64, (n_seq,), kv.device)
    _launch(_native.load_library().gguf_hip_kv4_load, kv.device, kv.data_ptr(), lp, kp, vp,
            shape[-2], n_layers, n_seq, n_kv, hd, slots)


def evict_workspace(kv: torch.Tensor) -> torch.Tensor:
    """Device workspace of ``evict`` calls on caches of this shape."""
    n_layers, n_seq, n_kv, hd, slots = _shape(kv, layers=True)
    lib = _native.load_library()
    n = _native.check(lib.gguf_hip_kv4_evict_workspace(n_layers, n_seq, n_kv, hd, slots), lib)
    return torch.empty(n, dtype=torch.uint8, device=kv.device)


def evict(kv: torch.Tensor, weights: torch.Tensor, positions: torch.Tensor, lengths: torch.Tensor,
          pos: torch.Tensor, keep: int, work: torch.Tensor, recent: int = 0, sinks: int = 0,
          trigger: Optional[int] = None, weights_out: Optional[torch.Tensor] = None,
          positions_out: Optional[torch.Tensor] = None,
          lengths_out: Optional[torch.Tensor] = None) -> None:
    """Cut every sequence longer than ``keep`` slots (and not below ``trigger``) back to the
    ``keep`` slots of largest weight, per layer and KV head.

    Slots with ``positions >= pos[s] - recent`` or ``< sinks`` are kept before all others
    (``recent + sinks <= keep``); of equal weights the lower slot stays, NaN counts least.
    The kept slots from ``keep`` on move into the slots given up below it, in order: slots
    are no longer in the order of their positions, which attention does not need.
    ``weights``, ``positions`` and ``lengths`` are updated in place, or written to the
    ``*_out`` tensors.  ``kv``, ``weights`` and ``positions`` may have a leading dimension of
    layers, which share ``lengths``.  Two launches."""
    n_layers, n_seq, n_kv, hd, slots = _shape(kv, layers=True)
    dev, shape = kv.device, (*kv.shape[:-2], slots)
    weights_out = weights if weights_out is None else weights_out
    positions_out = positions if positions_out is None else positions_out
    lengths_out = lengths if lengths_out is None else lengths_out
    wp = _tensor("weights", weights, torch.float32, shape, dev)
    pp = _tensor("positions", positions, torch.int32, shape, dev)
    lp = _tensor("lengths", lengths, torch.int64, (n_seq,), dev)
    np_ = _tensor("pos", pos, torch.int64, (n_seq,), dev)
    wo = _tensor("weights_out", weights_out, torch.float32, shape, dev)
    po = _tensor("positions_out", positions_out, torch.int32, shape, dev)
    lo = _tensor("lengths_out", lengths_out, torch.int64, (n_seq,), dev)
    if work.device != dev or not work.is_contiguous():
        raise ValueError("kv4: the workspace must be a contiguous tensor on the cache's device")
    _launch(_native.load_library().gguf_hip_kv4_evict, kv.device, kv.data_ptr(), wp, pp, lp, np_,
            keep, keep + 1 if trigger is None else trigger, recent, sinks, wo, po, lo, n_layers,
            n_seq, n_kv, hd, slots, work.data_ptr(), work.numel() * work.element_size())
