"""Sampling a token per row of logits from given random numbers (libgguf_hip).

The reference draws on the host from logits that it reads back (webgpu/src/engine/generate.ts);
``glue.argmax`` is its greedy case on the device.  Here a row's tokens, in descending order of
their logits (equal ones by index), are weighted ``exp((logit - largest) / temperature)``; the
shortest run that ``top_k``, ``top_p`` and ``min_p`` ask for is kept, and the drawn token is the
first at which the running sum exceeds ``u`` times the kept sum.  The exact rules are in
include/gguf_hip_sample.h.
"""

from __future__ import annotations

from typing import Optional, Union

import torch

from . import _native


def workspace(rows: int, vocab: int, device="cuda") -> torch.Tensor:
    """Device workspace of ``sample`` calls of up to ``rows`` rows of ``vocab`` logits."""
    lib = _native.load_library()
    n = _native.check(lib.gguf_hip_sample_workspace(rows, vocab), lib)
    return torch.empty(n, dtype=torch.uint8, device=device)


def _array(name: str, t: torch.Tensor, dtype, shape, device: int) -> int:
    if (t.dtype is dtype and t.shape == shape and t.is_contiguous() and t.get_device() == device):
        return t.data_ptr()
    raise ValueError(f"sample: {name} must be a contiguous {dtype} tensor {tuple(shape)} on device "
                     f"{device}, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _setting(name: str, v, dtype, shape, device: int):
    """The address of a setting (0: the same for every row), and its value."""
    if isinstance(v, torch.Tensor):
        return _array(name, v, dtype, shape, device), 0
    return 0, v


def sample(logits: torch.Tensor, u: torch.Tensor, out: torch.Tensor, work: torch.Tensor,
           temperature: Union[float, torch.Tensor] = 1.0, top_k: Union[int, torch.Tensor] = 0,
           top_p: Union[float, torch.Tensor] = 1.0, min_p: Union[float, torch.Tensor] = 0.0,
           probs: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out[r] (int64) = a token drawn from row r of ``logits`` (f32 ``[rows, vocab]``, unit column
    stride) with the random number ``u[r]`` (f32, 0 <= u < 1).

    Each setting is a value for every row or a device tensor ``[rows]`` (f32; ``top_k`` int32).
    ``top_k`` <= 0, ``top_p`` >= 1 and ``min_p`` <= 0 keep everything; ``temperature`` <= 0 draws
    the first of the largest.  ``probs`` (f32 ``[rows]``): the drawn tokens' probabilities among
    the kept ones.  ``work``: from ``workspace``, for calls that do not overlap.  Allocates and
    synchronises nothing."""
    if _native.direct().sample(logits, u, out, work, temperature, top_k, top_p, min_p, probs):
        return out
    dev = logits.get_device()
    if logits.dim() != 2 or logits.dtype is not torch.float32 or dev < 0:
        raise ValueError("sample: logits must be float32 device rows [rows, vocab]")
    rows, vocab = logits.shape
    ld, step = logits.stride()
    if rows <= 1:
        ld = max(vocab, 1)
    if (vocab > 1 and step != 1) or ld < vocab:
        raise ValueError("sample: logits must be rows with unit column stride")
    n = (rows,)
    up = _array("u", u, torch.float32, n, dev)
    op = _array("out", out, torch.int64, n, dev)
    tp, tv = _setting("temperature", temperature, torch.float32, n, dev)
    kp, kv = _setting("top_k", top_k, torch.int32, n, dev)
    pp, pv = _setting("top_p", top_p, torch.float32, n, dev)
    mp, mv = _setting("min_p", min_p, torch.float32, n, dev)
    qp = 0 if probs is None else _array("probs", probs, torch.float32, n, dev)
    if work.get_device() != dev or not work.is_contiguous():
        raise ValueError("sample: the workspace must be a contiguous tensor on the logits' device")
    _native.call(_native.SAMPLE, dev, logits.data_ptr(), ld, rows, vocab, up, tp, tv, kp,
                 max(0, min(int(kv), 2 ** 31 - 1)), pp, pv, mp, mv, op, qp, work.data_ptr(), work.nbytes)
    return out
