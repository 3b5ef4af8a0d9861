"""Llama-style decoder whose every projection is a quantized GGUF matmul.

This is the caller of the dequant-matmul path in the reference's engine: the
per-layer loop of webgpu/src/engine/forward-pass.ts:2925-3297 (input RMSNorm,
Q/K/V projections, rotate_half RoPE, GQA causal attention over a KV cache,
output projection and residual, FFN RMSNorm, gate+up projection, gate_silu,
down projection and residual), the final norm and LM head
(forward-pass.ts:3642-3644), and greedy argmax or drawn tokens (``sampling``).

Glue semantics follow the reference's shaders:
* RMSNorm  ``x * 1/sqrt(mean(x^2) + eps) * w``           rmsnorm.wgsl:1-9,58-67
* RoPE     rotate_half pairing of ``i`` with ``i + d/2``,
           ``theta = pos / base^(2i/d)``                  rope.wgsl:1-10
* SwiGLU   ``up * silu(gate)``                            elementwise.wgsl:96-102 (gate_silu)
* tok/s    generated tokens / decode wall time, prefill excluded (generate.ts:1155-1160)

Every projection goes through ``dispatch_matmul_gguf`` (libgguf_hip): Q/K/V are
one row-concatenated weight and gate/up another (the reference's gate+up
fusion, forward-pass.ts:740-791, applied to Q/K/V too; byte-identical to
separate dispatches).  A decode step runs the glue as libgguf_hip kernels
(``glue.py``: the input norms and SwiGLU run as prologues of the projections
that consume them, the residual adds as accumulate epilogues of the output
and down projections, RoPE + KV append + GQA attention as one launch whose
records the output projection merges, argmax) over preallocated buffers: five
launches per layer (six with caches of more than 2048 slots, whose records the
attention call merges).  Prefill (many positions at once) runs the glue as
libgguf_hip kernels too: RMSNorm rows, each residual add fused with the
RMSNorm after it, RoPE + KV append + causal GQA attention of all rows
(``glue.attention_prefill``, the reference's attention.wgsl with
new_seq_len > 1), SwiGLU rows.  ``hip_glue=False`` runs the prefill glue as
torch f32 ops instead, and ``fused=False`` does the same for decode steps.
A decode step keeps
the token and position in device tensors, so it can be captured once in a HIP
graph and replayed for every generated token without host synchronization.

``kv_bits=4`` holds the caches in 4 bits (``kv4``): a prompt's rows attend in f32 to what the
cache holds (read back) and to each other, and are stored quantized; a decode step stores its
row and attends over the codes.  With ``kv_keep`` the caches have a fixed number of slots,
independent of ``max_seq``: each slot's attention weight is accumulated (the last rows of a
prompt, then every step), and a full cache is cut back to the ``kv_keep`` slots of largest
weight, the latest and the first positions always among them.
"""

from __future__ import annotations

import dataclasses
import math
import time
from typing import Optional, Union

import numpy as np
import torch

from . import glue, kv4, quantize, sampling
from .ggml import FUSED_TYPES, Q4_K, Q6_K, TILE_ROWS, raw_row_bytes
from .linear import (GGUFWeight, LayerWeights, QuantEmbedding, concat_rows, dispatch_matmul_gguf,
                     interleave_tiles, repack_gguf_for_gpu, split_interleaved)


@dataclasses.dataclass
class DecoderConfig:
    n_layers: int = 32
    d_model: int = 4096
    n_heads: int = 32
    n_kv_heads: int = 8
    head_dim: int = 128
    ffn: int = 14336
    vocab: int = 151936
    rope_base: float = 1_000_000.0
    eps: float = 1e-6
    max_seq: int = 512
    attn_type: int = Q4_K      # q, k, v, o
    gate_up_type: int = Q4_K
    down_type: int = Q6_K
    lm_head_type: int = Q6_K
    rope_freq_factors: Optional[tuple] = None   # per-pair divisors of theta (llama rope_freqs)

    @property
    def qkv_rows(self) -> int:
        return (self.n_heads + 2 * self.n_kv_heads) * self.head_dim

    def weight_bytes_per_token(self) -> int:
        """Quantized weight bytes one decode step streams from HBM."""
        d, f = self.d_model, self.ffn
        per_layer = (self.qkv_rows * raw_row_bytes(self.attn_type, d)
                     + d * raw_row_bytes(self.attn_type, self.n_heads * self.head_dim)
                     + 2 * f * raw_row_bytes(self.gate_up_type, d)
                     + d * raw_row_bytes(self.down_type, f))
        return self.n_layers * per_layer + self.vocab * raw_row_bytes(self.lm_head_type, d)


@dataclasses.dataclass
class DecoderWeights:
    """Per-layer ``LayerWeights`` slots: ``qkv_gg`` (Q, K, V rows concatenated) or,
    when the three have different GGUF types, ``qkv_parts = [q, k, v]``; the FFN
    input as ``gateUpI_gg`` (gate and up tiles interleaved, ``interleave_tiles``:
    the decode step then applies SwiGLU in the projection's epilogue),
    ``gateUp_gg`` (rows concatenated) or ``gateUp_parts = [gate, up]``; ``o_gg``,
    ``down_gg`` and the f32 norms ``attn_norm`` / ``ffn_norm``.  ``embed`` is a
    dense ``[vocab, d_model]`` table or a ``QuantEmbedding`` of raw GGUF rows."""
    layers: list
    final_norm: torch.Tensor
    lm_head_gg: GGUFWeight
    embed: Union[torch.Tensor, QuantEmbedding]

    def weight_bytes_per_token(self) -> int:
        """Quantized bytes one decode step streams (projections and LM head)."""
        def nb(w):
            return w.n * raw_row_bytes(w.ggml_type, w.k)
        total = nb(self.lm_head_gg)
        for lw in self.layers:
            for slot in ("qkv", "gateUp"):
                total += sum(nb(w) for w in parts(lw, slot))
            total += nb(lw.o_gg) + nb(lw.down_gg)
        return total


def all_weights(w: DecoderWeights) -> list:
    """Every quantized projection of the model, the LM head included."""
    out = [w.lm_head_gg]
    for lw in w.layers:
        for slot in ("qkv", "gateUp"):
            out += parts(lw, slot)
        out += [lw.o_gg, lw.down_gg]
    return out


def parts(lw: LayerWeights, slot: str) -> list:
    """The weights of a slot: ``[<slot>_gg]``, ``[<slot>I_gg]`` (tile-interleaved)
    or ``<slot>_parts``."""
    for name in (f"{slot}_gg", f"{slot}I_gg"):
        w = lw.get(name)
        if w is not None:
            return [w]
    return list(lw.get(f"{slot}_parts"))


def _quantized(ggml_type: int, n: int, k: int, seed: int, device) -> GGUFWeight:
    w = quantize.synthetic_weight(n, k, seed=seed)
    return repack_gguf_for_gpu(ggml_type, quantize.quantize(w, ggml_type), n, k, device=device)


def _tiled_rows(ggml_type: int, unique_rows: int, n: int, k: int, seed: int, device) -> GGUFWeight:
    """An ``[n, k]`` weight whose rows repeat a block of ``unique_rows`` quantized rows
    (``unique_rows`` a multiple of 16); every row still has its own bytes in HBM."""
    base = _quantized(ggml_type, unique_rows, k, seed, device)
    reps = -(-n // unique_rows)
    data = base.data[:base.nbytes].repeat(reps)
    full = GGUFWeight(data, ggml_type, reps * unique_rows, k)
    return full.rows(0, n) if full.n != n else full


def synthetic_weights(cfg: DecoderConfig, seed: int = 0, device="cuda",
                      distinct_layers: bool = False,
                      lm_head_unique_rows: Optional[int] = None) -> DecoderWeights:
    """Seeded N(0, 0.02) weights quantized in the configured GGUF types.

    Quantizing 32 layers on the host is slow, so unless ``distinct_layers`` the
    layers share one quantized set of values held in separate device buffers
    (each decode step still streams every layer's own bytes from HBM).  The LM
    head likewise repeats ``lm_head_unique_rows`` quantized rows when given."""
    d, hd = cfg.d_model, cfg.head_dim
    g = torch.Generator(device=device).manual_seed(seed)

    def layer_set(s):
        q = _quantized(cfg.attn_type, cfg.n_heads * hd, d, s + 1, device)
        k = _quantized(cfg.attn_type, cfg.n_kv_heads * hd, d, s + 2, device)
        v = _quantized(cfg.attn_type, cfg.n_kv_heads * hd, d, s + 3, device)
        o = _quantized(cfg.attn_type, d, cfg.n_heads * hd, s + 4, device)
        gate = _quantized(cfg.gate_up_type, cfg.ffn, d, s + 5, device)
        up = _quantized(cfg.gate_up_type, cfg.ffn, d, s + 6, device)
        down = _quantized(cfg.down_type, d, cfg.ffn, s + 7, device)
        return concat_rows(q, k, v), o, interleave_tiles(gate, up), down

    layers = []
    shared = None if distinct_layers else layer_set(seed * 1000)
    for l in range(cfg.n_layers):
        qkv, o, gu, down = layer_set(seed * 1000 + 10 * l) if distinct_layers else shared
        if not distinct_layers:
            qkv, o, gu, down = (GGUFWeight(w.data[w.byte_offset:w.byte_offset + w.nbytes].clone(),
                                           w.ggml_type, w.n, w.k) for w in shared)
        layers.append(LayerWeights(
            qkv_gg=qkv, o_gg=o, gateUpI_gg=gu, down_gg=down,
            attn_norm=1.0 + 0.02 * torch.randn(d, device=device, generator=g),
            ffn_norm=1.0 + 0.02 * torch.randn(d, device=device, generator=g)))
    if lm_head_unique_rows:
        lm = _tiled_rows(cfg.lm_head_type, lm_head_unique_rows, cfg.vocab, d, seed + 99, device)
    else:
        lm = _quantized(cfg.lm_head_type, cfg.vocab, d, seed + 99, device)
    embed = (torch.randn(cfg.vocab, d, device=device, generator=g)).half()
    final_norm = 1.0 + 0.02 * torch.randn(d, device=device, generator=g)
    return DecoderWeights(layers, final_norm, lm, embed)


def rms_norm(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    """rmsnorm.wgsl:58-67 with a direct weight (use_residual_weight = 0)."""
    return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w


def rope_tables(cfg: DecoderConfig, device) -> tuple[torch.Tensor, torch.Tensor]:
    half = cfg.head_dim // 2
    inv = 1.0 / (cfg.rope_base ** (torch.arange(half, dtype=torch.float64) * 2.0 / cfg.head_dim))
    if cfg.rope_freq_factors is not None:
        f = torch.tensor(cfg.rope_freq_factors, dtype=torch.float64)
        if f.numel() != half:
            raise ValueError(f"rope_freq_factors has {f.numel()} entries, head_dim/2 = {half}")
        inv = inv / f
    ang = torch.arange(cfg.max_seq, dtype=torch.float64)[:, None] * inv[None, :]
    return ang.cos().float().to(device), ang.sin().float().to(device)


def apply_rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """rotate_half RoPE (rope.wgsl:1-10): x [M, H, D], cos/sin [M, D/2]."""
    half = x.shape[-1] // 2
    x1, x2 = x[..., :half], x[..., half:]
    c, s = cos[:, None, :], sin[:, None, :]
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], dim=-1)


def glue_shapes(cfg: DecoderConfig) -> bool:
    """Whether the glue kernels take the configuration: head_dim 64, 128 or 256,
    at most 8 query heads per KV head, rows of a multiple of 4 values."""
    return (cfg.head_dim in (64, 128, 256) and cfg.n_heads % cfg.n_kv_heads == 0
            and cfg.n_heads // cfg.n_kv_heads <= 8 and cfg.d_model % 4 == 0
            and cfg.ffn % 4 == 0)


def kv_cache_slots(cfg: DecoderConfig, fused: bool, kv_bits: int, kv_slots: Optional[int],
                   kv_keep: Optional[int], kv_recent: int, kv_sinks: int) -> int:
    """The slots per KV head of a ``QuantDecoder``'s cache; ValueError for options that do not go
    together.  ``fused``: the decoder has the fused decode step and the HIP glue."""
    if kv_bits != 4:
        if kv_bits != 32 or kv_slots is not None or kv_keep is not None:
            raise ValueError(f"kv_bits {kv_bits} not 32 or 4, or kv_slots / kv_keep without 4")
        return cfg.max_seq
    if not fused:
        raise ValueError("kv_bits=4 needs the fused decode step and the HIP glue")
    slots = -(-(cfg.max_seq if kv_slots is None else kv_slots) // kv4.TILE) * kv4.TILE
    kv4.cache_bytes(1, cfg.n_kv_heads, cfg.head_dim, slots)
    if kv_keep is not None and not (0 <= kv_recent and 0 <= kv_sinks
                                    and max(1, kv_recent + kv_sinks) <= kv_keep < slots):
        raise ValueError(f"kv_keep {kv_keep}: kv_recent {kv_recent} + kv_sinks {kv_sinks} must fit "
                         f"it, and it must be above 0 and below the {slots} slots")
    return slots


class LayerStack:
    """The layers of a decoder over many rows: ``cfg``, ``w`` (``DecoderWeights``) and ``device``,
    and ``_attend_rows`` of the subclass, which holds the cache."""

    cfg: DecoderConfig
    w: DecoderWeights
    device: torch.device

    def _attend_rows(self, l: int, qkv: torch.Tensor, pos: torch.Tensor, att: torch.Tensor,
                     held: int) -> None:
        """Attention of layer l's rows ``[q | k | v]`` into ``att``."""
        raise NotImplementedError

    def _proj(self, x: torch.Tensor, w: GGUFWeight, label: str) -> torch.Tensor:
        M = x.shape[0]
        y = torch.empty(M, w.n, device=self.device)
        dispatch_matmul_gguf(x, w, y, M, w.n, w.k, label)
        return y

    def _proj_slot(self, x: torch.Tensor, lw: LayerWeights, slot: str, label: str) -> torch.Tensor:
        ws = parts(lw, slot)
        if len(ws) == 1:
            return self._proj(x, ws[0], label)
        return torch.cat([self._proj(x, w, f"{label}{i}") for i, w in enumerate(ws)], dim=1)

    def _embed(self, tok: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        e = self.w.embed
        if isinstance(e, QuantEmbedding):
            return e.gather(tok, out)
        x = e.index_select(0, tok).float()
        if out is None:
            return x
        out.copy_(x)
        return out

    def _layers_glue(self, x: torch.Tensor, pos: torch.Tensor, held: int = 0) -> torch.Tensor:
        """All layers over the M rows of ``x`` (updated in place) with the glue as
        libgguf_hip kernels; returns the rows after the final RMSNorm.  ``pos`` and ``held``
        (the slots in use before the rows) are ``_attend_rows``'s."""
        cfg, layers = self.cfg, self.w.layers
        M = x.shape[0]
        h = torch.empty_like(x)
        att = torch.empty(M, cfg.n_heads * cfg.head_dim, device=self.device)
        a = torch.empty(M, cfg.ffn, device=self.device)
        glue.rmsnorm(x, layers[0].attn_norm, cfg.eps, h)
        for l, lw in enumerate(layers):
            qkv = self._proj_slot(h, lw, "qkv", f"L{l}-qkv")
            self._attend_rows(l, qkv, pos, att, held)
            glue.add_rmsnorm(x, self._proj(att, lw.o_gg, f"L{l}-o"), lw.ffn_norm, cfg.eps, h)
            w = lw.get("gateUpI_gg")
            if w is not None:  # tile-interleaved gate / up columns -> [gate | up] rows, one copy
                gu = torch.empty(M, 2, cfg.ffn // TILE_ROWS, TILE_ROWS, device=self.device)
                gu.copy_(self._proj(h, w, f"L{l}-gateUp").view(M, -1, 2, TILE_ROWS).transpose(1, 2))
                gu = gu.view(M, 2 * cfg.ffn)
            else:
                gu = self._proj_slot(h, lw, "gateUp", f"L{l}-gateUp")
            glue.swiglu(gu, a)
            nxt = layers[l + 1].attn_norm if l + 1 < len(layers) else self.w.final_norm
            glue.add_rmsnorm(x, self._proj(a, lw.down_gg, f"L{l}-down"), nxt, cfg.eps, h)
        return h


class QuantDecoder(LayerStack):
    """Decoder of one sequence over ``DecoderWeights`` with an f32 or 4-bit KV cache in HBM; its
    tokens are the largest logits' or drawn (``set_sampling``).

    ``kv_bits`` 4: ``kv_slots`` (default: enough for ``max_seq``) slots per KV head, rounded up
    to a multiple of 32; ``kv_keep``: a full cache is cut back to that many slots, of which the
    last ``kv_recent`` and the first ``kv_sinks`` positions are never given up.  ``max_seq``
    then bounds the positions only.  A prompt longer than the cache goes on, after the first
    cut, in chunks of ``kv_slots - kv_keep`` tokens, each a pass of the model that reads the
    kept rows back: a ``kv_keep`` near ``kv_slots`` suits short prompts only."""

    WINDOW = 32  # rows at a prompt's end whose attention weights are counted

    def __init__(self, cfg: DecoderConfig, weights: DecoderWeights, device="cuda",
                 fused: bool = True, hip_glue: bool = True, kv_bits: int = 32,
                 kv_slots: Optional[int] = None, kv_keep: Optional[int] = None,
                 kv_recent: int = 64, kv_sinks: int = 4):
        # a weight of a type without fused decode-step kernels runs the step unfused
        grid = any(w.ggml_type not in FUSED_TYPES for w in all_weights(weights))
        self.cfg, self.w, self.device = cfg, weights, torch.device(device)
        self.fused = fused and not grid
        self.hip_glue = hip_glue and glue_shapes(cfg)
        L, kv, T, hd = cfg.n_layers, cfg.n_kv_heads, cfg.max_seq, cfg.head_dim
        self.kv_bits, self.kv_keep = kv_bits, kv_keep
        slots = kv_cache_slots(cfg, self.fused and self.hip_glue, kv_bits, kv_slots, kv_keep,
                               kv_recent, kv_sinks)
        if kv_bits == 4:
            self._init_kv4(slots, kv_keep, kv_recent, kv_sinks)
        else:
            self.k_cache = torch.zeros(L, kv, T, hd, device=self.device)
            self.v_cache = torch.zeros(L, kv, T, hd, device=self.device)
            self.cos, self.sin = rope_tables(cfg, self.device)
        self.t_idx = torch.arange(T, device=self.device)
        self._graph = None
        # static buffers of the fused decode step
        e = lambda n: torch.empty(1, n, device=self.device)  # noqa: E731
        d = cfg.d_model
        self.b_x, self.b_h, self.b_qkv = e(d), e(d), e(cfg.qkv_rows)
        self.b_att, self.b_o = e(cfg.n_heads * hd), e(d)
        self.b_gu, self.b_a, self.b_d = e(2 * cfg.ffn), e(cfg.ffn), e(d)
        self.b_logits = e(cfg.vocab)
        if kv_bits == 32:
            self.w_att = glue.attention_workspace(cfg.n_heads, cfg.n_kv_heads, hd, T, self.device)
        self.w_arg = glue.argmax_workspace(self.device)
        self._draw = self._u = None
        self._chosen: dict = {}             # set_sampling's arguments

    # -- the choice of the next token --
    def set_sampling(self, temperature: float = 0.0, top_k: int = 0, top_p: float = 1.0,
                     min_p: float = 0.0, seed: int = 0) -> None:
        """How the next tokens are chosen (``sampling.sample``); ``temperature`` 0: the largest
        logit.  The random numbers, one for each position, follow from ``seed``.  Steps captured
        before keep the settings that they were captured with, and read the new random numbers."""
        choice = dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, seed=seed)
        self._set_sampling(**choice)
        self._chosen = choice

    def _set_sampling(self, temperature: float = 0.0, top_k: int = 0, top_p: float = 1.0,
                      min_p: float = 0.0, seed: int = 0) -> None:
        if not temperature > 0:
            self._draw = None
            return
        g = torch.Generator(device=self.device).manual_seed(seed)
        self._draw = dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
        if self._u is None:
            self._u = torch.empty(self.cfg.max_seq, device=self.device)
            self._u_now = torch.empty(1, device=self.device)
            self._w_draw = sampling.workspace(1, self.cfg.vocab, self.device)
        self._u.copy_(torch.rand(self.cfg.max_seq, device=self.device, generator=g))

    def _choose(self, logits: torch.Tensor, tok: torch.Tensor, pos: torch.Tensor) -> None:
        """The token after position ``pos`` [1] into ``tok`` [1], by ``logits`` [1, vocab]."""
        if self._draw is None:
            glue.argmax(logits, tok, self.w_arg)
            return
        # a step past the last position has NaN logits or no meaning, but no index out of range
        torch.index_select(self._u, 0, pos.clamp(0, self._u.numel() - 1), out=self._u_now)
        sampling.sample(logits, self._u_now, tok, self._w_draw, **self._draw)

    # -- the 4-bit cache --
    def _init_kv4(self, slots, keep, recent, sinks) -> None:
        cfg, dev = self.cfg, self.device
        L, nkv, hd = cfg.n_layers, cfg.n_kv_heads, cfg.head_dim
        self.kv_slots, self.kv_recent, self.kv_sinks = slots, recent, sinks
        self.kv4 = kv4.empty(1, nkv, hd, slots, dev, n_layers=L)
        # the slots in use, and the position after the last one (with eviction further on)
        self.kv_state = torch.zeros(2, dtype=torch.long, device=dev)
        self.kv_lengths = self.kv_state[:1]
        # one layer's rows in f32, for the attention of a prompt
        self.k_cache = torch.zeros(nkv, slots, hd, device=dev)
        self.v_cache = torch.zeros(nkv, slots, hd, device=dev)
        # a prompt's slot t stands at position t + an offset below max_seq
        self.cos, self.sin = rope_tables(
            dataclasses.replace(cfg, max_seq=cfg.max_seq + slots), dev)
        self.kv_weights = self.kv_positions = None
        if keep is not None:
            self.kv_weights = torch.zeros(L, 1, nkv, slots, device=dev)
            self.kv_positions = torch.zeros(L, 1, nkv, slots, dtype=torch.int32, device=dev)
            self.w_evict = kv4.evict_workspace(self.kv4)
        # of steps, and of a prompt's last rows
        self.w_att = kv4.attention_workspace(self.kv4[0], cfg.n_heads,
                                             rows=1 if keep is None else self.WINDOW,
                                             weights=keep is not None)

    def _kv_slot(self, l: int):
        """Layer l's positions and weights (None without eviction)."""
        if self.kv_keep is None:
            return dict(positions=None, weights=None)
        return dict(positions=self.kv_positions[l], weights=self.kv_weights[l])

    def _evict(self, pos: torch.Tensor) -> None:
        """Cut the caches back if they are full (decided on the device)."""
        kv4.evict(self.kv4, self.kv_weights, self.kv_positions, self.kv_lengths, pos, self.kv_keep,
                  self.w_evict, recent=self.kv_recent, sinks=self.kv_sinks, trigger=self.kv_slots)

    def _cache_state(self) -> list:
        """The tensors that a step changes, besides token and position."""
        if self.kv_bits == 32:
            return [self.k_cache, self.v_cache]
        return [t for t in (self.kv4, self.kv_state, self.kv_weights, self.kv_positions)
                if t is not None]

    def _attend_rows(self, l: int, qkv: torch.Tensor, pos: torch.Tensor, att: torch.Tensor,
                     held: int) -> None:
        """Attention of a prompt's rows in layer l; ``held`` slots are in use before them."""
        cfg = self.cfg
        if self.kv_bits == 32:
            glue.attention_prefill(qkv, pos, self.cos, self.sin, self.k_cache[l], self.v_cache[l],
                                   att, cfg.n_heads, cfg.n_kv_heads, cfg.head_dim)
            return
        m, cache = qkv.shape[0], self.kv4[l]
        first = pos[:1]
        if held:
            kv4.load(cache, self.kv_lengths, self.k_cache[None], self.v_cache[None])
        off = self._prompt_pos - held
        glue.attention_prefill(qkv, pos - off, self.cos.narrow(0, off, self.kv_slots),
                               self.sin.narrow(0, off, self.kv_slots), self.k_cache, self.v_cache,
                               att, cfg.n_heads, cfg.n_kv_heads, cfg.head_dim)
        kv4.append(qkv, self.kv_lengths, first, self.cos, self.sin, cache, cfg.n_heads,
                   **self._kv_slot(l))
        if self.kv_keep is not None:
            w = min(m, self.WINDOW)
            kv4.attention(qkv[m - w:], self.kv_lengths + (m - w), first + (m - w), self.cos,
                          self.sin, cache, torch.empty_like(att[:w]), cfg.n_heads,
                          self.w_att, store=False, weights=self.kv_weights[l],
                          accumulate=True)

    def _prefill_kv4(self, tokens: torch.Tensor, pos0: int) -> torch.Tensor:
        if tokens.numel() == 0:
            raise ValueError("an empty prompt has no logits")
        held, follows = self.kv_state.tolist() if pos0 else (0, 0)
        if pos0 != follows:
            raise ValueError(f"position {pos0} does not follow what the 4-bit cache holds: "
                             f"{held} slots, position {follows} is the next")
        if self.kv_keep is None and held + tokens.numel() > self.kv_slots:
            raise ValueError(f"sequence of {held + tokens.numel()} exceeds the cache's "
                             f"{self.kv_slots} slots (kv_keep bounds it)")
        if pos0 == 0:
            self.kv_state.zero_()
        done, h = 0, None
        while done < tokens.numel():
            m = min(tokens.numel() - done, self.kv_slots - held)
            self._prompt_pos = pos0 + done
            pos = torch.arange(pos0 + done, pos0 + done + m, device=self.device)
            h = self._layers_glue(self._embed(tokens[done:done + m]), pos, held)
            self.kv_state += m
            held, done = held + m, done + m
            if self.kv_keep is not None and held == self.kv_slots:
                self._evict(pos[-1:] + 1)
                held = self.kv_keep
        return self._proj(h[-1:], self.w.lm_head_gg, "lm_head")

    # -- one pass of all layers over M tokens at positions ``pos`` (device [M]) as torch ops --
    def _gate_up(self, h: torch.Tensor, lw: LayerWeights, label: str):
        """(gate, up) projections of the FFN input ``h``."""
        w = lw.get("gateUpI_gg")
        if w is not None:
            return split_interleaved(self._proj(h, w, label))
        gu = self._proj_slot(h, lw, "gateUp", label)
        return gu[:, :self.cfg.ffn], gu[:, self.cfg.ffn:]

    def _layers(self, x: torch.Tensor, pos: torch.Tensor) -> torch.Tensor:
        cfg = self.cfg
        M, nh, nkv, hd = x.shape[0], cfg.n_heads, cfg.n_kv_heads, cfg.head_dim
        grp = nh // nkv
        cos, sin = self.cos.index_select(0, pos), self.sin.index_select(0, pos)
        # causal mask over cache slots: query at position p sees slots t <= p
        mask = torch.where(self.t_idx[None, :] <= pos[:, None], 0.0, float("-inf"))  # [M, T]
        mask = mask.repeat_interleave(grp, dim=0)[None]                            # [1, M*grp, T]
        scale = 1.0 / math.sqrt(hd)
        for l, lw in enumerate(self.w.layers):
            h = rms_norm(x, lw.attn_norm, cfg.eps)
            qkv = self._proj_slot(h, lw, "qkv", f"L{l}-qkv")
            q = qkv[:, :nh * hd].view(M, nh, hd)
            k = qkv[:, nh * hd:(nh + nkv) * hd].view(M, nkv, hd)
            v = qkv[:, (nh + nkv) * hd:].view(M, nkv, hd)
            q, k = apply_rope(q, cos, sin), apply_rope(k, cos, sin)
            self.k_cache[l].index_copy_(1, pos, k.transpose(0, 1))
            self.v_cache[l].index_copy_(1, pos, v.transpose(0, 1))
            # GQA: query head h reads KV head h // grp
            qg = q.view(M, nkv, grp, hd).permute(1, 0, 2, 3).reshape(nkv, M * grp, hd)
            s = torch.matmul(qg, self.k_cache[l].transpose(1, 2)) * scale + mask
            o = torch.matmul(torch.softmax(s, dim=-1), self.v_cache[l])           # [nkv, M*grp, hd]
            o = o.view(nkv, M, grp, hd).permute(1, 0, 2, 3).reshape(M, nh * hd)
            x = x + self._proj(o, lw.o_gg, f"L{l}-o")
            h = rms_norm(x, lw.ffn_norm, cfg.eps)
            gate, up = self._gate_up(h, lw, f"L{l}-gateUp")
            a = up * torch.nn.functional.silu(gate)
            x = x + self._proj(a, lw.down_gg, f"L{l}-down")
        return x

    def _logits(self, x_last: torch.Tensor) -> torch.Tensor:
        h = rms_norm(x_last, self.w.final_norm, self.cfg.eps)
        return self._proj(h, self.w.lm_head_gg, "lm_head")

    @torch.no_grad()
    def prefill(self, tokens: torch.Tensor, pos0: int = 0) -> torch.Tensor:
        """Run ``tokens`` (device int64 [M]) at positions pos0.. and return the
        last position's logits [1, vocab].  With a 4-bit cache ``pos0`` is 0 (a new
        sequence) or the position after the last one."""
        M = tokens.numel()
        if pos0 + M > self.cfg.max_seq:
            raise ValueError(f"sequence of {pos0 + M} exceeds max_seq {self.cfg.max_seq}")
        if self.kv_bits == 4:
            return self._prefill_kv4(tokens, pos0)
        pos = torch.arange(pos0, pos0 + M, device=self.device)
        x = self._embed(tokens)
        if self.hip_glue:
            h = self._layers_glue(x, pos)
            return self._proj(h[-1:], self.w.lm_head_gg, "lm_head")
        x = self._layers(x, pos)
        return self._logits(x[-1:])

    def _proj_into(self, x: torch.Tensor, w: GGUFWeight, y: torch.Tensor, label: str) -> None:
        dispatch_matmul_gguf(x, w, y, 1, w.n, w.k, label)

    def _step_fused(self, tok: torch.Tensor, pos: torch.Tensor) -> torch.Tensor:
        """Five launches per layer: Q/K/V projection with the input RMSNorm as its
        prologue, attention (partial-softmax records only), output projection
        that merges the records as its prologue and accumulates into the
        residual, gate/up projection with the FFN RMSNorm prologue and the
        SwiGLU epilogue (interleaved gate / up tiles), down projection
        accumulated into the residual.  With concatenated or split gate / up
        weights, SwiGLU runs as the down projection's prologue instead; with
        n_heads * head_dim above 8192 the attention merges its own records.  A 4-bit
        cache's attention writes its output (a second launch where the slots are
        split), is NaN beforehand, and adds the length's limit or an eviction's two
        launches to the step."""
        cfg, W = self.cfg, self.w
        x = self.b_x
        merge = cfg.n_heads * cfg.head_dim <= 8192 and self.kv_bits == 32
        self._embed(tok, x)
        if self.kv_bits == 4:
            self.b_att.fill_(float("nan"))  # stays where the row has no slot or no position
        for l, lw in enumerate(W.layers):
            self._fused_slot(x, lw, "qkv", self.b_qkv, lw.attn_norm)
            if self.kv_bits == 4:
                kv4.attention(self.b_qkv, self.kv_lengths, pos, self.cos, self.sin, self.kv4[l],
                              self.b_att, cfg.n_heads, self.w_att, accumulate=True,
                              **self._kv_slot(l))
            else:
                glue.attention_decode(self.b_qkv, pos, self.cos, self.sin, self.k_cache[l],
                                      self.v_cache[l], None if merge else self.b_att, cfg.n_heads,
                                      cfg.n_kv_heads, cfg.head_dim, self.w_att)
            if merge:
                glue.matmul_attn_merge(self.w_att, pos, lw.o_gg, x, cfg.n_heads, cfg.n_kv_heads,
                                       cfg.head_dim, cfg.max_seq, accumulate=True)
            else:
                glue.matmul_fused(self.b_att, lw.o_gg, x, accumulate=True)
            gui = lw.get("gateUpI_gg")
            if gui is not None:
                glue.matmul_fused(x, gui, self.b_a, glue.PROLOGUE_RMSNORM, lw.ffn_norm, cfg.eps,
                                  epilogue=glue.EPILOGUE_SWIGLU)
                glue.matmul_fused(self.b_a, lw.down_gg, x, accumulate=True)
            else:
                self._fused_slot(x, lw, "gateUp", self.b_gu, lw.ffn_norm)
                glue.matmul_fused(self.b_gu, lw.down_gg, x, glue.PROLOGUE_SWIGLU,
                                  accumulate=True)
        glue.matmul_fused(x, W.lm_head_gg, self.b_logits, glue.PROLOGUE_RMSNORM, W.final_norm,
                          cfg.eps)
        self._choose(self.b_logits, tok, pos)
        if self.kv_bits == 32:
            pos.add_(1)
            return self.b_logits
        torch._foreach_add_([pos, self.kv_state], 1)  # one launch
        if self.kv_keep is not None:
            self._evict(pos)
        else:
            self.kv_state.clamp_(max=self.kv_slots)
        return self.b_logits

    def _fused_slot(self, x, lw, slot, y, norm_w) -> None:
        """RMSNorm-prologue projection of a concatenated slot into ``y`` (one launch
        per part; the parts write consecutive column ranges of ``y``)."""
        c = 0
        for w in parts(lw, slot):
            glue.matmul_fused(x, w, y[:, c:c + w.n], glue.PROLOGUE_RMSNORM, norm_w, self.cfg.eps)
            c += w.n

    @torch.no_grad()
    def step(self, tok: torch.Tensor, pos: torch.Tensor) -> torch.Tensor:
        """One decode step in place: reads token ``tok`` [1] at position
        ``pos`` [1], writes the next token into ``tok`` and advances ``pos``.
        Touches no host state, so it can be captured in a graph.  With a 4-bit cache ``pos``
        is the position after the last one; a step for which it has no slot left stores
        nothing, and its logits are NaN."""
        if self.fused:
            return self._step_fused(tok, pos)
        x = self._embed(tok)
        x = self._layers(x, pos)
        logits = self._logits(x)
        if self._draw is None:
            tok.copy_(torch.argmax(logits, dim=-1))
        else:
            self._choose(logits, tok, pos)
        pos.add_(1)
        return logits

    @torch.no_grad()
    def capture(self, tok: torch.Tensor, pos: torch.Tensor) -> None:
        """Capture ``step(tok, pos)`` in a HIP graph (tok / pos are the static inputs).
        The capture run itself executes one step, so it is made on a copy."""
        s = torch.cuda.Stream(device=self.device)
        s.wait_stream(torch.cuda.current_stream(self.device))
        t0, p0 = tok.clone(), pos.clone()
        saved = [t.clone() for t in self._cache_state()]

        def restore():
            tok.copy_(t0)
            pos.copy_(p0)
            for t, before in zip(self._cache_state(), saved):
                t.copy_(before)

        with torch.cuda.stream(s):
            self.step(tok, pos)                    # warm-up outside the graph
        torch.cuda.current_stream(self.device).wait_stream(s)
        restore()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            self._graph_logits = self.step(tok, pos)
        restore()
        self._graph = g

    @torch.no_grad()
    def generate(self, prompt: torch.Tensor, n_new: int, graph: bool = True,
                 temperature: Optional[float] = None, top_k: Optional[int] = None,
                 top_p: Optional[float] = None, min_p: Optional[float] = None,
                 seed: Optional[int] = None) -> dict:
        """Generation, greedy or sampled: returns the new token ids and prefill / decode timings.
        What is not given of the settings is what ``set_sampling`` chose; what is given holds until
        the next call of either.  tok/s = n_new / decode wall time (prefill excluded,
        generate.ts:1155-1160)."""
        dev = self.device
        given = dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, seed=seed)
        if prompt.numel() + n_new > self.cfg.max_seq:
            raise ValueError(f"prompt {prompt.numel()} + {n_new} new tokens exceed max_seq "
                             f"{self.cfg.max_seq}")
        if (self.kv_bits == 4 and self.kv_keep is None
                and prompt.numel() + n_new > self.kv_slots + 1):
            raise ValueError(f"prompt {prompt.numel()} + {n_new} new tokens exceed the cache's "
                             f"{self.kv_slots} slots (kv_keep bounds it)")
        self._set_sampling(**{**self._chosen, **{k: v for k, v in given.items() if v is not None}})
        if self.kv_bits == 32:
            self.k_cache.zero_()
            self.v_cache.zero_()
        torch.cuda.synchronize(dev)
        t0 = time.perf_counter()
        logits = self.prefill(prompt, 0)
        tok = torch.argmax(logits, dim=-1).view(1)
        if self._draw is not None:
            self._choose(logits, tok, torch.full((1,), prompt.numel() - 1, dtype=torch.long, device=dev))
        torch.cuda.synchronize(dev)
        t_prefill = time.perf_counter() - t0
        pos = torch.full((1,), prompt.numel(), dtype=torch.long, device=dev)
        out = torch.empty(n_new, dtype=torch.long, device=dev)
        out[0] = tok[0]
        if graph:
            self.capture(tok, pos)
        torch.cuda.synchronize(dev)
        t1 = time.perf_counter()
        for i in range(1, n_new):
            if graph:
                self._graph.replay()
            else:
                self.step(tok, pos)
            out[i] = tok[0]
        torch.cuda.synchronize(dev)
        t_decode = time.perf_counter() - t1
        steps = max(n_new - 1, 1)
        return {"tokens": out, "prefill_s": t_prefill, "decode_s": t_decode,
                "decode_steps": steps, "tok_s": steps / t_decode,
                "prefill_tok_s": prompt.numel() / t_prefill}
