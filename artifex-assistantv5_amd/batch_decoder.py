"""Several sequences of one model decoded together over a KV cache in pages.

``QuantDecoder`` runs one sequence over a cache of its own.  Here ``n_seq`` sequences share the
layers' projections of a step (one row each) and a pool of pages (``paged``): a prompt is run once
and forked into as many continuations as are asked for, which share its pages and copy only the one
they go on writing in.  A step makes room for the next rows, runs the layers
(``glue`` kernels and ``dispatch_matmul_gguf`` of ``n_seq`` rows), and draws each sequence's token
(``sampling``); it touches no host state, so it can be captured in a HIP graph.

Per sequence: ``lengths`` (slots in use, which is the position of the next row), ``tables`` and
``refs`` as ``paged`` has them, ``tok`` (the token that its next step reads) and ``rows`` (1: it
takes part in steps; 0: it rests).  The prompt's own rows attend in f32, the cached ones as
rounded to the pages' type.
"""

from __future__ import annotations

import dataclasses
import time
from typing import Optional, Sequence, Union

import torch

from . import _native, glue, paged, sampling
from .decoder import DecoderConfig, DecoderWeights, LayerStack, glue_shapes, rope_tables

Setting = Union[float, int, Sequence, torch.Tensor]


def check_batch(cfg: DecoderConfig, n_seq: int, n_pages: Optional[int], page: int,
                dtype: torch.dtype) -> tuple:
    """(table columns, pages) of a ``BatchDecoder``; ValueError for options that it cannot have."""
    if not glue_shapes(cfg):
        raise ValueError("BatchDecoder needs a model that the glue kernels take: head_dim 64, 128 or "
                         "256, at most 8 query heads per KV head, rows of a multiple of 4 values")
    if not 1 <= n_seq <= 4096:
        raise ValueError(f"BatchDecoder: {n_seq} sequences not in 1..4096")
    if dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"BatchDecoder: pages are float16 or bfloat16, not {dtype}")
    paged.pool_bytes(1, cfg.n_kv_heads, cfg.head_dim, page)
    columns = -(-cfg.max_seq // page)
    n_pages = n_seq * columns if n_pages is None else n_pages
    paged.pool_bytes(n_pages, cfg.n_kv_heads, cfg.head_dim, page)
    if not 1 <= cfg.n_layers <= 65535:
        raise ValueError(f"BatchDecoder: {cfg.n_layers} layers not in 1..65535")
    # what the calls over its sequences, of a prompt and of a draw take
    lib = _native.load_library()
    heads = (cfg.n_heads, cfg.n_kv_heads, cfg.head_dim)
    _native.check(lib.gguf_hip_paged_attention_workspace(page, columns, n_seq, *heads), lib)
    _native.check(lib.gguf_hip_attention_workspace(*heads, columns * page), lib)
    _native.check(lib.gguf_hip_sample_workspace(n_seq, cfg.vocab), lib)
    return columns, n_pages


class BatchDecoder(LayerStack):
    """``n_seq`` sequences over a pool of ``n_pages`` pages (default: enough for all of
    ``max_seq`` tokens) of ``page`` slots in ``dtype``.

    A sequence for which the pool has no page, or past ``max_seq``, stores nothing in a step: its
    logits are NaN, its ``tok`` is 0 and its length stays.  The token that it was to store waits for
    the first step with room for it, unless ``tok`` has been given another one (not 0) by then."""

    def __init__(self, cfg: DecoderConfig, weights: DecoderWeights, n_seq: int,
                 n_pages: Optional[int] = None, page: int = 16,
                 dtype: torch.dtype = torch.float16, device="cuda"):
        columns, n_pages = check_batch(cfg, n_seq, n_pages, page, dtype)
        self.cfg, self.w, self.n_seq = cfg, weights, n_seq
        self.slots = columns * page
        self.kv = paged.empty(n_pages, cfg.n_kv_heads, cfg.head_dim, page, dtype, device,
                              n_layers=cfg.n_layers)
        dev = self.device = self.kv.device  # with its index: what is current may change
        self.tables, self.lengths, self.refs = paged.empty_tables(n_seq, columns, n_pages, dev)
        i64 = lambda n: torch.zeros(n, dtype=torch.int64, device=dev)  # noqa: E731
        self.rows, self.room, self.tok = i64(n_seq), i64(n_seq), i64(n_seq)
        self._waiting = i64(n_seq)          # tokens of sequences that had no room, 0: none
        self.live = i64(1)
        self.cos, self.sin = rope_tables(dataclasses.replace(cfg, max_seq=self.slots), dev)
        # one layer's rows of a sequence in f32, for the attention of a prompt
        self.k_cache = torch.zeros(cfg.n_kv_heads, self.slots, cfg.head_dim, device=dev)
        self.v_cache = torch.zeros_like(self.k_cache)
        self.w_att = paged.attention_workspace(self.kv[0], self.tables, cfg.n_heads)
        self.w_grow = paged.grow_workspace(self.kv, self.tables)
        self.w_compact = paged.compact_workspace(self.kv, self.tables)
        self.w_draw = sampling.workspace(n_seq, cfg.vocab, dev)
        self.probs = torch.zeros(n_seq, device=dev)
        self._seq = torch.arange(n_seq, device=dev)
        self._logits = self._side = None
        self._prompt = None                 # the sequence whose prompt runs; None: a step
        self._set_sampling()
        self._chosen: dict = {}             # set_sampling's arguments

    # -- the choice of the tokens --
    def set_sampling(self, temperature: Setting = 0.0, top_k: Setting = 0, top_p: Setting = 1.0,
                     min_p: Setting = 0.0, seed: int = 0, stop: Optional[int] = None) -> None:
        """How the next tokens are chosen (``sampling.sample``): values for all sequences or one for
        each.  A sequence whose token is ``stop`` rests from then on.  The random numbers follow from
        ``seed``, one for each position of each sequence: the same seed gives the same ones again,
        also to another prompt that takes a sequence's place, and another seed gives all sequences
        new ones.  Steps captured before read these settings too, but for a ``stop`` where they
        were captured without any."""
        self._set_sampling(temperature, top_k, top_p, min_p, seed, stop)
        self._chosen = dict(temperature=self._temperature.clone(), top_k=self._top_k.clone(),
                            top_p=self._top_p.clone(), min_p=self._min_p.clone(), seed=seed, stop=stop)

    def _set_sampling(self, temperature: Setting = 0.0, top_k: Setting = 0, top_p: Setting = 1.0,
                      min_p: Setting = 0.0, seed: int = 0, stop: Optional[int] = None) -> None:
        dev, n = self.device, self.n_seq

        def each(name, v, dtype):
            t = torch.as_tensor(v, dtype=dtype).to(dev)
            if t.dim() > 1 or (t.dim() == 1 and t.shape[0] != n):
                raise ValueError(f"{name} must be one value, or one for each of {n} sequences")
            return t.expand(n).contiguous()

        # a row of random numbers for each position; two sequences at one position have their own
        g = torch.Generator(device=dev).manual_seed(seed)
        new = dict(_temperature=each("temperature", temperature, torch.float32),
                   _top_k=each("top_k", top_k, torch.int32),
                   _top_p=each("top_p", top_p, torch.float32),
                   _min_p=each("min_p", min_p, torch.float32),
                   _stop_tok=torch.full((1,), -1 if stop is None else stop, dtype=torch.int64, device=dev),
                   _u=torch.rand(self.slots, n, device=dev, generator=g))
        for name, t in new.items():  # all of them fit; in place, for steps captured before
            old = getattr(self, name, None)
            setattr(self, name, t.clone() if old is None else old.copy_(t))
        self._stop = stop

    def _choose(self, logits: torch.Tensor, takes: torch.Tensor, stored: torch.Tensor) -> None:
        """The tokens after the last slots of the sequences for which ``takes`` (bool), by ``logits``
        [n_seq, vocab].  Where ``stored`` is 0 they are no draws, which ``stop`` could end."""
        at = (self.lengths - 1).clamp_(0, self.slots - 1)
        u = self._u[at, self._seq]
        tok = torch.empty_like(self.tok)
        probs = torch.empty_like(self.probs)
        sampling.sample(logits, u, tok, self.w_draw, self._temperature, self._top_k, self._top_p,
                        self._min_p, probs=probs)
        torch.where(takes, tok, self.tok, out=self.tok)
        torch.where(takes, probs, self.probs, out=self.probs)
        if self._stop is not None:
            self.rows.mul_((self.tok != self._stop_tok) | (stored == 0))

    # -- the cache --
    def reset(self) -> None:
        """No sequence holds anything, none takes part."""
        self.tables.fill_(-1)
        for t in (self.lengths, self.refs, self.rows, self.room, self.tok, self._waiting):
            t.zero_()

    @torch.no_grad()
    def fork(self, parents: Union[Sequence[int], torch.Tensor]) -> None:
        """Sequence ``s`` becomes a fork of sequence ``parents[s]`` as that was before (itself: it
        stays; -1: it is freed and rests): the parent's pages, token and part in steps."""
        p = torch.as_tensor(parents, dtype=torch.int64).to(self.device).contiguous()
        paged.fork(self.tables, self.lengths, self.refs, p)
        ok = (p >= 0) & (p < self.n_seq)
        src = torch.where(ok, p, 0)
        for t in (self.tok, self._waiting, self.rows, self.probs):
            t.copy_(torch.where(ok, t[src], torch.zeros_like(t)))

    @torch.no_grad()
    def compact(self) -> torch.Tensor:
        """The pages in use to the front of the pool; their number (device int64 [1])."""
        paged.compact(self.kv, self.tables, self.refs, self.live, self.w_compact)
        return self.live

    def _grow(self, rows: torch.Tensor) -> None:
        """Room for ``rows`` more rows of each sequence, up to ``max_seq``."""
        paged.grow(self.kv, self.tables, self.lengths, self.refs, rows, self.room, self.w_grow)
        if self.slots > self.cfg.max_seq:
            self.room.clamp_(max=self.cfg.max_seq)

    def _attend_rows(self, l: int, qkv: torch.Tensor, pos: torch.Tensor, att: torch.Tensor,
                     held: int) -> None:
        cfg, kv = self.cfg, self.kv[l]
        if self._prompt is None:
            if l == 0:
                att.fill_(float("nan"))  # stays where a sequence does not take part
            paged.attention(qkv, self.lengths, self.tables, self.cos, self.sin, kv, att, cfg.n_heads,
                            self.w_att, room=self.room)
            return
        s = slice(self._prompt, self._prompt + 1)
        if held:
            paged.load(kv, self.tables[s], self.lengths[s], self.k_cache[None], self.v_cache[None])
        glue.attention_prefill(qkv, pos, self.cos, self.sin, self.k_cache, self.v_cache, att,
                               cfg.n_heads, cfg.n_kv_heads, cfg.head_dim)
        paged.append(qkv, self.lengths[s], self.tables[s], self.cos, self.sin, kv, cfg.n_heads,
                     room=self.room[s])

    # -- prompts and steps --
    @torch.no_grad()
    def prefill(self, tokens: torch.Tensor, seq: int) -> torch.Tensor:
        """Run ``tokens`` (device int64 [M]) behind what sequence ``seq`` holds, and return the last
        one's logits [1, vocab].  ValueError if they do not fit ``max_seq`` or the pool; then nothing
        has changed."""
        m = tokens.numel()
        if not 0 <= seq < self.n_seq:
            raise ValueError(f"sequence {seq} not in 0..{self.n_seq - 1}")
        if m == 0:
            raise ValueError("an empty prompt has no logits")
        held = int(self.lengths[seq])
        if held + m > self.cfg.max_seq:
            raise ValueError(f"sequence of {held + m} exceeds max_seq {self.cfg.max_seq}")
        rows = torch.zeros_like(self.rows)
        rows[seq] = m
        table, refs = self.tables[seq].clone(), self.refs.clone()
        self._grow(rows)
        if int(self.room[seq]) < held + m:
            self.tables[seq] = table
            self.refs.copy_(refs)
            raise ValueError(f"the pool of {self.kv.shape[1]} pages has no room for {m} more rows")
        self._prompt = seq
        try:
            pos = torch.arange(held, held + m, device=self.device)
            h = self._layers_glue(self._embed(tokens), pos, held)
        finally:
            self._prompt = None
        self.lengths[seq] += m
        s = slice(seq, seq + 1)
        self.tok[s] = self._next_tok()[s]
        self._waiting[s] = 0
        return self._proj(h[-1:], self.w.lm_head_gg, "lm_head")

    def _next_tok(self) -> torch.Tensor:
        """The tokens that the next step reads."""
        return torch.where(self.tok != 0, self.tok, self._waiting)

    @torch.no_grad()
    def step(self) -> torch.Tensor:
        """One step of every sequence with ``rows`` 1, in place: its token ``tok`` is stored in the
        next slot and the one after it takes its place.  Returns the logits [n_seq, vocab], NaN
        where a sequence did not take part.  Touches no host state, so it can be captured."""
        self._grow(self.rows)
        tok = self._next_tok()
        h = self._layers_glue(self._embed(tok), self.lengths)
        logits = self._proj(h, self.w.lm_head_gg, "lm_head")
        stored = torch.minimum(self.rows, self.room - self.lengths)
        self.lengths.add_(stored)
        takes = self.rows > 0
        # tok where it was not stored, 0 where it was
        torch.where(takes, torch.addcmul(tok, tok, stored, value=-1), self._waiting, out=self._waiting)
        self._choose(logits, takes, stored)
        return logits

    @torch.no_grad()
    def capture(self) -> "torch.cuda.CUDAGraph":
        """A HIP graph of ``step``; the cache and the sequences are as they were before."""
        if self._side is None:  # of this device, whichever is current or was captured on first
            self._side = torch.cuda.Stream(device=self.device)
        s, now = self._side, torch.cuda.current_stream(self.device)
        s.wait_stream(now)
        rows = self.rows.clone()
        with torch.cuda.stream(s):
            self.rows.zero_()
            self.step()                    # warm-up outside the graph, in which no sequence takes part
            self.rows.copy_(rows)
        now.wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.device(self.device), torch.cuda.graph(graph, stream=s):
            self._logits = self.step()
        return graph

    @torch.no_grad()
    def generate(self, prompts: Sequence[torch.Tensor], n_new: int, samples: int = 1,
                 graph: bool = True, **choice) -> dict:
        """``samples`` continuations of each prompt (device int64 [M]), ``n_new`` tokens each, from
        an empty cache; ``choice``: ``set_sampling``'s arguments, for sequence ``i * samples + j``
        the j-th continuation of prompt i, which hold until the next call of either; those that are
        not given are what ``set_sampling`` chose.  Returns their tokens [sequences, n_new] (after
        ``stop``: ``stop``), the probabilities they were drawn with, and prefill / decode timings."""
        dev, n = self.device, len(prompts) * samples
        if samples < 1 or n_new < 1 or not 0 < n <= self.n_seq:
            raise ValueError(f"{len(prompts)} prompts of {samples} continuations of {n_new} tokens for "
                             f"{self.n_seq} sequences")
        for p in prompts:
            if p.numel() == 0:
                raise ValueError("an empty prompt has no logits")
            if p.numel() + n_new - 1 > self.cfg.max_seq:
                raise ValueError(f"prompt {p.numel()} + {n_new} new tokens exceed max_seq "
                                 f"{self.cfg.max_seq}")
        page = self.kv.shape[-2]
        need = 0
        for p in prompts:  # the pages that a prompt's continuations share, and their own
            shared = p.numel() // page if n_new > 1 else -(-p.numel() // page)
            need += shared + samples * (-(-(p.numel() + n_new - 1) // page) - shared)
        if need > self.kv.shape[1]:
            raise ValueError(f"the sequences need {need} pages, the pool has {self.kv.shape[1]}")
        self._set_sampling(**{**self._chosen, **choice})
        self.reset()
        torch.cuda.synchronize(dev)
        t0 = time.perf_counter()
        first = torch.zeros(self.n_seq, self.cfg.vocab, device=dev)
        for i, p in enumerate(prompts):
            first[i * samples:(i + 1) * samples] = self.prefill(p, i * samples)
        parents = [s // samples * samples if s < n else s for s in range(self.n_seq)]
        self.fork(parents)
        self.rows[:n] = 1
        self._choose(first, self.rows > 0, self.rows)
        del first
        out = torch.empty(n_new, n, dtype=torch.int64, device=dev)
        probs = torch.empty(n_new, n, device=dev)
        out[0], probs[0] = self.tok[:n], self.probs[:n]
        torch.cuda.synchronize(dev)
        t_prefill = time.perf_counter() - t0
        replay = self.capture().replay if graph and n_new > 1 else self.step
        torch.cuda.synchronize(dev)
        t1 = time.perf_counter()
        for i in range(1, n_new):
            replay()
            out[i], probs[i] = self.tok[:n], self.probs[:n]
        torch.cuda.synchronize(dev)
        t_decode = time.perf_counter() - t1
        return {"tokens": out.t(), "probs": probs.t(), "prefill_s": t_prefill, "decode_s": t_decode,
                "decode_steps": n_new - 1, "tok_s": n * (n_new - 1) / t_decode,
                "prefill_tok_s": sum(p.numel() for p in prompts) / t_prefill}
