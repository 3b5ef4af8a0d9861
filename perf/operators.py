"""The operators of the 4-bit KV cache as measurable cases, each with its plain form.

A case is a dict of plain values with a ``kind``:

* ``attend``  one attention call of a decode loop: RoPE of the new rows' queries and keys, the
              new rows stored in the cache, attention of each query head over the slots that
              its row sees, and (``weights``) each slot's attention weight, summed over the
              rows and the query heads that share its KV head;
* ``fill``    a chunk of one or more prompts: the rows stored in the caches, and every cached
              row read back as f32 for the attention of the chunk that follows;
* ``evict``   the caches of all layers cut back to ``keep`` slots by attention weight.

A cache of one layer is ``[sequences, KV heads, slots / 32, 36 * head_dim]`` bytes.  32 slots of
a KV head form a tile: K codes, V codes, K scales, V scales.  32 channels share an f16 scale d; a
4-bit code c stands for ``d * (c - 8)``.  The bytes of a tile, with NB = head_dim / 32:

* K codes ``[slot 32][g 4][block NB][4]``: byte i holds channels 32 block + 8 g + i (low nibble)
  and + 4 + i (high nibble);
* V codes ``[group 8][n 16][block NB][slot of the group 4]``: channels 32 block + n (low nibble)
  and + 16 + n (high nibble) of slot 4 group + s;
* K scales and V scales, each ``[group 8][block NB][slot of the group 4]`` f16.

The cache's bytes are a call's state; where they are returned they are compared as they are.
"""

from __future__ import annotations

import importlib
import math
import random

import torch

own = False
DEV = "cuda"
TILE = 32


# --------------------------------------------------------------------------
# the cases
# --------------------------------------------------------------------------


def _attend(name, seqs, heads, kv, hd, slots, low, high, rows=1, weights=False):
    return dict(name=name, kind="attend", seqs=seqs, heads=heads, kv=kv, hd=hd, slots=slots,
                low=low, high=high, rows=rows, weights=weights)


def _fill(name, seqs, heads, kv, hd, slots, low, high, new_low, new_high):
    return dict(name=name, kind="fill", seqs=seqs, heads=heads, kv=kv, hd=hd, slots=slots,
                low=low, high=high, new_low=new_low, new_high=new_high)


def _evict(name, layers, seqs, kv, hd, slots, low, high, keep, recent, sinks):
    return dict(name=name, kind="evict", layers=layers, seqs=seqs, kv=kv, hd=hd, slots=slots,
                low=low, high=high, keep=keep, recent=recent, sinks=sinks)


def listed() -> list:
    return [
        # one token early in a chat, the benchmark decoder's heads and cache: latency only
        _attend("attend-300", 1, 32, 8, 128, 512, 300, 300),
        # one token over a long document
        _attend("attend-6000", 1, 32, 8, 128, 8192, 6000, 6000),
        # one token at the end of a very long context: the cache's bytes are all that counts
        _attend("attend-130000", 1, 32, 8, 128, 131072, 130000, 130000),
        # sixteen sequences of different lengths decoded together
        _attend("attend-16x4k", 16, 32, 8, 128, 4096, 37, 4095),
        # a small model without grouped heads, eight sequences
        _attend("attend-8x2k-hd64", 8, 8, 8, 64, 2048, 500, 2047),
        # wide heads, eight to a KV head, with the weights that eviction goes by
        _attend("attend-4x9k-hd256", 4, 16, 2, 256, 9216, 7001, 9001, weights=True),
        # the last 32 rows of a long prompt asked for their weights before an eviction
        _attend("window-20000", 1, 32, 8, 128, 20480, 20000, 20000, rows=32, weights=True),
        # one new token in each of two dozen short caches, read back: launches and latency
        _fill("fill-24x1", 24, 12, 4, 128, 320, 1, 300, 1, 1),
        # five packed prompts' next chunks behind what their caches hold
        _fill("fill-5x900", 5, 32, 8, 128, 2048, 0, 900, 211, 1100),
        # a cache at its limit loses one slot per step: 2049 to 2048, four layers
        _evict("evict-step", 4, 1, 8, 128, 2080, 2049, 2049, 2048, 256, 4),
        # a long prompt cut to an eighth before decoding starts, all layers of the benchmark
        _evict("evict-prompt", 32, 1, 8, 128, 16384, 15999, 15999, 2000, 250, 4),
        # a batch of long caches, some of them still below the limit
        _evict("evict-6x60k", 2, 6, 4, 64, 61440, 4000, 61001, 10007, 1000, 16),
    ]


def _log(rng, lo: float, hi: float) -> int:
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))


def _room(n: int) -> int:
    return -(-n // TILE) * TILE


def draw(rng) -> dict:
    """One more case of the same ranges; never more work than the largest listed ones."""
    kind = rng.choice(("attend",) * 6 + ("fill",) * 2 + ("evict",) * 2)
    hd = rng.choice((64, 128, 128, 128, 256))
    kv = rng.choice((1, 2, 4, 8, 8))
    heads = kv * rng.choice((1, 2, 3, 4, 4, 4, 7, 8))
    seqs = rng.choice((1, 1, 1, _log(rng, 2, 64)))
    if kind == "attend":
        most = min(131072, 131072 * 1024 // (seqs * kv * hd))
        high = _log(rng, 32, most)
        low = rng.choice((high, rng.randint(0, high)))
        rows = rng.choice((1, 1, 1, 1, _log(rng, 2, 32)))
        if rows > 1:
            high = min(high, 2600000000 // (rows * seqs * heads * hd))
            low = min(low, high)
        slots = _room(high + rows + rng.choice((0, rng.randint(0, high))))
        case = _attend("", seqs, heads, kv, hd, slots, low, high, rows, rng.random() < 0.4)
    elif kind == "fill":
        new_high = _log(rng, 1, max(8, 2800 * 1024 // (seqs * kv * hd)))
        high = rng.choice((0, rng.randint(0, 2 * new_high)))
        case = _fill("", seqs, heads, kv, hd, _room(high + new_high + rng.randint(0, 100)),
                     rng.randint(0, high), high, rng.randint(1, new_high), new_high)
    else:
        layers = rng.choice((1, 4, 32))
        high = _log(rng, 64, min(65536, 14 * 16384 * 1024 // (layers * seqs * kv * hd)))
        keep = rng.randint(1, high)
        sinks = rng.randint(0, min(8, keep))
        case = _evict("", layers, seqs, kv, hd, _room(high + rng.randint(0, 64)),
                      rng.randint(high // 2, high), high, keep,
                      rng.randint(0, (keep - sinks) // 2), sinks)
    del case["name"]
    return case


def _spread(case: dict, low: int, high: int, salt: int) -> list:
    """One length per sequence, the same for every seed."""
    rng = random.Random(1000003 * low + 101 * high + 7 * case["seqs"] + salt)
    return [rng.randint(low, high) for _ in range(case["seqs"])]


def _lengths(case: dict) -> list:
    return _spread(case, case["low"], case["high"], 0)


def _new_rows(case: dict) -> list:
    if case["kind"] == "fill":
        return _spread(case, case["new_low"], case["new_high"], 1)
    return [case.get("rows", 0)] * case["seqs"]


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------


def _quantize(x):
    """Codes (uint8, 0 .. 15) and f16 scales of f32 ``x`` in blocks of 32 channels: d is the
    element of largest magnitude (the first of several) over -8, rounded to f16, and a code is
    x / d rounded to the nearest integer, plus 8."""
    b = x.unflatten(-1, (-1, TILE))
    a, lane = b.abs(), torch.arange(TILE, device=x.device)
    at = torch.where(a == a.amax(-1, keepdim=True), lane, TILE).amin(-1, keepdim=True)
    d = (b.gather(-1, at) / -8).half()
    df = d.float()
    c = torch.where(df != 0, torch.round(b / df), torch.zeros_like(b)) + 8
    return c.clamp(0, 15).to(torch.uint8).flatten(-2), d.squeeze(-1)


def _channels_k(hd: int):
    """Channels of a slot in the order of its K code bytes: low nibbles, high nibbles."""
    nb = hd // TILE
    c = torch.arange(hd, device=DEV).reshape(nb, 4, 2, 4)          # block, g, half, i
    c = c.permute(1, 0, 3, 2).reshape(-1, 2)                        # (g, block, i), half
    return c[:, 0], c[:, 1]


def _channels_v(hd: int):
    """Channels of a slot in the order of its V code bytes: low nibbles, high nibbles."""
    nb = hd // TILE
    c = torch.arange(hd, device=DEV).reshape(nb, 2, 16).permute(2, 0, 1).reshape(-1, 2)
    return c[:, 0], c[:, 1]                                         # (n, block), half


def _places(slot, hd: int):
    """Byte offsets, within the cache of one KV head, of a slot's K codes, V codes, K scales and
    V scales (the last two as offsets of 2-byte values), along a new last dimension."""
    nb, bytes_tile = hd // TILE, 36 * hd
    slot = slot.unsqueeze(-1)
    tile, j = slot // TILE * bytes_tile, slot % TILE
    e = torch.arange(hd // 2, device=slot.device)
    b = torch.arange(nb, device=slot.device)
    k = tile + j * (hd // 2) + e
    v = tile + 16 * hd + (j // 4) * (2 * hd) + e * 4 + j % 4
    ks = tile + 32 * hd + ((j // 4) * nb + b) * 8 + (j % 4) * 2
    return k, v, ks // 2, (ks + 2 * hd) // 2


def _rope_tables(n: int, hd: int):
    """cos / sin of the angles, f64 on the device, held as f32."""
    inv = 1e6 ** (-torch.arange(hd // 2, dtype=torch.float64, device=DEV) * 2.0 / hd)
    ang = torch.arange(n, dtype=torch.float64, device=DEV)[:, None] * inv
    return ang.cos().float(), ang.sin().float()


def _gen(seed: int):
    return torch.Generator(device=DEV).manual_seed(seed)


def _cached_rows(case: dict, seed: int):
    """Codes and scales of the rows that the caches hold: K with a few strong channels."""
    g = _gen(seed + 1)
    shape = (case["seqs"], case["kv"], _room(max(_lengths(case) + [1])), case["hd"])
    strong = torch.exp(0.7 * torch.randn(case["hd"], device=DEV, generator=g))
    out = []
    for scale in (strong, 1.0):
        x = torch.randn(shape, device=DEV, generator=g) * scale
        out.append(_quantize(x))
    return out


def _pack(case: dict, rows) -> torch.Tensor:
    """A layer's cache with the cached rows in its first slots; the others hold codes of 8
    and scales of 0."""
    (kc, kd), (vc, vd) = rows
    hd, seqs, kv = case["hd"], case["seqs"], case["kv"]
    n = kc.shape[2]
    nb, t = hd // TILE, n // TILE
    kc = kc.reshape(seqs, kv, t, TILE, nb, 4, 2, 4)
    vc = vc.reshape(seqs, kv, t, 8, 4, nb, 2, 16)
    k = kc.permute(0, 1, 2, 3, 5, 4, 7, 6)                          # slot, g, block, i, half
    v = vc.permute(0, 1, 2, 3, 7, 5, 4, 6)                          # group, n, block, s, half
    parts = [(k[..., 0] | (k[..., 1] << 4)).flatten(3), (v[..., 0] | (v[..., 1] << 4)).flatten(3)]
    for d in (kd, vd):
        d = d.reshape(seqs, kv, t, 8, 4, nb).transpose(4, 5).contiguous()
        parts.append(d.view(torch.uint8).flatten(3))
    out = torch.zeros(seqs, kv, case["slots"] // TILE, 36 * hd, dtype=torch.uint8, device=DEV)
    out[..., :32 * hd] = 0x88
    out[:, :, :t] = torch.cat(parts, dim=-1)
    return out


def _qkv(case: dict, seed: int):
    """The projections' rows: queries twice as wide as the keys, so that attention picks."""
    g = _gen(seed + 2)
    heads, kv, hd = case["heads"], case["kv"], case["hd"]
    x = torch.randn(sum(_new_rows(case)), (heads + 2 * kv) * hd, device=DEV, generator=g)
    x[:, :heads * hd] *= 2
    return x


def _weights(case: dict, seed: int):
    """Accumulated attention weights of the cached slots: heavy-tailed, and zero where no row
    has looked yet."""
    g = _gen(seed + 3)
    shape = (case["layers"], case["seqs"], case["kv"], case["slots"])
    w = torch.exp(2.0 * torch.randn(shape, device=DEV, generator=g) - 6.0)
    return torch.where(torch.rand(shape, device=DEV, generator=g) < 0.05, torch.zeros_like(w), w)


def _evict_cache(case: dict, seed: int) -> torch.Tensor:
    """Every layer's cache: random codes and scales."""
    g = _gen(seed + 4)
    hd = case["hd"]
    shape = (case["layers"], case["seqs"], case["kv"], case["slots"] // TILE)
    kv = torch.randint(0, 256, (*shape, 36 * hd), dtype=torch.uint8, device=DEV, generator=g)
    d = 0.05 + 0.2 * torch.rand((*shape, 2 * hd), device=DEV, generator=g)
    kv[..., 32 * hd:] = d.half().view(torch.uint8)
    return kv


def _int64(v) -> torch.Tensor:
    return torch.tensor(v, dtype=torch.int64, device=DEV)


def prepare(case: dict, seed: int) -> dict:
    c, lengths = case, _lengths(case)
    pos = [n + 3 * (n // 40) for n in lengths]    # ahead of the slots by what evictions took
    st = dict(case=c, lengths=_int64(lengths), pos=_int64(pos))
    if c["kind"] == "evict":
        shape = (c["layers"], c["seqs"], c["kv"], c["slots"])
        steps = torch.arange(c["slots"], device=DEV)
        positions = (steps + 3 * (steps // 40)).int().expand(shape).contiguous()
        w = _weights(c, seed)
        return dict(st, kv=_evict_cache(c, seed), weights=w, positions=positions,
                    weights_out=w.clone(), positions_out=positions.clone(),
                    lengths_out=torch.empty_like(st["lengths"]), work=None)
    new = _new_rows(c)
    cos, sin = _rope_tables(max(pos) + max(new), c["hd"])
    st.update(kv=_pack(c, _cached_rows(c, seed)), qkv=_qkv(c, seed), cos=cos, sin=sin)
    if c["kind"] == "fill":
        ends = [0]
        for n in new:
            ends.append(ends[-1] + n)
        shape = (c["seqs"], c["kv"], c["slots"], c["hd"])
        return dict(st, starts=_int64(ends), filled=_int64([a + b for a, b in zip(lengths, new)]),
                    k=torch.zeros(shape, device=DEV), v=torch.zeros(shape, device=DEV))
    st["out"] = torch.empty(c["seqs"] * c["rows"], c["heads"] * c["hd"], device=DEV)
    if c["weights"]:
        st["weights"] = torch.zeros(c["seqs"], c["kv"], c["slots"], device=DEV)
    return dict(st, work=None)


# --------------------------------------------------------------------------
# the plain forms
# --------------------------------------------------------------------------


def _unpack(kv, hd: int):
    """A layer's cache as f32 keys and values [sequences, KV heads, slots, head_dim]."""
    nb = hd // TILE
    lead = kv.shape[:-1]
    k = kv[..., :16 * hd].reshape(*lead, TILE, 4, nb, 4)            # slot, g, block, i
    v = kv[..., 16 * hd:32 * hd].reshape(*lead, 8, 16, nb, 4)       # group, n, block, s
    d = kv[..., 32 * hd:].contiguous().view(torch.float16).reshape(*lead, 2, 8, nb, 4)
    d = d.transpose(-1, -2).float().reshape(*lead, 2, TILE, nb, 1)  # K / V, slot, block
    k = torch.stack([k & 15, k >> 4], dim=-2)                       # slot, g, block, half, i
    k = k.transpose(-3, -4).reshape(*lead, TILE, nb, TILE)
    v = torch.stack([v & 15, v >> 4], dim=-3)                       # group, n, half, block, s
    v = v.permute(*range(len(lead)), -5, -1, -2, -3, -4).reshape(*lead, TILE, nb, TILE)
    # [sequences, KV heads, tiles, 32, blocks, 32] -> [sequences, KV heads, slots, head_dim]
    return [((c.float() - 8) * d[..., i, :, :, :]).flatten(4, 5).flatten(2, 3)
            for i, c in enumerate((k, v))]


def _rope(x, cos, sin):
    """rotate_half RoPE of [rows, heads, head_dim]; every product and sum is rounded to f32."""
    a, b = x.chunk(2, dim=-1)
    c, s = cos.unsqueeze(1), sin.unsqueeze(1)
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def _store(kv, seq, slot, k, v, hd: int) -> None:
    """Rows [rows, KV heads, head_dim] quantized into slot ``slot`` of sequence ``seq``."""
    flat = kv.view(kv.shape[0], kv.shape[1], -1)
    halves = flat.view(torch.float16)
    at = _places(slot, hd)
    s = seq.unsqueeze(-1)
    for x, order, code_at, scale_at in ((k, _channels_k(hd), at[0], at[2]),
                                        (v, _channels_v(hd), at[1], at[3])):
        c, d = _quantize(x)
        flat[s, :, code_at] = (c[..., order[0]] | (c[..., order[1]] << 4)).transpose(1, 2)
        halves[s, :, scale_at] = d.transpose(1, 2)


def _new_kv(st: dict, row_pos):
    """The new rows' roped keys, and their values, [rows, KV heads, head_dim]."""
    c = st["case"]
    heads, kv, hd = c["heads"], c["kv"], c["hd"]
    x = st["qkv"].unflatten(1, (heads + 2 * kv, hd))
    roped = _rope(x[:, :heads + kv], st["cos"][row_pos], st["sin"][row_pos])
    return roped[:, :heads], roped[:, heads:], x[:, heads + kv:]


def _plain_attend(st: dict) -> dict:
    c = st["case"]
    seqs, rows, heads, kv, hd, slots = (c[n] for n in ("seqs", "rows", "heads", "kv", "hd",
                                                       "slots"))
    step = torch.arange(rows, device=DEV)
    seq = torch.arange(seqs, device=DEV).repeat_interleave(rows)
    slot = (st["lengths"][:, None] + step).flatten()
    q, k, v = _new_kv(st, (st["pos"][:, None] + step).flatten())
    _store(st["kv"], seq, slot, k, v, hd)
    keys, values = _unpack(st["kv"], hd)
    grp = heads // kv
    q = q.reshape(seqs, rows, kv, grp, hd).transpose(1, 2).reshape(seqs, kv, rows * grp, hd)
    s = torch.matmul(q, keys.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(hd))
    seen = torch.arange(slots, device=DEV) <= slot.reshape(seqs, rows, 1)
    seen = seen.repeat_interleave(grp, dim=1).unsqueeze(1)
    s = s.masked_fill(~seen, -math.inf)
    p = torch.exp(s - s.max(dim=-1, keepdim=True).values)
    p = p / p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p, values).reshape(seqs, kv, rows, grp, hd).transpose(1, 2)
    got = dict(out=o.reshape(seqs * rows, heads * hd), kv=st["kv"])
    if c["weights"]:
        got["weights"] = p.sum(dim=2)
    return got


def _plain_fill(st: dict) -> dict:
    c = st["case"]
    r = torch.arange(st["qkv"].shape[0], device=DEV)
    seq = torch.bucketize(r, st["starts"][1:], right=True)
    i = r - st["starts"][seq]
    _, k, v = _new_kv(st, st["pos"][seq] + i)
    _store(st["kv"], seq, st["lengths"][seq] + i, k, v, c["hd"])
    held = torch.arange(c["slots"], device=DEV) < st["filled"][:, None]
    held = held[:, None, :, None]
    keys, values = _unpack(st["kv"], c["hd"])
    return dict(k=keys * held, v=values * held)


def _plain_evict(st: dict) -> dict:
    c = st["case"]
    keep, slots = c["keep"], c["slots"]
    at = torch.arange(slots, device=DEV)
    lengths = st["lengths"][:, None, None]
    held = at < lengths
    p = st["positions"]
    last = (st["pos"] - c["recent"])[:, None, None]
    score = torch.where((p < c["sinks"]) | (p >= last), math.inf, st["weights"])
    score = torch.where(held, score, -math.inf)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, at.expand_as(order).contiguous())
    kept = held & ((rank < keep) | (lengths <= keep))
    hole, moved = ~kept & (at < keep) & held, kept & (at >= keep) & (lengths > keep)
    behind = torch.sort((~moved).byte(), dim=-1, stable=True).indices   # the moved ones first
    src = behind.gather(-1, (hole.cumsum(-1) - 1).clamp(min=0))
    src = torch.where(hole, src, at)[..., :keep]
    now = torch.minimum(st["lengths"], torch.tensor(keep, device=DEV))
    live = at[:keep] < now[:, None, None]
    out = dict(kv=st["kv"], lengths=now)
    for n in ("weights", "positions"):
        t = st[n].clone()
        t[..., :keep] = torch.where(live, t.gather(-1, src), t[..., :keep])
        out[n] = t
    flat = st["kv"].flatten(3)
    halves = flat.view(torch.float16)
    dst_at, src_at = _places(at[:keep], c["hd"]), _places(src, c["hd"])
    for i, buf in ((0, flat), (1, flat), (2, halves), (3, halves)):
        here = dst_at[i].flatten()
        buf[..., here] = buf.gather(-1, src_at[i].flatten(3))
    return out


# --------------------------------------------------------------------------
# what is measured
# --------------------------------------------------------------------------


def run(state: dict):
    st, c = state, state["case"]
    if not own:
        return {"attend": _plain_attend, "fill": _plain_fill, "evict": _plain_evict}[c["kind"]](st)
    kv4 = importlib.import_module("artifex-assistantv5_amd.kv4")
    if c["kind"] == "attend":
        if st["work"] is None:
            st["work"] = kv4.attention_workspace(st["kv"], c["heads"], rows=c["rows"],
                                                 weights=c["weights"])
        kv4.attention(st["qkv"], st["lengths"], st["pos"], st["cos"], st["sin"], st["kv"],
                      st["out"], c["heads"], st["work"], weights=st.get("weights"))
        got = dict(out=st["out"], kv=st["kv"])
        if c["weights"]:
            got["weights"] = st["weights"]
        return got
    if c["kind"] == "fill":
        kv4.append(st["qkv"], st["lengths"], st["pos"], st["cos"], st["sin"], st["kv"],
                   c["heads"], starts=st["starts"])
        kv4.load(st["kv"], st["filled"], st["k"], st["v"])
        return dict(k=st["k"], v=st["v"])
    if st["work"] is None:
        st["work"] = kv4.evict_workspace(st["kv"])
    kv4.evict(st["kv"], st["weights"], st["positions"], st["lengths"], st["pos"], c["keep"],
              st["work"], recent=c["recent"], sinks=c["sinks"], weights_out=st["weights_out"],
              positions_out=st["positions_out"], lengths_out=st["lengths_out"])
    return dict(kv=st["kv"], weights=st["weights_out"], positions=st["positions_out"],
                lengths=st["lengths_out"])


def _exact_evict(c: dict, seed: int) -> dict:
    """The weights after the eviction, one list of slots at a time."""
    weights, lengths, keep = _weights(c, seed).double().cpu(), _lengths(c), c["keep"]
    for layer in weights:
        for n, heads in zip(lengths, layer):
            if n <= keep:
                continue
            at = torch.arange(n)
            p = at + 3 * (at // 40)
            stays = (p < c["sinks"]) | (p >= n + 3 * (n // 40) - c["recent"])
            for w in heads:
                # ascending by (-weight, slot): the first `keep` stay
                order = torch.sort(-w[:n].masked_fill(stays, math.inf), stable=True).indices
                stay = order[:keep]
                holes = torch.sort(order[keep:][order[keep:] < keep]).values
                w[holes] = w[torch.sort(stay[stay >= keep]).values].clone()
    return dict(kv=None, weights=weights, positions=None, lengths=None)


def exact(case: dict, seed: int):
    """The definition in 64 bits from the inputs' own codes, one sequence and head at a time."""
    c = case
    if c["kind"] == "evict":
        return _exact_evict(c, seed)
    heads, kv, hd, lengths, new = c["heads"], c["kv"], c["hd"], _lengths(c), _new_rows(c)
    held = _cached_rows(c, seed)
    x = _qkv(c, seed).double().unflatten(1, (heads + 2 * kv, hd))
    pos = [n + 3 * (n // 40) for n in lengths]
    cos, sin = _rope_tables(max(p + n for p, n in zip(pos, new)), hd)
    shape = (c["seqs"], kv, c["slots"], hd)
    if c["kind"] == "fill":
        got = [torch.zeros(shape, dtype=torch.float64, device=DEV) for _ in range(2)]
    else:
        out = torch.empty(c["seqs"], c["rows"], heads, hd, dtype=torch.float64, device=DEV)
        weights = torch.zeros(shape[:3], dtype=torch.float64, device=DEV)
    first = 0
    for s, (n, m, p) in enumerate(zip(lengths, new, pos)):
        turn = torch.complex(cos[p:p + m].double(), sin[p:p + m].double())[:, None]
        y = x[first:first + m]
        z = torch.complex(y[:, :heads + kv, :hd // 2], y[:, :heads + kv, hd // 2:]) * turn
        roped = torch.cat([z.real, z.imag], dim=-1)
        first += m
        for h in range(kv):
            rows = []
            for i, fresh in enumerate((roped[:, heads + h], y[:, heads + kv + h])):
                codes, d = held[i][0][s, h, :n].double(), held[i][1][s, h, :n].double()
                old = ((codes.view(n, hd // TILE, TILE) - 8) * d[..., None]).view(n, hd)
                b = fresh.reshape(m, hd // TILE, TILE)
                big = b.abs().argmax(-1, keepdim=True)
                e = (b.gather(-1, big) / -8).float().half().double()
                q = torch.where(e != 0, torch.round(b / e).clamp(-8, 7), torch.zeros_like(b))
                rows.append(torch.cat([old, (q * e).reshape(m, hd)]))
            if c["kind"] == "fill":
                for i in range(2):
                    got[i][s, h, :n + m] = rows[i]
                continue
            grp = heads // kv
            q = roped[:, h * grp:(h + 1) * grp].reshape(m * grp, hd)
            score = q @ rows[0].t().contiguous() / math.sqrt(hd)
            sees = n + torch.arange(m, device=DEV).repeat_interleave(grp)
            score[torch.arange(n + m, device=DEV) > sees[:, None]] = -math.inf
            prob = torch.softmax(score, dim=-1)
            out[s, :, h * grp:(h + 1) * grp] = (prob @ rows[1]).reshape(m, grp, hd)
            weights[s, h, :n + m] = prob.sum(0)
    if c["kind"] == "fill":
        return dict(k=got[0], v=got[1])
    return dict(out=out.reshape(c["seqs"] * c["rows"], heads * hd), kv=None,
                **({"weights": weights} if c["weights"] else {}))


def work(case: dict) -> dict:
    c, lengths, new = case, _lengths(case), _new_rows(case)
    kv, hd = c["kv"], c["hd"]
    slot = 9 * hd // 8                                     # bytes of a slot's codes and scales
    if c["kind"] == "evict":
        total = 0
        for n in lengths:
            total += 8 * n                                 # weights and positions read
            if n > c["keep"]:
                # the slots behind `keep` that stay: the recent ones, and of the others as
                # many as their share; each is read and written with its weight and position
                rest = max(0, n - c["recent"])
                late = max(0, rest - c["keep"])
                free = c["keep"] - min(n, c["recent"])
                moved = min(n - c["keep"], c["recent"]) + free * late / max(1, rest)
                total += moved * 2 * slot + 8 * min(n, c["keep"])
        return dict(bytes=c["layers"] * kv * total, flops=0)
    rows, seen = sum(new), sum(lengths) + sum(new)
    if c["kind"] == "fill":
        return dict(bytes=rows * 8 * kv * hd + seen * kv * (slot + 8 * hd), flops=rows * 6 * kv * hd)
    heads, m = c["heads"], c["rows"]
    pairs = sum(m * n + m * (m + 1) // 2 for n in lengths)
    return dict(bytes=seen * kv * (slot + (4 if c["weights"] else 0))
                + rows * 4 * (2 * heads + 2 * kv) * hd, flops=4 * pairs * heads * hd)
