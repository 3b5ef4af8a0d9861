"""The KV cache in pages on the GPU against the plain restatement of paged_model.py.

Tolerances.  Stored rows, tables, counts, moved bytes and read-back values are equal.  An
attention output differs from float64 by what its roundings allow:
* a query channel after RoPE and scaling: four f32 roundings of terms of up to |x1 c| + |x2 s|,
  and its parts (2^-22 of it, or 2^-35 of the row's largest): below 2^-21 of the terms' sum plus
  2^-35 of the largest;
* a score: at most 2 head_dim / 32 + 1 accumulations and a rotation's addition, each with the
  rounding of a few f32 sums, below (2 head_dim / 32 + 2) 2^-22 of sum |q| |k|;
together an error e of the score, a factor within 1 +- 2 e of each p.  The exponential (2^-22), p's
parts (2^-22), sums over up to n / 32 units of p and p v (2^-23 each) and the division (2^-23) add
(n / 32 + 8) 2^-23.  Both act on sum p |v|, once above and once below the fraction.
"""
import importlib
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import paged_model as model  # noqa: E402

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def paged(pkg):
    return importlib.import_module("artifex-assistantv5_amd.paged")


def _tables(n, hd, base=10000.0):
    inv = base ** (-np.arange(hd // 2) * 2.0 / hd)
    ang = np.arange(n)[:, None] * inv
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


def _cuda(x, dtype=None):
    return torch.tensor(np.asarray(x), dtype=dtype, device="cuda")


def _i64(v):
    return _cuda(v, torch.int64)


def _bits(t):
    return t.cpu().view(torch.int16)


def _pool(rng, n_pages, kv, page, hd, dtype, waste=float("nan")):
    """A CPU pool: random pages; ``waste`` is put behind the sequences' ends by the caller."""
    x = rng.standard_normal((n_pages, 2, kv, page, hd)).astype(np.float32)
    x[:, 0] *= np.exp(0.5 * rng.standard_normal(hd)).astype(np.float32)
    return torch.from_numpy(x).to(dtype)


def _spoil(pool, tables, lengths, value=float("nan")):
    """Every slot that no sequence uses holds ``value``."""
    n_pages, _, kv, page, hd = pool.shape
    used = np.zeros((n_pages, page), bool)
    for table, n in zip(tables, lengths):
        for c in range(-(-max(0, n) // page)):
            if 0 <= table[c] < n_pages:
                used[table[c], :max(0, min(page, n - c * page))] = True
    for p in range(n_pages):
        for j in np.flatnonzero(~used[p]):
            for h in range(kv):
                model.put(pool, p, h, j, torch.full((hd,), value), torch.full((hd,), value))


def _store(pool, table, slot, row, cos, sin, heads, kv, hd):
    """The new row of a sequence into a CPU pool."""
    page = pool.shape[3]
    x = row.reshape(heads + 2 * kv, hd)
    for h in range(kv):
        k = model.rounded(model.rope(x[heads + h], cos[slot], sin[slot]), pool.dtype)
        v = model.rounded(x[heads + kv + h], pool.dtype)
        model.put(pool, int(table[slot // page]), h, slot % page, k, v)


def _stored(table, slot, columns, page, n_pages, rope_rows, room=None):
    return (0 <= slot < min(columns * page, rope_rows, columns * page if room is None else room)
            and 0 <= table[slot // page] < n_pages)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv,hd,page,lengths,starts,rows,rope,room", [
    (8, 2, 128, 16, [0, 15, 40], [0, 1, 40, 64], 64, 150, None),       # packed prompts
    (4, 4, 64, 32, [5, 0, 63, 64], [0, 3, 3, 5, 9], 12, 150, None),    # an empty one, padding rows
    (8, 1, 256, 64, [30, 9], [2, 9, 12], 14, 33, None),                # RoPE tables end first
    (6, 2, 128, 16, [-1, 3, 20], None, 9, 150, [100, 5, -7]),          # the same number each; room
    (2, 2, 64, 16, [1, 1], [-(1 << 62), 3, 5], 6, 150, None),          # starts far before the rows
    # by whole blocks: aligned and not, empty ones, padding rows, what ends first, many heads
    (2, 2, 64, 16, [0, 16, 3, 9], [0, 32, 64, 64, 67], 70, 150, None),
    (9, 9, 128, 32, [7, -1, 60], [-5, 20, 30, 61], 60, 70, None),
    (8, 1, 256, 64, [30, 9], [2, 40, 102], 110, 230, [55, 1 << 40]),
    (4, 4, 64, 16, [70, 2, 11], None, 90, 150, [80, -(1 << 62), 30]),
    (2, 2, 64, 16, [1, 1, 5], [-(1 << 62), -3, 5, 1 << 62], 48, 150, None),
])
def test_append_is_exact(paged, dtype, heads, kv, hd, page, lengths, starts, rows, rope, room):
    rng = np.random.default_rng(hd + rows)
    seqs, columns, n_pages = len(lengths), 5, 24
    cos, sin = _tables(rope, hd)
    tables, _ = model.shared_tables(rng, seqs, columns, n_pages, [columns - 1] * seqs, 0)
    tables[0, 1] = n_pages + 3                                        # names no page
    qkv = rng.standard_normal((rows, (heads + 2 * kv) * hd + 4)).astype(np.float32) * 3
    qkv[0, heads * hd:][:4] = (70000.0, -65519.0, 1e-9, 0.0)          # f16: infinite, the last finite
    pool = _pool(rng, n_pages, kv, page, hd, TYPES[dtype])
    dev = pool.cuda()
    paged.append(_cuda(qkv)[:, :-4], _i64(lengths), _cuda(tables), _cuda(cos), _cuda(sin), dev, heads,
                 starts=None if starts is None else _i64(starts),
                 room=None if room is None else _i64(room))
    at = starts or [s * (rows // seqs) for s in range(seqs + 1)]
    for s, n in enumerate(lengths):
        for r in range(max(0, at[s]), min(at[s + 1], rows)):
            slot = n + r - at[s]
            if n >= 0 and _stored(tables[s], slot, columns, page, n_pages, rope,
                                  None if room is None else room[s]):
                _store(pool, tables[s], slot, qkv[r, :-4], cos, sin, heads, kv, hd)
    assert torch.equal(_bits(dev), _bits(pool))


def test_append_without_rows(paged):
    kv = paged.empty(4, 2, 64)
    t, n, _ = paged.empty_tables(2, 3, 4)
    cos, sin = (_cuda(x) for x in _tables(8, 64))
    paged.append(torch.empty(0, 6 * 64, device="cuda"), n, t, cos, sin, kv, 2)
    paged.append(torch.ones(2, 6 * 64, device="cuda"), n, t, cos, sin, kv, 2)   # no pages
    assert not kv.any()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hd,page,out_slots,lengths", [(64, 16, 80, [0, 1, 79]),
                                                      (128, 32, 40, [64, 39, -1]),
                                                      (256, 64, 250, [191, 7, 300])])
def test_load(paged, dtype, hd, page, out_slots, lengths):
    """Rows 0 .. min(length, out_slots) - 1; nothing behind them or without a page is written."""
    rng = np.random.default_rng(hd)
    columns, n_pages, kv = 192 // page if page > 16 else 5, 40, 2
    tables, _ = model.shared_tables(rng, 3, columns, n_pages, [columns] * 3, 1)
    tables[1, 0] = -1
    pool = _pool(rng, n_pages, kv, page, hd, TYPES[dtype])
    k = torch.full((3, kv, out_slots, hd), 9.0, device="cuda")
    v = k.clone()
    paged.load(pool.cuda(), _cuda(tables), _i64(lengths), k, v)
    want = np.full((2, 3, kv, out_slots, hd), 9.0)
    for s, n in enumerate(lengths):
        n = max(0, min(n, out_slots, columns * page))
        for h in range(kv):
            a, b, there = model.rows(pool, tables[s], n, h)
            want[0, s, h, :n][there], want[1, s, h, :n][there] = a[there], b[there]
    assert np.array_equal(k.cpu().double().numpy(), want[0])
    assert np.array_equal(v.cpu().double().numpy(), want[1])


def _reference(pool, tables, lengths, qkv, cos, sin, heads, kv, hd, room=None):
    """The pool after the call, outputs [seqs, heads, hd] (NaN where none) and their bounds."""
    n_pages, _, _, page, _ = pool.shape
    pool, seqs, columns, grp = pool.clone(), len(lengths), tables.shape[1], heads // kv
    takes = [_stored(tables[s], n, columns, page, n_pages, cos.shape[0],
                     None if room is None else room[s]) for s, n in enumerate(lengths)]
    for s, n in enumerate(lengths):
        if takes[s]:
            _store(pool, tables[s], n, qkv[s], cos, sin, heads, kv, hd)
    out, bound = np.full((2, seqs, heads, hd), np.nan)
    half = hd // 2
    for s, n in enumerate(lengths):
        if not takes[s]:
            continue
        c, t = cos[n].astype(np.float64), sin[n].astype(np.float64)
        for h in range(heads):
            x = qkv[s].reshape(heads + 2 * kv, hd)[h].astype(np.float64)
            q = np.concatenate([x[:half] * c - x[half:] * t, x[half:] * c + x[:half] * t])
            terms = np.tile(np.abs(x[:half]) + np.abs(x[half:]), 2)
            k, v, there = model.rows(pool, tables[s], n + 1, h // grp)
            o, spread = model.attend(q, k, v, there)
            ka = np.abs(k[there])
            e = (ka @ (terms * 2.0 ** -21 + np.abs(q).max() * 2.0 ** -35)
                 + (2 * hd / 32 + 2) * 2.0 ** -22 * (ka @ np.abs(q))).max() / math.sqrt(hd)
            out[s, h] = o
            bound[s, h] = 2 * (2 * e + (n / 32 + 8) * 2.0 ** -23) * spread + 1e-30
    return pool, out, bound


def _attend(paged, pool, tables, lengths, qkv, cos, sin, heads, out=None, room=None):
    dev = pool.cuda()
    n = len(lengths)
    out = torch.full((n, heads * pool.shape[-1]), float("nan"), device="cuda") if out is None else out
    t = _cuda(tables)
    work = paged.attention_workspace(dev, t, heads)
    work.fill_(0xFF)
    paged.attention(qkv, _i64(lengths), t, _cuda(cos), _cuda(sin), dev, out, heads, work,
                    room=None if room is None else _i64(room))
    return dev, out


CASES = [
    # heads, kv, hd, page, lengths, shared columns
    (8, 2, 128, 16, [0], 0),                                # only itself
    (4, 4, 64, 16, [1, 14, 15, 16, 17], 0),                 # around a page's end
    (3, 1, 128, 32, [30, 31, 32, 33], 1),                   # around a unit's end
    (32, 8, 128, 16, [300], 0),
    (8, 1, 256, 64, [63, 64, 200, 0], 1),
    (7, 1, 64, 128, [500, 127, 128], 0),                    # seven heads of eight columns
    (16, 2, 256, 256, [255, 256, 700], 0),
    (12, 4, 128, 16, [5, 900, 33, 0, 64, 257, 128], 0),     # many splits next to one
    (2, 2, 64, 16, [2049], 3),
]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv,hd,page,lengths,shared", CASES)
def test_attention(paged, dtype, heads, kv, hd, page, lengths, shared):
    """Against float64; what the sequences do not use is NaN, as is the rest of the tables' pages."""
    rng = np.random.default_rng(sum(lengths) + hd)
    seqs = len(lengths)
    used = [n // page + 1 for n in lengths]
    columns = max(used) + 1
    n_pages = sum(used) + 3
    tables, _ = model.shared_tables(rng, seqs, columns, n_pages, used,
                                    min(shared, min(n // page for n in lengths)))
    pool = _pool(rng, n_pages, kv, page, hd, TYPES[dtype])
    _spoil(pool, tables, lengths)
    cos, sin = _tables(max(lengths) + 1, hd)
    qkv = rng.standard_normal((seqs, (heads + 2 * kv) * hd)).astype(np.float32)
    qkv[:, :heads * hd] *= 2
    dev, out = _attend(paged, pool, tables, lengths, _cuda(qkv), cos, sin, heads)
    want_pool, want, bound = _reference(pool, tables, lengths, qkv, cos, sin, heads, kv, hd)
    assert torch.equal(_bits(dev), _bits(want_pool))
    err = np.abs(out.cpu().double().numpy().reshape(want.shape) - want)
    assert (err <= bound).all(), (err / bound).max()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attention_who_takes_part(paged, dtype):
    """Negative lengths, full tables, no page, room, RoPE tables that end; pages missing among the
    slots; strides of qkv and out; the rest of out and of the pages stays."""
    rng = np.random.default_rng(7)
    heads, kv, hd, page, columns, n_pages = 6, 2, 64, 16, 6, 60
    lengths = [-1, 96, 40, 95, 16, 70, 50, 33, 1 << 40, -(1 << 62), 60]
    room = [96, 96, 96, 96, 16, 71, 64, 96, 96, 96, -5]
    tables = (np.arange(columns) + 5 * np.arange(len(lengths))[:, None]).astype(np.int32) % n_pages
    tables[2, 2] = -1                                     # 40: no page for the row
    tables[5, 1], tables[5, 3] = n_pages, -(1 << 31)      # pages missing before the row
    tables[6, 0] = -1
    tables[7, 0], tables[7, 1] = -1, -1                   # none but the row's
    for i, s in enumerate((3, 5, 6, 7)):                  # those that store have pages of their own
        ok = (tables[s] >= 0) & (tables[s] < n_pages)
        tables[s][ok] = (36 + 6 * i + np.arange(columns))[ok]
    pool = _pool(rng, n_pages, kv, page, hd, TYPES[dtype])
    cos, sin = _tables(96, hd)
    qkv = rng.standard_normal((len(lengths), (heads + 2 * kv) * hd + 8)).astype(np.float32)
    wide = torch.full((len(lengths), heads * hd + 4), 5.0, device="cuda")
    dev, _ = _attend(paged, pool, tables, lengths, _cuda(qkv)[:, :-8], cos, sin, heads,
                     out=wide[:, :-4], room=room)
    want_pool, want, bound = _reference(pool, tables, lengths, qkv[:, :-8], cos, sin, heads, kv, hd,
                                        room=room)
    assert torch.equal(_bits(dev), _bits(want_pool))
    got = wide.cpu().double().numpy()
    assert (got[:, -4:] == 5).all()
    got = got[:, :-4].reshape(want.shape)
    takes = ~np.isnan(want[:, 0, 0])
    assert takes.tolist() == [n in (95, 70, 50, 33) for n in lengths]
    assert (got[~takes] == 5).all()
    err = np.abs(got - want)[takes]
    assert (err <= bound[takes]).all(), (err / bound[takes]).max()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attention_extremes(paged, dtype):
    """Scores that differ by hundreds, a slot of weight one far from the others; zeros; a NaN or an
    infinity in a slot reaches the sequence and KV head that see it and no other."""
    rng = np.random.default_rng(3)
    heads, kv, hd, page, lengths = 4, 2, 128, 16, [200, 200, 200]
    columns = n = 13
    tables, _ = model.shared_tables(rng, 3, columns, 3 * n, [n] * 3, 0)
    pool = _pool(rng, 3 * n, kv, page, hd, TYPES[dtype])
    cos, sin = _tables(201, hd)
    qkv = rng.standard_normal((3, (heads + 2 * kv) * hd)).astype(np.float32)
    qkv[0, :heads * hd] *= 60                              # one slot takes it all
    qkv[1] = 0                                             # all alike
    dev, out = _attend(paged, pool, tables, lengths, _cuda(qkv), cos, sin, heads)
    want_pool, want, bound = _reference(pool, tables, lengths, qkv, cos, sin, heads, kv, hd)
    assert torch.equal(_bits(dev), _bits(want_pool))
    err = np.abs(out.cpu().double().numpy().reshape(want.shape) - want)
    assert (err <= bound).all(), (err / bound).max()
    for value in (float("nan"), float("inf")):
        bad = pool.clone()
        bad[tables[1, 3], 0, 1, 5, 7] = value              # K of sequence 1, KV head 1
        bad[tables[2, 4], 1, 0].view(-1, hd, 16)[0, 9, 2] = value  # V of sequence 2, head 0, channel 9
        _, got = _attend(paged, bad, tables, lengths, _cuda(qkv), cos, sin, heads)
        got, out_ = got.cpu().reshape(3, heads, hd), out.cpu().reshape(3, heads, hd)
        assert torch.equal(got[0], out_[0]) and torch.equal(got[1, :2], out_[1, :2])
        assert not torch.isfinite(got[1, 2:]).any()
        assert torch.equal(got[2, 2:], out_[2, 2:])
        rest = torch.arange(hd) != 9
        assert torch.equal(got[2, :2][:, rest], out_[2, :2][:, rest])
        assert not torch.isfinite(got[2, :2, 9]).any()


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("n_seq,columns,n_pages", [(1, 1, 1), (7, 5, 40), (64, 300, 20000),
                                                   (4096, 3, 9000), (3, 70000, 150000)])
def test_fork(paged, in_place, n_seq, columns, n_pages):
    rng = np.random.default_rng(n_seq)
    used = rng.integers(0, columns + 1, n_seq).tolist()
    while sum(used) > n_pages:
        used = [u // 2 for u in used]
    tables, refs = model.shared_tables(rng, n_seq, columns, n_pages, used, 0)
    lengths = rng.integers(0, 1000, n_seq)
    t, n, r = _cuda(tables), _i64(lengths), _cuda(refs)
    for turn in range(3):                                  # shared pages from the second turn on
        parents = rng.integers(-1, n_seq + 1, n_seq)
        parents = np.where(rng.random(n_seq) < 0.3, np.arange(n_seq), parents)
        if n_seq > 4:
            parents[:2] = (1, 0)                           # a swap, and values far outside
            parents[2:4] = (1 << 40, -(1 << 62))
        want = model.fork(tables, lengths, refs, parents.tolist())
        if in_place:
            paged.fork(t, n, r, _i64(parents))
        else:
            before = [x.clone() for x in (t, n, r)]
            outs = [torch.full_like(x, -9) for x in (t, n, r)]
            paged.fork(t, n, r, _i64(parents), *outs)
            for x, y in zip((t, n, r), before):
                assert torch.equal(x, y)
            t, n, r = outs
        for got, w in zip((t, n, r), want):
            assert np.array_equal(got.cpu().numpy(), w)
        tables, lengths, refs = want


def _grow_case(paged, rng, tables, lengths, refs, rows, page, layers, kv=2, hd=64,
               dtype=torch.float16):
    n_pages = len(refs)
    pool = torch.stack([_pool(rng, n_pages, kv, page, hd, dtype) for _ in range(layers)])
    dev, t, r = pool.cuda(), _cuda(tables), _cuda(refs)
    room = torch.full((len(lengths),), -9, dtype=torch.int64, device="cuda")
    work = paged.grow_workspace(dev, t)
    work.fill_(0xFF)
    paged.grow(dev, t, _i64(lengths), r, _i64(rows), room, work)
    wt, wr, wroom, copies = model.grow(tables, np.asarray(lengths), refs, rows, page)
    assert np.array_equal(t.cpu().numpy(), wt)
    assert np.array_equal(r.cpu().numpy(), wr)
    assert np.array_equal(room.cpu().numpy(), wroom)
    want = pool.clone()
    for src, dst, blocks in copies:
        want[:, dst, :, :, :16 * blocks] = pool[:, src, :, :, :16 * blocks]   # whole blocks: K's rows
    assert torch.equal(_bits(dev), _bits(want))
    return wt, wr


@pytest.mark.parametrize("page", [16, 64, 256])
def test_grow(paged, page):
    """New pages, copies of shared ones, prompts of many pages, sequences that need none."""
    rng = np.random.default_rng(page)
    lengths = [0, 5, page - 1, page, page + 20, 3 * page, -1, 2 * page + 1, 7 * page]
    rows = [1, 0, 1, 1, 4 * page, 3, 5, -2, 4]
    used = [-(-max(n, 0) // page) for n in lengths]
    tables, refs = model.shared_tables(rng, len(lengths), 7, 60, used, 0)
    tables, refs = _grow_case(paged, rng, tables, lengths, refs, rows, page, 3)
    # forks of sequence 4 on every place that holds nothing else: their last pages are shared
    lengths = np.array([max(n, 0) for n in lengths])
    tables, lengths, refs = model.fork(tables, lengths, refs, [4, 1, 4, 3, 4, 4, -1, 7, 4])
    _grow_case(paged, rng, tables, lengths.tolist(), refs, [1] * 9, page, 2)
    _grow_case(paged, rng, tables, lengths.tolist(), refs, [0, 1, page, 0, 3, 0, 1, 1, 1], page, 1)


def test_grow_many_sequences_and_entries(paged):
    """More entries than one turn takes, free pages found over several turns."""
    rng = np.random.default_rng(5)
    n = 1500
    lengths = rng.integers(0, 100, n)
    used = [-(-int(x) // 16) for x in lengths]
    tables, refs = model.shared_tables(rng, n, 12, 30000, used, 0)
    parents = rng.integers(0, n, n)
    tables, lengths, refs = model.fork(tables, lengths, refs, parents.tolist())
    _grow_case(paged, rng, tables, lengths.tolist(), refs, rng.integers(-1, 70, n).tolist(), 16, 1, kv=1)


@pytest.mark.parametrize("free", [[39999], [3, 16383, 16384, 16385, 39000], list(range(20000, 22300))])
def test_grow_in_a_large_pool(paged, free):
    """The lowest free pages wherever they are, over several turns of entries; too few at the end."""
    rng = np.random.default_rng(len(free))
    refs = np.full(40000, 2, np.int32)                 # held elsewhere too
    refs[free] = 0
    refs[free[0]] = -1                                 # counts as free
    n = 1100
    tables = np.full((n, 3), -1, np.int32)
    tables[::2, 0] = rng.choice(np.flatnonzero(refs > 0), n // 2)
    _grow_case(paged, rng, tables, [5] * n, refs, [30] * n, 16, 1, kv=1)


@pytest.mark.parametrize("spare", [0, 1, 2, 5, 9])
def test_grow_when_the_pool_runs_out(paged, spare):
    """Sequences in order get what is left; a page that its other holders could not leave stays
    shared and is not to be written."""
    rng = np.random.default_rng(spare)
    tables = np.array([[0, 1, -1, -1], [0, 1, -1, -1], [0, 1, -1, -1], [0, 2, -1, -1],
                       [3, -1, -1, -1], [0, 1, -1, -1]], np.int32)
    refs = np.zeros(4 + spare, np.int32)
    refs[:4] = (5, 4, 1, 1)
    _grow_case(paged, rng, tables, [20, 20, 32, 25, 16, 20], refs, [1, 1, 1, 30, 40, 1], 16, 2)


@pytest.mark.parametrize("spare", [1, 2, 3])
def test_grow_keeps_what_the_others_left(paged, spare):
    """Sequences 0 and 3 hold one page each with 2 and 4; 1 takes what the pool has left.  Where 0 could
    leave its page, 2 keeps it alone, whatever the pool holds then; so do 3 and 4."""
    rng = np.random.default_rng(spare)
    tables = np.array([[0, -1, -1], [1, -1, -1], [0, -1, -1], [2, -1, -1], [2, -1, -1]], np.int32)
    refs = np.zeros(3 + spare, np.int32)
    refs[:3] = (2, 1, 2)
    _grow_case(paged, rng, tables, [7, 16, 9, 3, 12], refs, [1, 32, 1, 2, 3], 16, 2)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("n_pages,share,layers,page,hd", [(1, 1.0, 1, 16, 64), (50, 0.0, 2, 16, 64),
                                                          (50, 0.5, 2, 32, 128),
                                                          (3001, 0.3, 1, 16, 64), (40003, 0.4, 1, 16, 64),
                                                          (300, 0.97, 3, 16, 256)])
def test_compact(paged, in_place, n_pages, share, layers, page, hd):
    rng = np.random.default_rng(n_pages)
    n_seq, kv = 5, 1
    used = [int(n_pages * share) // n_seq + (n_pages == 1 and s == 0) for s in range(n_seq)]
    tables, refs = model.shared_tables(rng, n_seq, max(used) + 2, n_pages, used, min(2, min(used)))
    tables[0, -1] = n_pages + 5                            # names no page: stays as it is
    refs = np.bincount(tables[(tables >= 0) & (tables < n_pages)], minlength=n_pages).astype(np.int32)
    pool = torch.stack([_pool(rng, n_pages, kv, page, hd, torch.bfloat16) for _ in range(layers)])
    dev, t, r = pool.cuda(), _cuda(tables), _cuda(refs)
    live = _i64([-1])
    work = paged.compact_workspace(dev, t)
    work.fill_(0xFF)
    outs = {} if in_place else dict(tables_out=torch.full_like(t, -9), refs_out=torch.full_like(r, -9))
    paged.compact(dev, t, r, live, work, **outs)
    wt, wr, wlive, moves = model.compact(tables, refs)
    assert np.array_equal(outs.get("tables_out", t).cpu().numpy(), wt)
    assert np.array_equal(outs.get("refs_out", r).cpu().numpy(), wr)
    assert live.item() == wlive
    if not in_place:
        assert np.array_equal(t.cpu().numpy(), tables) and np.array_equal(r.cpu().numpy(), refs)
    want = pool.clone()
    for src, dst in moves:
        want[:, dst] = pool[:, src]
    assert torch.equal(_bits(dev), _bits(want))


def test_refusals(paged):
    kv = paged.empty(8, 2, 64, n_layers=2)
    t, n, r = paged.empty_tables(3, 4, 8)
    cos, sin = (_cuda(x) for x in _tables(64, 64))
    q, out = torch.zeros(3, 8 * 64, device="cuda"), torch.zeros(3, 4 * 64, device="cuda")
    work = paged.attention_workspace(kv[0], t, 4)
    call = lambda **o: paged.attention(**{**dict(qkv=q, lengths=n, tables=t, cos=cos, sin=sin,  # noqa: E731
                                                 kv=kv[0], out=out, n_heads=4, work=work), **o})
    call()
    for bad in (dict(qkv=q[:2]), dict(out=out[:2]), dict(lengths=n[:2]), dict(lengths=n.int()),
                dict(tables=t.long()), dict(tables=t[:, :3]), dict(tables=t[0]), dict(cos=cos[:5]),
                dict(sin=sin.double()), dict(kv=kv), dict(kv=kv[0].float()), dict(qkv=q.half()),
                dict(kv=kv[0, :, :, :, :8]), dict(work=work[:0]), dict(n_heads=17), dict(room=n[:1]),
                dict(qkv=q.t()), dict(work=work.cpu()), dict(out=out.cpu())):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(ValueError):
        paged.append(q, n, t, cos, sin, kv[0], 4, starts=n)
    with pytest.raises(ValueError):
        paged.load(kv[0], t, n, torch.zeros(3, 2, 5, 64, device="cuda"), torch.zeros(3, 2, 6, 64, device="cuda"))
    with pytest.raises(ValueError):
        paged.fork(t, n, r, n.int())
    with pytest.raises(ValueError, match="overlaps"):
        big = torch.zeros(4, 4, dtype=torch.int32, device="cuda")
        paged.fork(big[:3], n, r, n, tables_out=big[1:])
    with pytest.raises(ValueError):
        paged.grow(kv, t, n, r[:7], n, n.clone(), paged.grow_workspace(kv, t))
    with pytest.raises(ValueError):
        paged.compact(kv, t, r, n, paged.compact_workspace(kv, t))
    with pytest.raises(ValueError, match="workspace"):
        paged.compact(kv, t, r, n[:1].clone(), torch.empty(16, dtype=torch.uint8, device="cuda"))


def test_pages_past_4_gib(paged):
    """Pages whose bytes lie past 2^32, in every call."""
    heads, kv, hd, page, n_pages = 8, 8, 128, 64, 20000       # 262144 bytes a page: 5.2 GB
    rng = np.random.default_rng(11)
    dev = torch.empty(n_pages, 2, kv, page, hd, dtype=torch.bfloat16, device="cuda")
    last = n_pages - 8
    small = _pool(rng, 8, kv, page, hd, torch.bfloat16)
    dev[last:] = small.cuda()
    tables = np.array([[last + 7, last + 2, last + 5], [last + 1, last + 4, last]], np.int32)
    lengths = [130, 64]
    cos, sin = _tables(192, hd)
    qkv = rng.standard_normal((2, (heads + 2 * kv) * hd)).astype(np.float32)
    t, n = _cuda(tables), _i64(lengths)
    out = torch.empty(2, heads * hd, device="cuda")
    args = (_cuda(qkv), n, t, _cuda(cos), _cuda(sin), dev)
    paged.attention(*args, out, heads, paged.attention_workspace(dev, t, heads))
    want_pool, want, bound = _reference(small, tables - last, lengths, qkv, cos, sin, heads, kv, hd)
    assert torch.equal(_bits(dev[last:]), _bits(want_pool))
    err = np.abs(out.cpu().double().numpy().reshape(want.shape) - want)
    assert (err <= bound).all(), (err / bound).max()
    k, v = (torch.zeros(2, kv, 131, hd, device="cuda") for _ in range(2))
    paged.load(dev, t, n + 1, k, v)
    for s, m in enumerate(lengths):
        a, b, _ = model.rows(want_pool, tables[s] - last, m + 1, 3)
        assert np.array_equal(k[s, 3, :m + 1].cpu().double().numpy(), a)
        assert np.array_equal(v[s, 3, :m + 1].cpu().double().numpy(), b)
    more = rng.standard_normal((40, (heads + 2 * kv) * hd)).astype(np.float32)
    paged.append(_cuda(more), n + 1, t, *args[3:], heads)      # 20 rows each
    for s, m in enumerate(lengths):
        for i in range(20):
            _store(want_pool, tables[s] - last, m + 1 + i, more[20 * s + i], cos, sin, heads, kv, hd)
    assert torch.equal(_bits(dev[last:]), _bits(want_pool))
    refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    refs[t.flatten().long()] = 1
    refs[last + 3] = 2                                         # a shared page, copied to page 0
    t[0, 2] = last + 3
    refs[last + 5] = 0
    room = torch.empty_like(n)
    paged.grow(dev, t, n, refs, _i64([1, 0]), room, paged.grow_workspace(dev, t))
    assert t[0].tolist() == [last + 7, last + 2, 0] and room.tolist() == [192, 64]
    assert torch.equal(_bits(dev[0, :, :, :16]), _bits(want_pool[3, :, :, :16]))
    live = _i64([0])
    paged.compact(dev, t, refs, live, paged.compact_workspace(dev, t))
    order = [0, 1, 2, 3, 4, 7]                                 # of the last eight: moved to 1 .. 6
    assert int(live) == 7 and torch.equal(_bits(dev[1:7]), _bits(want_pool[order]))
    assert t.tolist() == [[6, 3, 0], [2, 5, 1]]


def test_captured_calls(paged):
    """Attention, forks, room and compaction in one graph, replayed with other lengths, tables and
    rows, eager work between, against the same calls made eagerly."""
    rng = np.random.default_rng(21)
    heads, kv, hd, page, seqs, columns, n_pages = 8, 2, 128, 16, 6, 80, 300
    cos, sin = (_cuda(x) for x in _tables(columns * page, hd))

    class Side:
        pass

    sides = []
    for _ in "ab":
        x = Side()
        x.kv = paged.empty(n_pages, kv, hd, page, n_layers=2)
        x.t, x.n, x.r = paged.empty_tables(seqs, columns, n_pages)
        x.rows, x.room, x.parents, x.live = (torch.zeros(m, dtype=torch.int64, device="cuda")
                                             for m in (seqs, seqs, seqs, 1))
        x.q = torch.zeros(seqs, (heads + 2 * kv) * hd, device="cuda")
        x.out = torch.zeros(2, seqs, heads * hd, device="cuda")
        x.w = paged.attention_workspace(x.kv[0], x.t, heads)
        x.wg, x.wc = paged.grow_workspace(x.kv, x.t), paged.compact_workspace(x.kv, x.t)
        sides.append(x)

    def calls(x):
        paged.fork(x.t, x.n, x.r, x.parents)
        paged.grow(x.kv, x.t, x.n, x.r, x.rows, x.room, x.wg)
        for l in range(2):
            paged.attention(x.q, x.n, x.t, cos, sin, x.kv[l], x.out[l], heads, x.w, room=x.room)
        torch.minimum(x.n + x.rows, x.room, out=x.n)
        paged.compact(x.kv, x.t, x.r, x.live, x.wc)

    a, b = sides
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for x in sides:
            x.parents.copy_(torch.arange(seqs))
        calls(a)                                          # nothing takes part: rows are 0
        calls(b)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        calls(a)
    torch.cuda.synchronize()
    for step in range(40):
        q = torch.from_numpy(rng.standard_normal(tuple(a.q.shape)).astype(np.float32))
        parents = torch.arange(seqs)
        if step % 5 == 4:
            parents = torch.from_numpy(rng.integers(0, seqs, seqs))
        if step % 11 == 10:
            parents[int(rng.integers(0, seqs))] = -1
        rows = torch.from_numpy(rng.integers(0, 2, seqs))
        for x in sides:
            x.q.copy_(q)
            x.parents.copy_(parents)
            x.rows.copy_(rows)
            if step % 7 == 3:                             # a prompt's rows, eagerly
                m = _i64([30 * int(i == step % seqs) for i in range(seqs)])
                paged.grow(x.kv, x.t, x.n, x.r, m, x.room, x.wg)
                more = torch.ones(30, x.q.shape[1], device="cuda") * (step + 1)
                at = _i64([0] * (step % seqs + 1) + [30] * (seqs - step % seqs))
                for l in range(2):
                    paged.append(more, x.n, x.t, cos, sin, x.kv[l], heads, starts=at, room=x.room)
                torch.minimum(x.n + m, x.room, out=x.n)
        g.replay()
        calls(b)
        torch.cuda.synchronize()
        for u, v in zip((a.t, a.n, a.r, a.room, a.live, a.out), (b.t, b.n, b.r, b.room, b.live, b.out)):
            assert torch.equal(u, v), step
        assert torch.equal(_bits(a.kv), _bits(b.kv)), step
    held = b.t[b.t >= 0].long()
    assert int(b.n.max()) > 3 * page and torch.equal(torch.bincount(held, minlength=n_pages), b.r.long())


def test_two_streams_at_once(paged):
    """Calls on two streams with workspaces of their own do not meet."""
    rng = np.random.default_rng(5)
    heads, kv, hd, page, n = 16, 4, 128, 16, 3000
    columns = n // page + 1
    cos, sin = (_cuda(x) for x in _tables(n + 1, hd))
    sets = []
    for i in range(2):
        tables = _cuda(np.random.default_rng(i).permutation(columns)[None].astype(np.int32))
        kv_ = _pool(rng, columns, kv, page, hd, torch.float16).cuda()
        q = _cuda(rng.standard_normal((1, (heads + 2 * kv) * hd)).astype(np.float32))
        sets.append((q, _i64([n]), tables, cos, sin, kv_, heads, paged.attention_workspace(kv_, tables, heads)))
    alone = []
    for q, m, t, c, s, kv_, h, w in sets:
        out = torch.empty(1, heads * hd, device="cuda")
        alone.append(paged.attention(q, m, t, c, s, kv_, out, h, w))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    outs = [[torch.empty(1, heads * hd, device="cuda") for _ in range(30)] for _ in sets]
    torch.cuda.synchronize()
    for j in range(30):
        for i, (q, m, t, c, s, kv_, h, w) in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                paged.attention(q, m, t, c, s, kv_, outs[i][j], h, w)
    torch.cuda.synchronize()
    for i in range(2):
        for out in outs[i]:
            assert torch.equal(out, alone[i])


def test_large_batches_by_norm(paged):
    """Random caches at the sizes that the kernels are made for, against float64 on the device: the
    norm of the errors below 2^-15 of the outputs' (a part of an operand left out is six times
    that)."""
    for seed, (seqs, heads, kv, hd, page, high, dtype) in enumerate([
            (150, 8, 2, 64, 16, 700, torch.float16), (24, 32, 8, 128, 32, 3000, torch.bfloat16),
            (1, 32, 8, 128, 64, 100000, torch.float16), (5, 16, 2, 256, 16, 5000, torch.bfloat16),
            (40, 20, 4, 128, 16, 1500, torch.bfloat16)]):
        g = torch.Generator(device="cuda").manual_seed(seed)
        lengths = torch.randint(0, high, (seqs,), device="cuda", generator=g)
        lengths[0] = high - 1
        columns = high // page + 1
        n_pages = seqs * columns
        tables = torch.randperm(n_pages, device="cuda", generator=g).view(seqs, columns).int()
        pool = torch.randn(n_pages, 2, kv, page, hd, device="cuda", generator=g).to(dtype)
        qkv = torch.randn(seqs, (heads + 2 * kv) * hd, device="cuda", generator=g)
        qkv[:, :heads * hd] *= 2
        cos, sin = (_cuda(x) for x in _tables(high + 1, hd))
        out = torch.empty(seqs, heads * hd, device="cuda")
        paged.attention(qkv, lengths, tables, cos, sin, pool, out, heads,
                        paged.attention_workspace(pool, tables, heads))
        err = norm = 0.0
        for s in range(seqs):
            n = int(lengths[s]) + 1
            got = pool[tables[s, :-(-n // page)].long()].double()
            k = got[:, 0].transpose(0, 1).reshape(kv, -1, hd)[:, :n]
            v = got[:, 1].reshape(-1, kv, page // 16, hd, 16).transpose(-1, -2)
            v = v.reshape(-1, kv, page, hd).transpose(0, 1).reshape(kv, -1, hd)[:, :n]
            q = qkv[s, :heads * hd].double().view(heads, hd)
            z = torch.complex(q[:, :hd // 2], q[:, hd // 2:]) * torch.complex(cos[n - 1].double(),
                                                                             sin[n - 1].double())
            q = torch.cat([z.real, z.imag], 1).view(kv, heads // kv, hd)
            p = torch.softmax(q @ k.transpose(1, 2).contiguous() / math.sqrt(hd), -1)
            want = (p @ v).reshape(-1)
            err += float((out[s].double() - want).square().sum())
            norm += float(want.square().sum())
        assert err < (2.0 ** -15) ** 2 * norm, (seed, (err / norm) ** 0.5)
