"""The 4-bit KV cache's kernels at the lengths and batches that they are made for: long lists in
several workgroups of several turns, many lists of different lengths, many records to join.

The caches hold random codes and scales (every slot counts; unused ones NaN scales), their values
are read through the offsets of kv4_model.py, and attention is taken in float64 over them.

Tolerances.  Each output and weight keeps the bound of test_gpu_kv4.py.  That is a worst case, so
the error's norm over a call's outputs is bounded beside it, at 2^-15 of the outputs' norm:

* a score is off by 2^-22 of each product (the queries' two f16 parts) and by f32 roundings of its
  2 head_dim / 32 partial sums, of either sign, 2^-24 of at most 40 each (the scores' standard
  deviation is 5): below 40 sqrt(16) 2^-24 < 2^-16, and it moves an output as much;
* p * scale is off by 2^-22 of it; the sums over a wave's turns (at most 16, two products of some
  four roundings each), 8 waves and at most 128 records in groups are under 2 * 16 * 4 + 8 + 16 =
  152 roundings of 2^-24 of partial sums no larger than the result's scale: below 2^-16.7 even if
  all had one sign.

An f16 part left out is off by 2^-12.3 of each product (f16's error, root mean square, 2^-11 /
sqrt(3) / 1.4) and the outputs' norm as much, six times the tolerance.
"""
import importlib

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import kv4_model as model  # noqa: E402
from test_gpu_kv4 import EPS, _cuda, _i64, _tables  # noqa: E402

pytestmark = pytest.mark.gpu

NORM = 2.0 ** -15


@pytest.fixture(scope="module")
def kv4(pkg):
    return importlib.import_module("artifex-assistantv5_amd.kv4")


def _at(hd, j):
    """Offsets of slot j's code bytes with their channels, and of its scales' bytes (K, V)."""
    ko, vo, ks, vs = model._offsets(hd, j)
    t = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
    return [(t(c[:, 0]), t(c[:, 1]), t(c[:, 2]), t(np.stack([s, s + 1], 1).ravel()))
            for c, s in ((ko, ks), (vo, vs))]


def _values(cache, hd):
    """f32 keys and values [..., slots, hd] of a device cache [..., tiles, 36 hd]."""
    out = torch.zeros(2, *cache.shape[:-1], 32, hd, device="cuda")
    for j in range(32):
        for i, (at, low, high, sc) in enumerate(_at(hd, j)):
            byte = cache[..., at]
            c = torch.zeros(*cache.shape[:-1], hd, device="cuda")
            c[..., low], c[..., high] = (byte & 15).float(), (byte >> 4).float()
            d = cache[..., sc].contiguous().view(torch.float16).float()
            out[i][..., j, :] = (c - 8) * d.repeat_interleave(32, dim=-1)
    return out.flatten(-3, -2)


def _cache(g, lengths, kv, hd, slots):
    """Random codes and scales; keys twice as large in the first slots as in the last, so that the
    tiles, taken from the last, raise a row's maximum again and again.  Slots from a sequence's
    length on hold 0xFF: scales that are NaN."""
    seqs, tiles = len(lengths), slots // 32
    c = torch.randint(0, 256, (seqs, kv, tiles, 36 * hd), dtype=torch.uint8, device="cuda",
                      generator=g)
    d = 0.05 + 0.25 * torch.rand(2, seqs, kv, tiles, hd, device="cuda", generator=g)
    d *= torch.where(torch.rand(d.shape, device="cuda", generator=g) < 0.5, -1.0, 1.0)
    d[0] *= torch.linspace(2, 1, tiles, device="cuda")[:, None]
    for i in range(2):
        c[..., (32 + 2 * i) * hd:(34 + 2 * i) * hd] = d[i].half().view(torch.uint8)
    unused = torch.arange(tiles, device="cuda") * 32 - _i64(lengths)[:, None]
    for j in range(32):
        free = (unused + j >= 0)[:, None, :, None]
        for at, _, _, sc in _at(hd, j):
            for x in (at, sc):
                c[..., x] = torch.where(free, torch.full((), 255, dtype=torch.uint8, device="cuda"),
                                        c[..., x])
    return c


CASES = {
    # heads, kv, hd, slots, lengths, rows
    # few query rows, 32 lists and more: small workgroups
    "8x8 lists of 64": (8, 8, 64, 2048, [2047, 1, 640, 0, 1999, 33, 1500, 777], 1),
    "4x8 lists of 64, groups of 4": (32, 8, 64, 8192, [8191, 5, 3333, 7000], 1),
    "16x8 lists of 128": (32, 8, 128, 4096, [4095, 37, 2500, 3999, 31, 0, 1024, 3100, 64, 2047, 905,
                                             -1, 4000, 63, 3777, 1800], 1),
    "4x4 lists of 256": (16, 4, 256, 9216, [9000, 9215, 4001, 7007], 1),
    # few query rows, few lists: large workgroups, many records
    "8 lists of 100000": (32, 8, 128, 100032, [100000], 1),
    "4 lists of 60000, 64 channels": (4, 4, 64, 60032, [60001], 1),
    # many query rows
    "32 rows over 20000": (32, 8, 128, 20480, [20000], 32),
    "32 rows of 64 channels": (16, 8, 64, 16384, [16000, 9001], 32),
    "groups of 8 over 30000": (64, 8, 128, 30016, [30000, 17003], 1),
    "3 rows of 64 channels": (8, 4, 64, 30016, [29000, 14001], 3),
    "groups of 8 of 256 channels": (16, 2, 256, 30016, [30000, 8, 21000, 29999], 1),
}


def _check(kv4, heads, kv, hd, slots, lengths, rows, scale_q, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    seqs, grp = len(lengths), heads // kv
    pos = [max(0, n) + 3 for n in lengths]
    cos, sin = (_cuda(t) for t in _tables(max(pos) + rows, hd, base=1e6))
    cache = _cache(g, lengths, kv, hd, slots)
    qkv = torch.randn(seqs * rows, (heads + 2 * kv) * hd, device="cuda", generator=g)
    qkv[:, :heads * hd] *= scale_q
    out = torch.full((seqs * rows, heads * hd), 7.0, device="cuda")
    weights = torch.full((seqs, kv, slots), 0.25, device="cuda")
    work = kv4.attention_workspace(cache, heads, rows=rows, weights=True)
    work.fill_(0xFF)
    args = (qkv, _i64(lengths), _i64(pos), cos, sin, cache, out, heads, work)
    kv4.attention(*args, weights=weights)
    got = out.view(seqs, rows, kv, grp, hd).double()
    wrong = size = wwrong = wsize = 0.0
    for s, n in enumerate(lengths):
        if n < 0 or n + rows > slots:
            assert (got[s] == 7).all() and (weights[s] == 0.25).all()
            continue
        x = qkv[s * rows:(s + 1) * rows].double().view(rows, heads + 2 * kv, hd)[:, :heads]
        turn = torch.complex(cos[pos[s]:pos[s] + rows].double(), sin[pos[s]:pos[s] + rows].double())
        z = torch.complex(x[..., :hd // 2], x[..., hd // 2:]) * turn[:, None]
        q = torch.cat([z.real, z.imag], -1).view(rows, kv, grp, hd).transpose(0, 1)
        sees = n + torch.arange(rows, device="cuda").repeat_interleave(grp)[:, None]
        for h in range(kv):
            last = (n + rows + 31) // 32
            k, v = (t[:n + rows].double() for t in _values(cache[s, h, :last], hd))
            qh = q[h].reshape(rows * grp, hd)
            score = qh @ k.t().contiguous() / hd ** 0.5
            score.masked_fill_(torch.arange(n + rows, device="cuda") > sees, -torch.inf)
            p = torch.softmax(score, dim=-1)
            top = qh.abs() @ k.abs().t().contiguous() / hd ** 0.5
            top.masked_fill_(torch.isinf(score), 0.0)
            err = (8 * EPS * top.amax(-1) + EPS)[:, None]
            least = 2.0 ** -34.9 * (n + rows) * (p * v.abs().amax(-1)).amax(-1, keepdim=True)
            ref, bound = p @ v, (p @ v.abs()) * err + least
            o = got[s, :, h].reshape(rows * grp, hd)
            off = (o - ref).abs()
            assert (off <= bound).all(), (s, h, (off / bound).max().item())
            wrong, size = wrong + (off ** 2).sum().item(), size + (ref ** 2).sum().item()
            w, wref = weights[s, h].double(), p.sum(0)
            assert (w[n + rows:] == 0.25).all()
            woff = (w[:n + rows] - wref).abs()
            assert (woff <= (p * err).sum(0) + 1e-30).all(), (s, h)
            wwrong, wsize = wwrong + (woff ** 2).sum().item(), wsize + (wref ** 2).sum().item()
    assert wrong <= NORM ** 2 * size, (wrong / size) ** 0.5
    assert wwrong <= NORM ** 2 * wsize, (wwrong / wsize) ** 0.5
    # again over the stored rows, without weights
    again = torch.full_like(out, 7.0)
    kv4.attention(qkv, _i64(lengths), _i64(pos), cos, sin, cache, again, heads,
                  kv4.attention_workspace(cache, heads, rows=rows), store=False)
    assert torch.equal(out, again)


@pytest.mark.parametrize("scale_q", [3.0, 1e-12], ids=["picking", "flat"])
@pytest.mark.parametrize("name", CASES)
def test_attention_of_long_lists(kv4, name, scale_q):
    """``flat``: equal probabilities, so that nothing but the products with V can be off."""
    _check(kv4, *CASES[name], scale_q, seed=len(name))


@pytest.mark.parametrize("heads,kv,hd,rows", [(4, 2, 64, 1), (8, 2, 128, 1), (4, 1, 256, 1),
                                              (4, 2, 64, 5), (8, 1, 128, 3)])
def test_attention_of_many_sequences(kv4, heads, kv, hd, rows):
    """150 sequences, active ones and others in every 64 of them, lengths from none to all."""
    rng = np.random.default_rng(hd + rows)
    slots = 1024
    lengths = rng.integers(0, slots - rows + 1, 150)
    lengths[rng.permutation(150)[:40]] = rng.integers(-2, 3, 40)
    lengths[[0, 63, 64, 127, 128, 149]] = [slots - rows, 900, slots, 0, 33, 500]
    _check(kv4, heads, kv, hd, slots, lengths.tolist(), rows, 3.0, seed=rows)


def _put(cache, seq, slots, k, v):
    """Rows [n, n_kv, hd] quantized into ``slots`` [n] of one sequence of a host cache."""
    hd = k.shape[-1]
    coded = [model.quantize(np.ascontiguousarray(x)) for x in (k, v)]
    for j in range(32):
        pick = np.nonzero(slots % 32 == j)[0]
        tile = slots[pick] // 32
        ko, vo, ks, vs = model._offsets(hd, j)
        for (c, d), at, sc in zip(coded, (ko, vo), (ks, vs)):
            c, d = c[pick], np.ascontiguousarray(d[pick]).view(np.uint8)
            d = d.reshape(len(pick), cache.shape[1], hd // 32, 2)
            for h in range(cache.shape[1]):
                rows = cache[seq, h]
                rows[tile[:, None], at[:, 0]] = c[:, h][:, at[:, 1]] | (c[:, h][:, at[:, 2]] << 4)
                rows[tile[:, None], sc], rows[tile[:, None], sc + 1] = d[:, h, :, 0], d[:, h, :, 1]


@pytest.mark.parametrize("heads,kv,hd,slots,lengths,starts,rows", [
    (8, 8, 128, 1024, [5, 0, 700], [3, 401, 402, 1090], 1101),  # behind 5 and 700 slots
    (4, 4, 64, 1600, [31, 63], [0, 1101, 2100], 2100),
    (5, 5, 128, 480, [-1, 9, 100, 30], None, 1640),             # units that end inside a wave's
    (8, 4, 256, 1024, [2, 33], [0, 1040, 2049], 2050),          # the last rows do not fit
])
def test_append_of_many_rows(kv4, heads, kv, hd, slots, lengths, starts, rows):
    """Rows times KV heads above 8192: several units per wave, stored bit for bit."""
    assert rows * kv >= 8192
    rng = np.random.default_rng(rows)
    seqs = len(lengths)
    pos = [max(0, n) + 11 for n in lengths]
    cos, sin = _tables(slots + 200, hd)
    qkv = (rng.standard_normal((rows, (heads + 2 * kv) * hd)) * 3).astype(np.float32)
    qkv[rng.integers(0, rows, 40), -32:] = 0
    cache = np.full((seqs, kv, slots // 32, 36 * hd), 0x5A, np.uint8)
    dev = _cuda(cache)
    positions = np.full((seqs, kv, slots), -7, np.int32)
    weights = np.full((seqs, kv, slots), 3.5, np.float32)
    dp, dw = _cuda(positions), _cuda(weights)
    kv4.append(_cuda(qkv), _i64(lengths), _i64(pos), _cuda(cos), _cuda(sin), dev, heads,
               starts=None if starts is None else _i64(starts), positions=dp, weights=dw)
    at = starts or [s * (rows // seqs) for s in range(seqs + 1)]
    x = qkv.reshape(rows, heads + 2 * kv, hd)
    for s, n in enumerate(lengths):
        m = min(at[s + 1] - at[s], slots - n)
        if n < 0 or m <= 0:
            continue
        r, to = np.arange(at[s], at[s] + m), np.arange(n, n + m)
        p = pos[s] + np.arange(m)
        _put(cache, s, to, model.rope(x[r, heads:heads + kv], cos[p][:, None], sin[p][:, None]),
             x[r, heads + kv:])
        positions[s][:, to], weights[s][:, to] = p, 0
    assert np.array_equal(dev.cpu().numpy(), cache)
    assert np.array_equal(dp.cpu().numpy(), positions)
    assert np.array_equal(dw.cpu().numpy(), weights)


@pytest.mark.parametrize("what", [float("nan"), float("inf")])
@pytest.mark.parametrize("heads,kv,hd,lengths,rows", [
    (4, 1, 64, [700], 1), (8, 2, 128, [700, 31], 1), (4, 1, 256, [700], 1),
    (8, 1, 64, [700], 3), (8, 1, 128, [0, 700], 4), (16, 2, 256, [700], 2)])
def test_a_bad_query_is_its_own(kv4, heads, kv, hd, lengths, rows, what):
    """A query of NaN or infinities leaves the other heads' and rows' outputs as near as they
    were: only the order in which their maximum is raised may change."""
    g = torch.Generator(device="cuda").manual_seed(hd + rows)
    slots, seqs = 1024, len(lengths)
    cache = _cache(g, lengths, kv, hd, slots)
    cos, sin = (_cuda(t) for t in _tables(slots, hd))
    qkv = torch.randn(seqs * rows, (heads + 2 * kv) * hd, device="cuda", generator=g)
    bad = qkv.clone()
    bad[rows - 1, hd:2 * hd] = what                  # head 1 of the first sequence's last row
    outs = []
    for x in (qkv, bad):
        out = torch.empty(seqs * rows, heads * hd, device="cuda")
        kv4.attention(x, _i64(lengths), _i64(lengths), cos, sin, cache, out, heads,
                      kv4.attention_workspace(cache, heads, rows=rows))
        outs.append(out.view(seqs * rows, heads, hd))
    assert torch.isnan(outs[1][rows - 1, 1]).all()
    for out in outs:
        out[rows - 1, 1] = 0
    assert torch.isfinite(outs[1]).all()
    assert (outs[1] - outs[0]).norm() <= 2 * NORM * outs[0].norm()   # each within NORM of exact
