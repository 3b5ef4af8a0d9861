"""Sampling on the GPU against its definition in float64.

Tokens are equal: the kernels sum w as multiples of 2^-43, so a running sum of n tokens is off by at
most n 2^-44 of the largest w, and a drawn token can differ only where u (or top_p) falls that
close to a border, which these inputs do not do (a row's border is met by chance once in 10^6
rows; where borders are meant to be met, w are whole numbers and every sum is exact).  A
probability is off by that, the roundings of f32 (2^-24) and the w's own 2^-44.
"""
import importlib
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sampling(pkg):
    return importlib.import_module("artifex-assistantv5_amd.sampling")


def expected(x, u, t=1.0, k=0, p=1.0, m=0.0):
    """(token, probability, kept) of a row by the header's rules."""
    x = x.astype(np.float64)
    x[np.isnan(x)] = -np.inf
    top = x.max()
    if top == -np.inf:
        return 0, 0.0, 0
    order = np.argsort(-x, kind="stable")
    if not t > 0:
        return int(order[0]), 1.0, 1
    if top == np.inf:
        w = (x[order] == np.inf).astype(np.float64)
    else:
        with np.errstate(invalid="ignore"):
            w = np.where(x[order] == -np.inf, 0.0, np.exp((x[order] - top) / t))
            w = np.where(x[order] == top, 1.0, w)
    n = len(w)
    if 0 < k < n:
        n = k
    cum = np.cumsum(w)
    keep = n
    if p < 1:
        keep = min(keep, int((cum < p * cum[n - 1]).sum()) + 1)
    if m > 0:
        keep = min(keep, max(1, int((w >= m).sum())))
    u = 0.0 if not u > 0 else min(u, float(np.nextafter(np.float32(1), np.float32(0))))
    at = min(int((cum <= u * cum[keep - 1]).sum()), keep - 1)
    return int(order[at]), w[at] / cum[keep - 1], keep


def check(sampling, x, u, t=1.0, k=0, p=1.0, m=0.0, ld=None):
    rows, vocab = x.shape
    each = [np.broadcast_to(np.asarray(v), (rows,)) for v in (t, k, p, m)]
    wide = torch.full((rows, ld or vocab), float("nan"))
    wide[:, :vocab] = torch.from_numpy(x)
    dev = wide.cuda()[:, :vocab]
    out = torch.full((rows,), -7, dtype=torch.int64, device="cuda")
    probs = torch.full((rows,), -7.0, device="cuda")
    work = sampling.workspace(rows, vocab)
    work.fill_(0xFF)
    kinds = (torch.float32, torch.int32, torch.float32, torch.float32)
    args = [v if np.ndim(v) == 0 else torch.tensor(v, dtype=d, device="cuda")
            for v, d in zip((t, k, p, m), kinds)]
    sampling.sample(dev, torch.tensor(u, dtype=torch.float32, device="cuda"), out, work, *args, probs=probs)
    u = np.float32(u)
    f = lambda v: float(np.float32(v))  # noqa: E731
    want = [expected(x[r].copy(), float(u[r]), f(each[0][r]), int(each[1][r]), f(each[2][r]),
                     f(each[3][r])) for r in range(rows)]
    assert out.tolist() == [w[0] for w in want]
    got = probs.cpu().double().numpy()
    ref = np.array([w[1] for w in want])
    assert (np.abs(got - ref) <= 2.0 ** -23 * ref + vocab * 2.0 ** -43).all(), (got, ref)
    return out, want


@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 63), (5, 64), (2, 1000), (1, 4097),
                                        (4, 32000), (1, 151936), (33, 5003), (130, 777),
                                        (2, 1 << 20)])
@pytest.mark.parametrize("k,p,m", [(0, 1.0, 0.0), (50, 1.0, 0.0), (0, 0.9, 0.0), (0, 1.0, 0.05),
                                   (40, 0.95, 0.02), (1, 0.5, 0.0), (2000, 0.6, 0.001)])
def test_against_definition(sampling, rows, vocab, k, p, m):
    rng = np.random.default_rng(rows * 7 + vocab + k)
    x = (rng.standard_normal((rows, vocab)) * rng.uniform(0.5, 3, (rows, 1))).astype(np.float32)
    x[:, rng.integers(0, vocab, min(vocab, 20))] += 5
    t = rng.uniform(0.3, 1.6, rows).astype(np.float32)
    check(sampling, x, rng.random(rows), t=t, k=k, p=p, m=m)


def test_settings_per_row_and_strides(sampling):
    rng = np.random.default_rng(1)
    rows, vocab = 37, 2500
    x = (rng.standard_normal((rows, vocab)) * 2).astype(np.float32)
    t = rng.uniform(0.2, 2, rows).astype(np.float32)
    t[::5] = 0
    k = rng.integers(-2, 3000, rows)
    p = rng.uniform(0, 1.3, rows).astype(np.float32)
    m = rng.uniform(-0.1, 0.3, rows).astype(np.float32)
    check(sampling, x, rng.random(rows), t=t, k=k, p=p, m=m, ld=2503)
    check(sampling, x, rng.random(rows), t=0.7, k=k, p=0.8, m=m)


@pytest.mark.parametrize("vocab", [5, 64, 3000, 100000])
def test_whole_weights(sampling, vocab):
    """Equal logits: w are ones, borders are met exactly; tokens go by index."""
    rng = np.random.default_rng(vocab)
    rows = 12
    x = np.full((rows, vocab), 2.5, np.float32)
    u = np.array([0, 0.5, 0.25, 1 - 2.0 ** -24] * 3)
    k = np.array([0, 0, 0, 0, 4, 4, 4, 4, vocab, vocab + 1, 1, 2])
    p = np.array([1, 1, 1, 1, 0.5, 0.25, 0.75, 1, 0.5, 0.5, 0.5, 0.5], np.float32)
    check(sampling, x, u, k=k, p=p)
    x[:, rng.integers(0, vocab, vocab // 2)] = -np.inf           # half of them masked
    check(sampling, x, u, k=k, p=p)


@pytest.mark.parametrize("vocab", [300, 40000])
def test_ties(sampling, vocab):
    """Logits of few values (as of 8-bit products): many equal ones at every border."""
    rng = np.random.default_rng(vocab)
    x = np.round(rng.standard_normal((40, vocab)) * 3).astype(np.float32) * 0.5
    x[::3] = np.where(x[::3] == 0, -0.0, x[::3])
    x[1::3][:, ::2] = -x[1::3][:, ::2]                           # zeros of both signs
    k = rng.integers(1, vocab, 40)
    k[::4] = 0
    check(sampling, x, rng.random(40), t=rng.uniform(0.5, 2, 40).astype(np.float32), k=k,
          p=rng.uniform(0.1, 1.1, 40).astype(np.float32), m=0.0)


def test_special_values(sampling):
    rng = np.random.default_rng(2)
    nan, inf = float("nan"), float("inf")
    x = rng.standard_normal((12, 700)).astype(np.float32)
    x[0, ::3] = nan
    x[1] = nan
    x[2] = -inf
    x[3, 5], x[3, 600], x[3, 300] = inf, inf, nan
    x[4] = -inf
    x[4, 699] = -3e38                                            # one left
    x[5] = 3e38
    x[5, 10] = -3e38
    x[6] *= 1e30
    x[7, 1:] = np.finfo(np.float32).min
    x[8] = np.float32(1e-45)
    x[8, 3] = 0
    x[9, 17] = inf
    x[10, :699] = -inf
    x[10, 699] = nan                                             # nothing left
    for t in (1.0, 1e-30, 1e30, inf, 0.0, -1.0, nan):
        for k, p, m in ((0, 1.0, 0.0), (3, 0.9, 0.1), (0, nan, nan), (0, 0.0, 2.0)):
            check(sampling, x, rng.random(12), t=t, k=k, p=1.0 if p != p else p, m=0.0 if m != m else m)


def test_nan_settings_are_off(sampling):
    rng = np.random.default_rng(4)
    x = torch.from_numpy(rng.standard_normal((2, 900)).astype(np.float32)).cuda()
    u = torch.tensor([0.3, 0.8], device="cuda")
    work, a, b = sampling.workspace(2, 900), *(torch.zeros(2, dtype=torch.int64, device="cuda") for _ in "ab")
    sampling.sample(x, u, a, work)
    sampling.sample(x, u, b, work, top_p=float("nan"), min_p=float("nan"), top_k=-5)
    assert torch.equal(a, b)


def test_random_numbers_outside(sampling):
    x = np.zeros((6, 10), np.float32)
    check(sampling, x, np.array([-1, float("nan"), 1.0, 7.0, float("inf"), -float("inf")]))


def test_frequencies(sampling):
    """10^5 draws with evenly spaced random numbers: each token's share is its probability to within
    one draw, by the definition."""
    n = 100000
    x = torch.tensor([1.0, 3.0, -1.0, 2.0, 0.0], device="cuda")
    u = (torch.arange(n, device="cuda") + 0.5) / n
    out = torch.empty(n, dtype=torch.int64, device="cuda")
    for r0 in range(0, n, 50000):
        part = x.expand(50000, 5).contiguous()
        sampling.sample(part, u[r0:r0 + 50000].contiguous(), out[r0:r0 + 50000],
                        sampling.workspace(50000, 5), temperature=1.5)
    share = torch.bincount(out, minlength=5).double().cpu() / n
    want = torch.softmax(x.double().cpu() / 1.5, 0)
    assert (share - want).abs().max() <= 2 / n


def test_greedy_equals_argmax(sampling, pkg):
    glue = importlib.import_module("artifex-assistantv5_amd.glue")
    x = torch.randn(1, 151936, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    a, b = (torch.zeros(1, dtype=torch.int64, device="cuda") for _ in "ab")
    glue.argmax(x[0], a, glue.argmax_workspace("cuda"))
    sampling.sample(x, torch.tensor([0.9], device="cuda"), b, sampling.workspace(1, 151936), temperature=0.0)
    assert torch.equal(a, b)


def test_refusals(sampling):
    x, u = torch.zeros(2, 10, device="cuda"), torch.zeros(2, device="cuda")
    out, work = torch.zeros(2, dtype=torch.int64, device="cuda"), sampling.workspace(2, 10)
    call = lambda **o: sampling.sample(**{**dict(logits=x, u=u, out=out, work=work), **o})  # noqa: E731
    call()
    for bad in (dict(logits=x.half()), dict(logits=x[0]), dict(logits=x.t()), dict(u=u[:1]),
                dict(u=u.double()), dict(out=out.int()), dict(work=work.cpu()), dict(work=work[:0]),
                dict(temperature=u[:1]), dict(top_k=u), dict(top_p=u.double()), dict(min_p=u[:1]),
                dict(probs=out), dict(logits=x.expand(5, 2, 10)), dict(logits=x[:, :0])):
        with pytest.raises(ValueError):
            call(**bad)


def test_captured_with_device_settings(sampling):
    """One graph of two calls that share a workspace, replayed with other logits, random numbers and
    settings, eager calls between."""
    rows, vocab = 5, 20000
    g = torch.Generator(device="cuda").manual_seed(1)
    x, u = torch.zeros(2, rows, vocab, device="cuda"), torch.zeros(2, rows, device="cuda")
    t, p, m = (torch.ones(rows, device="cuda") for _ in range(3))
    k = torch.zeros(rows, dtype=torch.int32, device="cuda")
    out = torch.zeros(2, rows, dtype=torch.int64, device="cuda")
    work, other = sampling.workspace(rows, vocab), sampling.workspace(rows, vocab)

    def calls(to, w):
        for i in range(2):
            sampling.sample(x[i], u[i], to[i], w, t, k, p, m)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        calls(out, work)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls(out, work)
    for step in range(12):
        x.copy_(torch.randn(x.shape, device="cuda", generator=g) * (1 + step % 3))
        u.copy_(torch.rand(u.shape, device="cuda", generator=g))
        t.copy_(torch.rand(rows, device="cuda", generator=g) * 1.5 - 0.1)
        k.copy_(torch.randint(-5, 900, (rows,), device="cuda", generator=g))
        p.copy_(torch.rand(rows, device="cuda", generator=g) + 0.2)
        m.copy_(torch.rand(rows, device="cuda", generator=g) * 0.2 - 0.1)
        graph.replay()
        want = torch.full_like(out, -1)
        calls(want, other)
        torch.cuda.synchronize()
        assert torch.equal(out, want), step
        for i in range(2):
            for r in range(rows):
                w = expected(x[i, r].cpu().numpy().astype(np.float64), float(u[i, r]), float(t[r]),
                             int(k[r]), float(p[r]), float(m[r]))
                assert int(out[i, r]) == w[0]


def test_a_workspace_serves_fewer_rows(sampling):
    """A workspace of many rows serves calls of any fewer, which are cut otherwise."""
    work = sampling.workspace(64, 151936)
    assert work.numel() < 64 * 151936 * 4                   # less than the logits
    g = torch.Generator(device="cuda").manual_seed(2)
    x, u = torch.randn(64, 151936, device="cuda", generator=g), torch.rand(64, device="cuda", generator=g)
    out = torch.zeros(64, dtype=torch.int64, device="cuda")
    sampling.sample(x, u, out, work, top_p=0.9)
    for rows in (1, 3, 27, 28, 40):
        got = torch.zeros(rows, dtype=torch.int64, device="cuda")
        sampling.sample(x[:rows], u[:rows].contiguous(), got, work, top_p=0.9)
        assert torch.equal(got, out[:rows])


@pytest.mark.parametrize("m", [0.0, 0.4, 1.0])
def test_more_equal_logits_than_are_sorted(sampling, m):
    """Tens of thousands of equal logits at every border, few and many of them asked for."""
    rng = np.random.default_rng(9)
    vocab = 60000
    x = rng.integers(0, 3, (14, vocab)).astype(np.float32)        # three values, 20000 of each
    x[7:] -= 1e4 * (rng.random((7, vocab)) < 0.5)                 # half of them of weight zero
    k = np.array([0, 1, 5, 512, 513, 25000, 59999] * 2)
    p = np.array([1.0, 0.9, 0.5, 0.999, 0.3, 0.7, 0.95] * 2, np.float32)
    check(sampling, x, rng.random(14), t=np.linspace(0.4, 3, 14).astype(np.float32), k=k, p=p, m=m)


def test_many_of_many(sampling):
    """top_k of thousands over a large vocabulary, narrow and wide rows, outliers at both ends."""
    rng = np.random.default_rng(10)
    x = (rng.standard_normal((9, 151936)) * np.array([[0.01, 0.1, 0.5, 1, 2, 4, 8, 1, 1]]).T)
    x = x.astype(np.float32)
    x[7, 77], x[8, 5] = 60, -1e30
    for k, p in ((4097, 1.0), (10000, 0.97), (150000, 0.999999), (513, 0.5)):
        check(sampling, x, rng.random(9), t=0.9, k=k, p=p)


@pytest.mark.parametrize("alike", [3700, 3797, 4096])
def test_a_full_bin_behind_others(sampling, alike):
    """A few hundred tokens, then as many equal ones as are just sorted, the top_k-th among them: what
    lies before them counts."""
    rng = np.random.default_rng(alike)
    x = np.full((6, 20000), -5.0, np.float32)
    for r in range(6):
        at = rng.permutation(20000)
        x[r, at[:300]] = 4 + 2 * rng.random(300)
        x[r, at[300:300 + alike]] = 3
    check(sampling, x, np.array([0.0, 0.2, 0.5, 0.9, 0.99, 0.9999]), k=np.array([299, 300, 301, 400, 512, 505]),
          p=np.array([1.0, 0.9, 1.0, 0.99, 1.0, 0.999], np.float32), m=np.array([0, 0, 0.01, 0, 0, 0.02], np.float32))
