"""Calls straight from tensors (_tensors): each equals the one that paged.py and sampling.py make by
their own checks, bit for bit, and refuses what those refuse.  What a wrong argument points to is at
least as large as the right one, so that even a call made by mistake stays in bounds."""
import importlib
import threading

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

S, COLUMNS, PAGES, PAGE, HEADS, KV, HD = 3, 4, 16, 16, 8, 2, 64


@pytest.fixture(scope="module")
def native():
    return importlib.import_module("artifex-assistantv5_amd._native")


@pytest.fixture(scope="module")
def ops():
    return {n: importlib.import_module("artifex-assistantv5_amd." + n) for n in ("paged", "sampling")}


def _i64(*x):
    return torch.tensor(x, dtype=torch.int64, device="cuda")


def _args(ops, name):
    """All arguments of a call, in the order of its Python function's."""
    p = ops["paged"]
    g = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
    kv = rand(PAGES, 2, KV, PAGE, HD).to(torch.bfloat16)
    tables = torch.arange(S * COLUMNS, dtype=torch.int32, device="cuda").view(S, COLUMNS).contiguous()
    refs = torch.zeros(PAGES, dtype=torch.int32, device="cuda")
    refs[:S * COLUMNS] = 1
    lengths, room = _i64(5, 40, 16), _i64(64, 64, 64)
    cos, sin = rand(64, HD // 2), rand(64, HD // 2)
    width = (HEADS + 2 * KV) * HD
    if name == "append":
        return [rand(9, width), lengths, tables, cos, sin, kv, HEADS, _i64(0, 2, 3, 9), room]
    if name == "attention":
        return [rand(S, width), lengths, tables, cos, sin, kv, rand(S, HEADS * HD), HEADS,
                p.attention_workspace(kv, tables, HEADS), room]
    if name == "load":
        return [kv, tables, lengths, rand(S, KV, 64, HD), rand(S, KV, 64, HD)]
    if name == "fork":
        return [tables, lengths, refs, _i64(1, 1, -1), torch.empty_like(tables), torch.empty_like(lengths),
                torch.empty_like(refs)]
    if name == "grow":
        tables[1, 3], refs[7] = -1, 0
        layers = rand(2, PAGES, 2, KV, PAGE, HD).half()
        return [layers, tables, lengths, refs, _i64(1, 24, 0), room, p.grow_workspace(layers, tables)]
    if name == "compact":
        refs[3:6] = 0
        layers = rand(2, PAGES, 2, KV, PAGE, HD).half()
        return [layers, tables, refs, _i64(0), p.compact_workspace(layers, tables),
                torch.empty_like(tables), torch.empty_like(refs)]
    n, vocab = 5, 300
    return [rand(n, vocab) * 3, torch.rand(n, device="cuda", generator=g), torch.zeros_like(_i64(*range(n))),
            ops["sampling"].workspace(n, vocab), torch.rand(n, device="cuda", generator=g) + 0.5,
            torch.full((n,), 40, dtype=torch.int32, device="cuda"), 0.9,
            torch.full((n,), 0.02, device="cuda"), torch.zeros(n, device="cuda")]


NAMES = ("append", "attention", "load", "fork", "grow", "compact", "sample")


def _call(ops, name, args):
    """By the Python function, whose optional arguments go by name."""
    m = ops["sampling" if name == "sample" else "paged"]
    if name == "attention":
        return m.attention(*args)
    return getattr(m, name)(*args)


class Refusing:
    def __getattr__(self, name):
        return lambda *args: False


@pytest.mark.parametrize("name", NAMES)
def test_equals_the_checked_call(native, ops, monkeypatch, name):
    direct, checked = _args(ops, name), _args(ops, name)
    assert getattr(native.direct(), name)(*direct) is True
    with monkeypatch.context() as m:
        m.setattr(native, "_tensors", Refusing())
        _call(ops, name, checked)
    again = _args(ops, name)
    with monkeypatch.context() as m:  # and it is what the Python function does
        for module in ops.values():
            if hasattr(module, "_call"):
                m.setattr(module, "_call", None)
        m.setattr(native, "call", None)
        _call(ops, name, again)
    torch.cuda.synchronize()
    work = {"attention": 8, "grow": 6, "compact": 4, "sample": 3}.get(name)
    for i, (x, y, z) in enumerate(zip(direct, checked, again)):
        if isinstance(x, torch.Tensor) and i != work:
            assert torch.equal(x, y) and torch.equal(x, z), i


def _wrong(x):
    """Arguments that are not as they should be, none smaller."""
    if not isinstance(x, torch.Tensor):
        return ["8", None, [8], 2 ** 40, 1e300]
    more = torch.zeros(2 * x.numel() + 64, dtype=x.dtype, device="cuda")
    wide = torch.zeros(*x.shape, 2, dtype=x.dtype, device="cuda")[..., 0]
    return [x.cpu(), torch.zeros(x.shape, dtype=torch.complex128, device="cuda"), more.expand(1, 1, 1, -1),
            wide, x.cpu().double().numpy(), "tensor", 3.5, torch.zeros(x.shape, device="cuda").to_sparse()]


@pytest.mark.parametrize("name", NAMES)
def test_refuses_what_the_checked_call_refuses(native, ops, name):
    f = getattr(native.direct(), name)
    good = _args(ops, name)
    before = [x.clone() if isinstance(x, torch.Tensor) else x for x in good]
    for i, x in enumerate(good):
        if isinstance(x, torch.Tensor) and x.dtype is torch.uint8:
            wrong = [x.cpu(), None, 7, torch.zeros(1, dtype=torch.uint8, device="cuda")]  # the workspace
        elif name == "sample" and i in (4, 5, 6, 7):
            wrong = ["1", None, 1e300 if i != 5 else 2 ** 40, x.cpu() if isinstance(x, torch.Tensor) else [1],
                     torch.zeros(64, dtype=torch.float64, device="cuda")]
        else:
            wrong = _wrong(x)
        if isinstance(x, torch.Tensor) and x.numel() == 1:  # whose strides do not matter
            wrong = [w for w in wrong if not (isinstance(w, torch.Tensor) and w.dtype is x.dtype)]
        for w in wrong:
            assert f(*good[:i], w, *good[i + 1:]) is False, (i, type(w))
    assert f(*good[:-1]) is False and f(*good, None) is False and f() is False
    torch.cuda.synchronize()
    for x, old in zip(good, before):
        if isinstance(x, torch.Tensor):
            assert torch.equal(x, old)


def test_messages_are_the_checks_own(ops):
    """What the direct call refuses is refused by name."""
    a = _args(ops, "attention")
    with pytest.raises(ValueError, match="lengths must be a contiguous torch.int64"):
        ops["paged"].attention(a[0], a[1].int(), *a[2:])
    with pytest.raises(ValueError, match="n_heads 7 must be 1..8 times"):
        ops["paged"].attention(*a[:7], 7, *a[8:])
    with pytest.raises(ValueError, match="workspace of 16 bytes, needs"):
        s = _args(ops, "sample")
        ops["sampling"].sample(*s[:3], torch.zeros(16, dtype=torch.uint8, device="cuda"), *s[4:])


def test_settings_as_numbers(native, ops):
    """Python's integers and floats, as the checked call takes them; no rows at all."""
    a = _args(ops, "sample")
    for t, k, p, m in ((1, 0, 1, 0), (0.5, True, 0.9, 0.1), (0, -5, 2.0, -1.0), (float("inf"), 2 ** 31 - 1, 1.0, 0.0)):
        assert native.direct().sample(*a[:4], t, k, p, m, None) is True
        want = torch.zeros_like(a[2])
        with pytest.MonkeyPatch.context() as mp:
            mp.setattr(native, "_tensors", Refusing())
            ops["sampling"].sample(a[0], a[1], want, a[3], t, k, p, m)
        assert torch.equal(a[2], want)
    ops["sampling"].sample(a[0], a[1], a[2], a[3], 1.0, 2 ** 40)  # beyond what the entry point takes
    assert ops["sampling"].sample(a[0][:0], a[1][:0], a[2][:0], a[3]).numel() == 0


def test_streams_and_threads(native, ops):
    """The current stream of the calling thread is the call's."""
    got = {}

    def run(k):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                a = _args(ops, "attention")
                ops["paged"].attention(*a)
            s.synchronize()
            got[k] = a[6]

    threads = [threading.Thread(target=run, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    a = _args(ops, "attention")
    ops["paged"].attention(*a)
    assert all(torch.equal(got[k], a[6]) for k in range(4))


@pytest.fixture
def answers(native):
    """Entry points that do nothing but return a code, and count their calls."""
    import ctypes

    signatures = {**native.PAGED_SIGNATURES, **native.SAMPLE_SIGNATURES}
    state = dict(rc=0, calls=0)

    def answer(*args):
        state["calls"] += 1
        return state["rc"]

    stubs = [ctypes.CFUNCTYPE(signatures[n][0], *signatures[n][1])(answer) for n in native.PACKED]
    lib, direct = native.load_library(), native.direct()
    address = lambda f: ctypes.cast(f, ctypes.c_void_p).value  # noqa: E731
    direct.bind(*map(address, stubs))
    yield state
    direct.bind(*(address(getattr(lib, n)) for n in native.PACKED))


@pytest.mark.parametrize("name", NAMES)
def test_a_call_that_failed_is_not_made_again(native, ops, answers, name):
    """A HIP error may come after the first of two launches: it is raised, and nothing more is done."""
    args = _args(ops, name)
    before = [x.clone() if isinstance(x, torch.Tensor) else x for x in args]
    for rc in (native.ERR_HIP, -99):
        answers.update(rc=rc, calls=0)
        with pytest.raises(native.GGUFHipError) as e:
            _call(ops, name, args)
        assert e.value.code == rc and answers["calls"] == 1
        for x, old in zip(args, before):
            if isinstance(x, torch.Tensor) and x.dtype is not torch.uint8:
                assert torch.equal(x, old)
    f = getattr(native.direct(), name)
    for rc in (native.ERR_TYPE, native.ERR_SHAPE, native.ERR_NULL, native.ERR_ALIGN, native.ERR_DTYPE,
               native.ERR_BYTES):
        answers.update(rc=rc, calls=0)
        assert f(*args) is False and answers["calls"] == 1
    answers.update(rc=0, calls=0)
    assert f(*args) is True and answers["calls"] == 1
