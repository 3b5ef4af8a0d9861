"""The 4-bit KV cache without a GPU: symbols, refusals, and the restatement's own layout."""
import ctypes
import importlib
import os
import re

import numpy as np
import pytest
import torch

import kv4_model as model

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def native(pkg):
    return importlib.import_module("artifex-assistantv5_amd._native")


@pytest.fixture(scope="module")
def lib(native):
    return native.load_library()


def test_exports_and_constants(lib, native):
    with open(os.path.join(ROOT, "include", "gguf_hip_kv4.h"), encoding="utf-8") as f:
        text = f.read()
    names = re.findall(r"^(?:int|int64_t)\s+(gguf_hip_kv4_\w+)\s*\(", text, re.M)
    assert set(names) == set(native.KV4_SIGNATURES) and len(names) == 7
    for n in names:
        assert hasattr(lib, n)
    d = {m[0]: int(m[1]) for m in re.findall(r"#define\s+GGUF_HIP_KV4_(\w+)\s+(\d+)", text)}
    assert (d["TILE"], d["MAX_SLOTS"], d["MAX_ROWS"]) == (native.KV4_TILE, native.KV4_MAX_SLOTS,
                                                          native.KV4_MAX_ROWS)
    assert (d["WEIGHTS_NONE"], d["WEIGHTS_STORE"], d["WEIGHTS_ADD"]) == (
        native.KV4_WEIGHTS_NONE, native.KV4_WEIGHTS_STORE, native.KV4_WEIGHTS_ADD)


def test_model_layout_covers_every_byte():
    """Every byte of a tile belongs to exactly one slot's codes or scales."""
    for hd in (64, 128, 256):
        seen = np.zeros(36 * hd, int)
        for j in range(32):
            k, v, ks, vs = model._offsets(hd, j)
            for at in (k[:, 0], v[:, 0], ks, ks + 1, vs, vs + 1):
                seen[at] += 1
            assert sorted(k[:, 1:].ravel()) == sorted(v[:, 1:].ravel()) == list(range(hd))
        assert (seen == 1).all()


def test_model_round_trip():
    rng = np.random.default_rng(0)
    cache = np.zeros((1, 2, 2, 36 * 64), np.uint8)
    k, v = rng.standard_normal((2, 64, 64)).astype(np.float32)
    for t in range(64):
        model.put(cache, 0, 1, t, k[t], v[t])
    got = model.get(cache, 64)
    for x, y in zip(got, (k, v)):
        assert np.array_equal(x[0, 1], model.values(*model.quantize(y)))
    assert not got[:, 0, 0].any()


A, B, C, D, W = 0x10000, 0x20000, 0x30000, 0x40000, 0x50000


def test_bytes(lib, native):
    assert lib.gguf_hip_kv4_bytes(3, 8, 128, 64) == 3 * 8 * 2 * 36 * 128
    for bad in ((1, 8, 96, 64), (1, 8, 128, 63), (1, 8, 128, 0), (0, 8, 128, 64), (1, 0, 128, 64),
                (1, 8, 128, (1 << 20) + 32), (8192, 8, 128, 64)):
        assert lib.gguf_hip_kv4_bytes(*bad) == native.ERR_SHAPE, bad
    assert "lists" in native.last_error(lib)


def _append(lib, **over):
    a = dict(qkv=A, ld=6144, rows=4, starts=B, lengths=B, pos=B, cos=C, sin=C, rope=100, kv=D,
             positions=A, weights=A, seqs=2, heads=32, kv_heads=8, hd=128, slots=64)
    a.update(over)
    return lib.gguf_hip_kv4_append(*a.values(), None)


def test_append_refusals(lib, native):
    for over in (dict(heads=33), dict(heads=72), dict(heads=0), dict(hd=32), dict(ld=6140),
                 dict(ld=6146), dict(rope=0), dict(rows=-1), dict(rows=3, starts=None),
                 dict(slots=33), dict(rows=1 << 40)):
        assert _append(lib, **over) == native.ERR_SHAPE, over
    for name in ("qkv", "lengths", "pos", "cos", "sin", "kv"):
        assert _append(lib, **{name: None}) == native.ERR_NULL, name
    for name, off in (("qkv", 4), ("lengths", 4), ("pos", 4), ("cos", 8), ("sin", 4), ("kv", 8),
                      ("positions", 2), ("weights", 2), ("starts", 4)):
        assert _append(lib, **{name: A + off}) == native.ERR_ALIGN, name
    assert _append(lib, rows=0, qkv=None, kv=None) == 0


def _attention(lib, **over):
    a = dict(qkv=A, ld=6144, rows=1, lengths=B, pos=B, cos=C, sin=C, rope=100, kv=D, store=1,
             positions=A, weights=A, mode=1, out=C, ldo=4096, seqs=2, heads=32, kv_heads=8, hd=128,
             slots=64, work=W)
    a.update(over)
    need = over.get("need", lib.gguf_hip_kv4_attention_workspace(
        a["rows"], a["mode"], a["seqs"], a["heads"], a["kv_heads"], a["hd"], a["slots"]))
    a.pop("need", None)
    return lib.gguf_hip_kv4_attention(*a.values(), need, None)


def test_attention_refusals(lib, native):
    for over in (dict(heads=12), dict(heads=72), dict(hd=48), dict(rows=0), dict(rows=65),
                 dict(mode=3), dict(mode=-1), dict(ldo=4092), dict(ldo=4098), dict(ld=100),
                 dict(slots=-32), dict(seqs=0), dict(rope=0)):
        assert _attention(lib, **over) == native.ERR_SHAPE, over
    for name in ("qkv", "lengths", "pos", "cos", "sin", "kv", "out", "work", "weights"):
        assert _attention(lib, **{name: None}) == native.ERR_NULL, name
    for name in ("qkv", "out", "work", "kv", "cos"):
        assert _attention(lib, **{name: A + 8}) == native.ERR_ALIGN, name
    good = lib.gguf_hip_kv4_attention_workspace(1, 1, 2, 32, 8, 128, 64)
    assert good > 0
    assert _attention(lib, need=good - 1) == native.ERR_BYTES
    assert "workspace" in native.last_error(lib)


def test_load_refusals(lib, native):
    f = lib.gguf_hip_kv4_load
    assert f(A, B, C, D, 10, 1, 2, 8, 100, 64, None) == native.ERR_SHAPE
    assert f(A, B, C, D, -1, 1, 2, 8, 128, 64, None) == native.ERR_SHAPE
    assert f(A, B, C, D, 10, 0, 2, 8, 128, 64, None) == native.ERR_SHAPE
    assert f(None, B, C, D, 10, 1, 2, 8, 128, 64, None) == native.ERR_NULL
    assert f(A, B, C + 4, D, 10, 1, 2, 8, 128, 64, None) == native.ERR_ALIGN
    assert f(None, None, None, None, 0, 1, 2, 8, 128, 64, None) == 0


def _evict(lib, **over):
    a = dict(kv=A, weights=B, positions=B, lengths=C, pos=C, keep=32, trigger=33, recent=8, sinks=4,
             wo=B, po=B, lo=C, layers=2, seqs=3, kv_heads=4, hd=64, slots=64, work=W)
    need = over.pop("need", 1 << 40)
    a.update(over)
    return lib.gguf_hip_kv4_evict(*a.values(), need, None)


def test_evict_refusals(lib, native):
    for over in (dict(keep=0), dict(keep=65), dict(recent=33), dict(sinks=25), dict(recent=-1),
                 dict(sinks=-1), dict(hd=72), dict(slots=40), dict(layers=0)):
        assert _evict(lib, **over) == native.ERR_SHAPE, over
    for name in ("kv", "weights", "positions", "lengths", "pos", "wo", "po", "lo", "work"):
        assert _evict(lib, **{name: None}) == native.ERR_NULL, name
    for name, off in (("kv", 8), ("weights", 2), ("positions", 2), ("lengths", 4), ("lo", 4),
                      ("work", 8)):
        assert _evict(lib, **{name: A + off}) == native.ERR_ALIGN, name
    good = lib.gguf_hip_kv4_evict_workspace(2, 3, 4, 64, 64)
    assert _evict(lib, need=good - 1) == native.ERR_BYTES
    assert lib.gguf_hip_kv4_evict_workspace(70000, 1, 1, 64, 64) == native.ERR_SHAPE


def test_python_refuses_host_tensors(pkg):
    kv4 = importlib.import_module("artifex-assistantv5_amd.kv4")
    kv = torch.zeros(1, 2, 2, 36 * 64, dtype=torch.uint8)
    with pytest.raises(ValueError, match="device"):
        kv4.attention_workspace(kv, 4)
    with pytest.raises(ValueError, match="device"):
        kv4.load(kv, torch.zeros(1, dtype=torch.int64), torch.zeros(1), torch.zeros(1))
    with pytest.raises(ValueError, match="slots"):
        kv4.empty(1, 2, 64, 33, device="cpu")


def test_append_row_limit(lib, native):
    """2^25 rows pass the check of their number (the next one, of the pointers, refuses)."""
    assert _append(lib, rows=(1 << 25) + 2) == native.ERR_SHAPE
    assert _append(lib, rows=1 << 25, qkv=None) == native.ERR_NULL


@pytest.fixture
def file_loader(pkg, tmp_path, monkeypatch):
    """load_decoder on a small model file whose tensors are never placed: True if it got there."""
    import gguf_models as gm

    gmodel = importlib.import_module("artifex-assistantv5_amd.gguf_model")

    class Placed(Exception):
        pass

    def place(*a, **k):
        raise Placed

    monkeypatch.setattr(gmodel, "load_gguf_model", place)

    def load(**options):
        p = str(tmp_path / "m.gguf")
        gm.write_model(p, gm.make_model(seed=1))
        try:
            gmodel.load_decoder(p, "cuda", max_seq=128, **options)
        except Placed:
            return True

    return load


def test_cache_options_are_checked_before_a_file_is_loaded(file_loader):
    """A cache that the decoder would refuse is refused before the tensors are placed."""
    assert file_loader()
    assert file_loader(kv_bits=4)
    assert file_loader(kv_bits=4, kv_slots=64, kv_keep=40, kv_recent=16, kv_sinks=2)
    with pytest.raises(TypeError):
        file_loader(kv_bit=4)
    for bad in (dict(kv_bits=8), dict(kv_slots=64), dict(kv_keep=32), dict(kv_bits=4, kv_slots=0),
                dict(kv_bits=4, kv_slots=64, kv_keep=64), dict(kv_bits=4, kv_keep=20, kv_recent=17),
                dict(kv_bits=4, kv_slots=64, kv_keep=0, kv_recent=0, kv_sinks=0),
                dict(kv_bits=4, kv_slots=(1 << 20) + 1), dict(kv_bits=4, fused=False)):
        with pytest.raises(ValueError):
            file_loader(**bad)
