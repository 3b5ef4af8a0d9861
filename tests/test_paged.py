"""The KV cache in pages without a GPU: symbols, refusals, and the restatement itself."""
import importlib
import os
import re

import numpy as np
import pytest
import torch

import paged_model as model

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def native(pkg):
    return importlib.import_module("artifex-assistantv5_amd._native")


@pytest.fixture(scope="module")
def lib(native):
    return native.load_library()


def test_exports_and_constants(lib, native):
    with open(os.path.join(ROOT, "include", "gguf_hip_paged.h"), encoding="utf-8") as f:
        text = f.read()
    names = re.findall(r"^(?:int|int64_t)\s+(gguf_hip_paged_\w+)\s*\(", text, re.M)
    assert set(names) == set(native.PAGED_SIGNATURES) and len(names) == 10
    for n in names:
        assert hasattr(lib, n)
    d = {m[0]: int(m[1]) for m in re.findall(r"#define\s+GGUF_HIP_PAGED_(\w+)\s+(\d+)", text)}
    assert (d["F16"], d["BF16"]) == (native.PAGED_F16, native.PAGED_BF16)
    assert (d["MAX_SEQS"], d["MAX_SLOTS"], d["MAX_PAGES"]) == (
        native.PAGED_MAX_SEQS, native.PAGED_MAX_SLOTS, native.PAGED_MAX_PAGES)


def test_model_layout_covers_every_value():
    pool = torch.zeros(2, 2, 3, 32, 64)
    for h in range(3):
        for j in range(32):
            model.put(pool, 1, h, j, torch.ones(64), torch.ones(64))
    assert (pool[1] == 1).all() and (pool[0] == 0).all()
    pool[1, 1, 2].view(2, 64, 16)[1, 7, 3] = 5
    assert model.get(pool, 1, 2, 19)[1][7] == 5


def test_model_fork_then_grow():
    """Two forks of a half-filled page: each that goes on copies it but the last one."""
    t = np.array([[3, 1], [-1, -1], [0, -1]], np.int32)
    n, refs = np.array([20, 0, 5]), np.array([1, 1, 0, 1, 0, 0], np.int32)
    t, n, refs = model.fork(t, n, refs, [0, 0, 0])
    assert t.tolist() == [[3, 1]] * 3 and n.tolist() == [20] * 3
    assert refs.tolist() == [0, 3, 0, 3, 0, 0]
    t, refs, room, copies = model.grow(t, n, refs, [1, 1, 1], 16)
    assert t.tolist() == [[3, 0], [3, 2], [3, 1]] and room.tolist() == [32] * 3
    assert copies == [(1, 0, 1), (1, 2, 1)] and refs.tolist() == [1, 1, 1, 3, 0, 0]


A, B, C, D, W = 0x10000, 0x20000, 0x30000, 0x40000, 0x50000


def test_bytes(lib, native):
    assert lib.gguf_hip_paged_bytes(7, 32, 8, 128) == 7 * 2 * 8 * 32 * 128 * 2
    for bad in ((0, 16, 8, 128), (7, 8, 8, 128), (7, 48, 8, 128), (7, 512, 8, 128), (7, 0, 8, 128),
                (7, -16, 8, 128), (7, 16, 0, 128), (7, 16, 1025, 128), (7, 16, 8, 96),
                ((1 << 24) + 1, 16, 8, 128)):
        assert lib.gguf_hip_paged_bytes(*bad) == native.ERR_SHAPE, bad


def _append(lib, **over):
    a = dict(qkv=A, ld=6144, rows=4, starts=B, lengths=B, room=B, tables=A, cos=C, sin=C, rope=100,
             kv=D, dtype=1, pages=10, page=16, columns=4, seqs=2, heads=32, kv_heads=8, hd=128)
    a.update(over)
    return lib.gguf_hip_paged_append(*a.values(), None)


SHAPES = (dict(hd=32), dict(kv_heads=0), dict(pages=0), dict(page=24), dict(columns=0),
          dict(columns=1 << 18, page=32), dict(seqs=0), dict(seqs=4097), dict(columns=-1))


def test_append_refusals(lib, native):
    for over in SHAPES + (dict(heads=33), dict(heads=72), dict(heads=0), dict(ld=6140),
                          dict(ld=6146), dict(rope=0), dict(rope=1 << 31), dict(rows=-1),
                          dict(rows=3, starts=None), dict(rows=1 << 40),
                          dict(seqs=4096, kv_heads=16, heads=16)):
        assert _append(lib, **over) == native.ERR_SHAPE, over
    assert _append(lib, dtype=0) == native.ERR_DTYPE
    assert "f16 (1) or bf16 (2)" in native.last_error(lib)
    for name in ("qkv", "lengths", "tables", "cos", "sin", "kv"):
        assert _append(lib, **{name: None}) == native.ERR_NULL, name
    for name, off in (("qkv", 4), ("lengths", 4), ("tables", 2), ("cos", 8), ("sin", 4), ("kv", 8),
                      ("starts", 4), ("room", 4)):
        assert _append(lib, **{name: A + off}) == native.ERR_ALIGN, name
    assert _append(lib, rows=0, qkv=None, kv=None) == 0


def _attention(lib, **over):
    a = dict(qkv=A, ld=6144, lengths=B, room=B, tables=A, cos=C, sin=C, rope=100, kv=D, dtype=2,
             out=C, ldo=4096, pages=10, page=16, columns=40, seqs=2, heads=32, kv_heads=8, hd=128,
             work=W)
    a.update(over)
    need = over.get("need", lib.gguf_hip_paged_attention_workspace(
        a["page"], a["columns"], a["seqs"], a["heads"], a["kv_heads"], a["hd"]))
    a.pop("need", None)
    return lib.gguf_hip_paged_attention(*a.values(), need, None)


def test_attention_refusals(lib, native):
    for over in SHAPES + (dict(heads=12), dict(heads=72), dict(ldo=4092), dict(ldo=4098),
                          dict(ld=100), dict(rope=0), dict(seqs=4096, kv_heads=16, heads=16)):
        assert _attention(lib, **over) == native.ERR_SHAPE, over
    assert _attention(lib, dtype=3) == native.ERR_DTYPE
    for name in ("qkv", "lengths", "tables", "cos", "sin", "kv", "out", "work"):
        assert _attention(lib, **{name: None}) == native.ERR_NULL, name
    for name, off in (("qkv", 4), ("lengths", 4), ("tables", 2), ("cos", 8), ("sin", 4), ("kv", 8),
                      ("room", 4), ("out", 4), ("work", 8)):
        assert _attention(lib, **{name: A + off}) == native.ERR_ALIGN, name
    assert _attention(lib, need=15) == native.ERR_BYTES


def _load(lib, **over):
    a = dict(kv=D, dtype=1, tables=A, lengths=B, k=C, v=C, out_slots=8, pages=10, page=16,
             columns=4, seqs=2, kv_heads=8, hd=128)
    a.update(over)
    return lib.gguf_hip_paged_load(*a.values(), None)


def test_load_refusals(lib, native):
    for over in SHAPES + (dict(out_slots=-1),):
        assert _load(lib, **over) == native.ERR_SHAPE, over
    assert _load(lib, dtype=0) == native.ERR_DTYPE
    for name in ("kv", "tables", "lengths", "k", "v"):
        assert _load(lib, **{name: None}) == native.ERR_NULL, name
        assert _load(lib, **{name: A + 2}) == native.ERR_ALIGN, name
    assert _load(lib, out_slots=0, kv=None) == 0


def _fork(lib, **over):
    a = dict(tables=A, lengths=B, refs=C, parents=D, tables_out=A, lengths_out=B, refs_out=C,
             pages=10, columns=4, seqs=2)
    a.update(over)
    return lib.gguf_hip_paged_fork(*a.values(), None)


def test_fork_refusals(lib, native):
    for over in (dict(pages=0), dict(columns=0), dict(columns=(1 << 18) + 1), dict(seqs=0),
                 dict(seqs=4097), dict(tables_out=A + 16), dict(lengths_out=B - 8),
                 dict(refs_out=C + 36)):
        assert _fork(lib, **over) == native.ERR_SHAPE, over
    assert "overlaps" in native.last_error(lib)
    for name in ("tables", "lengths", "refs", "parents", "tables_out", "lengths_out", "refs_out"):
        assert _fork(lib, **{name: None}) == native.ERR_NULL, name
        assert _fork(lib, **{name: W + 2}) == native.ERR_ALIGN, name


def _grow(lib, **over):
    a = dict(kv=D, tables=A, lengths=B, refs=C, rows=B, room=W, layers=2, pages=10, page=16,
             columns=4, seqs=2, kv_heads=8, hd=128, work=W, need=4096)
    a.update(over)
    return lib.gguf_hip_paged_grow(*a.values(), None)


def _compact(lib, **over):
    a = dict(kv=D, tables=A, refs=C, tables_out=A, refs_out=C, live=W, layers=2, pages=10, page=16,
             columns=4, seqs=2, kv_heads=8, hd=128, work=W, need=4096)
    a.update(over)
    return lib.gguf_hip_paged_compact(*a.values(), None)


@pytest.mark.parametrize("call,names", [
    (_grow, ("kv", "tables", "lengths", "refs", "rows", "room", "work")),
    (_compact, ("kv", "tables", "refs", "tables_out", "refs_out", "live", "work"))])
def test_grow_and_compact_refusals(lib, native, call, names):
    for over in SHAPES + (dict(layers=0), dict(layers=65536)):
        assert call(lib, **over) == native.ERR_SHAPE, over
    for name in names:
        assert call(lib, **{name: None}) == native.ERR_NULL, name
        assert call(lib, **{name: W + 2}) == native.ERR_ALIGN, name
    assert call(lib, need=15) == native.ERR_BYTES
    if call is _compact:
        assert call(lib, tables_out=A + 4) == native.ERR_SHAPE
        assert call(lib, refs_out=C - 4) == native.ERR_SHAPE


def test_grow_refuses_room_over_its_inputs(lib, native):
    """rows may be lengths (both are only read), room neither nor a part of them."""
    for over in (dict(room=B), dict(room=B + 8), dict(rows=A + 64, room=A + 64),
                 dict(rows=A + 64, room=A + 56)):
        assert _grow(lib, **over) == native.ERR_SHAPE, over
    assert "room overlaps" in native.last_error(lib)


def test_python_refusals_without_device_tensors(pkg):
    """What the Python layer can tell before the library is called."""
    paged = importlib.import_module("artifex-assistantv5_amd.paged")
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        paged.empty(4, 2, 64, dtype=torch.float32, device="cpu")
    with pytest.raises(ValueError, match="not 16, 32, 64, 128 or 256"):
        paged.empty(4, 2, 64, page=20, device="cpu")
    kv = paged.empty(4, 2, 64, device="cpu")
    t, n, r = paged.empty_tables(2, 3, 4, device="cpu")
    with pytest.raises(ValueError, match="device tensor"):
        paged.grow_workspace(kv, t)
    with pytest.raises(ValueError, match="device tensor"):
        paged.fork(t, n, r, n)


def _words(native, op, *args):
    return native._PACK[op](*args)


def test_packed_calls(lib, native):
    """The entry points by number: their own refusals, and those of the array."""
    with open(os.path.join(ROOT, "include", "gguf_hip_packed.h"), encoding="utf-8") as f:
        text = f.read()
    assert re.findall(r"^int\s+(gguf_hip_\w+)\(", text, re.M) == list(native.PACKED_SIGNATURES)
    d = {m[0].lower(): int(m[1]) for m in re.findall(r"#define\s+GGUF_HIP_PACKED_(\w+)\s+(\d+)", text)}
    assert d == {n[len("gguf_hip_"):]: i for i, n in enumerate(native.PACKED)}
    call = lib.gguf_hip_packed_call
    fork = [A, B, C, D, A, B, C, 10, 4, 2, 0]
    for change, want in (({7: 0}, native.ERR_SHAPE), ({9: 0}, native.ERR_SHAPE),
                         ({0: 0}, native.ERR_NULL), ({1: B + 4}, native.ERR_ALIGN),
                         ({9: 1 << 32}, native.ERR_SHAPE), ({9: -(1 << 31) - 1}, native.ERR_SHAPE)):
        words = _words(native, native.PAGED_FORK, *[change.get(i, v) for i, v in enumerate(fork)])
        assert call(native.PAGED_FORK, words, len(words)) == want, change
    assert "out of range" in native.last_error(lib)
    words = _words(native, native.PAGED_FORK, *fork)
    assert call(native.PAGED_FORK, words, len(words) - 8) == native.ERR_BYTES
    assert call(native.PAGED_FORK, None, len(words)) == native.ERR_NULL
    for op in (-1, len(native.PACKED)):
        assert call(op, words, len(words)) == native.ERR_SHAPE
    # every entry point takes as many words as it has arguments
    for op, name in enumerate(native.PACKED):
        signature = {**native.PAGED_SIGNATURES, **native.SAMPLE_SIGNATURES}[name][1]
        zeros = bytes(8 * len(signature))
        assert call(op, zeros, len(zeros)) in (native.ERR_SHAPE, 0), name
        assert call(op, zeros, len(zeros) + 8) == native.ERR_BYTES, name
    # floats and integers arrive as they are: the settings come after the counts that are refused
    sample = [A, 10, 2, 10, A, 0, 0.7, 0, 3, 0, 0.5, 0, 0.25, A, 0, W, 0, 0]
    words = _words(native, native.SAMPLE, *sample)
    assert call(native.SAMPLE, words, len(words)) == native.ERR_BYTES     # its workspace of 0 bytes
