"""ctypes binding of ``libgguf_hip.so`` (the C ABI in ``include/gguf_hip.h``).

The library is loaded after ``torch`` so that its ``libamdhip64.so.7``
dependency resolves (by SONAME) to the HIP runtime torch already loaded:
one runtime per process, so torch's device pointers and ``hipStream_t``
handles are valid in the library.  Loading refuses to continue if two HIP
runtimes end up mapped, and raises if the library has not been built — there
is no fallback path.
"""

from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import os
import struct

from .ggml import GGMLTypeError

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libgguf_hip.so")
ABI_VERSION = 18

ERR_TYPE, ERR_SHAPE, ERR_NULL, ERR_ALIGN, ERR_DTYPE, ERR_BYTES, ERR_HIP = -1, -2, -3, -4, -5, -6, -7
VARIANT_AUTO, VARIANT_DECODE, VARIANT_GEMM = 0, 1, 2
ONE_SHOT_MAX_K = 16384  # one row of up to this K needs no matmul workspace
PROLOGUE_NONE, PROLOGUE_RMSNORM, PROLOGUE_SWIGLU = 0, 1, 2
EPILOGUE_STORE, EPILOGUE_ACCUMULATE, EPILOGUE_SWIGLU = 0, 1, 2
DECODE_MAX_M = 32
NOALLOC_ATTENTION_BYTES = 8 << 20

# Every symbol include/gguf_hip.h declares: name -> (restype, argtypes)
_vp, _i32, _i64, _fp = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_void_p
SIGNATURES = {
    "gguf_hip_abi_version": (_i32, []),
    "gguf_hip_last_error": (ctypes.c_char_p, []),
    "gguf_hip_type_traits": (_i32, [_i32, ctypes.POINTER(_i32), ctypes.POINTER(_i32)]),
    "gguf_hip_raw_bytes": (_i64, [_i32, _i64, _i64]),
    "gguf_hip_tile_bytes": (_i64, [_i32, _i64, _i64]),
    "gguf_hip_repack": (_i32, [_vp, _i64, _i32, _i64, _i64, _vp, _i64, _vp]),
    "gguf_hip_dequant": (_i32, [_vp, _i32, _i64, _i64, _fp, _i64, _vp]),
    "gguf_hip_dequant_raw": (_i32, [_vp, _i32, _i64, _fp, _vp]),
    "gguf_hip_get_rows": (_i32, [_vp, _i32, _i64, _i64, _vp, _i64, _fp, _i64, _vp]),
    "gguf_hip_matmul": (_i32, [_vp, _i32, _i64, _vp, _i32, _i64, _i64, _fp, _i64, _i64, _vp]),
    "gguf_hip_matmul_variant": (_i32, [_vp, _i32, _i64, _vp, _i32, _i64, _i64, _fp, _i64, _i64,
                                       _i32, _vp]),
    "gguf_hip_matmul_ws": (_i32, [_vp, _i32, _i64, _vp, _i32, _i64, _i64, _fp, _i64, _i64, _i32,
                                  _vp, _i64, _vp]),
    "gguf_hip_matmul_workspace": (_i64, [_i32, _i32, _i64, _i64, _i64]),
    "gguf_hip_matmul_fused": (_i32, [_fp, _vp, _i32, _i64, _i64, _fp, _i32, _fp, ctypes.c_float,
                                     _i32, _vp]),
    "gguf_hip_rmsnorm": (_i32, [_fp, _fp, ctypes.c_float, _fp, _i64, _i64, _vp]),
    "gguf_hip_add_rmsnorm": (_i32, [_fp, _fp, _fp, ctypes.c_float, _fp, _i64, _i64, _vp]),
    "gguf_hip_swiglu": (_i32, [_fp, _fp, _i64, _i64, _vp]),
    "gguf_hip_attention_decode": (_i32, [_fp, _vp, _fp, _fp, _fp, _fp, _fp, _i32, _i32, _i32,
                                         _i64, _vp, _vp]),
    "gguf_hip_attention_workspace": (_i64, [_i32, _i32, _i32, _i64]),
    "gguf_hip_attention_decode_noalloc": (_i32, [_fp, _vp, _fp, _fp, _fp, _fp, _fp, _i32, _i32,
                                                 _i32, _i64, _vp]),
    "gguf_hip_attention_prefill": (_i32, [_fp, _i64, _vp, _i64, _fp, _fp, _fp, _fp, _fp, _i64,
                                          _i32, _i32, _i32, _i64, _vp]),
    "gguf_hip_matmul_attn_merge": (_i32, [_vp, _vp, _i32, _i32, _i32, _i64, _vp, _i32, _i64, _fp,
                                          _i32, _vp]),
    "gguf_hip_argmax": (_i32, [_fp, _i64, _vp, _vp, _vp]),
    "gguf_hip_argmax_workspace": (_i64, []),
}

# Every symbol include/gguf_hip_kv4.h declares (the 4-bit KV cache)
KV4_TILE, KV4_MAX_SLOTS, KV4_MAX_ROWS = 32, 1 << 20, 64
KV4_WEIGHTS_NONE, KV4_WEIGHTS_STORE, KV4_WEIGHTS_ADD = 0, 1, 2
KV4_SIGNATURES = {
    "gguf_hip_kv4_bytes": (_i64, [_i32, _i32, _i32, _i64]),
    "gguf_hip_kv4_append": (_i32, [_fp, _i64, _i64, _vp, _vp, _vp, _fp, _fp, _i64, _vp, _vp, _fp,
                                   _i32, _i32, _i32, _i32, _i64, _vp]),
    "gguf_hip_kv4_attention": (_i32, [_fp, _i64, _i32, _vp, _vp, _fp, _fp, _i64, _vp, _i32, _vp,
                                      _fp, _i32, _fp, _i64, _i32, _i32, _i32, _i32, _i64, _vp,
                                      _i64, _vp]),
    "gguf_hip_kv4_attention_workspace": (_i64, [_i32, _i32, _i32, _i32, _i32, _i32, _i64]),
    "gguf_hip_kv4_load": (_i32, [_vp, _vp, _fp, _fp, _i64, _i32, _i32, _i32, _i32, _i64, _vp]),
    "gguf_hip_kv4_evict": (_i32, [_vp, _fp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _fp, _vp, _vp,
                                  _i32, _i32, _i32, _i32, _i64, _vp, _i64, _vp]),
    "gguf_hip_kv4_evict_workspace": (_i64, [_i32, _i32, _i32, _i32, _i64]),
}

# Every symbol include/gguf_hip_paged.h declares (the KV cache in pages)
PAGED_F16, PAGED_BF16 = 1, 2
PAGED_MAX_SEQS, PAGED_MAX_SLOTS, PAGED_MAX_PAGES = 4096, 1 << 22, 1 << 24
PAGED_SIGNATURES = {
    "gguf_hip_paged_bytes": (_i64, [_i64, _i32, _i32, _i32]),
    "gguf_hip_paged_append": (_i32, [_fp, _i64, _i64, _vp, _vp, _vp, _vp, _fp, _fp, _i64, _vp, _i32,
                                     _i64, _i32, _i64, _i32, _i32, _i32, _i32, _vp]),
    "gguf_hip_paged_attention": (_i32, [_fp, _i64, _vp, _vp, _vp, _fp, _fp, _i64, _vp, _i32, _fp,
                                        _i64, _i64, _i32, _i64, _i32, _i32, _i32, _i32, _vp, _i64,
                                        _vp]),
    "gguf_hip_paged_attention_workspace": (_i64, [_i32, _i64, _i32, _i32, _i32, _i32]),
    "gguf_hip_paged_load": (_i32, [_vp, _i32, _vp, _vp, _fp, _fp, _i64, _i64, _i32, _i64, _i32,
                                   _i32, _i32, _vp]),
    "gguf_hip_paged_fork": (_i32, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _i32, _vp]),
    "gguf_hip_paged_grow": (_i32, [_vp, _vp, _vp, _vp, _vp, _vp, _i32, _i64, _i32, _i64, _i32, _i32,
                                   _i32, _vp, _i64, _vp]),
    "gguf_hip_paged_grow_workspace": (_i64, [_i64, _i32, _i64, _i32]),
    "gguf_hip_paged_compact": (_i32, [_vp, _vp, _vp, _vp, _vp, _vp, _i32, _i64, _i32, _i64, _i32,
                                      _i32, _i32, _vp, _i64, _vp]),
    "gguf_hip_paged_compact_workspace": (_i64, [_i64, _i64, _i32]),
}

# Every symbol include/gguf_hip_sample.h declares
SAMPLE_MAX_VOCAB, SAMPLE_MAX_ROWS = 1 << 20, 65535
SAMPLE_SIGNATURES = {
    "gguf_hip_sample": (_i32, [_fp, _i64, _i64, _i64, _fp, _fp, ctypes.c_float, _vp, ctypes.c_int32,
                               _fp, ctypes.c_float, _fp, ctypes.c_float, _vp, _fp, _vp, _i64, _vp]),
    "gguf_hip_sample_workspace": (_i64, [_i64, _i64]),
}

# Every symbol include/gguf_hip_packed.h declares, and the entry points it reaches: their number
# there and the struct format of their arguments, the stream's handle last.
PACKED_SIGNATURES = {"gguf_hip_packed_call": (_i32, [_i32, ctypes.c_char_p, _i64])}


def _format(signature):
    return struct.Struct("".join("f4x" if t is ctypes.c_float else ("Q" if t is _vp else "q")
                                 for t in signature[1]))


PACKED = ["gguf_hip_paged_append", "gguf_hip_paged_attention", "gguf_hip_paged_load",
          "gguf_hip_paged_fork", "gguf_hip_paged_grow", "gguf_hip_paged_compact", "gguf_hip_sample"]
(PAGED_APPEND, PAGED_ATTENTION, PAGED_LOAD, PAGED_FORK, PAGED_GROW, PAGED_COMPACT,
 SAMPLE) = range(len(PACKED))
_PACK = [_format({**PAGED_SIGNATURES, **SAMPLE_SIGNATURES}[name]).pack for name in PACKED]


class GGUFHipError(RuntimeError):
    """A HIP runtime or launch failure reported by the library."""

    def __init__(self, code: int, msg: str):
        super().__init__(msg)
        self.code = code


_lib = None


def _hip_runtimes_mapped() -> set[str]:
    paths = set()
    try:
        with open("/proc/self/maps", encoding="utf-8") as f:
            for line in f:
                p = line.split()[-1] if line.strip() else ""
                if os.path.basename(p).startswith("libamdhip64.so"):
                    paths.add(os.path.realpath(p))
    except OSError:
        pass
    return paths


def load_library(path: str | None = None) -> ctypes.CDLL:
    """Load (once) and return the native library; raises if it is missing."""
    global _lib
    if _lib is not None and path is None:
        return _lib
    import torch  # noqa: F401  — bind to torch's HIP runtime first

    p = path or LIB_PATH
    if not os.path.exists(p):
        raise RuntimeError(
            f"{p} is not built; run `python artifex-assistantv5_amd/build.py` "
            "(the GGUF HIP path has no CPU fallback)")
    lib = ctypes.CDLL(p, mode=ctypes.RTLD_GLOBAL)
    for name, (res, args) in {**SIGNATURES, **KV4_SIGNATURES, **PAGED_SIGNATURES,
                                **SAMPLE_SIGNATURES, **PACKED_SIGNATURES}.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    if lib.gguf_hip_abi_version() != ABI_VERSION:
        raise RuntimeError(f"libgguf_hip ABI {lib.gguf_hip_abi_version()} != {ABI_VERSION}")
    runtimes = _hip_runtimes_mapped()
    if len(runtimes) > 1:
        raise RuntimeError(f"two HIP runtimes mapped in this process: {sorted(runtimes)}")
    if path is None:
        _lib = lib
    return lib


_tensors = None


def direct():
    """The module of calls straight from tensors (csrc/tensors.cpp), which return False where their
    arguments do not fit and raise by ``check`` where the call failed; raises if it is missing."""
    global _tensors
    if _tensors is None:
        lib = load_library()
        path = os.path.join(os.path.dirname(LIB_PATH), "_tensors.so")
        if not os.path.exists(path):
            raise RuntimeError(f"{path} is not built; run `python artifex-assistantv5_amd/build.py`")
        loader = importlib.machinery.ExtensionFileLoader("_tensors", path)
        module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_tensors", loader))
        module.bind(*(ctypes.cast(getattr(lib, name), _vp).value for name in PACKED))
        module.on_failure(check)
        _tensors = module
    return _tensors


def last_error(lib=None) -> str:
    lib = lib or load_library()
    msg = lib.gguf_hip_last_error()
    return msg.decode() if msg else ""


def check(rc: int, lib=None) -> int:
    """Map a negative return code onto the exception the reference would throw."""
    if rc >= 0:
        return rc
    msg = last_error(lib) or f"libgguf_hip error {rc}"
    if rc == ERR_TYPE:
        raise GGMLTypeError(msg)
    if rc in (ERR_SHAPE, ERR_NULL, ERR_ALIGN, ERR_DTYPE, ERR_BYTES):
        raise ValueError(msg)
    raise GGUFHipError(rc, msg)


def call(op: int, device: int, *args) -> None:
    """Entry point ``PACKED[op]`` with ``args`` (addresses, 0 for none, and numbers) on the current
    stream of ``device``, which need not be the current one.  The arguments go as one array of words:
    passed one by one, they cost more than the call's checks and launches together."""
    import torch  # loaded before the library anyway

    packed = _PACK[op](*args, torch._C._cuda_getCurrentRawStream(device))
    lib = _lib or load_library()
    if torch._C._cuda_getDevice() == device:
        rc = lib.gguf_hip_packed_call(op, packed, len(packed))
    else:
        with torch.cuda.device(device):
            rc = lib.gguf_hip_packed_call(op, packed, len(packed))
    if rc:
        check(rc, lib)
