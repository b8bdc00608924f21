"""ctypes binding of libg4b_attn.so (declared in include/g4b_attn.h).

The library is the product: if it is missing or cannot be loaded every op raises, there is
no fallback path.  Tensor-like arguments are anything with ``.shape``, ``.stride`` (a
sequence or a callable), ``.dtype`` and ``.data_ptr()``, which is what the reference's
launcher accepts (g4b/kernels/utils.py:51-60,113-122).
"""
from __future__ import annotations

import ctypes
import os
import struct
import sys
from pathlib import Path

_LIB_PATH = Path(__file__).resolve().parent / "lib" / "libg4b_attn.so"

# enum G4bDtype
F32, F16, BF16, I32, I64, U8, FP8_E4M3 = 0, 1, 2, 3, 4, 5, 6

_DTYPE_NAMES = {
    "float32": F32, "f32": F32, "float": F32,
    "float16": F16, "f16": F16, "half": F16,
    "bfloat16": BF16, "bf16": BF16,
    "int32": I32, "i32": I32,
    "int64": I64, "i64": I64, "long": I64,
    "uint8": U8, "u8": U8,
    "float8_e4m3fn": FP8_E4M3, "fp8_e4m3": FP8_E4M3,
}


class G4bTensor(ctypes.Structure):
    _fields_ = [
        ("ptr", ctypes.c_void_p),
        ("shape", ctypes.c_int64 * 5),
        ("stride", ctypes.c_int64 * 5),
        ("ndim", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
    ]


class G4bAttnArgs(ctypes.Structure):
    _fields_ = [
        ("q", G4bTensor), ("k_cache", G4bTensor), ("v_cache", G4bTensor), ("o", G4bTensor),
        ("time_dim_sizes", G4bTensor), ("user_phase", G4bTensor),
        ("partial_o", G4bTensor), ("partial_l", G4bTensor), ("partial_m", G4bTensor),
        ("block_tables", G4bTensor),
        ("ctx_window_size", ctypes.c_int32), ("phase", ctypes.c_int32), ("stage", ctypes.c_int32),
        ("page_size", ctypes.c_int32), ("sliding_window", ctypes.c_int32),
        ("num_kv_splits", ctypes.c_int32), ("scale", ctypes.c_float), ("reserved", ctypes.c_int32),
    ]


class G4bCombineArgs(ctypes.Structure):
    _fields_ = [
        ("partial_o", G4bTensor), ("partial_l", G4bTensor), ("partial_m", G4bTensor), ("o", G4bTensor),
        ("user_phase", G4bTensor), ("num_splits", ctypes.c_int32), ("phase", ctypes.c_int32),
    ]


class G4bAppendArgs(ctypes.Structure):
    _fields_ = [
        ("x", G4bTensor), ("cache", G4bTensor), ("cache_offsets", G4bTensor), ("x_rsos", G4bTensor),
        ("user_phase", G4bTensor), ("block_tables", G4bTensor),
        ("rmsnorm_eps", ctypes.c_float), ("phase", ctypes.c_int32), ("page_size", ctypes.c_int32),
        ("reserved", ctypes.c_int32),
    ]


class G4bRopeAppendArgs(ctypes.Structure):
    _fields_ = [
        ("q", G4bTensor), ("k", G4bTensor), ("v", G4bTensor), ("q_out", G4bTensor), ("k_out", G4bTensor),
        ("rope_freqs", G4bTensor), ("cache_offsets", G4bTensor),
        ("q_rsos", G4bTensor), ("k_rsos", G4bTensor), ("v_rsos", G4bTensor),
        ("q_norm_w", G4bTensor), ("k_norm_w", G4bTensor),
        ("k_cache", G4bTensor), ("v_cache", G4bTensor),
        ("user_phase", G4bTensor), ("block_tables", G4bTensor),
        ("rmsnorm_eps", ctypes.c_float), ("phase", ctypes.c_int32), ("page_size", ctypes.c_int32),
        ("norm_qk", ctypes.c_int32), ("norm_v", ctypes.c_int32), ("reserved", ctypes.c_int32),
    ]


class G4bExchangeArgs(ctypes.Structure):
    _fields_ = [
        ("partial_o", G4bTensor), ("partial_l", G4bTensor), ("partial_m", G4bTensor), ("o", G4bTensor),
        ("user_phase", G4bTensor),
        ("xbuf", ctypes.c_void_p * 8), ("state", ctypes.c_void_p),
        ("xbuf_bytes", ctypes.c_int64),
        ("num_splits", ctypes.c_int32), ("phase", ctypes.c_int32), ("world", ctypes.c_int32), ("rank", ctypes.c_int32),
    ]


class G4bDecodeStepArgs(ctypes.Structure):
    _fields_ = [
        ("attn", G4bAttnArgs), ("k_new", G4bTensor), ("v_new", G4bTensor),
        ("xbuf", ctypes.c_void_p * 8), ("state", ctypes.c_void_p), ("xbuf_bytes", ctypes.c_int64),
        ("world", ctypes.c_int32), ("rank", ctypes.c_int32),
    ]


class G4bFp8AppendArgs(ctypes.Structure):
    _fields_ = [
        ("x", G4bTensor), ("cache", G4bTensor), ("scales", G4bTensor), ("cache_offsets", G4bTensor),
        ("x_rsos", G4bTensor), ("user_phase", G4bTensor), ("block_tables", G4bTensor),
        ("rmsnorm_eps", ctypes.c_float), ("headroom", ctypes.c_float), ("phase", ctypes.c_int32),
        ("page_size", ctypes.c_int32),
    ]


class G4bFp8DequantArgs(ctypes.Structure):
    _fields_ = [
        ("cache", G4bTensor), ("scales", G4bTensor), ("out", G4bTensor), ("block_tables", G4bTensor),
        ("time_dim_sizes", G4bTensor), ("user_phase", G4bTensor), ("phase", ctypes.c_int32), ("page_size", ctypes.c_int32),
    ]


class G4bAdvanceArgs(ctypes.Structure):
    _fields_ = [
        ("input_token_ids", G4bTensor), ("out_token_ids", G4bTensor), ("cache_offsets", G4bTensor),
        ("time_dim_sizes", G4bTensor), ("user_phase", G4bTensor),
    ]


class G4bRopePackedArgs(ctypes.Structure):
    _fields_ = [
        ("q", G4bTensor), ("k", G4bTensor), ("v", G4bTensor), ("q_out", G4bTensor), ("rope_freqs", G4bTensor),
        ("positions", G4bTensor), ("pair_axis", G4bTensor), ("q_starts", G4bTensor), ("time_dim_sizes", G4bTensor),
        ("q_norm_w", G4bTensor), ("k_norm_w", G4bTensor), ("k_pool", G4bTensor), ("v_pool", G4bTensor),
        ("block_tables", G4bTensor), ("rmsnorm_eps", ctypes.c_float), ("page_size", ctypes.c_int32),
        ("norm_qk", ctypes.c_int32), ("norm_v", ctypes.c_int32),
    ]


class G4bPackedAttnArgs(ctypes.Structure):
    _fields_ = [
        ("q", G4bTensor), ("o", G4bTensor), ("k_pool", G4bTensor), ("v_pool", G4bTensor), ("q_starts", G4bTensor),
        ("time_dim_sizes", G4bTensor), ("block_tables", G4bTensor), ("workspace", G4bTensor),
        ("page_size", ctypes.c_int32), ("stage", ctypes.c_int32), ("sliding_window", ctypes.c_int32), ("scale", ctypes.c_float),
    ]


class G4bPagePool(ctypes.Structure):
    _fields_ = [("ptr", ctypes.c_void_p), ("page_bytes", ctypes.c_int64)]


class G4bPageCopyArgs(ctypes.Structure):
    _fields_ = [
        ("pools", ctypes.POINTER(G4bPagePool)), ("num_pages", ctypes.c_int64), ("src_pages", G4bTensor),
        ("dst_pages", G4bTensor), ("num_pools", ctypes.c_int32), ("reserved", ctypes.c_int32),
    ]


# every symbol include/g4b_attn.h declares: name -> (restype, argtypes)
EXPORTS = {
    "g4b_flash_attention": (ctypes.c_int, [ctypes.POINTER(G4bAttnArgs), ctypes.c_void_p]),
    "g4b_attn_prefill": (ctypes.c_int, [ctypes.POINTER(G4bAttnArgs), ctypes.c_void_p]),
    "g4b_attn_decode": (ctypes.c_int, [ctypes.POINTER(G4bAttnArgs), ctypes.c_void_p]),
    "g4b_attn_decode_static_scratch": (ctypes.c_int, [ctypes.POINTER(G4bAttnArgs), ctypes.c_void_p]),
    "g4b_decode_step": (ctypes.c_int, [ctypes.POINTER(G4bDecodeStepArgs), ctypes.c_void_p]),
    "g4b_kv_append_fp8": (ctypes.c_int, [ctypes.POINTER(G4bFp8AppendArgs), ctypes.c_void_p]),
    "g4b_kv_dequant_fp8": (ctypes.c_int, [ctypes.POINTER(G4bFp8DequantArgs), ctypes.c_void_p]),
    "g4b_flash_attention_fp8": (ctypes.c_int, [ctypes.POINTER(G4bAttnArgs), ctypes.POINTER(G4bTensor),
                                               ctypes.POINTER(G4bTensor), ctypes.c_void_p]),
    "g4b_attn_combine": (ctypes.c_int, [ctypes.POINTER(G4bCombineArgs), ctypes.c_void_p]),
    "g4b_attn_combine_exchange": (ctypes.c_int, [ctypes.POINTER(G4bExchangeArgs), ctypes.c_void_p]),
    "g4b_exchange_buffer_bytes": (ctypes.c_int64, [ctypes.c_int, ctypes.c_int64, ctypes.c_int]),
    "g4b_select_kv_splits": (ctypes.c_int, [ctypes.c_int] * 4),
    "g4b_kv_append": (ctypes.c_int, [ctypes.POINTER(G4bAppendArgs), ctypes.c_void_p]),
    "g4b_rope_norm_append": (ctypes.c_int, [ctypes.POINTER(G4bRopeAppendArgs), ctypes.c_void_p]),
    "g4b_advance_decode_state": (ctypes.c_int, [ctypes.POINTER(G4bAdvanceArgs), ctypes.c_void_p]),
    "g4b_rope_norm_append_packed": (ctypes.c_int, [ctypes.POINTER(G4bRopePackedArgs), ctypes.c_void_p]),
    "g4b_flash_attention_packed": (ctypes.c_int, [ctypes.POINTER(G4bPackedAttnArgs), ctypes.c_void_p]),
    "g4b_packed_workspace_bytes": (ctypes.c_int64, [ctypes.c_int64, ctypes.c_int64, ctypes.c_int, ctypes.c_int]),
    "g4b_page_copy": (ctypes.c_int, [ctypes.POINTER(G4bPageCopyArgs), ctypes.c_void_p]),
    "g4b_last_error_string": (ctypes.c_char_p, []),
    "g4b_abi_version": (ctypes.c_int, []),
    "g4b_device_status": (ctypes.c_int, [ctypes.c_void_p, ctypes.POINTER(ctypes.c_int32)]),
    "g4b_set_validate_only": (None, [ctypes.c_int]),
}

_lib = None
_fast = None                # the module of csrc/views.cpp
_fast_looked_for = False
_address: dict = {}         # entry point -> its address in the loaded library


def lib_path() -> Path:
    return Path(os.environ.get("G4B_B200_LIB", str(_LIB_PATH)))


def load() -> ctypes.CDLL:
    """Loads the library once; raises if it has not been built (python -m g4b_b200.build)."""
    global _lib
    if _lib is None:
        path = lib_path()
        if not path.exists():
            raise RuntimeError(
                f"{path} is missing: build it with `python -m g4b_b200.build` (needs nvcc). "
                "There is no fallback implementation."
            )
        lib = ctypes.CDLL(str(path))
        for name, (restype, argtypes) in EXPORTS.items():
            fn = getattr(lib, name)
            fn.restype = restype
            fn.argtypes = argtypes
        _lib = lib
        _address.update({name: ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in EXPORTS})
        _load_fast()
    return _lib


def _load_fast() -> None:
    """The compiled argument packing, where it has been built for the torch and the Python that run and torch is in use
    (whether that was imported before the library was loaded or after); without it the Python code packs."""
    global _fast, _fast_looked_for
    torch = sys.modules.get("torch")
    if _fast_looked_for or not hasattr(torch, "__version__") or not hasattr(torch, "Tensor"):     # (not there, or being imported)
        return
    _fast_looked_for = True
    path = _LIB_PATH.parent / "_views.so"
    if not path.exists():
        return
    import importlib.util

    spec = importlib.util.spec_from_file_location("_views", path)
    try:
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
    except ImportError:          # symbols that this torch does not have
        return
    if getattr(module, "built_for", None) == f"{torch.__version__} {sys.version.split()[0]} {sys.implementation.cache_tag}":
        _fast = module


def pack_tail(packer: struct.Struct, *values) -> bytes:
    """The plain numbers at the end of an argument struct; ValueError for what does not fit their 32 bits."""
    try:
        return packer.pack(*values)
    except (struct.error, OverflowError) as e:
        raise ValueError(f"argument out of range: {e}") from None


def call(name: str, args_type, tensors: tuple, tail: bytes, stream) -> None:
    """Entry point ``name`` on an argument struct that is the views of ``tensors`` (None: not given) and ``tail``."""
    lib = _lib if _lib is not None else load()
    if not _fast_looked_for:
        _load_fast()
    if _fast is not None:
        rc = _fast.call(_address[name], _validate_only_depth == 0, stream if stream is None or type(stream) is int else current_stream(stream),
                        tail, tensors)
        if rc is not None:
            if rc != 0:
                check(rc)
            return
    a = args_type.from_buffer_copy(views(*tensors) + tail)
    check(getattr(lib, name)(ctypes.byref(a), current_stream(stream)))


_dtype_codes: dict = {}     # dtype objects seen so far: spelling one out costs more than the rest of a view


def page_copy(pools: list, src_pages, dst_pages, stream) -> bool:
    """``g4b_page_copy`` through the compiled packing; False where that is for the Python code (or an error of its)."""
    if _lib is None:
        load()
    if not _fast_looked_for:
        _load_fast()
    if _fast is None:
        return False
    rc = _fast.page_copy(_address["g4b_page_copy"], _validate_only_depth == 0,
                         stream if stream is None or type(stream) is int else current_stream(stream), pools, src_pages, dst_pages)
    if rc is None:
        return False
    check(rc)
    return True


def dtype_code(dt) -> int:
    try:
        code = _dtype_codes.get(dt)
    except TypeError:            # a dtype that cannot be a key
        code = None
    if code is not None:
        return code
    name = getattr(dt, "name", None) or str(dt)
    name = name.replace("torch.", "").replace("numpy.", "").lower()
    if name not in _DTYPE_NAMES:
        raise TypeError(f"unsupported dtype {dt!r}")
    code = _DTYPE_NAMES[name]
    if type(dt).__module__ == "torch":
        _dtype_codes[dt] = code
    return code


def _strides(t) -> list[int]:
    if isinstance(t.stride, (list, tuple)):
        return list(t.stride)
    if callable(t.stride):
        return [t.stride(i) for i in range(len(t.shape))]
    raise RuntimeError("Failed to normalize tensor stride into list[int]")


_validate_only_depth = 0


class validate_only:
    """``with _cabi.validate_only():`` -- the library checks arguments and launches nothing
    (g4b_set_validate_only), and the wrappers accept host tensors.  For tests of the argument
    checks on machines without a GPU; a call that passes every check returns normally."""

    def __enter__(self):
        global _validate_only_depth
        _validate_only_depth += 1
        load().g4b_set_validate_only(1)
        return self

    def __exit__(self, *exc):
        global _validate_only_depth
        _validate_only_depth -= 1
        if _validate_only_depth == 0:
            load().g4b_set_validate_only(0)
        return False


def _check_device(t) -> None:
    """A kernel given a host pointer, or a pointer into another GPU's memory that is not
    mapped here, faults.  Torch tensors say where they live, so refuse them here; other
    tensor-likes (the reference's own Tensor class) carry no device and pass."""
    is_cuda = getattr(t, "is_cuda", None)
    if is_cuda is None or _validate_only_depth > 0:
        return
    if not is_cuda:
        raise ValueError("expected a CUDA tensor, got one in host memory")
    import torch

    cur = torch.cuda.current_device()
    if t.device.index is not None and t.device.index != cur:
        raise ValueError(f"tensor lives on cuda:{t.device.index} but the current device is cuda:{cur}; "
                         "make its device current (torch.cuda.device) before the call")


# a G4bTensor as bytes: pointer, 5 extents, 5 strides, rank, dtype.  Packed in one go: field by
# field a view costs three times as much, and a call packs a dozen.
_VIEW = struct.Struct("@P5q5qii")
_VIEW_OF_RANK = [struct.Struct(f"@P{n}q{8 * (5 - n)}x{n}q{8 * (5 - n)}xii") for n in range(6)]     # (pad bytes are zeros)
_ABSENT = bytes(_VIEW.size)
assert _VIEW.size == ctypes.sizeof(G4bTensor)


def _view_bytes(t) -> bytes:
    """The C view of one tensor-like that is not a torch tensor."""
    if not (hasattr(t, "shape") and hasattr(t, "stride") and hasattr(t, "dtype") and hasattr(t, "data_ptr")):
        raise TypeError(f"expected a tensor-like with shape/stride/dtype/data_ptr, got {type(t).__name__}")
    _check_device(t)
    shape, strides = [int(x) for x in t.shape], [int(x) for x in _strides(t)]
    n = len(shape)
    if n > 5:
        raise ValueError("tensors of rank > 5 are not supported")
    strides = strides[:n] + [0] * (n - len(strides))
    return _VIEW_OF_RANK[n].pack(int(t.data_ptr()), *shape, *strides, n, dtype_code(t.dtype))


def views(*tensors) -> bytes:
    """The C views of tensor-likes (None: not given) behind one another, as bytes."""
    if not _fast_looked_for:
        _load_fast()
    if _fast is not None:
        packed = _fast.views(_validate_only_depth == 0, tensors)
        if packed is not None:
            return packed
    torch = sys.modules.get("torch")
    if torch is None:
        return b"".join([_ABSENT if t is None else _view_bytes(t) for t in tensors])
    Tensor, packers, codes = torch.Tensor, _VIEW_OF_RANK, _dtype_codes
    current = -1 if _validate_only_depth else None          # the current device, asked for once
    out = []
    for t in tensors:
        if t is None:
            out.append(_ABSENT)
        elif isinstance(t, Tensor):
            if current != -1:
                device = t.get_device()
                if device != current:
                    if current is None and device >= 0:
                        current = torch.cuda.current_device()
                    if device != current:
                        _check_device(t)
            shape = t.shape
            n = len(shape)
            if n > 5:
                raise ValueError("tensors of rank > 5 are not supported")
            code = codes.get(t.dtype)
            out.append(packers[n].pack(t.data_ptr(), *shape, *t.stride(), n, dtype_code(t.dtype) if code is None else code))
        else:
            out.append(_view_bytes(t))
    return b"".join(out)


def as_tensor(t) -> G4bTensor:
    """Packs a tensor-like (or None) into the C view; strides are in elements."""
    return G4bTensor.from_buffer_copy(views(t))


def current_stream(stream=None) -> int:
    """Raw cudaStream_t: an int, an object with .cuda_stream, or torch's current stream."""
    if stream is None:
        torch = sys.modules.get("torch")
        if torch is None:
            import torch
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)      # (without the Stream object: 0.1 us instead of 3.3)
        return int(raw(torch.cuda.current_device()) if raw is not None else torch.cuda.current_stream().cuda_stream)
    if isinstance(stream, int):
        return stream
    for attr in ("cuda_stream", "handle"):
        if hasattr(stream, attr):
            return int(getattr(stream, attr))
    raise TypeError(f"cannot take a CUDA stream from {stream!r}")


_VALUE_ERRORS = {-1, -2, -3, -4, -7}


def check(rc: int) -> None:
    """Maps a G4B_ERR_* code to ValueError (bad arguments) or RuntimeError (CUDA / device)."""
    if rc == 0 or rc == 1:      # 1 = G4B_VALIDATED (validate-only mode)
        return
    msg = load().g4b_last_error_string().decode("utf-8", "replace")
    if rc in _VALUE_ERRORS:
        raise ValueError(msg)
    raise RuntimeError(f"libg4b_attn error {rc}: {msg}")


def device_status(stream=None) -> int:
    """Synchronises the stream and returns (and clears) the device status word."""
    out = ctypes.c_int32(0)
    rc = load().g4b_device_status(ctypes.c_void_p(current_stream(stream)), ctypes.byref(out))
    if rc != -6:                # G4B_ERR_DEVICE_WAIT only says that the word was not zero
        check(rc)
    return int(out.value)
