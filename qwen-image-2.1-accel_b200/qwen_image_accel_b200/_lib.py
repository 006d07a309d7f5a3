"""ctypes binding of libqia_b200.so (the C ABI declared in include/qia_b200.h).

The library is loaded from this package directory. There is no fallback: if
the shared library is missing or fails to load, every op raises.
"""
from __future__ import annotations

import ctypes
import threading
from pathlib import Path

import torch

LIB_PATH = Path(__file__).resolve().parent / "libqia_b200.so"

_P = ctypes.c_void_p
_I = ctypes.c_int64
_F = ctypes.c_float



class GemmProblem(ctypes.Structure):
    """qia_mxfp8_gemm_problem: one GEMM of a qia_mxfp8_gemm_grouped launch."""
    _fields_ = [("a_values", _P), ("a_scales", _P), ("b_values", _P), ("b_scales", _P), ("bias", _P),
                ("gate", _P), ("resid", _P), ("out", _P), ("ldo", _I), ("q_values", _P), ("q_scales", _P),
                ("m", _I), ("rows_per_batch", _I)]


EPI_BF16, EPI_GELU_QUANT, EPI_GATE_RESIDUAL, EPI_GELU_BF16 = 0, 1, 2, 3


class LnProblem(ctypes.Structure):
    """qia_ln_mod_quant_problem: one problem of a qia_ln_mod_quant_grouped launch."""
    _fields_ = [("x", _P), ("scale", _P), ("shift", _P), ("q_values", _P), ("q_scales", _P), ("rows", _I),
                ("rows_per_batch", _I)]

# name -> argument types (all return int status)
SIGNATURES: dict[str, list] = {
    "qia_mxfp8_gemm_grouped": [ctypes.c_int, _P, ctypes.c_int, _I, _I, _P],
    "qia_ln_mod_quant_grouped": [_P, ctypes.c_int, _I, _F, _P],
    "qia_adaln_modulation": [_P, _P, _P, _P, _I, _I, _I, _I, _P],
    "qia_cfg_euler": [_P, _P, _P, _P, _I, _I, _F, _F, _P],
    "qia_cfg_euler_sched": [_P, _P, _P, _P, _I, _I, _F, _P, _P],
    "qia_rope21_table": [_P, _I, _P, _I, _P, _P, _P, _I, _I, _I, _I, _I, _P, _P],
    "qia_proj_out_cfg_euler": [_P, _P, _P, _P, _P, _I, _I, _I, _F, _P, _P],
    "qia_ln_mod": [_P, _P, _P, _P, _I, _I, _I, _F, _P],
    "qia_ln_mod_quant": [_P, _P, _P, _P, _P, _I, _I, _I, _F, _P],
    "qia_gated_residual": [_P, _P, _P, _P, _I, _I, _I, _P],
    "qia_adaln_residual": [_P, _P, _P, _P, _P, _P, _I, _I, _I, _F, _P],
    "qia_rms_norm": [_P, _P, _P, _I, _I, _F, _P],
    "qia_rope_qk": [_P, _P, _P, _P, _P, _I, _I, _I, _I, _P],
    "qia_qknorm_rope_pack": [_P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _F, _F, _P],
    "qia_qknorm_rope_segment": [_P, _I, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _F, _F, _P],
    "qia_swiglu": [_P, _P, _P, _I, _P],
    "qia_swiglu_quant": [_P, _P, _P, _P, _I, _I, _P],
    "qia_gelu_tanh": [_P, _P, _I, _P],
    "qia_mxfp8_quantize": [_P, _I, _P, _P, _I, _I, _P],
    "qia_mxfp8_gemm": [_P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _P],
    "qia_mxfp8_gemm_gelu": [_P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _P],
    "qia_mxfp8_gemm_gelu_quant": [_P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _P],
    "qia_mxfp8_gemm_gate_residual": [_P, _P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _P],
    "qia_device_error": [_P],
    "qia_sage_attention": [_P, _P, _P, _P, _I, _I, _I, _I, _I, _P, _F, _P, _I, _P],
    "qia_mxfp8_gemm_swiglu_quant": [_P, _P, _P, _P, _P, _P, _I, _I, _I, _P],
    "qia_sage_attention_prefill": [_P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _P, _F, _P, _I, _P],
    "qia_sage_attention_split": [_P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _P, _F, _P, _I, _P],
    "qia_sage_attention_split_mx": [_P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _P, _F, _P, _I, _P],
    "qia_sage_attention_noalloc": [_P, _P, _P, _P, _I, _I, _I, _I, _I, _P, _F, _P],
    "qia_sage_quantize": [_P, _P, _P, _I, _I, _I, _I, _I, _P, _P, _I, _P],
    "qia_sage_quantize_joint": [_P, _I, _P, _I, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _F, _P, _I, _P],
    "qia_sage_attention_joint_mx": [_P, _I, _P, _I, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I,
                                    _F, _F, _P, _I, _P],
    "qia_sage_attn_quantized": [_P, _P, _I, _I, _I, _I, _I, _P, _F, _P],
}

SIGNATURES.update({
    "qia_ipc_alloc": [_I, ctypes.POINTER(ctypes.c_void_p), _P],
    "qia_ipc_open": [_P, ctypes.POINTER(ctypes.c_void_p)],
    "qia_ipc_close": [_P],
    "qia_ipc_free": [_P],
    "qia_ulysses_scatter_qkv": [_P, _I, _I, _I, _I, _P, _P, _P, _I, _I, _P],
    "qia_ulysses_wait": [_P, _P, _I, _I, _I, _P],
    "qia_sage_attn_quantized_peers": [_P, _I, _I, _I, _I, _P, _P, _I, _I, _I, _I, _P, _I, _F, _P],
})

SIGNATURES.update({
    "qia_kv_cache_write": [_P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _P, _P, _P],
    "qia_kv_cache_read": [_P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _P, _P],
    "qia_cached_attention": [_P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _I, _P, _I, _F, _P, _P],
    "qia_lora_add": [_P, _P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _P, _P, _P],
})

# entry points that do not return a status code: name -> (restype, argtypes)
RAW_SIGNATURES: dict[str, tuple] = {
    "qia_sage_workspace_bytes": (ctypes.c_int64, [_I, _I, _I, _I]),
    "qia_ipc_handle_bytes": (ctypes.c_int64, []),
    "qia_cached_attention_workspace_bytes": (ctypes.c_int64, [_I, _I, _I, _I, _I, _I]),
    "qia_lora_workspace_bytes": (ctypes.c_int64, [_I, _I, _I]),
    "qia_sage_attn_ctas": (ctypes.c_int64, [_I, _I, _I]),
}

_lock = threading.Lock()
_lib: ctypes.CDLL | None = None
_launches: ctypes.c_int64 | None = None      # qia_launches of the loaded library


class QiaError(RuntimeError):
    """A qia_* entry point returned a non-zero status."""

    def __init__(self, name: str, code: int, message: str):
        super().__init__(f"{name} failed with status {code}: {message}")
        self.code = code


def load() -> ctypes.CDLL:
    global _lib, _launches
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not LIB_PATH.exists():
                raise RuntimeError(f"{LIB_PATH} is missing: build it with "
                                   "`python qwen-image-2.1-accel_b200/build.py` (no CPU fallback exists)")
            lib = ctypes.CDLL(str(LIB_PATH))
            lib.qia_last_error_string.restype = ctypes.c_char_p
            lib.qia_last_error_string.argtypes = []
            lib.qia_abi_version.restype = ctypes.c_int
            for name, args in SIGNATURES.items():
                fn = getattr(lib, name)
                fn.argtypes = args
                fn.restype = ctypes.c_int
            for name, (res, args) in RAW_SIGNATURES.items():
                fn = getattr(lib, name)
                fn.argtypes = args
                fn.restype = res
            _launches = ctypes.c_int64.in_dll(lib, "qia_launches")
            _lib = lib
    return _lib


def declared_symbols() -> list[str]:
    return ["qia_last_error_string", "qia_abi_version", *SIGNATURES, *RAW_SIGNATURES]


# kernels each entry point queues (for launch accounting); default 1, None where the
# library counts them itself
KERNELS_PER_CALL = {"qia_sage_attention": 4, "qia_sage_attention_split": 4, "qia_sage_quantize": 3,
                    "qia_sage_attention_split_mx": 4, "qia_sage_quantize_joint": 3, "qia_sage_attention_joint_mx": 4,
                    "qia_sage_attention_noalloc": 4, "qia_sage_attention_prefill": 4,
                    "qia_device_error": 0,
                    **dict.fromkeys(("qia_kv_cache_write", "qia_kv_cache_read", "qia_cached_attention",
                                     "qia_lora_add"))}
launch_count = 0


def call(name: str, *args) -> None:
    """Invoke a qia_* entry point and raise QiaError on a non-zero status."""
    global launch_count
    lib = _lib or load()
    kernels = KERNELS_PER_CALL.get(name, 1)
    if kernels is None:
        before = _launches.value
        rc = getattr(lib, name)(*args)
        launch_count += _launches.value - before
    else:
        launch_count += kernels
        rc = getattr(lib, name)(*args)
    if rc != 0:
        msg = lib.qia_last_error_string().decode(errors="replace")
        raise QiaError(name, rc, msg)


def device_error() -> int:
    """Read and clear the device-side error word (synchronises the device)."""
    v = ctypes.c_int(0)
    call("qia_device_error", ctypes.byref(v))
    return v.value


def ptr(t: torch.Tensor | None):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def stream(device: torch.device | None = None):
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


# handle of the current stream of a device index, without the Stream object
# around it (2.4 us of a small op's call); None in a torch without CUDA, which can
# import this package but calls nothing
raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def used_strides(strides, *shapes) -> list[int]:
    """The leading strides of tensors (one after another, as many of each as its
    entry of `shapes` has sizes) with 0 for dimensions of size 1: nothing is ever
    that far apart, so what a view has there need not be a multiple of anything."""
    return [0 if n == 1 else s for n, s in zip((n for shape in shapes for n in shape), strides)]


def overlaps(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors of one element size share an element (exact: columns
    of one buffer that lie beside each other do not)."""
    at, other = a.data_ptr(), b.data_ptr()
    if at > other:
        a, b, at, other = b, a, other, at
    size, end = a.element_size(), 1
    for n, s in zip(a.shape, a.stride()):
        end += (n - 1) * s
    if at + end * size <= other or not a.numel() or not b.numel():
        return False
    # b's first element is at sum stride x of a minus the same of b, 0 <= x < size; with
    # b's x counted from their ends every term is positive, and terms of one stride add up
    target = (other - at) // size
    most: dict[int, int] = {}
    for n, s in zip(a.shape, a.stride()):
        if n > 1 and s:
            most[s] = most.get(s, 0) + n - 1
    for n, s in zip(b.shape, b.stride()):
        if n > 1 and s:
            most[s] = most.get(s, 0) + n - 1
            target += s * (n - 1)
    rest = sum(s * m for s, m in most.items())
    if not 0 <= target <= rest:
        return False
    terms = sorted(most.items(), reverse=True)

    def reached(i: int, target: int, rest: int) -> bool:
        if i == len(terms):
            return target == 0
        s, m = terms[i]
        rest -= s * m
        return any(reached(i + 1, target - s * x, rest)
                   for x in range(max(0, -((rest - target) // s)), min(m, target // s) + 1))

    return reached(0, target, rest)


def require_cuda(*tensors: torch.Tensor | None) -> None:
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise ValueError("qwen_image_accel_b200 ops run on CUDA tensors only (no CPU path)")
