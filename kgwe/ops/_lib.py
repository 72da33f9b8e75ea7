"""ctypes binding of ``libkgwe_ops.so`` (hand-written gfx950 HIP kernels).

The library exports a plain C ABI; every launcher takes device pointers and
the caller's ``hipStream_t`` so launches land on PyTorch's current stream
(and are therefore captured by ``torch.cuda.graph``).

Loading policy: on a machine with a GPU the library MUST load — a missing or
stale build raises instead of silently falling back to eager PyTorch.  On a
CPU-only host the ops dispatch to the fp32 PyTorch references in
``kgwe.ops.reference`` (used by the CPU test-suite and the control plane).
"""
from __future__ import annotations

import ctypes
import os
import struct
from pathlib import Path

import torch
from torch.autograd import forward_ad

# KGWE_OPS_LIB: load another build of the kernels (same-box A/B runs only).
_LIB_PATH = (Path(os.environ["KGWE_OPS_LIB"]) if os.environ.get("KGWE_OPS_LIB")
             else Path(__file__).resolve().parent.parent / "_lib" / "libkgwe_ops.so")
_lib = None

c_void_p = ctypes.c_void_p
c_int = ctypes.c_int
c_int64 = ctypes.c_int64
c_float = ctypes.c_float

_SIGS = {
    "kgwe_rmsnorm_fwd": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                 c_int, c_int, c_float, c_void_p]),
    "kgwe_rmsnorm_bwd": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                 c_void_p, c_void_p, c_void_p, c_int, c_int, c_void_p]),
    "kgwe_rmsnorm_bwd_grid": (c_int, [c_int]),
    "kgwe_swiglu_fwd": (c_int, [c_void_p, c_void_p, c_int64, c_void_p, c_int64, c_int, c_void_p]),
    "kgwe_swiglu_bwd": (c_int, [c_void_p, c_void_p, c_int64, c_void_p, c_void_p, c_void_p,
                                c_int64, c_int64, c_int, c_void_p]),
    "kgwe_swiglu_bwd_t": (c_int, [c_void_p, c_void_p, c_int64, c_void_p, c_void_p, c_void_p,
                                  c_int64, c_void_p, c_int64, c_int, c_void_p]),
    "kgwe_rope_qkv_fwd": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                  c_int64, c_int, c_int, c_int, c_int, c_void_p]),
    "kgwe_rope_qkv_bwd": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                  c_int64, c_int, c_int, c_int, c_int, c_void_p]),
    "kgwe_cross_entropy_fwd": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_int64,
                                       c_int64, c_void_p]),
    "kgwe_cross_entropy_bwd": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                       c_int64, c_int64, c_int64, c_void_p]),
    "kgwe_adamw_step": (c_int, [c_void_p, c_int, c_float, c_float, c_float, c_float,
                                c_float, c_int, c_float, c_int, c_void_p]),
    "kgwe_transpose_bf16": (c_int, [c_void_p, c_void_p, c_int64, c_int64, c_void_p]),
    "kgwe_adamw_chunk_elems": (c_int, []),
    "kgwe_decode_rope_append": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                        c_void_p, c_int, c_int, c_int, c_int, c_int, c_void_p]),
    "kgwe_decode_attn": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int,
                                 c_int, c_int, c_int, c_int, c_int, c_float, c_void_p]),
    "kgwe_decode_attn_rope": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                      c_void_p, c_int, c_int, c_int, c_int, c_int, c_int, c_float, c_void_p]),
    "kgwe_decode_attn_workspace": (c_int64, [c_int, c_int, c_int, c_int]),
    "kgwe_decode_attn_splits": (c_int, [c_int, c_int, c_int]),
    "kgwe_decode_gemv": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_float, c_void_p, c_void_p,
                                 c_void_p, c_int, c_int, c_int, c_int, c_int, c_int, c_void_p]),
    "kgwe_decode_argmax_finish": (c_int, [c_void_p, c_void_p, c_int, c_int, c_void_p]),
    "kgwe_decode_argmax_slots": (c_int, [c_int, c_int, c_int]),
    "kgwe_decode_skinny": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_float, c_void_p, c_void_p,
                                   c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_int, c_void_p]),
    "kgwe_decode_skinny_workspace": (c_int64, [c_int, c_int, c_int, c_int]),
    "kgwe_decode_skinny_blocks": (c_int, [c_int]),
    "kgwe_decode_skinny_slices": (c_int, [c_int, c_int, c_int]),
    "kgwe_decode_skinny_max_m": (c_int, []),
    "kgwe_adamw_tensor_bytes": (c_int, []),
    "kgwe_wgrad_bf16": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int,
                                c_int, c_int, c_int, c_int, c_void_p]),
    "kgwe_wgrad_splits": (c_int, [c_int, c_int, c_int]),
    "kgwe_wgrad_workspace": (c_int64, [c_int, c_int, c_int]),
    "kgwe_norm_rope_bwd_blocks": (c_int, [c_int, c_int, c_int, c_int]),
    "kgwe_packed_plan_jobs": (c_int, [c_int, c_int]),
    "kgwe_packed_plan": (c_int, [c_void_p, c_int, c_int, c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_void_p,
                                 c_void_p]),
    "kgwe_packed_attn_bwd_workspace": (c_int64, [c_int] * 5),
    "kgwe_prefix_attn_workspace": (c_int64, [c_int] * 6),
}
_OPTIONAL_SIGS = {
    "kgwe_flash_attn_fwd": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                    c_int, c_int, c_int, c_int, c_int, c_float, c_int,
                                    c_void_p]),
    "kgwe_flash_attn_bwd": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                    c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                    c_void_p, c_int, c_int, c_int, c_int, c_int, c_float,
                                    c_int, c_void_p]),
    "kgwe_flash_attn_bwd_workspace": (c_int64, [c_int, c_int, c_int, c_int, c_int]),
}


# Entries that take one packed record and the stream (the record's C struct
# stands beside the entry): pointers, then int64, then int32, then fp32 fields.
RECORDS = {name: struct.Struct(f"@{p}Q{q}q{i}i{f}f0q") for name, (p, q, i, f) in {
    "kgwe_packed_attn_fwd": (9, 10, 8, 1),
    "kgwe_packed_attn_bwd": (13, 6, 7, 1),
    "kgwe_norm_rope_fwd": (12, 1, 10, 1),
    "kgwe_norm_rope_bwd": (13, 1, 8, 1),
    "kgwe_prefix_attn": (8, 2, 7, 1),
}.items()}


class KernelLibraryMissing(RuntimeError):
    pass


def gpu_available() -> bool:
    return torch.cuda.is_available()


def lib():
    """Return the loaded library, raising if it is missing on a GPU host."""
    global _lib
    if _lib is not None:
        return _lib
    if not _LIB_PATH.exists():
        raise KernelLibraryMissing(
            f"{_LIB_PATH} not built; run `python -m kgwe._build` (hipcc, gfx950)")
    L = ctypes.CDLL(str(_LIB_PATH), mode=os.RTLD_NOW | os.RTLD_GLOBAL)
    for name, (res, args) in _SIGS.items():
        fn = getattr(L, name)
        fn.restype = res
        fn.argtypes = args
    for name, (res, args) in _OPTIONAL_SIGS.items():
        fn = getattr(L, name, None)
        if fn is not None:
            fn.restype = res
            fn.argtypes = args
    for name, rec in RECORDS.items():
        fn, size = getattr(L, name), getattr(L, name + "_bytes")
        fn.restype, fn.argtypes = c_int, [ctypes.c_char_p, c_void_p]
        size.restype, size.argtypes = c_int, []
        if size() != rec.size:
            raise KernelLibraryMissing(f"{_LIB_PATH}: {name} takes {size()} bytes, expected {rec.size}; rebuild it")
    _lib = L
    return L


def has_symbol(name: str) -> bool:
    try:
        return getattr(lib(), name, None) is not None
    except KernelLibraryMissing:
        return False


def stream(t: torch.Tensor | None = None) -> int:
    dev = t.device if t is not None else None
    return torch.cuda.current_stream(dev).cuda_stream


def ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def check(rc: int, what: str) -> None:
    if rc != 0:
        raise RuntimeError(f"{what} failed with code {rc}")


# Type codes of the kernels that take more than one 16-bit type (native/ops/half_types.h).
HALF_TYPES = {torch.bfloat16: 0, torch.float16: 1}


_FAR = 1 << 22  # elements between rows that the kernels' 32-bit offsets inside a tile of rows reach


def rows16(t: torch.Tensor) -> torch.Tensor:
    """t (2 or 3 dimensions) itself where its last dimension is dense and every row starts on 16
    bytes, behind the one before and not too far from it (what the strided kernels read), else a
    contiguous copy."""
    s = t.stride()
    if s[-1] == 1 and not t.data_ptr() & 15 and not (s[0] | s[-2]) & 7 and t.shape[-1] <= s[-2] <= _FAR:
        return t
    return _plain_strides(dense16(t))


def token_view(t: torch.Tensor) -> tuple:
    """(tensor, address, row stride, head stride) of [T, H, D] as the strided
    kernels read it: t itself where its last dimension is dense and every row
    starts on 16 bytes, behind the one before (a row stride of 0 is a broadcast
    input) and no further than the kernels' 32-bit offsets reach, else a
    contiguous copy."""
    s0, s1, s2 = t.stride()
    at = t.data_ptr()
    if s2 != 1 or (s0 | s1) & 7 or at & 15 or not t.shape[2] <= s0 <= _FAR:
        t = _plain_strides(dense16(t))
        (s0, s1, _), at = t.stride(), t.data_ptr()
    return t, at, s0, s1


def _plain_strides(t: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor with the strides of its shape (torch calls one
    contiguous whatever the strides of its dimensions of size 1)."""
    return t.view(-1).view(t.shape)


def dense16(t: torch.Tensor) -> torch.Tensor:
    """t itself where it is contiguous from a 16-byte boundary on, else a copy."""
    if t.is_contiguous() and not t.data_ptr() & 15:
        return t
    t = t.contiguous()
    return t.clone(memory_format=torch.contiguous_format) if t.data_ptr() & 15 else t


raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def launch(name: str, device: torch.device, *fields) -> None:
    """Call the record entry ``name`` on the current stream of ``device``, with
    ``device`` current whatever the caller's current device is.  (Small calls
    are host-bound: the device is switched only where it differs, the raw stream
    handle stands in for a Stream object, and one packed record for up to 29
    arguments that ctypes converts one by one.)"""
    fn, record, index = getattr(_lib or lib(), name), RECORDS[name].pack(*fields), device.index
    if index == torch.cuda.current_device():
        rc = fn(record, raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(record, raw_stream(index))
    if rc != 0:
        raise RuntimeError(f"{name} failed with code {rc}")


def addr(t: torch.Tensor | None) -> int:
    """Address for a record field: 0 for no tensor."""
    return 0 if t is None else t.data_ptr()


def no_tangents(what: str, *tensors: torch.Tensor | None) -> None:
    """Refuse tensors with a forward-mode derivative: the kernels have none, and to reverse mode such a tensor looks
    like one that wants no gradient.  Holds under torch.no_grad() too, which leaves forward mode on.  (Outside a
    dual level there are no tangents: one comparison.)"""
    if forward_ad._current_level >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError(f"{what} has no forward-mode derivative")


def use_hip(*tensors: torch.Tensor) -> bool:
    """True when the tensors live on a GPU: then the HIP kernels are mandatory."""
    return any(t is not None and t.is_cuda for t in tensors)
