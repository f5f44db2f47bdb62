"""ctypes binding of libnvm_attn.so (the C ABI declared in include/nvm_attn.h).

There is no CPU path: every operator raises if the library is missing or the
tensors are not on a CUDA device.  The library is built in-tree by
``nano-vllm-metal_b200/build.py`` (``__graft_entry__.build()`` calls it).
"""

from __future__ import annotations

import contextlib
import ctypes
import os
import threading

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libnvm_attn.so")

NVM_F32, NVM_F16, NVM_BF16, NVM_I8, NVM_I32, NVM_I64, NVM_U4 = 0, 1, 2, 3, 4, 5, 6
NVM_OK = 0
NVM_ERR_WORKSPACE = -3

_DTYPE_CODE = {
    torch.float32: NVM_F32,
    torch.float16: NVM_F16,
    torch.bfloat16: NVM_BF16,
    torch.int8: NVM_I8,
    torch.int32: NVM_I32,
    torch.int64: NVM_I64,
    torch.uint8: NVM_U4,  # pages of packed 4-bit codes
}
U4_GROUP = 64  # elements of a 4-bit row that share a scale and an offset

# Every exported symbol of include/nvm_attn.h with (restype, argtypes).
_P, _I, _I64, _F, _SZ, _CP = (ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float,
                              ctypes.c_size_t, ctypes.c_char_p)
SIGNATURES = {
    "nvm_status_string": (_CP, [_I]),
    "nvm_last_error": (_CP, []),
    "nvm_version": (_CP, []),
    "nvm_device_error": (_I, [_P, _I]),
    "nvm_selftest_wait_expiry": (_I, [_I64, _P, _P]),
    "nvm_paged_attention": (_I, [_P, _I, _P, _P, _I, _P, _P, _I, _P, _P, _P, _I, _I64, _I64, _I64, _I64, _I64,
                                 _I64, _I64, _I64, _F, _I, _P, _SZ, _P]),
    "nvm_paged_attention_workspace_size": (_SZ, [_I64, _I64, _I64, _I64, _I64, _I64, _I64, _I]),
    "nvm_paged_attention_noalloc": (_I, [_P, _I, _P, _P, _I, _P, _P, _I, _P, _P, _P, _I, _I64, _I64, _I64, _I64,
                                         _I64, _I64, _I64, _I64, _F, _I, _P]),
    "nvm_flash_attention": (_I, [_P, _P, _P, _I, _P, _I64, _I64, _I64, _P, _I, _I64, _I64, _I64, _I64, _I64,
                                 _I64, _F, _I, _P]),
    "nvm_paged_attention_window": (_I, [_P, _I, _P, _P, _I, _P, _P, _I, _P, _P, _P, _I, _I64, _I64, _I64, _I64, _I64,
                                        _I64, _I64, _I64, _F, _I, _I64, _I64, _P, _I64, _I64, _I64, _P, _SZ, _P]),
    "nvm_paged_attention_window_workspace_size": (_SZ, [_I64, _I64, _I64, _I64, _I64, _I64, _I64, _I, _I64, _I64, _I]),
    "nvm_flash_attention_window": (_I, [_P, _P, _P, _I, _P, _I, _I64, _I64, _I64, _I64, _I64, _I64, _F, _I, _I64,
                                        _I64, _P]),
    "nvm_paged_evict": (_I, [_P, _P, _I, _P, _P, _I, _P, _P, _P, _P, _I64, _I64, _I64, _P, _I64, _I64, _I64, _I64,
                             _I64, _I64, _I64, _I64, _I64, _I64, _I64, _P, _P, _P, _P, _P, _P]),
    "nvm_stream_capture_id": (_I, [_P, _P]),
    "nvm_reshape_and_cache": (_I, [_P, _P, _I, _I64, _I64, _P, _P, _I, _P, _P, _I, _P, _I64, _I64, _I64, _I64,
                                   _I64, _P]),
    "nvm_read_slots": (_I, [_P, _P, _I, _P, _P, _I, _P, _P, _P, _I, _I64, _I64, _I64, _I64, _I64, _P]),
    "nvm_paged_append": (_I, [_P, _P, _P, _P, _P, _P, _P, _P, _I64, _P, _I64, _I64, _I64, _I64, _P]),
    "nvm_paged_rewind": (_I, [_P, _P, _P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _P]),
    "nvm_paged_attach": (_I, [_P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _P]),
    "nvm_spec_verify_accept": (_I, [_P, _P, _I64, _I64, _I, _P, _P, _P, _P, _P, _P, _P, _P, _P]),
    "nvm_w4a16_matmul": (_I, [_P, _I, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _P]),
    "nvm_qk_norm_rope_write": (_I, [_P, _P, _P, _I, _I64, _I64, _P, _P, _F, _P, _P, _I64, _I, _P, _P, _I64, _P,
                                    _P, _I, _P, _P, _I, _P, _I64, _I64, _I64, _I64, _I64, _I64, _P]),
}

_lib = None
_lock = threading.Lock()


def lib() -> ctypes.CDLL:
    """Load libnvm_attn.so once; raise if it has not been built."""
    global _lib
    if _lib is None:
        with _lock:
            if _lib is None:
                if not os.path.exists(LIB_PATH):
                    raise RuntimeError(
                        f"libnvm_attn.so not found at {LIB_PATH}; build it with "
                        "`python nano-vllm-metal_b200/build.py` (nvcc, sm_100a)")
                handle = ctypes.CDLL(LIB_PATH)
                for name, (res, args) in SIGNATURES.items():
                    fn = getattr(handle, name)
                    fn.restype = res
                    fn.argtypes = args
                _lib = handle
    return _lib


def dtype_code(dtype: torch.dtype) -> int:
    try:
        return _DTYPE_CODE[dtype]
    except KeyError:
        raise RuntimeError(f"nvm: unsupported dtype {dtype}") from None


def check(status: int) -> None:
    """Raise RuntimeError carrying the library's message for a failed call."""
    if status != NVM_OK:
        L = lib()
        msg = L.nvm_last_error().decode() or L.nvm_status_string(status).decode()
        raise RuntimeError(f"{msg} [{L.nvm_status_string(status).decode()}]")


def require_cuda(op: str, *tensors: torch.Tensor) -> torch.device:
    """All tensors must live on one CUDA device; returns it."""
    dev = None
    for t in tensors:
        if t is None:
            continue
        i = t.get_device()  # -1 on the host
        if i < 0 or not t.is_cuda:
            raise RuntimeError(f"{op}: tensors must be on a CUDA device (libnvm_attn has no CPU path)")
        if dev is None:
            dev, index = t.device, i
        elif i != index:
            raise RuntimeError(f"{op}: all tensors must be on the same CUDA device")
    if dev is None:
        raise RuntimeError(f"{op}: no tensor given")
    return dev


def require_u4(op: str, D: int, key_pages: torch.Tensor, value_pages: torch.Tensor, key_scales: torch.Tensor | None,
               value_scales: torch.Tensor | None) -> None:
    """The pools of a 4-bit cache of head dim D: uint8 [P, Hkv, page_size, D/2] with scales and offsets
    [P, Hkv, page_size, D/32], all contiguous."""
    if D != 128 and D != 64:
        raise RuntimeError(f"{op}: 4-bit pages need a head dimension of 64 or 128 (got {D})")
    shape = key_pages.shape
    if value_pages.dtype is not torch.uint8 or len(shape) != 4 or value_pages.shape != shape or shape[3] * 2 != D:
        raise RuntimeError(f"{op}: 4-bit key_pages and value_pages must be uint8 [P, Hkv, page_size, D / 2]")
    if key_scales is None or value_scales is None:
        raise RuntimeError(f"{op}: 4-bit pages need key_scales and value_scales")
    scales = key_scales.shape
    if scales != (*shape[:3], 2 * D // U4_GROUP) or value_scales.shape != scales:
        raise RuntimeError(f"{op}: scales of 4-bit pages must be [P, Hkv, page_size, {2 * D // U4_GROUP}] (a scale and an offset "
                           f"for every {U4_GROUP} elements)")
    dtype = key_scales.dtype
    if dtype is not value_scales.dtype or (dtype is not torch.bfloat16 and dtype is not torch.float16):
        raise RuntimeError(f"{op}: scales of 4-bit pages must both be float16 or both bfloat16")
    if not (key_pages.is_contiguous() and value_pages.is_contiguous() and key_scales.is_contiguous()
            and value_scales.is_contiguous()):
        raise RuntimeError(f"{op}: 4-bit pages and their scales must be contiguous")


def packed(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """x as contiguous numbers of a type; x itself where it is that already (two calls fewer, 1 us)."""
    return x if x.dtype is dtype and x.is_contiguous() else x.to(dtype).contiguous()


def ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def stream_ptr(device: torch.device) -> int:
    """The current stream's handle, without building a torch.cuda.Stream (2 us a call)."""
    index = device.index if device.index is not None else torch.cuda.current_device()
    return torch._C._cuda_getCurrentRawStream(index)


_HERE_ALREADY = contextlib.nullcontext()


def on_device(device: torch.device):
    """torch.cuda.device(device), or nothing to do when it is the current device."""
    if device.index is None or device.index == torch._C._cuda_getDevice():
        return _HERE_ALREADY
    return torch.cuda.device(device)


# Split-K workspace: one zero-filled buffer per (device, stream), grown on demand.
# Successful calls leave its ticket region zero; calls on one stream never overlap on
# the GPU.  A call whose bounded wait expired may leave tickets non-zero, so
# device_error() re-zeroes every workspace of the device after a non-zero word.
_workspaces: dict[tuple[int, int], torch.Tensor] = {}
# A call that uses the workspace may launch several kernels, the later ones on what the first left
# there, and ctypes drops the interpreter lock meanwhile: host threads that share a stream take turns.
# Reentrant, since a signal handler or a finaliser may call from inside a call of its own thread.
_workspace_locks: dict = {}  # (device, stream) -> threading.RLock


def _workspace_key(device: torch.device) -> tuple[int, int]:
    return device.index if device.index is not None else torch.cuda.current_device(), stream_ptr(device)


def workspace_lock(device: torch.device):
    """To be held from ``workspace(device, ...)`` until the call that uses it has returned."""
    return _workspace_locks.setdefault(_workspace_key(device), threading.RLock())


def workspace(device: torch.device, nbytes: int) -> torch.Tensor | None:
    if nbytes == 0:
        return None
    key = _workspace_key(device)
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
        _workspaces[key] = ws
    return ws


# The workspace of the capture that runs (or ran last) on a stream, with that capture's id.
_captured: dict[tuple[int, int], tuple[int, torch.Tensor]] = {}


def capture_id(stream: int) -> int:
    """The id of the CUDA graph capture on a stream, different for every capture (0: none)."""
    out = ctypes.c_uint64(0)
    check(lib().nvm_stream_capture_id(stream, ctypes.byref(out)))
    return out.value


def call_with_workspace(device: torch.device, size, call) -> None:
    """Run ``call(pointer, nbytes, stream) -> status`` with a workspace of ``size()`` bytes.

    The buffer cached for (device, stream) is offered first, whatever its size: a call that
    needs more says so before any GPU work, and only then is the size asked for and the buffer
    grown.  Threads on one stream take turns (0.5 us).

    While a CUDA graph is being captured, the calls of one capture and stream share a buffer of
    their graph's memory pool instead, whose tickets a node of the graph zeroes in front of the
    first of them (1.3-2 us a replay): a graph replays with the addresses it captured, on any
    stream, beside any other graph, and after eager calls that needed a larger buffer."""
    key = _workspace_key(device)
    stream = key[1]
    with _workspace_locks.get(key) or workspace_lock(device):
        if torch.cuda.is_current_stream_capturing():
            graph = capture_id(stream)
            held, ws = _captured.get(key, (0, None))
            if held != graph:
                ws = None
            status = call(ptr(ws), 0 if ws is None else ws.numel(), stream)
            if status == NVM_ERR_WORKSPACE:
                ws = torch.empty(size(), dtype=torch.uint8, device=device)
                ws[:1 << 20].zero_()
                _captured[key] = graph, ws
                status = call(ptr(ws), ws.numel(), stream)
        else:
            ws = _workspaces.get(key)
            status = call(ptr(ws), 0 if ws is None else ws.numel(), stream)
            if status == NVM_ERR_WORKSPACE:
                nbytes = size()
                status = call(ptr(workspace(device, nbytes)), nbytes, stream)
    check(status)


def device_error(device: torch.device, clear: bool = True) -> int:
    """Synchronise and read the device error word (0 = no bounded wait expired).

    After a non-zero word (a kernel gave up on a wait and returned early), the split-K
    workspaces cached for this device are zero-filled again once the device is idle,
    so the next call cannot merge a half-finished call's tickets or partials.
    """
    with torch.cuda.device(device):
        word = int(lib().nvm_device_error(stream_ptr(device), 1 if clear else 0))
        if word != 0:
            index = device.index if device.index is not None else torch.cuda.current_device()
            torch.cuda.synchronize(device)
            for (dev_index, _), ws in list(_workspaces.items()):
                if dev_index == index:
                    ws.zero_()
            torch.cuda.synchronize(device)
        return word
