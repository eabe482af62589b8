"""ctypes binding of libictc_cuda.so (the C ABI declared in include/ictc_cuda.h).

The library is loaded from this folder only.  There is no fallback: if it is
missing or was built for another ABI version, every CUDA-backend operation
raises.  Tensor arguments are passed as raw device pointers; the stream is
torch's current stream for the tensors' device.
"""
import ctypes
import os
import threading

import torch

LIBRARY_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libictc_cuda.so")
ABI_VERSION = 3

_p = ctypes.c_void_p
_i = ctypes.c_int
_i64 = ctypes.c_int64
_u64 = ctypes.c_uint64
_f = ctypes.c_float
_d = ctypes.c_double

# name -> argtypes (all return int status unless listed in _RESTYPES)
_SIGNATURES = {
    "ictc_version": [],
    "ictc_last_error": [],
    "ictc_tp_plan_create": [_i, _i, _i, _i, _i, _i, _p, _p, _i64, _i, _i, ctypes.POINTER(_p)],
    "ictc_tp_plan_destroy": [_p],
    "ictc_tp_plan_info": [_p, ctypes.POINTER(_i64), _i],
    "ictc_tp_plan_status": [_p, ctypes.POINTER(ctypes.c_int32), _i],
    "ictc_tp_forward": [_p, _p, _p, _p, _p, _p, _i64, _p],
    "ictc_tp_backward": [_p, _p, _p, _p, _p, _p, _p, _p, _p, _i64, _p],
    "ictc_tp_message_forward": [_p, _p, _p, _p, _p, _p, _p, _p, _p, _p, _i64, _p],
    "ictc_tp_message_backward": [_p, _p, _p, _p, _p, _p, _p, _p, _p, _p, _p, _p, _p, _i64, _p],
    "ictc_harmonics_table_size": [_i],
    "ictc_sc_table_rows": [_i, _i, _i],
    "ictc_sc_fold": [_p, _p, _p, _i, _i, _i, _i, _i64, _i64, _i, _p],
    "ictc_sc_directional": [_p, _p, _p, _p, _p, _i64, _p, _i, _i, _i, _i, _p],
    "ictc_sc_hvp": [_p, _p, _p, _p, _p, _i64, _p, _p, _i, _i, _i, _i, _p],
    "ictc_sc_table_grad": [_p, _p, _p, _p, _p, _i64, _p, _i, _i, _i, _i, _i, _p],
    "ictc_sc_tile_nodes": [],
    "ictc_sc_forward": [_p, _p, _p, _p, _i64, _p, _i, _i, _i, _i, _p],
    "ictc_sc_backward": [_p, _p, _p, _p, _i64, _p, _p, _i, _i, _i, _i, _p],
    "ictc_neighbor_workspace_bytes": [_i64, _p, ctypes.c_float],
    "ictc_neighbor_count": [_p, _i64, _p, ctypes.c_float, _p, _i64, _p, _p],
    "ictc_neighbor_fill": [_p, _i64, _p, ctypes.c_float, _p, _i64, _p, _p, _p, _p, _p],
    "ictc_neighbor_count_receivers": [_p, _i64, _i64, _p, ctypes.c_float, _p, _i64, _p, _p],
    "ictc_neighbor_fill_receivers": [_p, _i64, _i64, _p, ctypes.c_float, _p, _i64, _p, _p, _p, _p, _p],
    "ictc_neighbor_noalloc_scratch_bytes": [],
    "ictc_neighbor_list_noalloc": [_p, _i64, _p, ctypes.c_float, _p, _p, _p, _p, _i64, _p],
    "ictc_direction_harmonics": [_p, _p, _p, _p, _p, _p, _i64, _i, _i, _p],
    "ictc_edge_geometry": [_p, _i64, ctypes.c_float, _i, _i, _i, _p, _p, _p, _p],
    "ictc_edge_geometry_backward": [_p, _p, _p, _i64, ctypes.c_float, _i, _i, _i, _p, _p],
    "ictc_channel_mix_tile_nodes": [],
    "ictc_channel_mix": [_p, _i64, _i64, _p, _p, _p, _i64, _p, _i64, _i64, _i64, _i, _i, _i, ctypes.c_float, _i,
                         _p],
    "ictc_radial_image_bytes": [_i, _i, _i],
    "ictc_wait_selftest": [_p, _i64, _i, _p],
    "ictc_radial_pack": [_p, _p, _p, _p, _i, _i, _i, _p, _i64],
    "ictc_radial_forward": [_p, _p, _p, _i64, _i, _i, _i, _p, _p],
    "ictc_radial_backward": [_p, _p, _p, _p, _p, _i64, _i, _i, _i, _p, _p],
    "ictc_adamw_turn_values": [],
    "ictc_adamw_workspace_bytes": [],
    "ictc_adamw_grad_norm": [_p, _i, _p, _p, _i, _f, _i, _i, _p, _p],
    "ictc_adamw_step": [_p, _p, _i, _i, _p, _p, _i, _i, _p, _p, _p, _p, _p, _p, _p, _d, _d, _d, _d, _d, _d, _u64, _i, _p,
                        _p],
    "ictc_block_partial_floats": [_i, _i],
    "ictc_block_supported": [_i, _i],
    "ictc_block_wait_limit": [_u64],
    "ictc_block_status_word": [_p],
    "ictc_block_status": [_i, _p, _p],
    "ictc_block_forward": [_p] * 6 + [_i, _i64, _i, _i, _i, _f] + [_p] * 6,
    "ictc_block_backward": [_p] * 10 + [_i64, _i, _i, _i] + [_p] * 9,
    "ictc_block_second": [_p] * 13 + [_i64, _i, _i, _i] + [_p] * 11,
    "ictc_adamw_decode": [_p, _p, _p, _p, _i64, _p, _p, _p],
}
_RESTYPES = {"ictc_last_error": ctypes.c_char_p, "ictc_sc_table_rows": _i64,
             "ictc_neighbor_workspace_bytes": _i64, "ictc_neighbor_noalloc_scratch_bytes": _i64,
             "ictc_radial_image_bytes": _i64, "ictc_adamw_workspace_bytes": _i64,
             "ictc_block_partial_floats": _i64}

_lock = threading.Lock()
_lib = None


class NativeError(RuntimeError):
    pass


def library():
    """Load (once) and return the ctypes handle of libictc_cuda.so."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        if not os.path.exists(LIBRARY_PATH):
            raise NativeError(f"libictc_cuda.so not found at {LIBRARY_PATH}; run __graft_entry__.build()")
        lib = ctypes.CDLL(LIBRARY_PATH)
        for name, args in _SIGNATURES.items():
            fn = getattr(lib, name)
            fn.argtypes = args
            fn.restype = _RESTYPES.get(name, _i)
        version = lib.ictc_version()
        if version != ABI_VERSION:
            raise NativeError(f"libictc_cuda.so ABI {version} != expected {ABI_VERSION}; rebuild it")
        _lib = lib
        return lib


def exported_symbols():
    return tuple(_SIGNATURES)


def check(status, what):
    if status != 0:
        message = library().ictc_last_error().decode(errors="replace")
        raise NativeError(f"{what} failed (status {status}): {message}")


def ptr(tensor):
    """Device pointer of a contiguous tensor, or NULL for None."""
    if tensor is None:
        return None
    return ctypes.c_void_p(tensor.data_ptr())


def stream_of(tensor):
    return ctypes.c_void_p(torch.cuda.current_stream(tensor.device).cuda_stream)


def host_tensors():
    """The extension module that reads many tensors' addresses at once (csrc/host_tensors.cpp)."""
    try:
        from . import _host_tensors
    except ImportError as error:
        raise NativeError(f"_host_tensors is missing or was built for another torch ({error}); "
                          "run __graft_entry__.build()") from error
    if getattr(_host_tensors, "torch_version", None) != str(torch.__version__):      # it reads torch's own structures
        raise NativeError(f"_host_tensors was built for another torch than {torch.__version__}; "
                          "run __graft_entry__.build()")
    return _host_tensors


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


_Tensor = torch.Tensor


def _no_address(name):
    # a host tensor in the place of a number (a size under torch.jit.trace) would pass its address as that number
    raise TypeError(f"{name} takes addresses of CUDA tensors only")


def launch(device, name, *args):
    """``call`` with ``device`` current and its current stream as the last argument; CUDA tensors may be
    given for their addresses (None: NULL)."""
    args = [(a.data_ptr() if a.is_cuda else _no_address(name)) if isinstance(a, _Tensor) else a for a in args]
    if torch.cuda.current_device() != device.index:
        with torch.cuda.device(device):
            return launch(device, name, *args)
    stream = torch.cuda.current_stream(device).cuda_stream if _raw_stream is None else _raw_stream(device.index)
    status = getattr(_lib or library(), name)(*args, stream)
    if status != 0:
        check(status, name)


def call(name, *args):
    check(getattr(library(), name)(*args), name)
