"""ctypes binding of liblbq.so (C ABI declared in include/lbq.h).

The library is loaded on first use; if it is missing or fails to load, every call raises — there is
no fallback implementation.
"""
import ctypes
import os
import threading

import torch

_PKG = os.path.dirname(os.path.abspath(__file__))
# LBQ_DEBUG_LIB=1: the debug build (device-side index checks recording 0x3xx status codes)
LIB_PATH = os.path.join(_PKG, "liblbq_debug.so" if os.environ.get("LBQ_DEBUG_LIB") == "1" else "liblbq.so")

_i32, _i64, _f32, _vp, _sz = ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_void_p, ctypes.c_size_t
_u64 = ctypes.c_uint64

# name -> (restype, argtypes)
SIGNATURES = {
    "lbq_abi_version": (_i32, []),
    "lbq_last_error": (ctypes.c_char_p, []),
    "lbq_device_status": (_i32, [_i32, ctypes.POINTER(_i32)]),
    "lbq_kv_block_stats": (_i32, [_vp, _i64, _i64, _i64, _vp, _i64, _i64, _i64, _i32, _i32, _i64, _i32, _i32,
                                  _i64, _vp, _vp, _i64, _i64, _i64, _vp]),
    "lbq_kv_window_sums": (_i32, [_vp, _vp, _i32, _i32, _i32, _i32, _i64, _vp, _vp, _vp]),
    "lbq_quant_q": (_i32, [_vp, _i64, _i64, _i64, _i32, _i32, _i32, _vp, _vp, _vp]),
    "lbq_rope_quant_q": (_i32, [_vp, _i64, _i64, _i64, _vp, _vp, _i64, _i64, _i32, _i32, _i32, _vp, _vp, _vp]),
    "lbq_cache_write": (_i32, [_vp, _i64, _i64, _i64, _vp, _i64, _i64, _i64, _vp, _vp, _i64, _i64,
                               _vp, _i64, _i64, _i64, _vp, _i64, _i64, _i64, _i32, _i32, _i64, _i64, _i64, _i64,
                               _vp, _vp, _i64, _i64, _i64, _vp]),
    "lbq_quant_kv": (_i32, [_vp, _i64, _i64, _i64, _vp, _i64, _i64, _i64, _i32, _i32, _i64, _i32, _i32, _i32, _i32,
                            _i64, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i32, _vp]),
    "lbq_quant_qkv_workspace": (_sz, [_i32, _i32, _i64]),
    "lbq_quant_qkv": (_i32, [_vp, _i64, _i64, _i64, _i32, _vp, _i64, _i64, _i64, _vp, _i64, _i64, _i64, _i64,
                             _i32, _i32, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _sz, _i32, _vp]),
    "lbq_quant_qkv_static": (_i32, [_vp, _i64, _i64, _i64, _i32, _vp, _i64, _i64, _i64, _vp, _i64, _i64, _i64, _i64,
                                    _i32, _i32, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i32, _vp]),
    "lbq_requant_cache": (_i32, [_vp, _i64, _i64, _i64, _vp, _i64, _i64, _i64, _i32, _i32, _i64, _i64, _vp, _vp,
                                 _vp, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _vp]),
    "lbq_attn_fwd": (_i32, [_vp, _vp, _i32, _vp, _vp, _vp, _vp, _i64, _i32, _i32, _i32, _i32, _f32, _i32, _vp, _i64,
                            _i64, _i64, _i32, _vp, _vp, ctypes.POINTER(_i32), _i32, _vp]),
    "lbq_fp8_quant_rows": (_i32, [_vp, _i64, _i32, _i32, _i32, _vp, _i64, _vp, _vp]),
    "lbq_fp8_gemm": (_i32, [_vp, _i64, _vp, _vp, _i64, _vp, _vp, _i32, _i32, _i32, _vp, _i64, _i32, _vp]),
    "lbq_splitkv_combine": (_i32, [_vp, _vp, _i32, _vp, _i32, _i32, _i32, _vp, _i64, _i64, _i64, _i32, _vp]),
    "lbq_peer_export": (_i32, [_vp, _vp, ctypes.POINTER(ctypes.c_uint64)]),
    "lbq_peer_open": (_i32, [_vp, ctypes.POINTER(_vp)]),
    "lbq_peer_close": (_i32, [_vp]),
    "lbq_exchange_bytes": (_i64, [_i32, _i32, _i32]),
    "lbq_share_totals_push": (_i32, [_vp, _vp, _i64, _i32, _i32, _i32, _i32, _vp, _i32, _i32, _i64, _vp]),
    "lbq_chunk_totals": (_i32, [_vp, _i32, _i32, _i64, _i32, _i32, _vp, _vp, _vp, _vp, _u64, _vp]),
    "lbq_share_push": (_i32, [_vp, _i64, _i64, _i64, _vp, _i64, _i64, _i64, _i32, _i32, _i32, _i32, _vp, _i32, _i32,
                              _i64, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _i32, _vp]),
    "lbq_share_quant_push": (_i32, [_vp, _i64, _i64, _i64, _vp, _i64, _i64, _i64, _i32, _i32, _i32, _i32, _i32,
                                    _i32, _i32, _i32, _i64, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i32, _vp, _i32,
                                    _i32, _i64, _i32, _vp]),
    "lbq_peer_wait": (_i32, [_vp, _i32, _i32, _i64, _i32, _u64, _vp]),
    "lbq_quant_kv_tiles": (_i32, [_vp, _i64, _i64, _i64, _vp, _i64, _i64, _i64, _i32, _i32, _i64, _i32, _i32, _i32,
                                  _i32, _i64, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i32, _i32, _i32, _vp]),
    "lbq_attn_fwd_keys": (_i32, [_vp, _vp, _i32, _i32, _vp, _vp, _vp, _i32, _i32, _i32, _i32, _f32, _vp, _vp, _vp,
                                 _vp, _i32, _i32, _i64, _i32, _i64, _i64, _vp]),
    "lbq_keys_combine": (_i32, [_vp, _vp, _i32, _i32, _i32, _vp, _i32, _i32, _vp, _i64, _i64, _i64, _vp]),
    "lbq_rope": (_i32, [_vp, _i64, _i64, _i64, _vp, _i64, _i64, _i64, _i32, _vp, _i64, _i64, _i64, _vp, _i64, _i64,
                        _i64, _i32, _i32, _i32, _i32, _vp, _vp, _i64, _i64, _i32, _i32, _vp, _i32, _i64, _i64, _i64,
                        _i32, _i32, _vp]),
    "lbq_page_write": (_i32, [_vp, _i64, _i64, _i64, _vp, _i64, _i64, _i64, _vp, _vp, _vp, _vp, _i64, _i32, _i32, _vp,
                              _i64, _i32, _vp, _i64, _vp, _i32, _i32, _vp, _vp, _i64, _i64, _i32, _i32, _vp, _i32,
                              _i64, _i64, _i32, _vp]),
    "lbq_page_read": (_i32, [_vp, _vp, _vp, _vp, _i64, _i32, _i32, _vp, _i64, _i32, _vp, _i64, _vp, _i32, _i32, _vp,
                             _i64, _i64, _i64, _vp, _i64, _i64, _i64, _i32, _vp]),
    "lbq_page_copy": (_i32, [_vp, _vp, _vp, _vp, _i64, _i32, _i32, _i64, _i64, _vp, _vp, _i32, _vp]),
    "lbq_paged_attn_splits": (_i32, [_i32, _i32, _i32, _i32, _i64, _i32]),
    "lbq_paged_attn_workspace": (_sz, [_i32, _i32, _i32, _i32, _i32]),
    "lbq_paged_attn": (_i32, [_vp, _i64, _i64, _i64, _vp, _vp, _vp, _vp, _i64, _i32, _i32, _vp, _i64, _i32, _vp, _i64,
                              _vp, _i32, _i32, _i32, _i32, _f32, _vp, _i64, _i64, _i64, _vp, _i32, _vp, _sz, _i32,
                              _vp]),
    "lbq_q_push": (_i32, [_vp, _vp, _i32, _i32, _i32, _i32, _i32, _i64, _i64, _vp, _i32, _i32, _i64, _i32, _vp]),
}

_lock = threading.Lock()
_lib = None
_entry = {}
_fast = None


class LbqError(RuntimeError):
    """An lbq_* entry point returned a non-zero status."""


def load():
    """Load liblbq.so once and declare every exported signature."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not os.path.exists(LIB_PATH):
                raise ImportError(f"{LIB_PATH} is missing: build it with `python -m lingbot_b200.build` "
                                  "(add --debug for the debug library; nvcc, sm_100a); there is no fallback "
                                  "implementation")
            lib = ctypes.CDLL(LIB_PATH)
            for name, (res, args) in SIGNATURES.items():
                fn = getattr(lib, name)
                fn.restype = res
                fn.argtypes = args
            _lib = lib
    return _lib


def fast():
    """The calls straight from torch tensors (_torchcall), bound to the loaded library's entries. They return None where
    a call is not of the usual form, else their result or an entry's status code."""
    global _fast
    if _fast is None:
        lib = load()
        try:
            from . import _torchcall
        except ImportError as e:
            raise ImportError("lingbot_b200/_torchcall.so is missing or does not load: build it with `python -m "
                              f"lingbot_b200.build` ({e})") from e
        _torchcall.init(*(ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in
                          ("lbq_rope", "lbq_page_write", "lbq_page_read", "lbq_paged_attn", "lbq_paged_attn_splits",
                           "lbq_paged_attn_workspace", "lbq_page_copy")))
        _fast = _torchcall
    return _fast


def check(name, rc):
    """Raise LbqError for a status code other than 0."""
    if rc != 0:
        raise LbqError(f"{name} failed ({rc}): {_lib.lbq_last_error().decode(errors='replace')}")


def call(name, *args):
    """Call an lbq_* entry point that returns a status code; raise LbqError on failure."""
    lib = load()
    rc = getattr(lib, name)(*args)
    if rc != 0:
        msg = lib.lbq_last_error().decode(errors="replace")
        raise LbqError(f"{name} failed ({rc}): {msg}")
    return rc


def call_on(device, name, *args):
    """`call` with the current stream of `device` as the last argument, made with that device current. (The raw stream
    handle and one attribute lookup: of a small launch's 15 us on the host, torch.cuda.current_stream() was 3.)"""
    index = device.index
    fn = _entry.get(name)
    if fn is None:
        fn = _entry[name] = getattr(load(), name)
    if index == torch.cuda.current_device():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    check(name, rc)


def device_status(clear=True):
    """Read (and by default clear) the current device's status word: 0 unless a kernel's bounded
    wait gave up."""
    out = _i32(0)
    call("lbq_device_status", int(bool(clear)), ctypes.byref(out))
    return out.value


def check_sizes(name, t):
    """The entries take 32-bit sizes, which ctypes would cut (an expanded dimension needs no memory to be longer)."""
    if any(n > 1 << 28 for n in t.shape):
        raise ValueError(f"{name}: {tuple(t.shape)} has a dimension of more than 2^28")


def no_gradient(what, *tensors):
    """Refuses tensors through which a gradient is wanted, backward or forward: the kernels record none."""
    for t in tensors:
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{what} records no gradient: call it under torch.no_grad()")
        if torch.autograd.forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{what} records no gradient, and its result would carry no tangent: pass the primal")


def _reaches(dims, at, width, zero):
    """Whether some sum of c * stride over dims (stride, least c, most c) lies nearer than `width` to `at`; with zero False,
    one whose c are not all 0. Strides far apart, as a tensor's are, leave one or two c to try at each; a case of very many
    counts as reached."""
    dims = sorted(dims, reverse=True)
    below = [(0, 0)]                                             # least and most of the smaller strides' sums
    for st, lo, hi in reversed(dims):
        below.append((below[-1][0] + lo * st, below[-1][1] + hi * st))
    below.reverse()
    todo = [(0, at, zero)]
    for _ in range(10000):
        if not todo:
            return False
        i, d, ok = todo.pop()
        if i == len(dims):
            if ok and -width < d < width:
                return True
            continue
        st, lo, hi = dims[i]
        least, most = below[i + 1]
        lo = max(lo, -((most + width - 1 - d) // st))
        hi = min(hi, (d + width - 1 - least) // st)
        todo += [(i + 1, d - c * st, ok or c != 0) for c in range(lo, min(hi, lo + 10000) + 1)]
    return True


def self_overlap(t):
    """Whether elements of a tensor with unit last stride share memory with one another."""
    if t.is_contiguous():
        return False
    if any(n > 1 and st == 0 for n, st in zip(t.shape, t.stride())):
        return True
    dims = [(st, 1 - n, n - 1) for n, st in zip(t.shape[:-1], t.stride()[:-1]) if n > 1]
    return t.numel() > 0 and _reaches(dims, 0, t.shape[-1], False)


def share_memory(a, b):
    """Whether two tensors of one type and one last dimension, of unit stride, have elements in common memory; not where
    their addresses alternate, as those of views of one buffer do."""
    if not a.numel() or not b.numel():
        return False
    size, width = a.element_size(), a.shape[-1] * a.element_size()
    at, dims = b.data_ptr() - a.data_ptr(), {}
    for t, sign in ((a, 1), (b, -1)):
        for n, st in zip(t.shape[:-1], t.stride()[:-1]):
            if n > 1 and st > 0:
                lo, hi = dims.get(st * size, (0, 0))
                dims[st * size] = (lo, hi + n - 1) if sign == 1 else (lo - n + 1, hi)
    return _reaches([(st, lo, hi) for st, (lo, hi) in dims.items()], at, width, True)
