"""KernelIntrinsics for B200: the host-side mirror of KernelIntrinsics.jl's API over libki_b200.so.

Names and argument meanings follow the reference (epilliat/KernelIntrinsics.jl v0.1.6):

* type lattices ``Workgroup/Device/System``, ``Weak/Volatile/Relaxed/Acquire/Release/AcqRel/SeqCst``
  (src/scopes_orderings.jl:13-120), ``Up/Down/Xor/Idx`` and ``All/AnyLane/Uni/Ballot``
  (src/warp.jl:16-106);
* ``shfl``, ``warpreduce``, ``warpfold``, ``vote`` run the warp intrinsics over every warp of a CUDA
  tensor (lanes are consecutive elements); ``Idx`` lanes and ``laneid`` are 1-based as in Julia;
* ``vload`` / ``vstore`` / ``vload_multi`` / ``vstore_multi`` take 1-based indices;
* ``access`` / ``fence`` validate scope/ordering like ``@access`` / ``@fence`` and raise
  ``KIArgumentError`` (a ``ValueError``) where the reference raises ``ArgumentError``;
* device-wide operations built from them: ``vcopy`` (copyto!), ``warpfold_reduce`` (sum),
  ``warpreduce_scan`` (cumsum), ``vote_compact`` (filter/findall), ``fp8_gemm``;
* the operators of a state-space layer served in 8 bits (no counterpart in the reference): ``quantize_rows``,
  ``int8_gemm``, ``causal_conv`` / ``causal_conv_step``, ``selective_scan`` / ``selective_scan_step``.

Every operation runs a hand-written sm_100a kernel from libki_b200.so; tensors are torch CUDA tensors
(torch provides device memory and streams only).  There is no CPU path.
"""
from __future__ import annotations

import ctypes
import threading
from typing import Optional

from . import _abi
from ._abi import KIArgumentError, KIError, KITimeoutError

__all__ = [
    "Workgroup", "Device", "System", "Weak", "Volatile", "Relaxed", "Acquire", "Release", "AcqRel", "SeqCst",
    "Up", "Down", "Xor", "Idx", "All", "AnyLane", "Uni", "Ballot", "KIError", "KIArgumentError",
    "KITimeoutError", "Context", "context", "warpsize", "get_warpsize", "devices", "shfl", "warpreduce",
    "warpfold", "vote", "vload", "vstore", "vload_multi", "vstore_multi", "generate_partN", "access",
    "message_pass", "vcopy", "vcopy_host", "reduce", "reduce_rows", "scan", "compact", "warpfold_reduce", "reduce_sum_i64", "warpreduce_scan", "warpreduce_scan_host", "vote_compact",
    "fp8_gemm", "quantize_rows", "int8_gemm", "causal_conv", "causal_conv_step", "selective_scan",
    "selective_scan_step", "fill_uniform", "fill_int_range", "fill_bytes", "fill_normal", "fill_e4m3_uniform",
]


# ---------------------------------------------------------------------------------------------
# type lattices (singletons, used like the reference's types)
# ---------------------------------------------------------------------------------------------
class Scope:
    key = "default"


class Workgroup(Scope):
    key = "workgroup"


class Device(Scope):
    key = "device"


class System(Scope):
    key = "system"


class Ordering:
    key = "default"


class Weak(Ordering):
    key = "weak"


class Volatile(Ordering):
    key = "volatile"


class Relaxed(Ordering):
    key = "relaxed"


class Acquire(Ordering):
    key = "acquire"


class Release(Ordering):
    key = "release"


class AcqRel(Ordering):
    key = "acqrel"


class SeqCst(Ordering):
    key = "seqcst"


class Direction:
    key = ""


class Up(Direction):
    key = "up"


class Down(Direction):
    key = "down"


class Xor(Direction):
    key = "xor"


class Idx(Direction):
    key = "idx"


class Mode:
    key = ""


class All(Mode):
    key = "all"


class AnyLane(Mode):
    key = "any"


class Uni(Mode):
    key = "uni"


class Ballot(Mode):
    key = "ballot"


# ---------------------------------------------------------------------------------------------
# context
# ---------------------------------------------------------------------------------------------
_torch_module = None


def _torch():
    global _torch_module
    if _torch_module is None:
        import torch

        _torch_module = torch
    return _torch_module


class Context:
    """One libki_b200 context (scratch + device status word) on one device (0-based ``device``)."""

    def __init__(self, device: int = 0):
        self.lib = _abi.load()
        h = ctypes.c_void_p()
        st = self.lib.ki_ctx_create(int(device), ctypes.byref(h))
        if st != _abi.KI_OK:
            raise _abi.status_error(st, f"ki_ctx_create(device={device}): "
                                        f"{self.lib.ki_status_string(st).decode()}")
        self.handle = h
        self.device = int(device)

    def close(self) -> None:
        if getattr(self, "handle", None):
            self.lib.ki_ctx_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _raise(self, st: int, what: str) -> None:
        msg = self.lib.ki_last_error_string(self.handle).decode(errors="replace")
        raise _abi.status_error(st, f"{what}: {msg or self.lib.ki_status_string(st).decode()}")

    def call(self, name: str, *args) -> None:
        st = getattr(self.lib, name)(self.handle, *args)
        if st != _abi.KI_OK:
            self._raise(st, name)

    def check(self, stream=None) -> None:
        """Synchronise ``stream`` and raise if a bounded device-side wait of this context ran out, or a kernel met an offset
        or a slot number in device memory that was out of range."""
        st = self.lib.ki_ctx_check(self.handle, _stream_ptr(stream, self.device))
        if st != _abi.KI_OK:
            self._raise(st, "ki_ctx_check")

    def set_wait_timeout(self, seconds: float) -> None:
        self.call("ki_ctx_set_wait_timeout_ns", ctypes.c_uint64(int(seconds * 1e9)))


_ctx_lock = threading.Lock()
_ctx_by_key: dict = {}


def context(device: Optional[int] = None) -> Context:
    """The calling thread's context on ``device`` (default: torch's current device)."""
    if device is None:
        device = _torch().cuda.current_device()
    key = (threading.get_ident(), int(device))
    c = _ctx_by_key.get(key)  # only this thread makes the entry
    if c is None:
        with _ctx_lock:
            c = _ctx_by_key[key] = Context(int(device))
    return c


def _stream_ptr(stream, device: int):
    torch = _torch()
    if stream is None:
        stream = torch.cuda.current_stream(device)
    return ctypes.c_void_p(stream.cuda_stream)


def _dev(t) -> int:
    if not t.is_cuda:
        raise KIArgumentError(_abi.KI_ERR_ARG, "tensor must be on a CUDA device (there is no CPU path)")
    return t.device.index


def _ptr(t) -> ctypes.c_void_p:
    return ctypes.c_void_p(t.data_ptr())


def _dtype_code(t) -> int:
    name = str(t.dtype).replace("torch.", "")
    if name not in _abi.DTYPE:
        raise KIArgumentError(_abi.KI_ERR_ARG, f"unsupported dtype {t.dtype}")
    return _abi.DTYPE[name]


# ---------------------------------------------------------------------------------------------
# device queries (src/device.jl, ext/CUDA/device.jl): 1-based device ids as in the reference
# ---------------------------------------------------------------------------------------------
def devices() -> list:
    lib = _abi.load()
    n = ctypes.c_int(0)
    lib.ki_device_count(ctypes.byref(n))
    return list(range(1, n.value + 1))


def get_warpsize(device: int = 1) -> int:
    lib = _abi.load()
    ws = ctypes.c_int(0)
    st = lib.ki_device_info(int(device) - 1, None, ctypes.byref(ws), None, None)
    if st != _abi.KI_OK:
        raise _abi.status_error(st, "ki_device_info")
    return ws.value


warpsize = get_warpsize


# ---------------------------------------------------------------------------------------------
# warp intrinsics over whole warps
# ---------------------------------------------------------------------------------------------
def shfl(direction, x, src: int, out=None):
    """@shfl(direction, val, src) on every warp of ``x`` (x.numel() % 32 == 0).

    ``src``: offset for Up/Down, lane mask for Xor, 1-BASED source lane for Idx.  Works on any
    element type, including structured numpy-style records viewed as bytes (element size 1..64).
    """
    torch = _torch()
    d = _dev(x)
    out = torch.empty_like(x) if out is None else out
    arg = int(src)
    if direction is Idx:
        if not 1 <= arg <= 32:
            raise KIArgumentError(_abi.KI_ERR_ARG, "Idx lane must be in 1..32")
        arg -= 1
    esz = x.element_size()
    n = x.numel()
    if x.dim() >= 2 and x.dtype == torch.uint8:  # rows of raw bytes = one element per row
        esz = x.shape[-1]
        n = x.numel() // esz
    context(d).call("ki_warp_shfl", _abi.DIR[direction.key], _ptr(x), _ptr(out), esz, n, arg,
                    _stream_ptr(None, d))
    return out


def warpreduce(x, op: str = "+", out=None):
    """@warpreduce(val, op): inclusive scan inside each warp (src/warp.jl:226-237)."""
    torch = _torch()
    d = _dev(x)
    out = torch.empty_like(x) if out is None else out
    context(d).call("ki_warp_reduce", _abi.OP[op], _dtype_code(x), _ptr(x), _ptr(out), x.numel(),
                    _stream_ptr(None, d))
    return out


def warpfold(x, op: str = "+", form: str = "xor", out=None):
    """@warpfold(val, op).  form="down" is the reference's exact Down fold (lane 1 holds the total);
    form="xor" gives every lane the total."""
    torch = _torch()
    d = _dev(x)
    out = torch.empty_like(x) if out is None else out
    f = {"xor": 0, "down": 1}[form]
    context(d).call("ki_warp_fold", _abi.OP[op], _dtype_code(x), f, _ptr(x), _ptr(out), x.numel(),
                    _stream_ptr(None, d))
    return out


def vote(mode, pred, out=None):
    """@vote(mode, pred) on every warp; ``pred`` is a bool/uint8 tensor.  Returns uint32 per lane
    (0/1 for All/AnyLane/Uni; the UInt32 ballot mask for Ballot, bit i = 0-based lane i)."""
    torch = _torch()
    d = _dev(pred)
    p = pred.to(torch.uint8) if pred.dtype != torch.uint8 else pred
    out = torch.empty(p.shape, dtype=torch.uint32, device=p.device) if out is None else out
    context(d).call("ki_warp_vote", _abi.MODE[mode.key], _ptr(p), _ptr(out), p.numel(), _stream_ptr(None, d))
    return out


# ---------------------------------------------------------------------------------------------
# vector access (1-based indices, as the reference)
# ---------------------------------------------------------------------------------------------
def vload(a, idx: int, nitem: int, rebase: bool = True, elem_bytes: Optional[int] = None):
    """vload(A, idx, Val(N), Val(Rebase)) -> tensor of N elements (src/vectorization.jl:135-199).

    rebase=True: ``idx`` is a 1-based block index (elements (idx-1)*N+1 .. idx*N);
    rebase=False: ``idx`` is the 1-based first element.  ``elem_bytes`` views a uint8 tensor as
    records of that size (non power-of-two sizes take the scalar path)."""
    torch = _torch()
    d = _dev(a)
    esz = elem_bytes or a.element_size()
    out = torch.empty(nitem * esz, dtype=torch.uint8, device=a.device)
    context(d).call("ki_vload", _ptr(a), esz, int(idx) - 1, int(nitem), int(bool(rebase)), _ptr(out),
                    _stream_ptr(None, d))
    if elem_bytes is None:
        return out.view(a.dtype)
    return out.view(nitem, esz)


def vstore(a, idx: int, values, rebase: bool = True, elem_bytes: Optional[int] = None) -> None:
    """vstore!(A, idx, values, Val(Rebase)) (src/vectorization.jl:218-300)."""
    d = _dev(a)
    esz = elem_bytes or a.element_size()
    nitem = values.numel() * values.element_size() // esz
    context(d).call("ki_vstore", _ptr(a), esz, int(idx) - 1, int(nitem), int(bool(rebase)),
                    _ptr(values.contiguous()), _stream_ptr(None, d))


def vload_multi(a, i: int, nitem: int):
    """vload_multi(a, i, Val(N)): N elements from 1-based element i with the generate_partN pieces."""
    return vload(a, i, nitem, rebase=False)


def vstore_multi(a, i: int, values) -> None:
    """vstore_multi!(a, i, values)."""
    vstore(a, i, values, rebase=False)


def generate_partN(N: int) -> tuple:
    """The reference's piece patterns (src/vectorization.jl:306-338), index = residue (0-based)."""
    if N <= 0 or N & (N - 1):
        raise KIArgumentError(_abi.KI_ERR_ARG, "N must be a positive power of 2")
    out = [(N,)]
    for r in range(1, N):
        pat, remaining, pos = [], N, r
        while remaining > 0:
            m = N // 2
            while m > 0 and not (pos % m == 0 and m <= remaining):
                m //= 2
            m = max(m, 1)
            pat.append(m)
            remaining -= m
            pos = (pos + m) % N
        out.append(tuple(pat))
    return tuple(out)


# ---------------------------------------------------------------------------------------------
# @access / @fence
# ---------------------------------------------------------------------------------------------
def _split_scope_order(args):
    """scope_ordering (src/macros.jl:130-196): 0-2 arguments, one Scope and/or one Ordering, any order."""
    if len(args) > 2:
        raise KIArgumentError(_abi.KI_ERR_ARG, f"Too many arguments: expected 0-2, got {len(args)}.")
    scope = order = None
    for a in args:
        if isinstance(a, type) and issubclass(a, Scope) and a is not Scope and scope is None:
            scope = a
        elif isinstance(a, type) and issubclass(a, Ordering) and a is not Ordering and order is None:
            order = a
        else:
            raise KIArgumentError(_abi.KI_ERR_ARG, "Arguments must be one Scope and one Ordering (in any order).")
    return scope, order


def access(slot, value, *args, fence_args=()):
    """@access store of ``value`` into ``slot[0]``, @fence, then @access load back; returns the value.

    ``args`` are the @access scope/ordering for both accesses, e.g. ``access(t, 5, Device, Relaxed)``;
    the store ordering defaults to Release and the load to Acquire.  ``fence_args`` likewise for
    @fence (default Device, AcqRel)."""
    torch = _torch()
    d = _dev(slot)
    scope, order = _split_scope_order(args)
    fscope, forder = _split_scope_order(fence_args)
    so = lo = _abi.ORDER[order.key] if order else 0
    if order in (Acquire, Release):  # one explicit ordering applies to the access it names
        so = _abi.ORDER["release"] if order is Release else 0
        lo = _abi.ORDER["acquire"] if order is Acquire else 0
    val = torch.tensor([value], dtype=slot.dtype, device=slot.device)
    rb = torch.empty(1, dtype=slot.dtype, device=slot.device)
    context(d).call("ki_access_roundtrip", _dtype_code(slot), _abi.SCOPE[scope.key] if scope else 0, so, lo,
                    _abi.SCOPE[fscope.key] if fscope else 0, _abi.ORDER[forder.key] if forder else 0,
                    _ptr(slot), _ptr(val), _ptr(rb), _stream_ptr(None, d))
    return rb


def message_pass(data, flag, seen, payload: int, produce: bool = True, timeout_s: float = 1.0):
    """Release/acquire message passing across blocks (the reference's @access producer/consumer
    example, src/macros.jl:84-97) with bounded waits.  ``seen[b]`` gets the payload, or -1 if the
    wait of consumer block b ran out (then ``Context.check`` raises KITimeoutError)."""
    d = _dev(data)
    context(d).call("ki_flag_message_pass", _ptr(data), _ptr(flag), _ptr(seen), seen.numel(), int(payload),
                    int(bool(produce)), ctypes.c_uint64(int(timeout_s * 1e9)), _stream_ptr(None, d))


# ---------------------------------------------------------------------------------------------
# device-wide operations
# ---------------------------------------------------------------------------------------------
def vcopy(dst, src, nbytes: Optional[int] = None, dst_offset: int = 0, src_offset: int = 0, stream=None):
    """copyto!: copy ``nbytes`` bytes from ``src`` (+src_offset bytes) to ``dst`` (+dst_offset bytes)
    with 128-bit vector accesses at any alignment."""
    d = _dev(dst)
    if nbytes is None:
        nbytes = min(src.numel() * src.element_size() - src_offset, dst.numel() * dst.element_size() - dst_offset)
    if src_offset + nbytes > src.numel() * src.element_size() or dst_offset + nbytes > dst.numel() * dst.element_size():
        raise KIArgumentError(_abi.KI_ERR_ARG, "vcopy: range outside the tensors")
    context(d).call("ki_vcopy", ctypes.c_void_p(dst.data_ptr() + dst_offset),
                    ctypes.c_void_p(src.data_ptr() + src_offset), int(nbytes), _stream_ptr(stream, d))
    return dst


def vcopy_2d(dst, dpitch: int, src, spitch: int, width: int, height: int, dst_offset: int = 0, src_offset: int = 0,
             stream=None):
    """copyto! of ``height`` rows of ``width`` bytes: row r from byte src_offset + r*spitch of ``src`` to
    byte dst_offset + r*dpitch of ``dst`` (any alignment, any pitch >= width)."""
    d = _dev(dst)
    if width > 0 and height > 0:
        last_d = dst_offset + (height - 1) * dpitch + width
        last_s = src_offset + (height - 1) * spitch + width
        if min(dst_offset, src_offset) < 0 or last_d > dst.numel() * dst.element_size() or \
                last_s > src.numel() * src.element_size():
            raise KIArgumentError(_abi.KI_ERR_ARG, "vcopy_2d: range outside the tensors")
    context(d).call("ki_vcopy_2d", ctypes.c_void_p(dst.data_ptr() + dst_offset), int(dpitch),
                    ctypes.c_void_p(src.data_ptr() + src_offset), int(spitch), int(width), int(height),
                    _stream_ptr(stream, d))
    return dst


def vcopy_strided(dst, dst_stride: int, src, src_stride: int, count: int, dst_start: int = 0, src_start: int = 0,
                  elem_bytes: Optional[int] = None, stream=None):
    """dst[dst_start + i*dst_stride] = src[src_start + i*src_stride] for i < count, in elements of the
    tensors' (equal) element size, or of ``elem_bytes`` bytes (a struct type held in byte tensors);
    strides of either sign, as Julia's strided and reversed views."""
    d = _dev(dst)
    if elem_bytes is None:
        es = dst.element_size()
        if src.element_size() != es:
            raise KIArgumentError(_abi.KI_ERR_ARG, "vcopy_strided: element sizes differ")
    else:
        es = int(elem_bytes)
        if es <= 0:
            raise KIArgumentError(_abi.KI_ERR_ARG, "vcopy_strided: element size must be positive")
    if count > 0:
        for t, st, n0 in ((dst, dst_stride, dst_start), (src, src_stride, src_start)):
            last = n0 + (count - 1) * st
            if min(n0, last) < 0 or (max(n0, last) + 1) * es > t.numel() * t.element_size():
                raise KIArgumentError(_abi.KI_ERR_ARG, "vcopy_strided: range outside the tensors")
    context(d).call("ki_vcopy_strided", ctypes.c_void_p(dst.data_ptr() + dst_start * es), int(dst_stride),
                    ctypes.c_void_p(src.data_ptr() + src_start * es), int(src_stride), es, int(count),
                    _stream_ptr(stream, d))
    return dst


def copyto(dst, src, stream=None):
    """copyto!(dst, src) for device views of the same shape and element size: contiguous ranges go
    through vcopy, 1-D strided views through vcopy_strided, 2-D views with contiguous rows through
    vcopy_2d (one row per leading index)."""
    if tuple(dst.shape) != tuple(src.shape) or dst.element_size() != src.element_size():
        raise KIArgumentError(_abi.KI_ERR_ARG, "copyto: shapes or element sizes differ")
    es = dst.element_size()
    if dst.numel() == 0:
        return dst
    if dst.is_contiguous() and src.is_contiguous():
        return _copy_raw("ki_vcopy", dst, src, dst.numel() * es, stream)
    if dst.dim() == 1:
        return _copy_raw("ki_vcopy_strided", dst, src, dst.numel(), stream, dst.stride(0), src.stride(0), es)
    if dst.dim() == 2 and dst.stride(1) == 1 and src.stride(1) == 1:
        return _copy_raw("ki_vcopy_2d", dst, src, dst.shape[1] * es, stream, dst.stride(0) * es, src.stride(0) * es,
                         dst.shape[0])
    raise KIArgumentError(_abi.KI_ERR_ARG, "copyto: 1-D views, or 2-D views with contiguous rows")


def _copy_raw(fn, dst, src, n, stream, *extra):
    d = _dev(dst)
    pd, ps = ctypes.c_void_p(dst.data_ptr()), ctypes.c_void_p(src.data_ptr())
    s = _stream_ptr(stream, d)
    if fn == "ki_vcopy":
        context(d).call(fn, pd, ps, int(n), s)
    elif fn == "ki_vcopy_strided":
        dstride, sstride, es = extra
        context(d).call(fn, pd, int(dstride), ps, int(sstride), int(es), int(n), s)
    else:
        dpitch, spitch, height = extra
        context(d).call(fn, pd, int(dpitch), ps, int(spitch), int(n), int(height), s)
    return dst


def vcopy_host(dst, src, nbytes: Optional[int] = None, dst_offset: int = 0, src_offset: int = 0, device: int = 0,
               stream=None):
    """copyto! between two host (CPU) tensors through device ``device``: chunks go to the device, are
    copied by the vectorised copy kernel and come back, both directions overlapped.  Pinned host
    tensors make the call asynchronous; it is complete when ``stream`` is."""
    if dst.is_cuda or src.is_cuda:
        raise KIArgumentError(_abi.KI_ERR_ARG, "vcopy_host: host tensors expected")
    if nbytes is None:
        nbytes = min(src.numel() * src.element_size() - src_offset, dst.numel() * dst.element_size() - dst_offset)
    if src_offset + nbytes > src.numel() * src.element_size() or dst_offset + nbytes > dst.numel() * dst.element_size():
        raise KIArgumentError(_abi.KI_ERR_ARG, "vcopy_host: range outside the tensors")
    context(device).call("ki_vcopy_host", ctypes.c_void_p(dst.data_ptr() + dst_offset),
                         ctypes.c_void_p(src.data_ptr() + src_offset), int(nbytes), _stream_ptr(stream, device))
    return dst


def warpfold_reduce(x, out_f64=None, out_f32=None, stream=None):
    """sum(x) for Float32 ``x`` (Float64 accumulation).  Returns the Float64 device scalar."""
    torch = _torch()
    d = _dev(x)
    if x.dtype != torch.float32:
        raise KIArgumentError(_abi.KI_ERR_ARG, "warpfold_reduce: Float32 input")
    if out_f64 is None:
        out_f64 = torch.empty((), dtype=torch.float64, device=x.device)
    context(d).call("ki_reduce_sum_f32", _ptr(x), x.numel(), _ptr(out_f32) if out_f32 is not None else None,
                    _ptr(out_f64), _stream_ptr(stream, d))
    return out_f64


def reduce_sum_i64(x, out=None, stream=None):
    """sum(x) for Int64 ``x`` with wrap-around.  Returns the Int64 device scalar."""
    torch = _torch()
    d = _dev(x)
    out = torch.empty((), dtype=torch.int64, device=x.device) if out is None else out
    context(d).call("ki_reduce_sum_i64", _ptr(x), x.numel(), _ptr(out), _stream_ptr(stream, d))
    return out


def warpreduce_scan(x, out=None, seed: int = 0, stream=None):
    """cumsum(x) for Int64 ``x`` (inclusive, single-pass decoupled lookback), plus ``seed``."""
    torch = _torch()
    d = _dev(x)
    if x.dtype != torch.int64:
        raise KIArgumentError(_abi.KI_ERR_ARG, "warpreduce_scan: Int64 input")
    out = torch.empty_like(x) if out is None else out
    context(d).call("ki_scan_inclusive_i64", _ptr(x), _ptr(out), x.numel(), ctypes.c_int64(int(seed)),
                    _stream_ptr(stream, d))
    return out


def warpreduce_scan_host(x, out=None, seed: int = 0, device: int = 0, stream=None):
    """cumsum of a HOST Int64 tensor through GPU ``device`` (chunks cross PCIe, are scanned there and come
    back, both directions overlapped).  Pinned tensors make it asynchronous; it is complete when
    ``stream`` (of ``device``) is."""
    torch = _torch()
    if x.is_cuda or x.dtype != torch.int64 or not x.is_contiguous():
        raise KIArgumentError(_abi.KI_ERR_ARG, "warpreduce_scan_host: contiguous Int64 host tensor")
    out = torch.empty_like(x) if out is None else out
    if out.is_cuda or out.dtype != torch.int64 or out.numel() != x.numel() or not out.is_contiguous():
        raise KIArgumentError(_abi.KI_ERR_ARG, "warpreduce_scan_host: output must match the input, on the host")
    context(device).call("ki_scan_inclusive_i64_host", _ptr(x), _ptr(out), x.numel(), ctypes.c_int64(int(seed)),
                         _stream_ptr(stream, device))
    return out


def _result_dtype(dtype, op: str):
    """Base's result type: sums and products (add_sum / mul_prod) widen integers narrower than 64
    bits to Int64 / UInt64; every other operator keeps the element type."""
    torch = _torch()
    if op in ("+", "add", "*", "mul"):
        if dtype in (torch.int8, torch.int16, torch.int32):
            return torch.int64
        if dtype in (torch.uint8, torch.uint16, torch.uint32):
            return torch.uint64
    return dtype


_GENERIC_OPS = {"+": 0, "add": 0, "max": 1, "min": 2, "|": 3, "or": 3, "&": 4, "and": 4, "xor": 5, "*": 6, "mul": 6}


def _np_dtype(t):
    import numpy as np

    name = str(t).replace("torch.", "")
    if name not in _abi.DTYPE:
        raise KIArgumentError(_abi.KI_ERR_ARG, f"unsupported dtype {t}")
    return np.dtype(name)


def reduce(x, op: str = "+", out=None, stream=None):
    """sum / prod / maximum / minimum / reduce(|, &, xor) of Int8 ... UInt64, Float32 or Float64 ``x``
    with Julia Base semantics (the device-wide @warpfold): sums and products of narrower integers
    widen to 64 bits, Float32 sums and products accumulate in Float64, maximum/minimum propagate
    NaN; the bitwise operators take integers.  Returns a device scalar."""
    torch = _torch()
    d = _dev(x)
    if op not in _GENERIC_OPS:
        raise KIArgumentError(_abi.KI_ERR_ARG, f"reduce: op must be one of {sorted(_GENERIC_OPS)}")
    x = x.contiguous()
    out = torch.empty((), dtype=_result_dtype(x.dtype, op), device=x.device) if out is None else out
    context(d).call("ki_reduce", _GENERIC_OPS[op], _dtype_code(x), _ptr(x), x.numel(), _ptr(out),
                    _stream_ptr(stream, d))
    return out


_MAPS = {None: 0, "identity": 0, "abs": 1, "abs2": 2}


def mapreduce(f, op: str, x, out=None, stream=None):
    """mapreduce(f, op, x) for f in abs, abs2 (computed in the element type, as Base does) and op in
    +, max, min: sum(abs2, x), maximum(abs, x).  Result types as ``reduce``."""
    torch = _torch()
    d = _dev(x)
    if f not in _MAPS:
        raise KIArgumentError(_abi.KI_ERR_ARG, "mapreduce: f must be 'abs', 'abs2' or None")
    if op not in _GENERIC_OPS:
        raise KIArgumentError(_abi.KI_ERR_ARG, f"mapreduce: op must be one of {sorted(_GENERIC_OPS)}")
    x = x.contiguous()
    out = torch.empty((), dtype=_result_dtype(x.dtype, op), device=x.device) if out is None else out
    context(d).call("ki_mapreduce", _MAPS[f], _GENERIC_OPS[op], _dtype_code(x), _ptr(x), x.numel(), _ptr(out),
                    _stream_ptr(stream, d))
    return out


def reduce_rows(x, op: str = "+", out=None, stream=None):
    """One reduction per row (the operators of ``reduce``) of a 2-D ``x`` whose rows are contiguous
    (``x.stride(1) == 1``; ``x.stride(0)`` is the leading dimension).  Result types as ``reduce``."""
    torch = _torch()
    d = _dev(x)
    if op not in _GENERIC_OPS:
        raise KIArgumentError(_abi.KI_ERR_ARG, f"reduce_rows: op must be one of {sorted(_GENERIC_OPS)}")
    if x.dim() != 2 or (x.shape[1] > 1 and x.stride(1) != 1):
        raise KIArgumentError(_abi.KI_ERR_ARG, "reduce_rows: 2-D input with contiguous rows")
    rows, cols = x.shape
    ld = x.stride(0) if rows > 1 else cols
    out = torch.empty(rows, dtype=_result_dtype(x.dtype, op), device=x.device) if out is None else out
    context(d).call("ki_reduce_rows", _GENERIC_OPS[op], _dtype_code(x), _ptr(x), rows, cols, max(ld, cols), _ptr(out),
                    _stream_ptr(stream, d))
    return out


def scan(x, op: str = "+", exclusive: bool = False, init=None, out=None, stream=None):
    """accumulate(op, x; init) / cumsum / cumprod for the operators and types of ``reduce`` (the
    device-wide @warpreduce).  The result has Base's type (widened for sums and products of narrower
    integers); ``exclusive`` shifts it by one element and starts at ``init`` (the identity when None)."""
    import numpy as np

    torch = _torch()
    d = _dev(x)
    if op not in _GENERIC_OPS:
        raise KIArgumentError(_abi.KI_ERR_ARG, f"scan: op must be one of {sorted(_GENERIC_OPS)}")
    rd = _result_dtype(x.dtype, op)
    out = torch.empty(x.shape, dtype=rd, device=x.device) if out is None else out
    init_buf = None
    if init is not None:
        init_buf = np.array([init], dtype=_np_dtype(rd))
    context(d).call("ki_scan", _GENERIC_OPS[op], _dtype_code(x), int(bool(exclusive)), _ptr(x), _ptr(out), x.numel(),
                    ctypes.c_void_p(init_buf.ctypes.data) if init_buf is not None else None, _stream_ptr(stream, d))
    return out


def scan_rows(x, op: str = "+", exclusive: bool = False, init=None, out=None, stream=None):
    """accumulate(op, x; dims) along each row of a 2-D ``x`` whose rows are contiguous
    (``x.stride(1) == 1``; ``x.stride(0)`` is the leading dimension), every row starting from ``init``.
    Operators and result types as ``scan``; ``out`` (rows contiguous) may have its own row stride."""
    import numpy as np

    torch = _torch()
    d = _dev(x)
    if op not in _GENERIC_OPS:
        raise KIArgumentError(_abi.KI_ERR_ARG, f"scan_rows: op must be one of {sorted(_GENERIC_OPS)}")
    if x.dim() != 2 or (x.shape[1] > 1 and x.stride(1) != 1):
        raise KIArgumentError(_abi.KI_ERR_ARG, "scan_rows: 2-D input with contiguous rows")
    rows, cols = x.shape
    rd = _result_dtype(x.dtype, op)
    out = torch.empty((rows, cols), dtype=rd, device=x.device) if out is None else out
    if out.shape != x.shape or out.dtype != rd or (cols > 1 and out.stride(1) != 1):
        raise KIArgumentError(_abi.KI_ERR_ARG, "scan_rows: output of the input's shape, result type and contiguous rows")
    init_buf = None if init is None else np.array([init], dtype=_np_dtype(rd))
    ld_in = x.stride(0) if rows > 1 else cols
    ld_out = out.stride(0) if rows > 1 else cols
    context(d).call("ki_scan_rows", _GENERIC_OPS[op], _dtype_code(x), int(bool(exclusive)), _ptr(x), max(ld_in, cols),
                    _ptr(out), max(ld_out, cols), rows, cols,
                    ctypes.c_void_p(init_buf.ctypes.data) if init_buf is not None else None, _stream_ptr(stream, d))
    return out


_PREDS = {">": 0, ">=": 1, "<": 2, "<=": 3, "==": 4, "!=": 5}


def compact(x, pred: str, threshold, out_vals=None, out_idx=None, count=None, index_base: int = 1, stream=None,
            trim: bool = True, f=None):
    """filter(v -> f(v) pred threshold, x) and findall for Int32/UInt32/Int64/UInt64/Float32/Float64 ``x``
    (IEEE comparisons; f None, 'abs' or 'abs2', applied in the element type; the kept elements are
    x's own).  Returns (vals, idx, count) like ``vote_compact``."""
    import numpy as np

    torch = _torch()
    d = _dev(x)
    if pred not in _PREDS:
        raise KIArgumentError(_abi.KI_ERR_ARG, f"compact: pred must be one of {sorted(_PREDS)}")
    if f not in _MAPS:
        raise KIArgumentError(_abi.KI_ERR_ARG, "compact: f must be 'abs', 'abs2' or None")
    x = x.contiguous()
    n = x.numel()
    thr = np.array([threshold], dtype=_np_dtype(x.dtype))
    out_vals = torch.empty(n, dtype=x.dtype, device=x.device) if out_vals is None else out_vals
    out_idx = torch.empty(n, dtype=torch.int32, device=x.device) if out_idx is None else out_idx
    count = torch.zeros((), dtype=torch.uint64, device=x.device) if count is None else count
    context(d).call("ki_compact_map", _MAPS[f], _PREDS[pred], _dtype_code(x), _ptr(x), n, ctypes.c_void_p(thr.ctypes.data),
                    _ptr(out_vals), _ptr(out_idx), ctypes.c_int64(int(index_base)), _ptr(count), _stream_ptr(stream, d))
    if trim:
        k = int(count.item())
        return out_vals[:k], out_idx[:k], count
    return out_vals, out_idx, count


def count(x, pred: str, threshold, f=None, out=None, stream=None):
    """count(v -> f(v) pred threshold, x): the compaction pipeline with no outputs.  Returns a UInt64
    device scalar."""
    import numpy as np

    torch = _torch()
    d = _dev(x)
    if pred not in _PREDS or f not in _MAPS:
        raise KIArgumentError(_abi.KI_ERR_ARG, "count: unknown predicate or map")
    x = x.contiguous()
    thr = np.array([threshold], dtype=_np_dtype(x.dtype))
    out = torch.zeros((), dtype=torch.uint64, device=x.device) if out is None else out
    context(d).call("ki_compact_map", _MAPS[f], _PREDS[pred], _dtype_code(x), _ptr(x), x.numel(),
                    ctypes.c_void_p(thr.ctypes.data), None, None, ctypes.c_int64(1), _ptr(out), _stream_ptr(stream, d))
    return out


def vote_compact(x, threshold: float, out_vals=None, out_idx=None, count=None, index_base: int = 1,
                 stream=None, trim: bool = True):
    """filter(v -> v > threshold, x) and findall (1-based Int32 indices by default).

    Returns (vals, idx, count) with ``count`` a device uint64 scalar; with trim=True the outputs are
    sliced to the count (one device-to-host read)."""
    torch = _torch()
    d = _dev(x)
    if x.dtype != torch.float32:
        raise KIArgumentError(_abi.KI_ERR_ARG, "vote_compact: Float32 input")
    n = x.numel()
    out_vals = torch.empty(n, dtype=torch.float32, device=x.device) if out_vals is None else out_vals
    out_idx = torch.empty(n, dtype=torch.int32, device=x.device) if out_idx is None else out_idx
    count = torch.zeros((), dtype=torch.uint64, device=x.device) if count is None else count
    context(d).call("ki_compact_gt_f32", _ptr(x), n, ctypes.c_float(threshold), _ptr(out_vals), _ptr(out_idx),
                    ctypes.c_int64(int(index_base)), _ptr(count), _stream_ptr(stream, d))
    if trim:
        k = int(count.item())
        return out_vals[:k], out_idx[:k], count
    return out_vals, out_idx, count


def fp8_gemm(A, B, C=None, scale_a: float = 1.0, scale_b: float = 1.0, stream=None):
    """C = scale_a*scale_b * A @ B for e4m3 A (MxK) and B (KxN), both row-major; Float32 C."""
    torch = _torch()
    d = _dev(A)
    M, K = A.shape
    K2, N = B.shape
    if K != K2:
        raise KIArgumentError(_abi.KI_ERR_ARG, "fp8_gemm: inner dimensions differ")
    C = torch.empty((M, N), dtype=torch.float32, device=A.device) if C is None else C
    context(d).call("ki_gemm_e4m3_f32", _ptr(A), _ptr(B), _ptr(C), M, N, K, ctypes.c_float(scale_a),
                    ctypes.c_float(scale_b), _stream_ptr(stream, d))
    return C


# ---------------------------------------------------------------------------------------------
# operators of a state-space layer served in 8 bits.  Single-token calls take less time on the GPU
# than in Python, so these checks read each tensor's properties once and build messages only to raise.
# These are served forms without gradients: a tensor that requires one is refused while torch records gradients,
# rather than its gradient lost.
# ---------------------------------------------------------------------------------------------
_float_codes: dict = {}


def _bad(what: str):
    return KIArgumentError(_abi.KI_ERR_ARG, what)


def _float_code(name: str, dtype) -> int:
    if not _float_codes:
        _float_codes.update({getattr(_torch(), k): v for k, v in _abi.FLOAT_DTYPE.items()})
    code = _float_codes.get(dtype)
    if code is None:
        raise _bad(f"{name}: float32, float16 or bfloat16 elements, not {dtype}")
    return code


def _index(name: str, t) -> int:
    d = t.get_device()
    if d < 0:
        raise _bad(f"{name}: tensors must be on a CUDA device (there is no CPU path)")
    return d


def _refuse(name: str, what: str, t, shape: tuple, dtype, d: int, how: str):
    if t.get_device() != d:
        raise _bad(f"{name}: {what} is on {t.device}, not on cuda:{d}")
    if t.dtype != dtype or t.shape != shape:
        raise _bad(f"{name}: {what} must be {dtype} {list(shape)}, not {t.dtype} {list(t.shape)}")
    raise _bad(f"{name}: {what} must {how}")


def _no_gradient(name: str, what: str):
    if _torch().is_grad_enabled():
        raise _bad(f"{name}: {what} requires a gradient, and this operator has none: detach it or call under torch.no_grad()")


def _rows(name: str, what: str, t, shape: tuple, dtype, d: int) -> int:
    """The row stride of a 2-D ``t`` of this shape and type on device ``d`` whose rows are contiguous."""
    if t.dtype is not dtype or t.shape != shape or t.get_device() != d:
        _refuse(name, what, t, shape, dtype, d, "")
    rows, cols = shape
    ld, inner = t.stride()
    if (inner != 1 and cols > 1) or (ld < cols and rows > 1):
        _refuse(name, what, t, shape, dtype, d, "have contiguous rows that do not overlap")
    if t.requires_grad:
        _no_gradient(name, what)
    return ld if rows > 1 else cols


def _flat(name: str, what: str, t, shape: tuple, dtype, d: int):
    """A pointer to ``t``, contiguous, of this shape and type and on device ``d``; None stays None."""
    if t is None:
        return None
    if t.dtype is not dtype or t.shape != shape or t.get_device() != d or not t.is_contiguous():
        _refuse(name, what, t, shape, dtype, d, "be contiguous")
    if t.requires_grad:
        _no_gradient(name, what)
    return t.data_ptr()


def _new(shape: tuple, dtype, like, stream):
    """A new tensor on ``like``'s device that belongs to the stream that writes it."""
    if stream is None:
        return like.new_empty(shape, dtype=dtype)
    with _torch().cuda.stream(stream):
        return like.new_empty(shape, dtype=dtype)


def _like(x, dtype, stream):
    """A new tensor of ``x``'s shape (whose rows are contiguous), with contiguous rows that follow each other."""
    if stream is None:
        return _torch().empty_like(x, dtype=dtype)
    with _torch().cuda.stream(stream):
        return _torch().empty_like(x, dtype=dtype)


_current_raw_stream = None


def _raw_stream(stream, d: int) -> int:
    global _current_raw_stream
    if stream is not None:
        if stream.device.index != d:
            raise _bad(f"stream of cuda:{stream.device.index} for tensors on cuda:{d}")
        return stream.cuda_stream
    if _current_raw_stream is None:
        _current_raw_stream = _torch()._C._cuda_getCurrentRawStream
    return _current_raw_stream(d)


def _state(name: str, state, first: int, second: int, dtype, d: int, slots, count: int):
    """(pointer, elements between slots, slots, pointer to the slot numbers) of a cache of states."""
    if state is None:
        if slots is not None:
            raise _bad(f"{name}: slots without a state")
        return None, 0, 0, None
    if state.dtype is not dtype or state.dim() != 3 or state.shape[1:] != (first, second) or state.get_device() != d:
        raise _bad(f"{name}: state must be {dtype} [slots, {first}, {second}] on cuda:{d}")
    if state.requires_grad:
        _no_gradient(name, "state")
    n, held = state.shape[0], first * second
    ld = held
    if not state.is_contiguous():
        ld, mid, inner = state.stride()
        if (inner != 1 and second > 1) or (mid != second and first > 1):
            raise _bad(f"{name}: every slot of the state must be contiguous")
        if n <= 1:
            ld = held
        elif ld < held:
            raise _bad(f"{name}: slots of the state overlap")
    if slots is None:
        if n < count:
            raise _bad(f"{name}: {n} state slots for {count} sequences")
        return state.data_ptr(), ld, n, None
    return state.data_ptr(), ld, n, _flat(name, "slots", slots, (count,), _torch().int32, d)


def _sequences(name: str, offsets, initial, state, d: int):
    """(sequences, pointer to the offsets, pointer to the initial flags)."""
    torch = _torch()
    count = 1
    if offsets is not None:
        if offsets.dim() != 1 or offsets.shape[0] < 1:
            raise _bad(f"{name}: offsets must hold one value more than there are sequences")
        count = offsets.shape[0] - 1
    at = _flat(name, "offsets", offsets, (count + 1,), torch.int32, d)
    if initial is not None:
        if state is None:
            raise _bad(f"{name}: initial without a state")
        if initial.dtype not in (torch.bool, torch.uint8):
            raise _bad(f"{name}: initial must be bool or uint8")
        initial = _flat(name, "initial", initial, (count,), initial.dtype, d)
    return count, at, initial


def _silu(name: str, activation) -> int:
    if activation is None:
        return 0
    if activation != "silu":
        raise _bad(f"{name}: activation must be 'silu' or None")
    return 1


def _matrix(name: str, what: str, t) -> tuple:
    shape = t.shape
    if len(shape) != 2:
        raise _bad(f"{name}: {what} must be 2-D")
    return shape


def quantize_rows(x, out=None, scale=None, stream=None):
    """int8 rows with one scale each: scale[r] = max|x[r]| * (1 / 127), out[r] = rint(x[r] / scale[r]) (ties
    to even, all in Float32), for a 2-D Float32, Float16 or BFloat16 ``x`` with contiguous rows.
    A row of zeros gives zeros and scale 0; a NaN or an infinity stays in the row's scale.  No gradient.
    Returns (out, scale): int8 of x's shape, Float32 per row."""
    torch = _torch()
    name = "quantize_rows"
    d = _index(name, x)
    rows, cols = shape = _matrix(name, "x", x)
    code = _float_code(name, x.dtype)
    ld = _rows(name, "x", x, shape, x.dtype, d)
    if out is None:
        out, ldq = _like(x, torch.int8, stream), cols
    else:
        ldq = _rows(name, "out", out, shape, torch.int8, d)
    if scale is None:
        scale = _new((rows,), torch.float32, x, stream)
        ps = scale.data_ptr()
    else:
        ps = _flat(name, "scale", scale, (rows,), torch.float32, d)
    context(d).call("ki_quantize_rows", code, x.data_ptr(), rows, cols, ld, out.data_ptr(), ldq, ps,
                    _raw_stream(stream, d))
    return out, scale


def int8_gemm(A, W, scale_a, scale_w, bias=None, out=None, dtype=None, stream=None):
    """out[m, n] = (sum_k A[m, k] W[n, k]) * scale_a[m] * scale_w[n] + bias[n] with exact Int32 sums on the
    tensor cores: int8 tokens ``A`` (M x K) and weights ``W`` (N x K) with contiguous rows, Float32 scales per
    token and per channel, Float32 ``bias`` or None.  ``out`` has ``dtype`` (bfloat16 unless given).  No gradient."""
    torch = _torch()
    name = "int8_gemm"
    d = _index(name, A)
    M, K = shape = _matrix(name, "A", A)
    N = _matrix(name, "W", W)[0]
    if dtype is None:
        dtype = torch.bfloat16 if out is None else out.dtype
    code = _float_code(name, dtype)
    lda = _rows(name, "A", A, shape, torch.int8, d)
    ldw = _rows(name, "W", W, (N, K), torch.int8, d)
    f32 = torch.float32
    pa = _flat(name, "scale_a", scale_a, (M,), f32, d)
    pw = _flat(name, "scale_w", scale_w, (N,), f32, d)
    pb = _flat(name, "bias", bias, (N,), f32, d)
    if out is None:
        out, ldc = _new((M, N), dtype, A, stream), N
    else:
        ldc = _rows(name, "out", out, (M, N), dtype, d)
    context(d).call("ki_gemm_i8", A.data_ptr(), lda, W.data_ptr(), ldw, pa, pw, pb, code, out.data_ptr(), ldc, M, N, K,
                    _raw_stream(stream, d))
    return out


def causal_conv(x, weight, bias=None, state=None, offsets=None, slots=None, initial=None, activation=None, out=None,
                stream=None):
    """Causal depthwise convolution of packed sequences: out[t, d] = act(bias[d] + sum_j weight[d, j] *
    x[t - (width-1) + j, d]) for ``x`` (tokens x channels, contiguous rows) and ``weight`` (channels x width,
    width 2 to 8), all of one type (Float32, Float16, BFloat16); activation None or 'silu'.

    ``offsets`` (int32, sequences + 1): sequence i holds rows offsets[i] to offsets[i+1]; None: one sequence.
    ``state`` (slots x (width-1) x channels, x's type): the last inputs of each sequence, oldest first, read
    before its first row and replaced; sequence i uses slot ``slots[i]`` (int32; None: slot i), negative
    numbers mark padding that is skipped, and no slot is named twice.  ``initial`` (bool or uint8): False
    starts the sequence from zeros.  Without a state every sequence starts from zeros.  Rows of no sequence
    are not written (a new output holds anything there).  A bad offset or slot number is reported by
    ``Context.check``.  No gradient."""
    name = "causal_conv"
    d = _index(name, x)
    tokens, channels = shape = _matrix(name, "x", x)
    width = _matrix(name, "weight", weight)[1]
    dtype = x.dtype
    code = _float_code(name, dtype)
    ldx = _rows(name, "x", x, shape, dtype, d)
    pw = _flat(name, "weight", weight, (channels, width), dtype, d)
    pb = _flat(name, "bias", bias, (channels,), dtype, d)
    count, at, flags = _sequences(name, offsets, initial, state, d)
    ps, state_ld, n, pslots = _state(name, state, width - 1, channels, dtype, d, slots, count)
    silu = _silu(name, activation)
    if out is None:
        out, ldy = _like(x, dtype, stream), channels
    else:
        ldy = _rows(name, "out", out, shape, dtype, d)
    context(d).call("ki_causal_conv", code, x.data_ptr(), ldx, pw, pb, ps, state_ld, n, pslots, flags, at, count,
                    out.data_ptr(), ldy, tokens, channels, width, silu, _raw_stream(stream, d))
    return out


def causal_conv_step(x, weight, bias=None, state=None, slots=None, activation=None, out=None, stream=None):
    """One token per row: row r of ``x`` (rows x channels) continues state slot ``slots[r]`` (None: slot r), which
    is updated; the arguments are those of ``causal_conv``."""
    name = "causal_conv_step"
    d = _index(name, x)
    rows, channels = shape = _matrix(name, "x", x)
    width = _matrix(name, "weight", weight)[1]
    dtype = x.dtype
    code = _float_code(name, dtype)
    if state is None:
        raise _bad(f"{name}: a state is needed")
    ldx = _rows(name, "x", x, shape, dtype, d)
    pw = _flat(name, "weight", weight, (channels, width), dtype, d)
    pb = _flat(name, "bias", bias, (channels,), dtype, d)
    ps, state_ld, n, pslots = _state(name, state, width - 1, channels, dtype, d, slots, rows)
    silu = _silu(name, activation)
    if out is None:
        out, ldy = _like(x, dtype, stream), channels
    else:
        ldy = _rows(name, "out", out, shape, dtype, d)
    context(d).call("ki_causal_conv_step", code, x.data_ptr(), ldx, pw, pb, ps, state_ld, n, pslots, out.data_ptr(), ldy,
                    rows, channels, width, silu, _raw_stream(stream, d))
    return out


def _per_state(name: str, what: str, t, rows: int, states: int, dtype, d: int) -> tuple:
    """(row stride, groups) of B or C: rows x states, or rows x groups x states with contiguous rows."""
    shape = t.shape
    if len(shape) == 2:
        return _rows(name, what, t, (rows, states), dtype, d), 1
    if len(shape) != 3:
        raise _bad(f"{name}: {what} must be 2-D or 3-D")
    groups = shape[1]
    if t.dtype is not dtype or shape[0] != rows or shape[2] != states or t.get_device() != d:
        _refuse(name, what, t, (rows, groups, states), dtype, d, "")
    ld, mid, inner = t.stride()
    if (inner != 1 and states > 1) or (mid != states and groups > 1) or (ld < groups * states and rows > 1):
        _refuse(name, what, t, shape, dtype, d, "have contiguous rows that do not overlap")
    if t.requires_grad:
        _no_gradient(name, what)
    return (ld if rows > 1 else groups * states), groups


def _scan_args(name, u, delta, A, B, C, D, z, delta_bias, d):
    f32 = _torch().float32
    rows, channels = shape = _matrix(name, "u", u)
    states = _matrix(name, "A", A)[1]
    dtype = u.dtype
    code = _float_code(name, dtype)
    ldu = _rows(name, "u", u, shape, dtype, d)
    ldd = _rows(name, "delta", delta, shape, dtype, d)
    pA = _flat(name, "A", A, (channels, states), f32, d)
    ldb, groups = _per_state(name, "B", B, rows, states, dtype, d)
    ldc, groups_c = _per_state(name, "C", C, rows, states, dtype, d)
    if groups != groups_c or groups < 1 or channels % groups:
        raise _bad(f"{name}: B and C need the same number of groups, a divisor of the channels")
    pD = _flat(name, "D", D, (channels,), f32, d)
    pbias = _flat(name, "delta_bias", delta_bias, (channels,), f32, d)
    ldz, pz = (0, None) if z is None else (_rows(name, "z", z, shape, dtype, d), z.data_ptr())
    return shape, states, groups, (code, u.data_ptr(), ldu, delta.data_ptr(), ldd, pA, B.data_ptr(), ldb, C.data_ptr(),
                                   ldc, pD, pz, ldz, pbias)


def selective_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, softplus=False, state=None, offsets=None,
                   slots=None, initial=None, out=None, stream=None):
    """Selective state space scan of packed sequences.  With s = delta + delta_bias (softplus'd if asked):

        h_t[d, n] = exp(s[t, d] A[d, n]) h_{t-1}[d, n] + s[t, d] u[t, d] B[t, g, n]
        out[t, d] = (sum_n C[t, g, n] h_t[d, n] + D[d] u[t, d]) * z[t, d] sigmoid(z[t, d])

    ``u``, ``delta``, ``z``: tokens x channels; ``B``, ``C``: tokens x states, or tokens x groups x states (channel d
    belongs to group d // (channels / groups)), all of one type (Float32, Float16, BFloat16) with contiguous
    rows; ``A``: channels x states, ``D``, ``delta_bias``: channels, Float32.  D, z and delta_bias may be None.
    ``state``: Float32 slots x channels x states; it, ``offsets``, ``slots`` and ``initial`` are as in ``causal_conv``.
    No gradient."""
    name = "selective_scan"
    d = _index(name, u)
    shape, states, groups, args = _scan_args(name, u, delta, A, B, C, D, z, delta_bias, d)
    rows, channels = shape
    count, at, flags = _sequences(name, offsets, initial, state, d)
    ps, state_ld, n, pslots = _state(name, state, channels, states, _torch().float32, d, slots, count)
    if out is None:
        out, ldy = _like(u, u.dtype, stream), channels
    else:
        ldy = _rows(name, "out", out, shape, u.dtype, d)
    context(d).call("ki_selective_scan", *args, 1 if softplus else 0, ps, state_ld, n, pslots, flags, at, count,
                    out.data_ptr(), ldy, rows, channels, states, groups, _raw_stream(stream, d))
    return out


def selective_scan_step(u, delta, A, B, C, D=None, z=None, delta_bias=None, softplus=False, state=None, slots=None,
                        out=None, stream=None):
    """One token per row: row r of ``u`` (rows x channels) continues state slot ``slots[r]`` (None: slot r), which
    is updated; the arguments are those of ``selective_scan``."""
    name = "selective_scan_step"
    d = _index(name, u)
    shape, states, groups, args = _scan_args(name, u, delta, A, B, C, D, z, delta_bias, d)
    rows, channels = shape
    if state is None:
        raise _bad(f"{name}: a state is needed")
    ps, state_ld, n, pslots = _state(name, state, channels, states, _torch().float32, d, slots, rows)
    if out is None:
        out, ldy = _like(u, u.dtype, stream), channels
    else:
        ldy = _rows(name, "out", out, shape, u.dtype, d)
    context(d).call("ki_selective_scan_step", *args, 1 if softplus else 0, ps, state_ld, n, pslots, out.data_ptr(), ldy,
                    rows, channels, states, groups, _raw_stream(stream, d))
    return out


# ---------------------------------------------------------------------------------------------
# synthetic inputs (splitmix64 streams; bit-identical to the host generator)
# ---------------------------------------------------------------------------------------------
def fill_uniform(out, seed: int, stream=None):
    d = _dev(out)
    context(d).call("ki_fill_uniform_f32", ctypes.c_uint64(seed), _ptr(out), out.numel(), _stream_ptr(stream, d))
    return out


def fill_int_range(out, seed: int, lo: int, hi: int, stream=None):
    d = _dev(out)
    context(d).call("ki_fill_int_range_i64", ctypes.c_uint64(seed), ctypes.c_int64(lo), ctypes.c_int64(hi),
                    _ptr(out), out.numel(), _stream_ptr(stream, d))
    return out


def fill_bytes(out, seed: int, stream=None):
    d = _dev(out)
    context(d).call("ki_fill_bytes", ctypes.c_uint64(seed), _ptr(out), out.numel() * out.element_size(),
                    _stream_ptr(stream, d))
    return out


def fill_normal(out, seed: int, stream=None):
    d = _dev(out)
    context(d).call("ki_fill_normal_f32", ctypes.c_uint64(seed), _ptr(out), out.numel(), _stream_ptr(stream, d))
    return out


def fill_e4m3_uniform(out, seed: int, scale: float, stream=None):
    d = _dev(out)
    context(d).call("ki_fill_e4m3_uniform", ctypes.c_uint64(seed), ctypes.c_float(scale), _ptr(out),
                    out.numel() * out.element_size(), _stream_ptr(stream, d))
    return out
