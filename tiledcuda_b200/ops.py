"""Operators of the tile-kernel path on torch CUDA tensors, each a thin call into the C ABI.

Tensors supply device memory and the current stream; all arithmetic happens in the sm_100a kernels
of libtiledcuda_b200.so. Outputs are written in place into caller-allocated tensors, as the
reference's ops do (include/kernels/flash_attn.hpp:35-37, include/kernels/scatter_nd.hpp:39-40).
Nothing here falls back to PyTorch: a CPU tensor, a wrong dtype or an unsupported shape raises.
"""
from __future__ import annotations

import ctypes
import math
import os
import re
from pathlib import Path

import torch

from . import _lib


import contextlib

_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_NO_GUARD = contextlib.nullcontext()


def _stream() -> ctypes.c_void_p:
    """The current CUDA stream of the current device as a raw handle."""
    if _raw_stream is not None:
        return ctypes.c_void_p(_raw_stream(torch.cuda.current_device()))
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _on(device: torch.device):
    """Context that makes `device` current for the call; free when it already is (the usual case)."""
    if device.index is None or device.index == torch.cuda.current_device():
        return _NO_GUARD
    return torch.cuda.device(device)


def _ptr(t: torch.Tensor | None) -> ctypes.c_void_p:
    return ctypes.c_void_p(0 if t is None else t.data_ptr())


def _need(t: torch.Tensor, name: str, dtype: torch.dtype, contiguous: bool = True) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (there is no CPU path)")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def gemm(a: torch.Tensor, b: torch.Tensor, c: torch.Tensor, max_sms: int = 0) -> None:
    """c[M,N] (fp32) = a[M,K] @ b[N,K].T with fp16 (or bf16) inputs and fp32 accumulation.

    `b` is the column-major [K,N] operand of the reference's GEMM stored as [N,K] rows, so the result
    equals `a @ b.t()` (examples/python/gemm/main.py:21). Row strides of a, b, c may exceed the row
    length (leading dimensions); the innermost stride must be 1. max_sms > 0 (fp16 only) runs the GEMM on
    at most that many SMs and leaves the rest to kernels running beside it (tc_gemm_f16_f32_sms).
    """
    in_dtype = torch.bfloat16 if isinstance(a, torch.Tensor) and a.dtype == torch.bfloat16 else torch.float16
    for t, name, dt in ((a, "a", in_dtype), (b, "b", in_dtype), (c, "c", torch.float32)):
        _need(t, name, dt, contiguous=False)
        if t.dim() != 2 or t.stride(1) != 1:
            raise ValueError(f"{name} must be 2-D with unit inner stride")
    m, k = a.shape
    n, kb = b.shape
    if kb != k or tuple(c.shape) != (m, n):
        raise ValueError(f"shape mismatch: a {tuple(a.shape)}, b {tuple(b.shape)}, c {tuple(c.shape)}")
    lib = _lib.load()
    if max_sms:
        if in_dtype != torch.float16:
            raise ValueError("max_sms is supported for fp16 inputs only")
        with _on(a.device):
            _lib.check("tc_gemm_f16_f32_sms",
                       lib.tc_gemm_f16_f32_sms(_ptr(a), _ptr(b), _ptr(c), m, n, k, a.stride(0), b.stride(0), c.stride(0),
                                               int(max_sms), _stream()))
        return
    fn_name = "tc_gemm_bf16_f32" if in_dtype == torch.bfloat16 else "tc_gemm_f16_f32"
    with _on(a.device):
        _lib.check(
            fn_name,
            getattr(lib, fn_name)(_ptr(a), _ptr(b), _ptr(c), m, n, k, a.stride(0), b.stride(0), c.stride(0), _stream()),
        )


_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 4}   # enum tc_type
_HALVES = (torch.float16, torch.bfloat16)
_INT8 = (torch.int8,)
_FLOAT = (torch.float32,)
_INTS = (torch.int32, torch.int64)


def _need_rows(t: torch.Tensor, name: str, shape: tuple, dtypes, device: int) -> bool:
    """A CUDA tensor of this shape on this device whose last dimension is dense; other strides are the caller's.
    device is -1 where the first operand of a call is not a CUDA tensor. Returns whether all of it is contiguous."""
    try:   # the usual case, in as few attribute reads as it takes (Tensor.stride alone is 0.4 us)
        if t.shape == shape and t.dtype in dtypes and t.get_device() == device >= 0:
            if t.is_contiguous():
                return True
            if shape[-1] <= 1 or t.stride(-1) == 1:
                return False
    except (AttributeError, TypeError):
        pass
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (there is no CPU path)")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} must have unit inner stride")
    raise ValueError(f"{name} is on {t.device}, the other operands are on cuda:{device}")


def _shape(t: torch.Tensor, name: str, dim: int) -> torch.Size:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dim() != dim:
        raise ValueError(f"{name} must be {dim}-D, got {list(t.shape)}")
    return t.shape


def _ld(t: torch.Tensor, shape: tuple, contiguous: bool, dim: int = 0, granule: int = 1) -> int:
    """Stride of a dimension in elements. That of a dimension of one element is never stepped over and may be anything,
    so it is replaced by the dense one, rounded up to what the kernels' loads are granular in."""
    if shape[dim] > 1 and not contiguous:
        return t.stride(dim)
    inner = shape[dim + 1] if dim + 2 == len(shape) else shape[dim + 1] * _ld(t, shape, contiguous, dim + 1, granule)
    return inner if shape[dim] > 1 else -(-max(1, inner) // granule) * granule


def _launch(name: str, device: int, *args) -> None:
    """Calls the C entry point `name` on the current stream of `device` and raises if it fails."""
    fn = getattr(_lib.load(), name)
    if device == torch.cuda.current_device():
        status = fn(*args, _raw_stream(device) if _raw_stream is not None else _stream())
    else:
        with torch.cuda.device(device):
            status = fn(*args, _stream())
    if status:
        _lib.check(name, status)


_OP_LIB = Path(__file__).resolve().parent / "libtiledcuda.so"
_registered_ops: dict | None = None
_direct_calls: dict = {}
_OP_FAILED = re.compile(r"tiledcuda::(\w+) failed with status (-?\d+): (.*)")   # how torch_bind.cc passes a status on


def _registered(name: str):
    """The op of that name in torch.ops.tiledcuda, or None where the op library has not been built. It makes the checks
    and the call of the functions below in C++: a call of gemm_i8 costs the host 4.7 us by that way, 3.4 past the dispatcher
    (_calls) and 8.2 by ctypes."""
    global _registered_ops
    if _registered_ops is None:
        _registered_ops = {}
        try:
            torch.ops.load_library(os.fspath(_OP_LIB))
        except OSError:
            pass   # not built, or for another torch
        else:
            for op in ("quantize_rows", "gemm_i8", "grouped_gemm", "grouped_gemm_i8", "grouped_gemm_dgrad", "grouped_gemm_wgrad"):
                packet = getattr(torch.ops.tiledcuda, op, None)   # not in a library built before the op was there
                if packet is not None:
                    _registered_ops[op] = packet.default
            try:
                from . import _calls
            except ImportError:
                pass
            else:
                _direct_calls.update((op, getattr(_calls, op)) for op in _registered_ops)
    return _registered_ops.get(name)


_DONE = Exception()


def _through_op(name: str, *args) -> Exception | None:
    """Makes the call through the registered op, or past the dispatcher where nothing would see it there (_calls), and returns _DONE.
    Returns None where there is no such op, and its error where it raised one: the checks of the function that called this then say
    in their own words what is wrong with the arguments, and _pass_on raises what they do not explain."""
    op = _registered(name)
    if op is None:
        return None
    try:
        direct = _direct_calls.get(name)
        if direct is None or not direct(*args):
            op(*args)
    except (RuntimeError, TypeError) as error:
        return error
    return _DONE


def _pass_on(error: Exception | None) -> None:
    """Raises the error of a registered op: what the C entry point said as the other way to it has it, anything else (a failure of a
    dispatch mode, say) as it is. None: there was no op, and the call is still to be made."""
    if error is None:
        return
    status = _OP_FAILED.match(str(error))
    if status is None:
        raise error
    raise _lib.TiledCudaError("tc_" + status[1], int(status[2]), status[3]) from error


def quantize_rows(x: torch.Tensor, q: torch.Tensor, scale: torch.Tensor) -> None:
    """q (int8 [M,K]) and scale (fp32 [M]) such that q[m] * scale[m] stands for x[m] (fp16, bf16 or fp32 [M,K]).

    scale = max(amax|x[m]| * (1/127), 2^-126) in fp32; q = x / scale rounded to nearest, ties to even. One scale per token for
    activations, one per output channel for a weight [N,K]. A row with an infinity or NaN gets that as its scale
    and q = 0. Row strides of x and q may exceed the row length.
    """
    refused = _through_op("quantize_rows", x, q, scale)
    if refused is _DONE:
        return
    shape = _shape(x, "x", 2)
    m, k = shape
    dev = x.get_device()
    dense_x = _need_rows(x, "x", shape, _TYPES, dev)
    dense_q = _need_rows(q, "q", shape, _INT8, dev)
    _need_rows(scale, "scale", (m,), _FLOAT, dev)
    _pass_on(refused)
    _launch("tc_quantize_rows", dev, x.data_ptr(), q.data_ptr(), scale.data_ptr(), m, k, _ld(x, shape, dense_x), _ld(q, shape, dense_q),
            _TYPES[x.dtype])


def gemm_i8(a: torch.Tensor, b: torch.Tensor, scale_a: torch.Tensor, scale_b: torch.Tensor, c: torch.Tensor) -> None:
    """c[M,N] (fp16, bf16 or fp32) = (a @ b.T) * scale_a[:, None] * scale_b[None, :], a int8 [M,K], b int8 [N,K].

    scale_a fp32 [M] (per token), scale_b fp32 [N] (per output channel). The integer sums are exact (K <= 131071);
    scaled in fp32 and rounded once. Row strides of a and b must be multiples of 16 bytes, K and N may be any size; M
    may be 0.
    """
    refused = _through_op("gemm_i8", a, b, scale_a, scale_b, c)
    if refused is _DONE:
        return
    sa, sb = _shape(a, "a", 2), _shape(b, "b", 2)
    m, k = sa
    n = sb[0]
    dev = a.get_device()
    dense_a = _need_rows(a, "a", sa, _INT8, dev)
    dense_b = _need_rows(b, "b", (n, k), _INT8, dev)
    _need_rows(scale_a, "scale_a", (m,), _FLOAT, dev)
    _need_rows(scale_b, "scale_b", (n,), _FLOAT, dev)
    dense_c = _need_rows(c, "c", (m, n), _TYPES, dev)
    _pass_on(refused)
    _launch("tc_gemm_i8", dev, a.data_ptr(), b.data_ptr(), scale_a.data_ptr(), scale_b.data_ptr(), c.data_ptr(), m, n, k,
            _ld(a, sa, dense_a, 0, 16), _ld(b, sb, dense_b, 0, 16), _ld(c, (m, n), dense_c), _TYPES[c.dtype])


def _need_offsets(offsets: torch.Tensor, experts: int, device: int) -> int:
    _need_rows(offsets, "offsets", (experts + 1,), _INTS, device)
    return int(offsets.dtype == torch.int64)


def grouped_gemm(a: torch.Tensor, b: torch.Tensor, offsets: torch.Tensor, c: torch.Tensor) -> None:
    """c[t] = a[t] @ b[e].T for the rows t of expert e, which are offsets[e] <= t < offsets[e + 1].

    a [T,K], rows sorted by expert; b [E,N,K]; both fp16 or both bf16; c [T,N] of the same type or fp32. offsets is a
    CUDA int32 / int64 tensor [E + 1], nondecreasing, within [0, T]; it is read on the device only. Experts may be
    empty; rows of c outside all groups stay as they were. Row strides of a and b must be multiples of 16 bytes. Like the other
    operators here it is not recorded by autograd; its gradients are grouped_gemm_dgrad and grouped_gemm_wgrad.
    """
    refused = _through_op("grouped_gemm", a, b, offsets, c)
    if refused is _DONE:
        return
    sa, sb = _shape(a, "a", 2), _shape(b, "b", 3)
    t, k = sa
    e, n, _ = sb
    dev = a.get_device()
    dense_a = _need_rows(a, "a", sa, _HALVES, dev)
    dense_b = _need_rows(b, "b", (e, n, k), (a.dtype,), dev)
    dense_c = _need_rows(c, "c", (t, n), (a.dtype, torch.float32), dev)
    wide = _need_offsets(offsets, e, dev)
    _pass_on(refused)
    _launch("tc_grouped_gemm", dev, a.data_ptr(), b.data_ptr(), offsets.data_ptr(), wide, c.data_ptr(), t, e, n, k, _ld(a, sa, dense_a, 0, 8),
            _ld(b, sb, dense_b, 1, 8), _ld(b, sb, dense_b, 0, 8), _ld(c, (t, n), dense_c), _TYPES[a.dtype], _TYPES[c.dtype])


def grouped_gemm_i8(a: torch.Tensor, b: torch.Tensor, scale_a: torch.Tensor, scale_b: torch.Tensor, offsets: torch.Tensor,
                    c: torch.Tensor) -> None:
    """grouped_gemm on int8 a [T,K] and b [E,N,K]: c[t] = (a[t] @ b[e].T) * scale_a[t] * scale_b[e].

    scale_a fp32 [T], scale_b fp32 [E,N] contiguous, c [T,N] fp16, bf16 or fp32; sums as in gemm_i8, offsets and
    rows outside all groups as in grouped_gemm. Strides of a and b must be multiples of 16 bytes.
    """
    refused = _through_op("grouped_gemm_i8", a, b, scale_a, scale_b, offsets, c)
    if refused is _DONE:
        return
    sa, sb = _shape(a, "a", 2), _shape(b, "b", 3)
    t, k = sa
    e, n, _ = sb
    dev = a.get_device()
    dense_a = _need_rows(a, "a", sa, _INT8, dev)
    dense_b = _need_rows(b, "b", (e, n, k), _INT8, dev)
    _need_rows(scale_a, "scale_a", (t,), _FLOAT, dev)
    _need_rows(scale_b, "scale_b", (e, n), _FLOAT, dev)
    if not scale_b.is_contiguous():
        raise ValueError("scale_b must be contiguous")
    dense_c = _need_rows(c, "c", (t, n), _TYPES, dev)
    wide = _need_offsets(offsets, e, dev)
    _pass_on(refused)
    _launch("tc_grouped_gemm_i8", dev, a.data_ptr(), b.data_ptr(), scale_a.data_ptr(), scale_b.data_ptr(), offsets.data_ptr(), wide,
            c.data_ptr(), t, e, n, k, _ld(a, sa, dense_a, 0, 16), _ld(b, sb, dense_b, 1, 16), _ld(b, sb, dense_b, 0, 16),
            _ld(c, (t, n), dense_c), _TYPES[c.dtype])


def grouped_gemm_dgrad(dc: torch.Tensor, b: torch.Tensor, offsets: torch.Tensor, da: torch.Tensor) -> None:
    """Gradient of grouped_gemm to a: da[t] = dc[t] @ b[e] for the rows t of expert e.

    dc [T,N] and b [E,N,K] of one type (fp16 or bf16), da [T,K] of that type or fp32; offsets and the rows outside all
    groups as in grouped_gemm. Row strides of dc and b must be multiples of 16 bytes.
    """
    refused = _through_op("grouped_gemm_dgrad", dc, b, offsets, da)
    if refused is _DONE:
        return
    sc, sb = _shape(dc, "dc", 2), _shape(b, "b", 3)
    t, n = sc
    e, _, k = sb
    dev = dc.get_device()
    dense_dc = _need_rows(dc, "dc", sc, _HALVES, dev)
    dense_b = _need_rows(b, "b", (e, n, k), (dc.dtype,), dev)
    dense_da = _need_rows(da, "da", (t, k), (dc.dtype, torch.float32), dev)
    wide = _need_offsets(offsets, e, dev)
    _pass_on(refused)
    _launch("tc_grouped_gemm_dgrad", dev, dc.data_ptr(), b.data_ptr(), offsets.data_ptr(), wide, da.data_ptr(), t, e, n, k,
            _ld(dc, sc, dense_dc, 0, 8), _ld(b, sb, dense_b, 1, 8), _ld(b, sb, dense_b, 0, 8), _ld(da, (t, k), dense_da), _TYPES[dc.dtype], _TYPES[da.dtype])


def grouped_gemm_wgrad(dc: torch.Tensor, a: torch.Tensor, offsets: torch.Tensor, db: torch.Tensor) -> None:
    """Gradient of grouped_gemm to b: db[e] = dc[rows of e].T @ a[rows of e], zeros for an expert without rows.

    dc [T,N] and a [T,K] of one type (fp16 or bf16), db [E,N,K] of that type or fp32, overwritten as a whole. Rows
    outside all groups take no part. Row strides of dc and a must be multiples of 16 bytes.
    """
    refused = _through_op("grouped_gemm_wgrad", dc, a, offsets, db)
    if refused is _DONE:
        return
    sc, sa, sb = _shape(dc, "dc", 2), _shape(a, "a", 2), _shape(db, "db", 3)
    t, n = sc
    k = sa[1]
    e = sb[0]
    dev = dc.get_device()
    dense_dc = _need_rows(dc, "dc", sc, _HALVES, dev)
    dense_a = _need_rows(a, "a", (t, k), (dc.dtype,), dev)
    dense_db = _need_rows(db, "db", (e, n, k), (dc.dtype, torch.float32), dev)
    wide = _need_offsets(offsets, e, dev)
    _pass_on(refused)
    _launch("tc_grouped_gemm_wgrad", dev, dc.data_ptr(), a.data_ptr(), offsets.data_ptr(), wide, db.data_ptr(), t, e, n, k,
            _ld(dc, sc, dense_dc, 0, 8), _ld(a, sa, dense_a, 0, 8), _ld(db, sb, dense_db, 1), _ld(db, sb, dense_db, 0), _TYPES[dc.dtype], _TYPES[db.dtype])


def gemm_host(a: torch.Tensor, b: torch.Tensor, c: torch.Tensor, workspace: torch.Tensor) -> None:
    """c (host, fp32 [M,N]) = a (host, fp16 [M,K]) @ b (host, fp16 [N,K]).T, copies pipelined against the kernel.

    a, b, c are contiguous CPU tensors (pinned for the copies to overlap); workspace is a CUDA uint8 tensor of
    at least gemm_host_workspace_bytes(M, N, K) bytes on the device that does the work. Everything is queued
    on return; synchronise the current stream of that device before reading c.
    """
    for t, name, dt in ((a, "a", torch.float16), (b, "b", torch.float16), (c, "c", torch.float32)):
        if t.is_cuda or t.dtype != dt or t.dim() != 2 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous 2-D CPU tensor of {dt}")
    if not workspace.is_cuda or not workspace.is_contiguous():
        raise ValueError("workspace must be a contiguous CUDA tensor")
    m, k = a.shape
    n, kb = b.shape
    if kb != k or tuple(c.shape) != (m, n):
        raise ValueError(f"shape mismatch: a {tuple(a.shape)}, b {tuple(b.shape)}, c {tuple(c.shape)}")
    lib = _lib.load()
    with _on(workspace.device):
        _lib.check(
            "tc_gemm_f16_f32_host",
            lib.tc_gemm_f16_f32_host(_ptr(a), _ptr(b), _ptr(c), m, n, k, _ptr(workspace),
                                     workspace.numel() * workspace.element_size(), _stream()),
        )


def gemm_host_workspace_bytes(m: int, n: int, k: int) -> int:
    return int(_lib.load().tc_gemm_host_workspace_bytes(m, n, k))


def back2back_gemm(a: torch.Tensor, b: torch.Tensor, d: torch.Tensor, e: torch.Tensor) -> None:
    """e (fp32 [.., M, P]) = fp16(a @ b.T) @ d.T, the intermediate kept on chip.

    a fp16 [batch, M, K] or [M, K]; b fp16 [.., N, K] (column-major [K,N]); d fp16 [.., P, N]
    (column-major [N,P]); as in KeFusedGemm (examples/cpp/02_fused_two_gemms/fused_gemm.hpp:98-181).
    """
    for t, name, dt in ((a, "a", torch.float16), (b, "b", torch.float16), (d, "d", torch.float16), (e, "e", torch.float32)):
        _need(t, name, dt)
    if a.dim() not in (2, 3) or b.dim() != a.dim() or d.dim() != a.dim() or e.dim() != a.dim():
        raise ValueError("a, b, d, e must all be 2-D or all be 3-D (batched)")
    batch = a.shape[0] if a.dim() == 3 else 1
    m, k = a.shape[-2:]
    n, kb = b.shape[-2:]
    p, nd = d.shape[-2:]
    if kb != k or nd != n or tuple(e.shape[-2:]) != (m, p):
        raise ValueError(f"shape mismatch: a {tuple(a.shape)}, b {tuple(b.shape)}, d {tuple(d.shape)}, e {tuple(e.shape)}")
    if a.dim() == 3 and not (b.shape[0] == d.shape[0] == e.shape[0] == batch):
        raise ValueError("batch sizes differ")
    lib = _lib.load()
    with _on(a.device):
        _lib.check("tc_b2b_gemm_f16", lib.tc_b2b_gemm_f16(_ptr(a), _ptr(b), _ptr(d), _ptr(e), m, n, k, p, batch, _stream()))


def flash_attn(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    o: torch.Tensor,
    scale: float | None = None,
    lse: torch.Tensor | None = None,
    v_is_transposed: bool = False,
    causal: bool = False,
    seq_major: bool = False,
) -> None:
    """o = softmax(scale * q k^T) v per (batch, head); fp32 statistics.

    q [B,H,Sq,D], k [B,H,Skv,D], o [B,H,Sq,Dv] fp16; v [B,H,Skv,Dv], or [B,H,Dv,Skv] when
    v_is_transposed. With seq_major the four tensors are [B,S,H,D] instead. scale defaults to
    1/sqrt(D). lse, if given, is fp32 [B,H,Sq]. causal: query row i sees KV rows
    j <= i + (Skv - Sq); a row that sees none comes back as zeros.
    """
    for t, name in ((q, "q"), (k, "k"), (v, "v"), (o, "o")):
        _need(t, name, torch.float16)
        if t.dim() != 4:
            raise ValueError(f"{name} must be 4-D [batch, heads, seq, dim]")
    if seq_major:
        if v_is_transposed:
            raise ValueError("a transposed v is not supported with seq_major operands")
        b, sq, h, d = q.shape
        skv = k.shape[1]
        dv = v.shape[3]
        k_expect, v_expect, o_expect = (b, skv, h, d), (b, skv, h, dv), (b, sq, h, dv)
    else:
        b, h, sq, d = q.shape
        skv = k.shape[2]
        dv = v.shape[2] if v_is_transposed else v.shape[3]
        k_expect = (b, h, skv, d)
        v_expect = (b, h, dv, skv) if v_is_transposed else (b, h, skv, dv)
        o_expect = (b, h, sq, dv)
    if tuple(k.shape) != k_expect or tuple(v.shape) != v_expect or tuple(o.shape) != o_expect:
        raise ValueError(f"shape mismatch: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}, o {tuple(o.shape)}")
    if lse is not None:
        _need(lse, "lse", torch.float32)
        if tuple(lse.shape) != (b, h, sq):
            raise ValueError("lse must be [batch, heads, seq_q]")
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    lib = _lib.load()
    with _on(q.device):
        if causal or seq_major:
            _lib.check(
                "tc_flash_attn_fwd_ex_f16",
                lib.tc_flash_attn_fwd_ex_f16(
                    _ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(lse), b, h, sq, skv, d, dv, float(scale),
                    int(bool(v_is_transposed)), int(bool(causal)), int(bool(seq_major)), _stream(),
                ),
            )
        else:
            _lib.check(
                "tc_flash_attn_fwd_f16",
                lib.tc_flash_attn_fwd_f16(
                    _ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(lse), b, h, sq, skv, d, dv, float(scale),
                    int(bool(v_is_transposed)), _stream(),
                ),
            )


def flash_attention_fwd(Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, O: torch.Tensor, m: int, n: int, k: int, p: int) -> None:
    """The reference's op, argument for argument (src/kernels/flash_attn.cu:424-456).

    Flattened fp16 buffers: Q is [m,k] row-major, K is [n,k] row-major (K as [seq, dim]), V is V^T
    = [p,n] row-major, O is [m,p]; one head, no softmax scale. Any m, n and k, p <= 128 that the
    kernel covers are accepted, not only the reference's three hard-coded shapes.
    """
    for t, name, numel in ((Q, "Q", m * k), (K, "K", n * k), (V, "V", n * p), (O, "O", m * p)):
        _need(t, name, torch.float16)
        if t.numel() != numel:
            raise ValueError(f"{name} has {t.numel()} elements, expected {numel}")
    lib = _lib.load()
    with torch.cuda.device(Q.device):
        _lib.check(
            "tc_flash_attn_fwd_f16",
            lib.tc_flash_attn_fwd_f16(_ptr(Q), _ptr(K), _ptr(V), _ptr(O), _ptr(None), 1, 1, m, n, k, p, 1.0, 1, _stream()),
        )


def lstm_cell(
    w: torch.Tensor,
    u: torch.Tensor,
    bias: torch.Tensor | None,
    x: torch.Tensor,
    h_prev: torch.Tensor,
    c_prev: torch.Tensor,
    h_out: torch.Tensor,
    c_out: torch.Tensor,
) -> None:
    """One LSTM cell step with gate order (i, f, g, o) as torch.nn.LSTMCell.

    gates = x @ w.T + h_prev @ u.T + bias; c_out = sigmoid(f) * c_prev + sigmoid(i) * tanh(g);
    h_out = sigmoid(o) * tanh(c_out). w fp16 [4H, I]; u fp16 [4H, H]; bias fp32 [4H] or None; x fp16
    [B, I]; h fp16 [B, H]; c fp32 [B, H].
    """
    _need(w, "w", torch.float16)
    _need(u, "u", torch.float16)
    _need(x, "x", torch.float16)
    _need(h_prev, "h_prev", torch.float16)
    _need(h_out, "h_out", torch.float16)
    _need(c_prev, "c_prev", torch.float32)
    _need(c_out, "c_out", torch.float32)
    if bias is not None:
        _need(bias, "bias", torch.float32)
    batch, inp = x.shape
    hidden = u.shape[1]
    if tuple(w.shape) != (4 * hidden, inp) or tuple(u.shape) != (4 * hidden, hidden):
        raise ValueError(f"weight shapes {tuple(w.shape)}, {tuple(u.shape)} do not match input {inp}, hidden {hidden}")
    for t, name in ((h_prev, "h_prev"), (h_out, "h_out"), (c_prev, "c_prev"), (c_out, "c_out")):
        if tuple(t.shape) != (batch, hidden):
            raise ValueError(f"{name} must be [{batch}, {hidden}]")
    if bias is not None and bias.numel() != 4 * hidden:
        raise ValueError("bias must have 4*hidden elements")
    if h_out.data_ptr() == h_prev.data_ptr():
        raise ValueError("h_out must not alias h_prev")
    lib = _lib.load()
    with _on(x.device):
        _lib.check(
            "tc_lstm_cell_f16",
            lib.tc_lstm_cell_f16(_ptr(w), _ptr(u), _ptr(bias), _ptr(x), _ptr(h_prev), _ptr(c_prev), _ptr(h_out),
                                 _ptr(c_out), batch, inp, hidden, _stream()),
        )


def lstm_chain(
    w: torch.Tensor,
    u: torch.Tensor,
    bias: torch.Tensor | None,
    x: torch.Tensor,
    h0: torch.Tensor,
    c0: torch.Tensor,
    h_all: torch.Tensor,
    c_out: torch.Tensor,
    workspace: torch.Tensor | None = None,
) -> None:
    """`steps` chained cells: x fp16 [T, B, I]; h_all fp16 [T, B, H] gets every h_t; c_out fp32 [B, H] gets c_T.

    With `workspace` (a CUDA tensor of at least lstm_chain_workspace_bytes(T, B, H) bytes) the input
    projections of all steps are computed first as one GEMM and each step only runs h @ U.T.
    """
    _need(w, "w", torch.float16)
    _need(u, "u", torch.float16)
    _need(x, "x", torch.float16)
    _need(h0, "h0", torch.float16)
    _need(h_all, "h_all", torch.float16)
    _need(c0, "c0", torch.float32)
    _need(c_out, "c_out", torch.float32)
    if bias is not None:
        _need(bias, "bias", torch.float32)
    steps, batch, inp = x.shape
    hidden = u.shape[1]
    if tuple(w.shape) != (4 * hidden, inp) or tuple(u.shape) != (4 * hidden, hidden):
        raise ValueError("weight shapes do not match x / hidden size")
    if tuple(h_all.shape) != (steps, batch, hidden) or tuple(h0.shape) != (batch, hidden):
        raise ValueError("h_all must be [steps, batch, hidden] and h0 [batch, hidden]")
    if tuple(c0.shape) != (batch, hidden) or tuple(c_out.shape) != (batch, hidden):
        raise ValueError("c0 and c_out must be [batch, hidden]")
    lib = _lib.load()
    with _on(x.device):
        if workspace is None:
            _lib.check(
                "tc_lstm_chain_f16",
                lib.tc_lstm_chain_f16(_ptr(w), _ptr(u), _ptr(bias), _ptr(x), _ptr(h0), _ptr(c0), _ptr(h_all), _ptr(c_out),
                                      steps, batch, inp, hidden, _stream()),
            )
        else:
            if not workspace.is_cuda or not workspace.is_contiguous():
                raise ValueError("workspace must be a contiguous CUDA tensor")
            _lib.check(
                "tc_lstm_chain_ws_f16",
                lib.tc_lstm_chain_ws_f16(_ptr(w), _ptr(u), _ptr(bias), _ptr(x), _ptr(h0), _ptr(c0), _ptr(h_all), _ptr(c_out),
                                         steps, batch, inp, hidden, _ptr(workspace), workspace.numel() * workspace.element_size(),
                                         _stream()),
            )


def lstm_chain_workspace_bytes(steps: int, batch: int, hidden: int) -> int:
    """Bytes of scratch memory lstm_chain needs to hoist the input projections out of the recurrence."""
    return int(_lib.load().tc_lstm_chain_workspace_bytes(steps, batch, hidden))


_SCATTER_ADD_TYPES = {torch.float32: 0, torch.float16: 1, torch.int32: 2, torch.float64: 3}


def _scatter_args(data: torch.Tensor, indices: torch.Tensor, updates: torch.Tensor):
    if not data.is_cuda or not indices.is_cuda or not updates.is_cuda:
        raise ValueError("scatter_nd needs CUDA tensors (there is no CPU path)")
    if indices.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"indices must be int32 or int64, got {indices.dtype}")
    if updates.dtype != data.dtype:
        raise TypeError("updates and data must have the same dtype")
    if not (data.is_contiguous() and indices.is_contiguous() and updates.is_contiguous()):
        raise ValueError("data, indices and updates must be contiguous")
    if indices.dim() < 1:
        raise ValueError("indices must have at least one dimension")
    k = indices.shape[-1]
    n = indices.numel() // k if k else 0
    if k < 1 or k > data.dim():
        raise ValueError(f"index tuple length {k} does not fit data of rank {data.dim()}")
    slice_elems = 1
    for s in data.shape[k:]:
        slice_elems *= s
    if updates.numel() != n * slice_elems:
        raise ValueError(f"updates has {updates.numel()} elements, expected {n} slices of {slice_elems}")
    dims = (ctypes.c_int64 * data.dim())(*data.shape)
    return dims, n, k


def scatter_nd(data: torch.Tensor, indices: torch.Tensor, updates: torch.Tensor) -> None:
    """data[indices[t, 0], ..., indices[t, k-1]] = updates[t] for every index tuple t (in place).

    data is N-D and contiguous; indices is int32 or int64 [..., k]; updates holds one slice
    data.shape[k:] per tuple. Tuples must be unique for a deterministic result. Argument order follows
    the reference's Python wrapper (pytiledcuda/__init__.py:6-8): data, indices, updates.
    """
    dims, n, k = _scatter_args(data, indices, updates)
    lib = _lib.load()
    with _on(data.device):
        _lib.check(
            "tc_scatter_nd",
            lib.tc_scatter_nd(_ptr(data), _ptr(updates), _ptr(indices), int(indices.dtype == torch.int64), dims,
                              data.dim(), n, k, data.element_size(), _stream()),
        )


def scatter_nd_add(data: torch.Tensor, indices: torch.Tensor, updates: torch.Tensor) -> None:
    """data[indices[t, 0], ..., indices[t, k-1]] += updates[t] (in place); repeated tuples add up.

    What the reference's kernel does with one atomicAdd per element (src/kernels/scatter_nd.cu:44-47).
    fp32, fp16, int32 and fp64 tables; arguments as scatter_nd.
    """
    if data.dtype not in _SCATTER_ADD_TYPES:
        raise TypeError(f"scatter_nd_add supports {sorted(str(t) for t in _SCATTER_ADD_TYPES)}, got {data.dtype}")
    dims, n, k = _scatter_args(data, indices, updates)
    lib = _lib.load()
    with _on(data.device):
        _lib.check(
            "tc_scatter_nd_add",
            lib.tc_scatter_nd_add(_ptr(data), _ptr(updates), _ptr(indices), int(indices.dtype == torch.int64), dims,
                                  data.dim(), n, k, _SCATTER_ADD_TYPES[data.dtype], _stream()),
        )
