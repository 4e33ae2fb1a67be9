"""Host-side drivers over the C ABI, operating on torch CUDA tensors.

These mirror what the reference's host programs do around their kernels
(rocWMMA samples/simple_hgemm.cpp:141-290 `gemm_test`, samples/perf_hgemm.cpp:716-944,
samples/simple_sgemv.cpp:157-270, samples/simple_dlrm.cpp:443-700): pick leading
dimensions, launch, hand back the result.  PyTorch is used for device memory
and streams only; every computation happens in this library's own kernels.

Storage conventions: fp16 -> torch.float16, bf16 -> torch.bfloat16,
e4m3 -> torch.uint8 (raw bits) or torch.float8_e4m3fn, i8 -> torch.int8,
f32/xf32 -> torch.float32, f64 -> torch.float64, i32 -> torch.int32.
Matrices are passed as flat (or 2-D contiguous) storage in the stated layout.
"""
from __future__ import annotations

import torch

from . import _lib as L
from ._lib import (BF16, COL_MAJOR, E4M3, E5M2, F16, F32, F64, I8, I32, MXF4, NVF4,  # noqa: F401
                   ROW_MAJOR, XF32, B200WmmaError)

_TORCH = {F16: torch.float16, BF16: torch.bfloat16, E4M3: torch.uint8, I8: torch.int8,
          F32: torch.float32, XF32: torch.float32, F64: torch.float64, I32: torch.int32,
          E5M2: torch.uint8}


def torch_dtype(code: int):
    return _TORCH[code]


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(stream=None):
    s = stream if stream is not None else torch.cuda.current_stream()
    return s.cuda_stream


def _require_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("device tensors required (this library has no CPU path)")


def _natural_ld(layout, rows, cols):
    return cols if layout == ROW_MAJOR else rows


def gemm_simple(in_t, out_t, m, n, k, a, b, c, alpha, beta, layout_a=ROW_MAJOR,
                layout_b=COL_MAJOR, layout_cd=ROW_MAJOR, block=16, lda=None, ldb=None, ldc=None,
                ldd=None, out=None, stream=None, compute=None, block_k=0):
    """D = alpha*A*B + beta*C, one fragment tile per warp (the simple_*gemm samples).
    compute: rocWMMA's ComputeT as a dtype code (None = the usual one for the input type);
    block_k: K extent of the fragments (0 = the usual one)."""
    _require_cuda(a, b, c)
    lda = lda or _natural_ld(layout_a, m, k)
    ldb = ldb or _natural_ld(layout_b, k, n)
    ldc = ldc or _natural_ld(layout_cd, m, n)
    ldd = ldd or _natural_ld(layout_cd, m, n)
    d = out if out is not None else torch.empty(
        (m if layout_cd == ROW_MAJOR else n) * ldd, dtype=_TORCH[out_t], device=a.device)
    if compute is None and block_k == 0:
        rc = L.lib().b200wmma_gemm_simple(in_t, out_t, m, n, k, _ptr(a), _ptr(b), _ptr(c), _ptr(d),
                                          lda, ldb, ldc, ldd, float(alpha), float(beta), layout_a,
                                          layout_b, layout_cd, block, _stream(stream))
    else:
        rc = L.lib().b200wmma_gemm_simple_ex(in_t, out_t, -1 if compute is None else compute, m, n,
                                             k, _ptr(a), _ptr(b), _ptr(c), _ptr(d), lda, ldb, ldc,
                                             ldd, float(alpha), float(beta), layout_a, layout_b,
                                             layout_cd, block, block_k, _stream(stream))
    L.check(rc, "b200wmma_gemm_simple")
    return d


def gemm(in_t, out_t, m, n, k, a, b, c, alpha, beta, layout_a=ROW_MAJOR, layout_b=COL_MAJOR,
         lda=None, ldb=None, ldc=None, ldd=None, out=None, stream=None):
    """D = alpha*A*B + beta*C through the block-cooperative tensor-core path; C/D row-major."""
    _require_cuda(a, b, c)
    lda = lda or _natural_ld(layout_a, m, k)
    ldb = ldb or _natural_ld(layout_b, k, n)
    ldc = ldc or n
    ldd = ldd or n
    d = out if out is not None else torch.empty(m * ldd, dtype=_TORCH[out_t], device=a.device)
    rc = L.lib().b200wmma_gemm(in_t, out_t, m, n, k, _ptr(a), _ptr(b), _ptr(c), _ptr(d), lda, ldb,
                               ldc, ldd, float(alpha), float(beta), layout_a, layout_b,
                               _stream(stream))
    L.check(rc, "b200wmma_gemm")
    return d


def gemm_noalloc(in_t, out_t, m, n, k, a, b, c, alpha, beta, layout_a=ROW_MAJOR,
                 layout_b=COL_MAJOR, lda=None, ldb=None, ldc=None, ldd=None, out=None,
                 stream=None):
    """gemm() through the entry point that never allocates device memory: the scratch for
    transposed operand layouts is a fixed 8 MiB array inside the library.  `out` must be
    given by callers that cannot allocate; problems whose transposed operands exceed the
    array raise B200WmmaError (status -6).  Calls on one device must not overlap."""
    _require_cuda(a, b, c)
    lda = lda or _natural_ld(layout_a, m, k)
    ldb = ldb or _natural_ld(layout_b, k, n)
    ldc = ldc or n
    ldd = ldd or n
    d = out if out is not None else torch.empty(m * ldd, dtype=_TORCH[out_t], device=a.device)
    rc = L.lib().b200wmma_gemm_noalloc(in_t, out_t, m, n, k, _ptr(a), _ptr(b), _ptr(c), _ptr(d),
                                       lda, ldb, ldc, ldd, float(alpha), float(beta), layout_a,
                                       layout_b, _stream(stream))
    L.check(rc, "b200wmma_gemm_noalloc")
    return d


def gemm_host(in_t, out_t, m, n, k, a, b, c, d, alpha, beta, layout_a=ROW_MAJOR,
              layout_b=COL_MAJOR, stream=None):
    """Same with HOST tensors (ideally pinned): copies in, computes, copies D back, waits."""
    for t in (a, b, c, d):
        if t is not None and t.is_cuda:
            raise ValueError("gemm_host takes host tensors")
    lda = _natural_ld(layout_a, m, k)
    ldb = _natural_ld(layout_b, k, n)
    rc = L.lib().b200wmma_gemm_host(in_t, out_t, m, n, k, _ptr(a), _ptr(b), _ptr(c), _ptr(d), lda,
                                    ldb, n, n, float(alpha), float(beta), layout_a, layout_b,
                                    _stream(stream))
    L.check(rc, "b200wmma_gemm_host")
    return d


def gemv(dtype, m, k, a, x, y, alpha, beta, lda=None, out=None, stream=None):
    """y_out = alpha*A*x + beta*y, A column-major (lda >= m)."""
    _require_cuda(a, x, y)
    out = out if out is not None else torch.empty_like(y)
    rc = L.lib().b200wmma_gemv(dtype, m, k, _ptr(a), _ptr(x), _ptr(y), _ptr(out), float(alpha),
                               float(beta), lda or m, _stream(stream))
    L.check(rc, "b200wmma_gemv")
    return out


def dlrm_fwd(x, m, k, batch, out=None, stream=None, dtype=F16):
    """[batch][m][k] -> [batch][k + m(m-1)/2]: row 0, then tril(X X^T, -1) row-major."""
    _require_cuda(x)
    out = out if out is not None else torch.empty(batch * (k + m * (m - 1) // 2),
                                                  dtype=_TORCH[dtype], device=x.device)
    rc = L.lib().b200wmma_dlrm_fwd(dtype, _ptr(x), _ptr(out), m, k, batch, _stream(stream))
    L.check(rc, "b200wmma_dlrm_fwd")
    return out


def dlrm_bwd(x, upstream, m, k, batch, grad=None, mlp_grad=None, stream=None, dtype=F16):
    """Returns (mlp_grad [batch][k], grad [batch][m][k])."""
    _require_cuda(x, upstream)
    grad = grad if grad is not None else torch.empty(batch * m * k, dtype=_TORCH[dtype],
                                                     device=x.device)
    mlp_grad = mlp_grad if mlp_grad is not None else torch.empty(batch * k, dtype=_TORCH[dtype],
                                                                 device=x.device)
    rc = L.lib().b200wmma_dlrm_bwd(dtype, _ptr(x), _ptr(upstream), _ptr(grad), _ptr(mlp_grad), m, k,
                                   batch, _stream(stream))
    L.check(rc, "b200wmma_dlrm_bwd")
    return mlp_grad, grad


def check_device(stream=None) -> None:
    """Waits for the stream; raises if a kernel gave up on a bounded device-side wait."""
    import ctypes as C
    detail = C.c_uint32(0)
    rc = L.lib().b200wmma_check_device(_stream(stream), C.byref(detail))
    if rc != L.OK:
        raise B200WmmaError(rc, f"b200wmma_check_device (wait code {detail.value})")


def shutdown() -> None:
    L.check(L.lib().b200wmma_shutdown(), "b200wmma_shutdown")


# ---- 4-bit block-scaled operands ------------------------------------------------------------
# An operand is a pair (codes, scales) of uint8 tensors, as the C header lays them out.

def _device_of(first, *others):
    """Index of the one device that the given tensors are on."""
    index = first.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            raise ValueError("tensors on several devices, or not on a device at all")
    if index < 0:
        raise ValueError("device tensors required (this library has no CPU path)")
    return index


def _launch(entry, index, stream, *args):
    """Calls the entry point with `stream`, or the current stream of the tensors' device, which
    need not be the current one.  (The raw handle: making a torch.cuda.Stream of the current
    stream takes 3 us, as long as the launch.)"""
    if stream is None:
        handle = torch._C._cuda_getCurrentRawStream(index)
    elif stream.device.index != index:
        raise ValueError(f"a stream of device {stream.device.index} for tensors on device {index}")
    else:
        handle = stream.cuda_stream
    if torch.cuda.current_device() == index:
        rc = getattr(L.lib(), entry)(*args, handle)
    else:
        with torch.cuda.device(index):
            rc = getattr(L.lib(), entry)(*args, handle)
    if rc:
        L.check(rc, entry)


def _empty(shape, dtype, device, stream):
    """A new tensor whose memory `stream` (None: the current stream) may use at once."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=device)


def _check(t, what, dtype, count):
    """A contiguous tensor of the type that holds what a call reads or writes of it."""
    if t.dtype != dtype:
        raise ValueError(f"{what}: {t.dtype}, expected {dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{what}: must be contiguous")
    if t.numel() < count:
        raise ValueError(f"{what}: {t.numel()} elements, {count} needed")


def mx_pitch(k):
    """Bytes of one row of codes."""
    return (k + 31) // 32 * 16


_GROUP = {MXF4: 128, NVF4: 64}  # values along k of one scale tile


def mx_scale_bytes(fmt, rows, k):
    """Bytes of the scales of a rows x k operand."""
    span = _GROUP.get(fmt)
    return (rows + 127) // 128 * ((k + span - 1) // span) * 512 if span else 0


def _operand(fmt, rows, k, codes, scales, ld):
    _check(codes, "codes", torch.uint8, (rows - 1) * ld + (k + 31) // 32 * 16)
    _check(scales, "scales", torch.uint8, mx_scale_bytes(fmt, rows, k))


def mx_quantize(fmt, in_t, rows, k, x, layout=ROW_MAJOR, exponent=0, ldx=None, ldq=None, out=None,
                stream=None):
    """Quantises rows x k values to MXF4 or NVF4; returns (codes, scales).
    layout: how x is stored (its k values contiguous, or its rows); ldx in elements, ldq in bytes."""
    ldx = ldx or _natural_ld(layout, rows, k)
    ldq = ldq or mx_pitch(k)
    if out is None:
        out = (_empty(rows * ldq, torch.uint8, x.device, stream),
               _empty(mx_scale_bytes(fmt, rows, k), torch.uint8, x.device, stream))
    device = _device_of(x, *out)
    _check(x, "x", _TORCH.get(in_t), (rows - 1) * ldx + k if layout == ROW_MAJOR else (k - 1) * ldx + rows)
    _operand(fmt, rows, k, *out, ldq)
    _launch("b200wmma_mx_quantize", device, stream, fmt, in_t, rows, k, x.data_ptr(), ldx, layout,
            exponent, out[0].data_ptr(), ldq, out[1].data_ptr())
    return out


def mx_dequantize(fmt, out_t, rows, k, codes, scales, exponent=0, ldq=None, ldo=None, out=None,
                  stream=None):
    """The values an operand stands for, times 2^exponent; row-major."""
    ldq = ldq or mx_pitch(k)
    ldo = ldo or k
    if out is None:
        out = _empty(rows * ldo, _TORCH.get(out_t), codes.device, stream)
    device = _device_of(codes, scales, out)
    _check(out, "out", _TORCH.get(out_t), (rows - 1) * ldo + k)
    _operand(fmt, rows, k, codes, scales, ldq)
    _launch("b200wmma_mx_dequantize", device, stream, fmt, out_t, rows, k, codes.data_ptr(), ldq,
            scales.data_ptr(), exponent, out.data_ptr(), ldo)
    return out


def mx_gemm(fmt, out_t, m, n, k, a, b, c, alpha, beta, lda=None, ldb=None, ldc=None, ldd=None,
            out=None, stream=None):
    """D = alpha*A*B + beta*C on 4-bit block-scaled operands: a = (codes, scales) of m rows x k,
    b of n rows x k (column-major B); C/D row-major.  lda, ldb in bytes."""
    lda = lda or mx_pitch(k)
    ldb = ldb or mx_pitch(k)
    ldc = ldc or n
    ldd = ldd or n
    d = out if out is not None else _empty(m * ldd, _TORCH.get(out_t), a[0].device, stream)
    device = _device_of(*a, *b, c, d)
    _operand(fmt, m, k, *a, lda)
    _operand(fmt, n, k, *b, ldb)
    _check(d, "out", _TORCH.get(out_t), (m - 1) * ldd + n)
    if c is not None and beta != 0:
        _check(c, "c", _TORCH.get(out_t), (m - 1) * ldc + n)
    _launch("b200wmma_mx_gemm", device, stream, fmt, out_t, m, n, k, a[0].data_ptr(), a[1].data_ptr(),
            b[0].data_ptr(), b[1].data_ptr(), _ptr(c), d.data_ptr(), lda, ldb, ldc, ldd, alpha, beta)
    return d


# ---- embedding --------------------------------------------------------------------------------

_CODE = {torch.float16: F16, torch.bfloat16: BF16, torch.float32: F32}


def _value_code(t, what):
    code = _CODE.get(t.dtype)
    if code is None:
        raise ValueError(f"{what} is {t.dtype}; float16, bfloat16 or float32 expected")
    return code


def _tokens(ids, first):
    """(outer, inner, id bytes, outer stride, inner stride) of ids; outer x inner tokens."""
    if ids.dtype == torch.int64:
        size = 8
    elif ids.dtype == torch.int32:
        size = 4
    else:
        raise ValueError(f"ids are {ids.dtype}; int32 or int64 expected")
    dims = ids.dim()
    if first is not None:
        if dims != 2 or first.dtype != torch.int64 or not first.is_contiguous() \
                or first.shape != (ids.shape[1] + 1,):
            raise ValueError("with first, ids are [outer, inner] and first inner + 1 int64 row numbers")
    elif dims == 1:
        return ids.shape[0], 1, size, ids.stride(0), 0
    elif dims != 2:
        if not ids.is_contiguous():
            raise ValueError("ids of this shape must be contiguous")
        return ids.numel(), 1, size, 1, 0
    return (*ids.shape, size, *ids.stride())


def _rows_of(t, ids_shape, dim, what):
    """Distances of t's rows along outer and inner, for t [*ids.shape, dim] with contiguous rows."""
    if t.shape != (*ids_shape, dim):
        raise ValueError(f"{what} is {tuple(t.shape)}, expected {(*ids_shape, dim)}")
    strides = t.stride()
    if dim > 1 and strides[-1] != 1:
        raise ValueError(f"the rows of {what} must be contiguous")
    if len(strides) == 3:
        return strides[:2]
    if len(strides) == 2:
        return strides[0], 0
    if not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous for ids of this shape")
    return dim, 0


def embedding(table, ids, scale=1.0, first=None, out_t=None, out=None, stream=None):
    """out[t, :] = scale * table[ids[t], :] for a table [rows, dim] (rows contiguous, any distance
    apart) and int32 / int64 ids of any shape; ids outside the table (-1: padding) give zeros.
    first: int64 [inner + 1] on the device; ids are [outer, inner], column i counts from row
    first[i] up to first[i + 1].  out: [*ids.shape, dim], may be a strided view such as the
    rows behind the dense one of dlrm_fwd's input; out_t: its type otherwise (the table's)."""
    rows, dim = table.shape
    ldt, step = table.stride()
    if dim > 1 and step != 1:
        raise ValueError("the rows of table must be contiguous")
    shape = ids.shape
    if out is None:
        out = _empty((*shape, dim), table.dtype if out_t is None else _TORCH.get(out_t), table.device,
                     stream)
    device = _device_of(table, ids, first, out)
    outer, inner, size, ids_outer, ids_inner = _tokens(ids, first)
    out_outer, out_inner = _rows_of(out, shape, dim, "out")
    if (not out_outer and outer > 1) or (not out_inner and inner > 1):
        raise ValueError("out must not hold a row twice")
    kinds = _value_code(table, "table"), _value_code(out, "out")
    if outer and inner:
        _launch("b200wmma_embedding", device, stream, *kinds, rows, dim, outer, inner, table.data_ptr(),
                ldt if rows > 1 else dim, ids.data_ptr(), size, ids_outer, ids_inner, _ptr(first),
                out.data_ptr(), out_outer, out_inner, scale)
    return out


def embedding_grad(grad, ids, rows, out_t=None, scale=1.0, first=None, out=None, accumulate=False,
                   workspace=None, stream=None):
    """Gradient [rows, dim] of embedding()'s table from grad [*ids.shape, dim] (strided like its
    out).  accumulate: add to `out`, whose rows without a token stay as they are; otherwise those
    become zero.  out_t: type of a new result (grad's).  workspace: a uint8 tensor of
    embedding_grad_workspace(...) bytes to use instead of a new one."""
    dim = grad.shape[-1]
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out")
        out = _empty((rows, dim), grad.dtype if out_t is None else _TORCH.get(out_t), grad.device, stream)
    ldt, step = out.stride()
    if out.shape != (rows, dim) or (dim > 1 and step != 1):
        raise ValueError(f"out must be {(rows, dim)} with contiguous rows")
    device = _device_of(grad, ids, first, out, workspace)
    outer, inner, size, ids_outer, ids_inner = _tokens(ids, first)
    grad_outer, grad_inner = _rows_of(grad, ids.shape, dim, "grad")
    kinds = _value_code(grad, "grad"), _value_code(out, "out")
    if not (outer and inner):
        if not accumulate:
            with torch.cuda.stream(stream):
                out.zero_()
        return out
    if workspace is None:
        workspace = _empty(L.lib().b200wmma_embedding_grad_workspace(rows, dim, outer, inner),
                           torch.uint8, grad.device, stream)
    elif workspace.dtype != torch.uint8 or not workspace.is_contiguous():
        raise ValueError("workspace must be a contiguous uint8 tensor")
    _launch("b200wmma_embedding_grad", device, stream, *kinds, rows, dim, outer, inner, grad.data_ptr(),
            grad_outer, grad_inner, ids.data_ptr(), size, ids_outer, ids_inner, _ptr(first),
            out.data_ptr(), ldt if rows > 1 else dim, scale, accumulate, workspace.data_ptr(),
            workspace.numel())
    return out


def embedding_grad_workspace(rows, dim, outer, inner=1):
    """Bytes of device memory that embedding_grad works in for outer x inner tokens."""
    return L.lib().b200wmma_embedding_grad_workspace(rows, dim, outer, inner)
