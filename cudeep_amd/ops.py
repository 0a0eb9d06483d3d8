"""Thin tensor-level wrappers over the C-ABI, for callers that hold
PyTorch-ROCm device tensors (tests, bench, the host layer).  PyTorch only
supplies device memory and the current stream; all arithmetic happens in
libcudeep_amd.so.  Every wrapper validates shapes / dtypes / devices on the
host before any launch, so a bad call raises instead of faulting.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib as L


# The current stream of the current device as an integer.  Asked for directly:
# torch.cuda.current_stream() builds a Stream object through several Python
# layers, 2.9 us of an 8 to 13 us call, against 0.2.
_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else None
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream() -> int:
    if _current_device is None or _raw_stream is None:
        return ctypes_stream(torch.cuda.current_stream())
    return _raw_stream(_current_device())


def ctypes_stream(s) -> int:
    return int(s.cuda_stream)


def _need(t: torch.Tensor, name: str, dtype=torch.float32):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")


def _ld(t: torch.Tensor, name: str) -> int:
    """Leading dimension of a row-major 2-D view (unit column stride)."""
    if t.dim() != 2:
        raise ValueError(f"{name} must be 2-D")
    ld, step = t.stride()
    cols = t.shape[1]
    if step != 1 and cols > 1:
        raise ValueError(f"{name} must have unit column stride")
    return ld if ld >= cols and ld >= 1 else max(cols, 1)


def _scratch(workspace, nbytes, device):
    """(pointer, bytes, keep-alive) of a call's scratch: the caller's
    `workspace`, else a block of torch's stream-ordered caching allocator
    sized by the library's query (no block when the call needs none; a block
    freed here is reused only by work queued after this call on the same
    stream).  Passing scratch in keeps the library off its own
    stream-ordered pool, whose allocate / free pair costs ~5 us between the
    kernels of back-to-back calls."""
    if workspace is not None:
        return workspace.data_ptr(), workspace.numel() * workspace.element_size(), workspace
    n = int(nbytes())
    if n <= 0:
        return None, 0, None
    t = torch.empty(n, dtype=torch.uint8, device=device)
    return t.data_ptr(), n, t


def gemm(A: torch.Tensor, B: torch.Tensor, *, precision: int = L.PREC_FP32,
         transA: bool = False, transB: bool = False, bias: torch.Tensor | None = None,
         bias_mode: int = L.BIAS_NONE, epilogue: int = L.EPI_NONE,
         out: torch.Tensor | None = None,
         workspace: torch.Tensor | None = None, aux: torch.Tensor | None = None,
         colsum: torch.Tensor | None = None) -> torch.Tensor:
    """C = epi(op(A) @ op(B) + bias).  A, B are row-major storage; transA /
    transB select the transpose, so x @ W.T is gemm(x, W, transB=True).
    `workspace` (at least gemm_workspace_bytes(...) bytes) makes the call
    allocation-free (cdx_gemm_ex_ws).  Fusions (cdx_gemm_fused): with an
    EPI_BWD_* epilogue, C = (op(A) @ op(B)) * act'(aux) (aux [M, N]); with
    `colsum` (a float32 [M] tensor), colsum[m] = sum_k op(A)[m, k] in the
    same launch (size the workspace with colsum=True)."""
    _need(A, "A")
    _need(B, "B")
    M, K = (A.shape[1], A.shape[0]) if transA else (A.shape[0], A.shape[1])
    K2, N = (B.shape[1], B.shape[0]) if transB else (B.shape[0], B.shape[1])
    if K != K2:
        raise ValueError(f"inner dimensions differ: {K} vs {K2}")
    if out is None:
        out = torch.empty((M, N), device=A.device, dtype=torch.float32)
    _need(out, "out")
    if tuple(out.shape) != (M, N):
        raise ValueError("out has the wrong shape")
    bptr = None
    if bias_mode != L.BIAS_NONE:
        if bias is None:
            raise ValueError("bias_mode set but bias is None")
        _need(bias, "bias")
        want = M if bias_mode == L.BIAS_ROW else N
        if bias.numel() != want or not bias.is_contiguous():
            raise ValueError("bias has the wrong size or is not contiguous")
        bptr = bias.data_ptr()
    if workspace is not None:
        _need(workspace, "workspace")
    ws_ptr, ws_bytes, _keep = _scratch(
        workspace, lambda: gemm_workspace_bytes(M, N, K, precision=precision, transA=transA,
                                                transB=transB, colsum=colsum is not None),
        A.device)
    if aux is None and colsum is None:
        L.call("cdx_gemm_ex_ws", precision, int(transA), int(transB), M, N, K,
               A.data_ptr(), _ld(A, "A"), B.data_ptr(), _ld(B, "B"),
               out.data_ptr(), _ld(out, "out"), bptr, bias_mode, epilogue, ws_ptr, ws_bytes,
               _stream())
        return out
    aux_ptr, ldaux = None, 0
    if aux is not None:
        _need(aux, "aux")
        if tuple(aux.shape) != (M, N):
            raise ValueError("aux must be [M, N]")
        aux_ptr, ldaux = aux.data_ptr(), _ld(aux, "aux")
    cs_ptr = None
    if colsum is not None:
        _need(colsum, "colsum")
        if colsum.numel() != M or not colsum.is_contiguous():
            raise ValueError("colsum must be a contiguous [M] tensor")
        cs_ptr = colsum.data_ptr()
    L.call("cdx_gemm_fused", precision, int(transA), int(transB), M, N, K,
           A.data_ptr(), _ld(A, "A"), B.data_ptr(), _ld(B, "B"),
           out.data_ptr(), _ld(out, "out"), bptr, bias_mode, epilogue, aux_ptr, ldaux, cs_ptr,
           ws_ptr, ws_bytes, _stream())
    return out


def gemm_workspace_bytes(M: int, N: int, K: int, *, precision: int = L.PREC_FP32,
                         transA: bool = False, transB: bool = False,
                         colsum: bool = False) -> int:
    """Scratch bytes gemm(..., workspace=) needs for op(A) [M, K] @ op(B) [K, N]
    (with colsum=True: for a call that also forms the row sums of op(A))."""
    if colsum:
        return int(L.lib().cdx_gemm_fused_workspace_size(precision, int(transA), int(transB),
                                                         M, N, K, 1))
    return int(L.lib().cdx_gemm_workspace_size(precision, int(transA), int(transB), M, N, K))


def gemm16(A: torch.Tensor, B: torch.Tensor, *, transA: bool = False, transB: bool = False,
           bias: torch.Tensor | None = None, bias_mode: int = L.BIAS_NONE,
           epilogue: int = L.EPI_NONE, out: torch.Tensor | None = None) -> torch.Tensor:
    """C = epi(op(A) @ op(B) + bias) for float16 or bfloat16 A, B (both the
    same type), fp32 accumulation and fp32 C (cdx_gemm16_ex)."""
    if not isinstance(A, torch.Tensor) or A.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("A must be a float16 or bfloat16 tensor")
    _need(A, "A", A.dtype)
    _need(B, "B", A.dtype)
    dt = L.DTYPE_F16 if A.dtype == torch.float16 else L.DTYPE_BF16
    M, K = (A.shape[1], A.shape[0]) if transA else (A.shape[0], A.shape[1])
    K2, N = (B.shape[1], B.shape[0]) if transB else (B.shape[0], B.shape[1])
    if K != K2:
        raise ValueError(f"inner dimensions differ: {K} vs {K2}")
    if out is None:
        out = torch.empty((M, N), device=A.device, dtype=torch.float32)
    _need(out, "out")
    if tuple(out.shape) != (M, N):
        raise ValueError("out has the wrong shape")
    bptr = None
    if bias_mode != L.BIAS_NONE:
        if bias is None:
            raise ValueError("bias_mode set but bias is None")
        _need(bias, "bias")
        want = M if bias_mode == L.BIAS_ROW else N
        if bias.numel() != want or not bias.is_contiguous():
            raise ValueError("bias has the wrong size or is not contiguous")
        bptr = bias.data_ptr()
    L.call("cdx_gemm16_ex", dt, int(transA), int(transB), M, N, K,
           A.data_ptr(), _ld(A, "A"), B.data_ptr(), _ld(B, "B"),
           out.data_ptr(), _ld(out, "out"), bptr, bias_mode, epilogue, _stream())
    return out


def hgemm(A, B, out=None):
    """C = A @ B for contiguous float16 A, B, fp32 C (cdx_hgemm_f16)."""
    _need(A, "A", torch.float16)
    _need(B, "B", torch.float16)
    if A.dim() != 2 or B.dim() != 2 or A.shape[1] != B.shape[0]:
        raise ValueError("hgemm: shape mismatch")
    if not (A.is_contiguous() and B.is_contiguous()):
        raise ValueError("hgemm: operands must be contiguous")
    M, K = A.shape
    N = B.shape[1]
    if out is None:
        out = torch.empty((M, N), device=A.device, dtype=torch.float32)
    _need(out, "out")
    L.call("cdx_hgemm_f16", A.data_ptr(), B.data_ptr(), out.data_ptr(), M, N, K, _stream())
    return out


def sgemm(A, B, out=None):
    """C = A @ B, FP32 products (cdx_sgemm_f32); A, B contiguous row-major."""
    _need(A, "A")
    _need(B, "B")
    if A.dim() != 2 or B.dim() != 2 or A.shape[1] != B.shape[0]:
        raise ValueError("sgemm: shape mismatch")
    if not (A.is_contiguous() and B.is_contiguous()):
        raise ValueError("sgemm: operands must be contiguous")
    M, K = A.shape
    N = B.shape[1]
    if out is None:
        out = torch.empty((M, N), device=A.device, dtype=torch.float32)
    L.call("cdx_sgemm_f32", A.data_ptr(), B.data_ptr(), out.data_ptr(), M, N, K, _stream())
    return out


def gemm_tf32mode(A, B, out=None):
    """C = A @ B in TF32 mode (bf16x3 split MFMA, cdx_gemm_tf32mode)."""
    _need(A, "A")
    _need(B, "B")
    if A.dim() != 2 or B.dim() != 2 or A.shape[1] != B.shape[0]:
        raise ValueError("gemm_tf32mode: shape mismatch")
    if not (A.is_contiguous() and B.is_contiguous()):
        raise ValueError("gemm_tf32mode: operands must be contiguous")
    M, K = A.shape
    N = B.shape[1]
    if out is None:
        out = torch.empty((M, N), device=A.device, dtype=torch.float32)
    L.call("cdx_gemm_tf32mode", A.data_ptr(), B.data_ptr(), out.data_ptr(), M, N, K, _stream())
    return out


def dgemm(A, B, transA=False, transB=False, out=None):
    _need(A, "A", torch.float64)
    _need(B, "B", torch.float64)
    M, K = (A.shape[1], A.shape[0]) if transA else (A.shape[0], A.shape[1])
    K2, N = (B.shape[1], B.shape[0]) if transB else (B.shape[0], B.shape[1])
    if K != K2:
        raise ValueError("dgemm: inner dimensions differ")
    if out is None:
        out = torch.empty((M, N), device=A.device, dtype=torch.float64)
    L.call("cdx_dgemm", int(transA), int(transB), M, N, K, A.data_ptr(), _ld(A, "A"),
           B.data_ptr(), _ld(B, "B"), out.data_ptr(), _ld(out, "out"), _stream())
    return out


def conv_out_size(i, k, s, p):
    return (i + 2 * p - k) // s + 1


def im2col(x, KH, KW, stride=(1, 1), padding=(0, 0), out=None):
    _need(x, "input")
    if x.dim() != 4 or not x.is_contiguous():
        raise ValueError("im2col: input must be contiguous NCHW")
    Bn, C, H, W = x.shape
    OH = conv_out_size(H, KH, stride[0], padding[0])
    OW = conv_out_size(W, KW, stride[1], padding[1])
    if OH <= 0 or OW <= 0:
        raise ValueError("im2col: kernel larger than padded input")
    shape = (C * KH * KW, Bn * OH * OW)
    if out is None:
        out = torch.empty(shape, device=x.device, dtype=torch.float32)
    if tuple(out.shape) != shape or not out.is_contiguous():
        raise ValueError("im2col: bad output buffer")
    L.call("cdx_im2col_f32", x.data_ptr(), out.data_ptr(), Bn, C, H, W, KH, KW,
           stride[0], stride[1], padding[0], padding[1], _stream())
    return out


def conv2d_forward(x, w, bias=None, stride=(1, 1), padding=(0, 0),
                   precision=L.PREC_FP32, workspace=None, out=None):
    _need(x, "input")
    _need(w, "weight")
    if x.dim() != 4 or w.dim() != 4 or not x.is_contiguous() or not w.is_contiguous():
        raise ValueError("conv2d: input / weight must be contiguous NCHW / OIHW")
    Bn, C, H, W = x.shape
    OC, C2, KH, KW = w.shape
    if C != C2:
        raise ValueError("conv2d: channel mismatch")
    OH = conv_out_size(H, KH, stride[0], padding[0])
    OW = conv_out_size(W, KW, stride[1], padding[1])
    if OH <= 0 or OW <= 0:
        raise ValueError("conv2d: kernel larger than padded input")
    if bias is not None:
        _need(bias, "bias")
        if bias.numel() != OC or not bias.is_contiguous():
            raise ValueError("conv2d: bias must have out_channels elements")
    if out is None:
        out = torch.empty((Bn, OC, OH, OW), device=x.device, dtype=torch.float32)
    ws_ptr, ws_bytes, _keep = _scratch(
        workspace, lambda: conv2d_workspace_bytes(x.shape, w.shape, stride, padding), x.device)
    L.call("cdx_conv2d_forward_f32", x.data_ptr(), w.data_ptr(),
           None if bias is None else bias.data_ptr(), out.data_ptr(), Bn, C, OC, H, W, KH, KW,
           stride[0], stride[1], padding[0], padding[1], precision, ws_ptr, ws_bytes, _stream())
    return out


def conv2d_implicit(x, w, bias=None, stride=(1, 1), padding=(0, 0), out=None):
    """NCHW convolution as an implicit GEMM, no column buffer
    (cdx_conv2d_forward_implicit_f32; FP32 products)."""
    _need(x, "input")
    _need(w, "weight")
    if x.dim() != 4 or w.dim() != 4 or not x.is_contiguous() or not w.is_contiguous():
        raise ValueError("conv2d_implicit: input / weight must be contiguous NCHW / OIHW")
    Bn, C, H, W = x.shape
    OC, C2, KH, KW = w.shape
    if C != C2:
        raise ValueError("conv2d_implicit: channel mismatch")
    OH = conv_out_size(H, KH, stride[0], padding[0])
    OW = conv_out_size(W, KW, stride[1], padding[1])
    if OH <= 0 or OW <= 0:
        raise ValueError("conv2d_implicit: kernel larger than padded input")
    if bias is not None:
        _need(bias, "bias")
        if bias.numel() != OC or not bias.is_contiguous():
            raise ValueError("conv2d_implicit: bias must have out_channels elements")
    if out is None:
        out = torch.empty((Bn, OC, OH, OW), device=x.device, dtype=torch.float32)
    L.call("cdx_conv2d_forward_implicit_f32", x.data_ptr(), w.data_ptr(),
           None if bias is None else bias.data_ptr(), out.data_ptr(), Bn, C, OC, H, W, KH, KW,
           stride[0], stride[1], padding[0], padding[1], _stream())
    return out


def conv2d_winograd(x, w, bias=None, padding=(0, 0), precision=L.PREC_FP32, workspace=None,
                    out=None):
    """3x3 stride-1 NCHW convolution by Winograd F(4x4, 3x3)
    (cdx_conv2d_forward_winograd_f32)."""
    _need(x, "input")
    _need(w, "weight")
    if x.dim() != 4 or w.dim() != 4 or not x.is_contiguous() or not w.is_contiguous():
        raise ValueError("conv2d_winograd: input / weight must be contiguous NCHW / OIHW")
    Bn, C, H, W = x.shape
    OC, C2, KH, KW = w.shape
    if C != C2 or KH != 3 or KW != 3:
        raise ValueError("conv2d_winograd: needs a 3x3 kernel and matching channels")
    OH, OW = H + 2 * padding[0] - 2, W + 2 * padding[1] - 2
    if OH <= 0 or OW <= 0:
        raise ValueError("conv2d_winograd: kernel larger than padded input")
    if bias is not None:
        _need(bias, "bias")
        if bias.numel() != OC or not bias.is_contiguous():
            raise ValueError("conv2d_winograd: bias must have out_channels elements")
    if out is None:
        out = torch.empty((Bn, OC, OH, OW), device=x.device, dtype=torch.float32)
    ws_ptr, ws_bytes, _keep = _scratch(
        workspace, lambda: conv2d_winograd_workspace_bytes(x.shape, OC, padding), x.device)
    L.call("cdx_conv2d_forward_winograd_f32", x.data_ptr(), w.data_ptr(),
           None if bias is None else bias.data_ptr(), out.data_ptr(), Bn, C, OC, H, W,
           padding[0], padding[1], precision, ws_ptr, ws_bytes, _stream())
    return out


def conv2d_winograd_workspace_bytes(x_shape, out_channels, padding=(0, 0)) -> int:
    Bn, C, H, W = x_shape
    return int(L.lib().cdx_conv2d_winograd_workspace_size(Bn, C, out_channels, H, W,
                                                          padding[0], padding[1]))


def conv2d_workspace_bytes(x_shape, w_shape, stride=(1, 1), padding=(0, 0)) -> int:
    Bn, C, H, W = x_shape
    _, _, KH, KW = w_shape
    return int(L.lib().cdx_conv2d_forward_workspace_size(
        Bn, C, H, W, KH, KW, stride[0], stride[1], padding[0], padding[1]))


def sum_reduce_rows(x, out=None, workspace=None):
    """Column sums of a contiguous 2-D tensor; `workspace` (at least
    sum_reduce_rows_workspace_bytes(rows, cols)) makes the call allocation-free."""
    _need(x, "input")
    if x.dim() != 2 or not x.is_contiguous():
        raise ValueError("sum_reduce_rows: input must be contiguous 2-D")
    rows, cols = x.shape
    if out is None:
        out = torch.empty((cols,), device=x.device, dtype=torch.float32)
    if workspace is not None:
        _need(workspace, "workspace")
    ws_ptr, ws_bytes, _keep = _scratch(
        workspace, lambda: sum_reduce_rows_workspace_bytes(rows, cols), x.device)
    L.call("cdx_sum_reduce_rows_f32", x.data_ptr(), out.data_ptr(), rows, cols, ws_ptr, ws_bytes,
           _stream())
    return out


def sum_reduce_rows_workspace_bytes(rows: int, cols: int) -> int:
    return int(L.lib().cdx_sum_reduce_rows_workspace_size(rows, cols))


def broadcast_add_row(m, row, out=None):
    _need(m, "matrix")
    _need(row, "row")
    if m.dim() != 2 or not m.is_contiguous() or row.numel() != m.shape[1]:
        raise ValueError("broadcast_add: shape mismatch")
    if out is None:
        out = torch.empty_like(m)
    L.call("cdx_broadcast_add_row_f32", m.data_ptr(), row.contiguous().data_ptr(),
           out.data_ptr(), m.shape[0], m.shape[1], _stream())
    return out


def activation(x, act, out=None, alpha=0.01):
    """act(x) elementwise; act is EPI_RELU / _GELU / _SILU / _SIGMOID, ACT_TANH or
    ACT_LEAKY_RELU (negative slope alpha)."""
    _need(x, "input")
    if not x.is_contiguous():
        raise ValueError("activation: input must be contiguous")
    if out is None:
        out = torch.empty_like(x)
    L.call("cdx_activation_forward_f32", x.data_ptr(), out.data_ptr(), x.numel(), act, alpha,
           _stream())
    return out


def activation_backward(grad_out, x, act, out=None, alpha=0.01):
    _need(grad_out, "grad_output")
    _need(x, "input")
    if grad_out.shape != x.shape or not (x.is_contiguous() and grad_out.is_contiguous()):
        raise ValueError("activation_backward: shape mismatch or non-contiguous")
    if out is None:
        out = torch.empty_like(x)
    L.call("cdx_activation_backward_f32", grad_out.data_ptr(), x.data_ptr(), out.data_ptr(),
           x.numel(), act, alpha, _stream())
    return out


def col2im(col, x_shape, KH, KW, stride=(1, 1), padding=(0, 0), out=None):
    _need(col, "col")
    Bn, C, H, W = x_shape
    OH = conv_out_size(H, KH, stride[0], padding[0])
    OW = conv_out_size(W, KW, stride[1], padding[1])
    if tuple(col.shape) != (C * KH * KW, Bn * OH * OW) or not col.is_contiguous():
        raise ValueError("col2im: col has the wrong shape")
    if out is None:
        out = torch.empty(tuple(x_shape), device=col.device, dtype=torch.float32)
    L.call("cdx_col2im_f32", col.data_ptr(), out.data_ptr(), Bn, C, H, W, KH, KW,
           stride[0], stride[1], padding[0], padding[1], _stream())
    return out


def _conv_geom(x_shape, w_shape, stride, padding):
    Bn, C, H, W = x_shape
    OC, C2, KH, KW = w_shape
    if C != C2:
        raise ValueError("conv2d: channel mismatch")
    OH = conv_out_size(H, KH, stride[0], padding[0])
    OW = conv_out_size(W, KW, stride[1], padding[1])
    if OH <= 0 or OW <= 0:
        raise ValueError("conv2d: kernel larger than padded input")
    return Bn, C, H, W, OC, KH, KW, OH, OW


def conv2d_backward_data(grad_out, w, x_shape, stride=(1, 1), padding=(0, 0),
                         precision=L.PREC_FP32, out=None, workspace=None):
    """`workspace` (at least conv2d_backward_data_workspace_bytes(...) bytes)
    makes the call allocation-free."""
    _need(grad_out, "grad_output")
    _need(w, "weight")
    Bn, C, H, W, OC, KH, KW, OH, OW = _conv_geom(tuple(x_shape), tuple(w.shape), stride, padding)
    if tuple(grad_out.shape) != (Bn, OC, OH, OW) or not grad_out.is_contiguous() \
            or not w.is_contiguous():
        raise ValueError("conv2d_backward_data: bad grad_output / weight")
    if out is None:
        out = torch.empty((Bn, C, H, W), device=w.device, dtype=torch.float32)
    ws_ptr, ws_bytes, _keep = _scratch(
        workspace, lambda: conv2d_backward_data_workspace_bytes(x_shape, w.shape, stride, padding),
        w.device)
    L.call("cdx_conv2d_backward_data_f32", grad_out.data_ptr(), w.data_ptr(), out.data_ptr(),
           Bn, C, OC, H, W, KH, KW, stride[0], stride[1], padding[0], padding[1], precision,
           ws_ptr, ws_bytes, _stream())
    return out


def conv2d_backward_data_workspace_bytes(x_shape, w_shape, stride=(1, 1),
                                         padding=(0, 0)) -> int:
    Bn, C, H, W, OC, KH, KW, _, _ = _conv_geom(tuple(x_shape), tuple(w_shape), stride, padding)
    return int(L.lib().cdx_conv2d_backward_data_workspace_size(
        Bn, C, OC, H, W, KH, KW, stride[0], stride[1], padding[0], padding[1]))


def conv2d_backward_data_winograd(grad_out, w, x_shape, padding=(0, 0), precision=L.PREC_FP32,
                                  workspace=None, out=None):
    """grad_input of a 3x3 stride-1 conv by Winograd F(4x4, 3x3) on the
    transposed convolution (cdx_conv2d_backward_data_winograd_f32)."""
    _need(grad_out, "grad_output")
    _need(w, "weight")
    Bn, C, H, W, OC, KH, KW, OH, OW = _conv_geom(tuple(x_shape), tuple(w.shape), (1, 1), padding)
    if (KH, KW) != (3, 3) or padding[0] > 2 or padding[1] > 2:
        raise ValueError("conv2d_backward_data_winograd: needs a 3x3 kernel and padding <= 2")
    if tuple(grad_out.shape) != (Bn, OC, OH, OW) or not grad_out.is_contiguous() \
            or not w.is_contiguous():
        raise ValueError("conv2d_backward_data_winograd: bad grad_output / weight")
    if out is None:
        out = torch.empty((Bn, C, H, W), device=w.device, dtype=torch.float32)
    ws_ptr, ws_bytes, _keep = _scratch(
        workspace, lambda: conv2d_backward_data_winograd_workspace_bytes(x_shape, OC, padding),
        w.device)
    L.call("cdx_conv2d_backward_data_winograd_f32", grad_out.data_ptr(), w.data_ptr(),
           out.data_ptr(), Bn, C, OC, H, W, padding[0], padding[1], precision,
           ws_ptr, ws_bytes, _stream())
    return out


def conv2d_backward_data_winograd_workspace_bytes(x_shape, out_channels, padding=(0, 0)) -> int:
    Bn, C, H, W = x_shape
    return int(L.lib().cdx_conv2d_backward_data_winograd_workspace_size(
        Bn, C, out_channels, H, W, padding[0], padding[1]))


def conv2d_backward_weight(grad_out, x, w_shape, stride=(1, 1), padding=(0, 0),
                           precision=L.PREC_FP32, out=None, workspace=None):
    """`workspace` (at least conv2d_backward_weight_workspace_bytes(...) bytes)
    makes the call allocation-free."""
    _need(grad_out, "grad_output")
    _need(x, "input")
    Bn, C, H, W, OC, KH, KW, OH, OW = _conv_geom(tuple(x.shape), tuple(w_shape), stride, padding)
    if tuple(grad_out.shape) != (Bn, OC, OH, OW) or not grad_out.is_contiguous() \
            or not x.is_contiguous():
        raise ValueError("conv2d_backward_weight: bad grad_output / input")
    if out is None:
        out = torch.empty(tuple(w_shape), device=x.device, dtype=torch.float32)
    ws_ptr, ws_bytes, _keep = _scratch(
        workspace, lambda: conv2d_backward_weight_workspace_bytes(x.shape, w_shape, stride, padding),
        x.device)
    L.call("cdx_conv2d_backward_weight_f32", grad_out.data_ptr(), x.data_ptr(), out.data_ptr(),
           Bn, C, OC, H, W, KH, KW, stride[0], stride[1], padding[0], padding[1], precision,
           ws_ptr, ws_bytes, _stream())
    return out


def conv2d_backward_weight_workspace_bytes(x_shape, w_shape, stride=(1, 1),
                                           padding=(0, 0)) -> int:
    Bn, C, H, W, OC, KH, KW, _, _ = _conv_geom(tuple(x_shape), tuple(w_shape), stride, padding)
    return int(L.lib().cdx_conv2d_backward_weight_workspace_size(
        Bn, C, OC, H, W, KH, KW, stride[0], stride[1], padding[0], padding[1]))


def conv2d_backward_bias(grad_out, out=None):
    _need(grad_out, "grad_output")
    if grad_out.dim() != 4 or not grad_out.is_contiguous():
        raise ValueError("conv2d_backward_bias: grad_output must be contiguous NCHW")
    Bn, OC, OH, OW = grad_out.shape
    if out is None:
        out = torch.empty((OC,), device=grad_out.device, dtype=torch.float32)
    L.call("cdx_conv2d_backward_bias_f32", grad_out.data_ptr(), out.data_ptr(), Bn, OC, OH * OW,
           _stream())
    return out


def _dtype_code(t):
    if t.dtype == torch.float32:
        return L.DTYPE_F32
    if t.dtype == torch.float64:
        return L.DTYPE_F64
    raise TypeError("only float32 / float64 tensors")


def strided_copy(view):
    """Contiguous copy of a strided device view (cdx_strided_copy)."""
    if not view.is_cuda:
        raise ValueError("device tensor expected")
    code = _dtype_code(view)
    out = torch.empty(tuple(view.shape), device=view.device, dtype=view.dtype)
    nd = view.dim()
    shape = (ctypes.c_int64 * max(nd, 1))(*view.shape)
    strides = (ctypes.c_int64 * max(nd, 1))(*view.stride())
    L.call("cdx_strided_copy", view.data_ptr(), out.data_ptr(), nd, shape, strides, code, _stream())
    return out


def fill(t, value):
    L.call("cdx_fill", t.data_ptr(), t.numel(), float(value), _dtype_code(t), _stream())
    return t


def binary(op, a, b, out=None):
    if a.shape != b.shape or a.dtype != b.dtype or not (a.is_contiguous() and b.is_contiguous()):
        raise ValueError("binary: operands must match and be contiguous")
    if out is None:
        out = torch.empty_like(a)
    L.call("cdx_binary", op, _dtype_code(a), a.data_ptr(), b.data_ptr(), out.data_ptr(),
           a.numel(), _stream())
    return out


def randn(shape, dtype=torch.float32, seed=0, offset=0):
    out = torch.empty(tuple(shape), device="cuda", dtype=dtype)
    L.call("cdx_randn", out.data_ptr(), out.numel(), _dtype_code(out), int(seed), int(offset),
           _stream())
    return out


def total_sum(x):
    if not x.is_contiguous():
        raise ValueError("sum: input must be contiguous")
    out = torch.empty((1,), device=x.device, dtype=x.dtype)
    L.call("cdx_sum", x.data_ptr(), out.data_ptr(), x.numel(), _dtype_code(x), None, 0, _stream())
    return out


# ---- layer norm and the 8-bit block-scaled format ------------------------------------------

_FLOATS = {torch.float32: L.DTYPE_F32, torch.float16: L.DTYPE_F16, torch.bfloat16: L.DTYPE_BF16}
_SCALES = {torch.float8_e8m0fnu: L.DTYPE_E8M0, torch.float32: L.DTYPE_F32}
_E4M3 = torch.float8_e4m3fn
_BLOCK = 128


def _float_code(t, name):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor")
    code = _FLOATS.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
    return code


def _rows(t, name):
    """(rows, columns, leading dimension) of a tensor seen as a matrix of its last
    dimension: any strides for two dimensions but a unit one in the last, dense beyond."""
    if t.is_contiguous():
        shape = t.shape
        if len(shape) == 2:
            return shape[0], shape[1], shape[1]
        if not shape:
            raise ValueError(f"{name} must have a last dimension")
        cols = shape[-1]
        rows = 1
        for d in shape[:-1]:
            rows *= d
        return rows, cols, cols
    if t.dim() != 2:
        raise ValueError(f"{name} must be contiguous (or 2-D with unit column stride)")
    rows, cols = t.shape
    ld, step = t.stride()
    if step != 1 and cols > 1:
        raise ValueError(f"{name} must have unit column stride")
    if rows > 1 and ld < cols:
        raise ValueError(f"{name}: rows overlap")
    return rows, cols, ld if rows > 1 else cols


def _new_like(t):
    """An uninitialised contiguous tensor of t's shape and type."""
    if t.is_contiguous():
        return torch.empty_like(t)   # (half the time of empty with a shape)
    return torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _workspace(workspace, nbytes, device):
    """_scratch with the caller's workspace checked."""
    if workspace is not None:
        if not isinstance(workspace, torch.Tensor) or not workspace.is_cuda \
                or not workspace.is_contiguous():
            raise ValueError("workspace must be a contiguous device tensor")
    return _scratch(workspace, nbytes, device)


def _out(out, shape, dtype):
    """Leading dimension of a caller's `out`, checked."""
    _need(out, "out", dtype)
    if out.shape != shape:
        raise ValueError("out has the wrong shape")
    return _rows(out, "out")[2]


def _param(p, name, dim, dtype):
    if not isinstance(p, torch.Tensor) or not p.is_cuda:
        raise ValueError(f"{name} must be a device tensor")
    if p.dtype != dtype and p.dtype != torch.float32:
        raise TypeError(f"{name} must be {dtype} or float32, got {p.dtype}")
    if p.dim() != 1 or p.shape[0] != dim or not p.is_contiguous():
        raise ValueError(f"{name} must be a contiguous [{dim}] tensor")
    return p.data_ptr()


def layer_norm(x, weight=None, bias=None, eps=1e-5, *, stats=False, out=None):
    """Layer norm over the last dimension of a float32, float16 or bfloat16 tensor (2-D: any
    row stride); sums in float32.  weight and bias are of x's type or float32 (both the
    same).  With stats, (y, mean, rstd), float32 [rows], as layer_norm_backward takes them.  `out`
    may be x itself."""
    code = _float_code(x, "input")
    rows, dim, ldx = _rows(x, "input")
    if dim < 1:
        raise ValueError("layer_norm: the last dimension is empty")
    if out is None:
        y, ldy = _new_like(x), dim
    else:
        y, ldy = out, _out(out, x.shape, x.dtype)
    wptr = bptr = None
    pcode = code
    if weight is not None:
        wptr = _param(weight, "weight", dim, x.dtype)
        pcode = _FLOATS[weight.dtype]
    if bias is not None:
        bptr = _param(bias, "bias", dim, x.dtype)
        if weight is not None and bias.dtype != weight.dtype:
            raise TypeError("weight and bias must have the same type")
        pcode = _FLOATS[bias.dtype]
    mean = rstd = None
    mptr = rptr = None
    if stats:
        mean = torch.empty((rows,), dtype=torch.float32, device=x.device)
        rstd = torch.empty_like(mean)
        mptr, rptr = mean.data_ptr(), rstd.data_ptr()
    L.call("cdx_layer_norm_forward", x.data_ptr(), ldx, wptr, bptr, y.data_ptr(), ldy, mptr, rptr,
           rows, dim, eps, code, pcode, _stream())
    return (y, mean, rstd) if stats else y


def layer_norm_backward(grad_out, x, mean, rstd, weight=None, *, params=True, param_dtype=None,
                        out=None, workspace=None):
    """(grad of x, of weight, of bias) of layer_norm, from the statistics it returned.  The
    parameters' gradients are of `param_dtype` (weight's type, else x's), None each without
    `params`.  `out` (x's gradient) may be x or grad_out itself.  `workspace`
    (layer_norm_backward_workspace_bytes) makes the call allocation-free."""
    code = _float_code(x, "input")
    _need(grad_out, "grad_out", x.dtype)
    if grad_out.shape != x.shape:
        raise ValueError("layer_norm_backward: grad_out and input differ in shape")
    rows, dim, ldx = _rows(x, "input")
    ldg = _rows(grad_out, "grad_out")[2]
    if dim < 1:
        raise ValueError("layer_norm_backward: the last dimension is empty")
    for t, name in ((mean, "mean"), (rstd, "rstd")):
        _need(t, name)
        if t.numel() != rows or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous tensor of {rows} elements")
    wptr = None
    pdtype = param_dtype or x.dtype
    if weight is not None:
        wptr = _param(weight, "weight", dim, x.dtype)
        if param_dtype is not None and param_dtype != weight.dtype:
            raise TypeError("param_dtype must be weight's type")
        pdtype = weight.dtype
    if pdtype != x.dtype and pdtype != torch.float32:
        raise TypeError(f"param_dtype must be {x.dtype} or float32")
    if out is None:
        dx, lddx = _new_like(x), dim
    else:
        dx, lddx = out, _out(out, x.shape, x.dtype)
    dw = db = None
    wsp, wsb, _keep = None, 0, None
    dwp = dbp = None
    if params:
        dw = torch.empty((dim,), dtype=pdtype, device=x.device)
        db = torch.empty_like(dw)
        dwp, dbp = dw.data_ptr(), db.data_ptr()
        wsp, wsb, _keep = _workspace(
            workspace, lambda: layer_norm_backward_workspace_bytes(rows, dim, x.dtype), x.device)
    L.call("cdx_layer_norm_backward", grad_out.data_ptr(), ldg, x.data_ptr(), ldx, wptr,
           mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(), lddx, dwp, dbp,
           rows, dim, code, _FLOATS[pdtype], wsp, wsb, _stream())
    return dx, dw, db


def layer_norm_backward_workspace_bytes(rows: int, dim: int, dtype=torch.float32) -> int:
    return int(L.lib().cdx_layer_norm_backward_workspace_size(rows, dim, _FLOATS[dtype]))


class Block8(NamedTuple):
    """A matrix in 8 bits: `q`, float8_e4m3fn [rows, cols], and `scale`, one for each 128
    columns of a row ([rows, ceil(cols / 128)], tile_rows 1) or each 128 x 128 tile
    ([ceil(rows / 128), ceil(cols / 128)], tile_rows 128), as float8_e8m0fnu (a power of two) or
    float32.  A value is q * scale."""
    q: torch.Tensor
    scale: torch.Tensor
    tile_rows: int = 1

    @property
    def shape(self):
        return self.q.shape


def _block8(b, name, tile_rows=None):
    """(rows, cols, q pointer, ld, scale pointer, ld, scale code) of a checked Block8."""
    if not isinstance(b, Block8):
        raise TypeError(f"{name} must be a Block8")
    q, s, tr = b
    if q.dtype != _E4M3:
        raise TypeError(f"{name}.q must be float8_e4m3fn, got {q.dtype}")
    code = _SCALES.get(s.dtype)
    if code is None:
        raise TypeError(f"{name}.scale must be float8_e8m0fnu or float32, got {s.dtype}")
    if not (q.is_cuda and s.is_cuda):
        raise ValueError(f"{name} must be on the device")
    if q.dim() != 2 or s.dim() != 2:
        raise ValueError(f"{name}: q and scale must be 2-D")
    if tr not in (1, _BLOCK) or (tile_rows is not None and tr != tile_rows):
        raise ValueError(f"{name}: tile_rows must be "
                         f"{tile_rows if tile_rows is not None else '1 or 128'}, got {tr}")
    rows, cols, ldq = _rows(q, f"{name}.q")
    srows, scols, lds = _rows(s, f"{name}.scale")
    if scols != -(-cols // _BLOCK) or srows != (rows if tr == 1 else -(-rows // _BLOCK)):
        raise ValueError(f"{name}.scale must hold one value for each block, got {list(s.shape)} "
                         f"for {[rows, cols]} (tile_rows {tr})")
    return rows, cols, q.data_ptr(), ldq, s.data_ptr(), lds, code


def _empty8(rows, cols, tile_rows, scale_dtype, device):
    """An uninitialised Block8 whose rows begin on 16-byte boundaries (what the products'
    wide loads want)."""
    ld = -(-cols // 16) * 16
    q = torch.empty((rows, ld), dtype=_E4M3, device=device)
    if ld != cols:
        q = q[:, :cols]
    tiles = rows if tile_rows == 1 else -(-rows // _BLOCK)
    return Block8(q, torch.empty((tiles, -(-cols // _BLOCK)), dtype=scale_dtype, device=device),
                  tile_rows), ld


def quantize8(x, tile_rows=1, *, scale_dtype=torch.float8_e8m0fnu):
    """x [rows, cols] (float32, float16, bfloat16) as a Block8: activations with a scale for
    each 128 columns of a row (tile_rows 1), weights with one for each 128 x 128 tile
    (tile_rows 128).  A scale is the least power of two under which the block's largest finite
    magnitude is at most 448 (1 for a block of zeros); infinities and NaN become NaN."""
    code = _float_code(x, "input")
    if x.dim() != 2:
        raise ValueError("quantize8: input must be 2-D")
    if tile_rows not in (1, _BLOCK):
        raise ValueError("quantize8: tile_rows must be 1 or 128")
    scode = _SCALES.get(scale_dtype)
    if scode is None:
        raise TypeError("quantize8: scale_dtype must be float8_e8m0fnu or float32")
    rows, cols, ldx = _rows(x, "input")
    b, ld = _empty8(rows, cols, tile_rows, scale_dtype, x.device)
    L.call("cdx_quantize_e4m3", x.data_ptr(), ldx, rows, cols, code, tile_rows, b.q.data_ptr(), ld,
           b.scale.data_ptr(), b.scale.shape[1], scode, _stream())
    return b


def dequantize8(b, dtype=torch.float32, out=None):
    """The values of a Block8, rounded to `dtype`."""
    rows, cols, q, ldq, s, lds, scode = _block8(b, "input")
    code = _FLOATS.get(dtype)
    if code is None:
        raise TypeError("dequantize8: dtype must be float32, float16 or bfloat16")
    if out is None:
        out, ldo = torch.empty((rows, cols), dtype=dtype, device=b.q.device), cols
    else:
        ldo = _out(out, (rows, cols), dtype)
    L.call("cdx_dequantize_e4m3", q, ldq, s, lds, scode, b.tile_rows, out.data_ptr(), ldo, rows,
           cols, code, _stream())
    return out


def _vector(bias, n, name="bias"):
    if bias is None:
        return None
    _need(bias, name)
    if bias.numel() != n or not bias.is_contiguous():
        raise ValueError(f"{name} has the wrong size or is not contiguous")
    return bias.data_ptr()


def gemm8(a, b, *, bias=None, epilogue=L.EPI_NONE, dtype=torch.bfloat16, out=None,
          workspace=None):
    """C = epi(A B^T + bias) of two Block8 matrices, A [M, K] with tile_rows 1 and B [N, K] (a
    Linear layer's weight) with tile_rows 128; C of `dtype`, bias float32.  Products are exact.  A
    float32 result has float32 sums; a 16-bit one, at twice the rate, loses up to 2^-10 of the
    largest of each eight products (consecutive k) before the float32 sums: usually far below its
    own rounding, more where sums cancel."""
    M, K, aq, lda, asc, ldsa, acode = _block8(a, "A", 1)
    N, K2, bq, ldb, bsc, ldsb, bcode = _block8(b, "B", _BLOCK)
    if K != K2:
        raise ValueError(f"inner dimensions differ: {K} vs {K2}")
    code = _FLOATS.get(dtype)
    if code is None:
        raise TypeError("gemm8: dtype must be float32, float16 or bfloat16")
    if out is None:
        out, ldo = torch.empty((M, N), dtype=dtype, device=a.q.device), N
    else:
        ldo = _out(out, (M, N), dtype)
    ws_ptr, ws_bytes, _keep = _workspace(
        workspace, lambda: L.lib().cdx_gemm_e4m3_workspace_size(M, N, K), a.q.device)
    L.call("cdx_gemm_e4m3", M, N, K, aq, lda, asc, ldsa, acode, bq, ldb, bsc, ldsb, bcode,
           out.data_ptr(), ldo, code, _vector(bias, N), epilogue, ws_ptr,
           ws_bytes, _stream())
    return out


def gemm8_workspace_bytes(M: int, N: int, K: int) -> int:
    return int(L.lib().cdx_gemm_e4m3_workspace_size(M, N, K))


def linear8(x, weight, bias=None, *, epilogue=L.EPI_NONE, dtype=None, out=None, workspace=None):
    """epi(x W^T + bias) with W a Block8 [N, K] (tile_rows 128) and x [M, K] quantised on the way
    in as quantize8(x) does; the result is of `dtype` (x's own by default), which also decides
    how sums are formed, as for gemm8.  `out` must not overlap x."""
    xcode = _float_code(x, "input")
    if x.dim() != 2:
        raise ValueError("linear8: input must be 2-D")
    M, K, ldx = _rows(x, "input")
    N, K2, bq, ldb, bsc, ldsb, bcode = _block8(weight, "weight", _BLOCK)
    if K != K2:
        raise ValueError(f"inner dimensions differ: {K} vs {K2}")
    dtype = dtype or x.dtype
    code = _FLOATS.get(dtype)
    if code is None:
        raise TypeError("linear8: dtype must be float32, float16 or bfloat16")
    if out is None:
        out, ldo = torch.empty((M, N), dtype=dtype, device=x.device), N
    else:
        ldo = _out(out, (M, N), dtype)
    ws_ptr, ws_bytes, _keep = _workspace(
        workspace, lambda: L.lib().cdx_linear_e4m3_workspace_size(M, N, K), x.device)
    L.call("cdx_linear_e4m3", M, N, K, x.data_ptr(), ldx, xcode, bq, ldb, bsc, ldsb, bcode,
           out.data_ptr(), ldo, code, _vector(bias, N), epilogue, ws_ptr,
           ws_bytes, _stream())
    return out


def linear8_workspace_bytes(M: int, N: int, K: int) -> int:
    return int(L.lib().cdx_linear_e4m3_workspace_size(M, N, K))


def activation8(z, act, *, alpha=0.01, scale_dtype=torch.float8_e8m0fnu, out=None):
    """(act(z), z as a Block8) in one pass over z [rows, cols]: what the backward pass keeps of
    an activation's input.  act as for `activation`; `out` may be z itself."""
    code = _float_code(z, "input")
    if z.dim() != 2:
        raise ValueError("activation8: input must be 2-D")
    scode = _SCALES.get(scale_dtype)
    if scode is None:
        raise TypeError("activation8: scale_dtype must be float8_e8m0fnu or float32")
    rows, cols, ldz = _rows(z, "input")
    if out is None:
        y, ldy = _new_like(z), cols
    else:
        y, ldy = out, _out(out, z.shape, z.dtype)
    b, ld = _empty8(rows, cols, 1, scale_dtype, z.device)
    L.call("cdx_activation_forward_e4m3", z.data_ptr(), ldz, y.data_ptr(), ldy,
           b.q.data_ptr(), ld, b.scale.data_ptr(), b.scale.shape[1], scode, rows, cols, code, act,
           alpha, _stream())
    return y, b


def activation_backward8(grad_out, z, act, *, alpha=0.01, out=None):
    """grad_out * act'(z) with z a Block8 (tile_rows 1); `out` may be grad_out itself."""
    code = _float_code(grad_out, "grad_out")
    rows, cols, q, ldq, s, lds, scode = _block8(z, "input", 1)
    if tuple(grad_out.shape) != (rows, cols):
        raise ValueError("activation_backward8: grad_out and input differ in shape")
    ldg = _rows(grad_out, "grad_out")[2]
    if out is None:
        out, ldo = _new_like(grad_out), cols
    else:
        ldo = _out(out, grad_out.shape, grad_out.dtype)
    L.call("cdx_activation_backward_e4m3", grad_out.data_ptr(), ldg, q, ldq, s, lds, scode,
           out.data_ptr(), ldo, rows, cols, code, act, alpha, _stream())
    return out


def linear_weight_grad8(grad_out, x, *, bias=True, workspace=None):
    """(weight gradient [N, K], bias gradient [N] or None) of a Linear layer from its output's
    gradient [M, N] (float32, float16, bfloat16) and its input kept as a Block8 [M, K] (tile_rows
    1, float8_e8m0fnu scales); both float32, exact products, float32 sums."""
    code = _float_code(grad_out, "grad_out")
    M, K, q, ldq, s, lds, scode = _block8(x, "input", 1)
    if scode != L.DTYPE_E8M0:
        raise TypeError("linear_weight_grad8: the input's scales must be float8_e8m0fnu")
    if grad_out.dim() != 2 or grad_out.shape[0] != M:
        raise ValueError(f"linear_weight_grad8: grad_out must be [{M}, out_features]")
    N = grad_out.shape[1]
    ldg = _rows(grad_out, "grad_out")[2]
    dw = torch.empty((N, K), dtype=torch.float32, device=grad_out.device)
    db = torch.empty((N,), dtype=torch.float32, device=grad_out.device) if bias else None
    ws_ptr, ws_bytes, _keep = _workspace(
        workspace, lambda: L.lib().cdx_linear_weight_grad_e4m3_workspace_size(M, N, K, code),
        grad_out.device)
    L.call("cdx_linear_weight_grad_e4m3", grad_out.data_ptr(), ldg, code, q, ldq, s, lds,
           dw.data_ptr(), db.data_ptr() if bias else None, M, N, K, ws_ptr, ws_bytes, _stream())
    return dw, db


def linear_weight_grad8_workspace_bytes(M: int, N: int, K: int, dtype=torch.float32) -> int:
    return int(L.lib().cdx_linear_weight_grad_e4m3_workspace_size(M, N, K, _FLOATS[dtype]))
