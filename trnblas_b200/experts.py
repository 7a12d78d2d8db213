"""Products grouped by expert: `grouped_gemm` and the gradient of its weights,
`grouped_gemm_wgrad`.

The rows of one operand fall into groups of any length (the tokens a router
sent to each expert), and every group has its own matrix. They stand beside
`batched_gemm`, whose entries all have one size; the reference has no
counterpart. The sizes stay on the device: no call on device operands synchronises,
and a captured graph follows the sizes of each replay. bfloat16 and float16 on
the sm_100a kernels through the C ABI; other dtypes raise TypeError.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _native as N
from ._flags import trans_flag
from .level3 import _add_c, _cuda_device, _fuse_c, _home, _mixed_dtype_error

DTYPES = (torch.bfloat16, torch.float16)
MAX_GROUPS = 1024


def call_on(dev: torch.device, fn, *args) -> int:
    """fn(*args, stream) on dev's current stream, with dev the current device."""
    stream = N.stream_ptr(dev)
    if dev.index == torch.cuda.current_device():
        return fn(*args, stream)
    with torch.cuda.device(dev):
        return fn(*args, stream)


def empty(shape, dtype, dev) -> torch.Tensor:
    """torch.empty for a 1-D or 2-D shape, by the entry that takes strides (half
    the host time of torch.empty's parsing)."""
    return torch.empty_strided(shape, (shape[1], 1) if len(shape) == 2 else (1,), dtype=dtype, device=dev)


def _same_cuda_device(*ts) -> bool:
    """Every tensor (or None) on one CUDA device: nothing to move."""
    d = ts[0].get_device()
    if d < 0:
        return False
    for t in ts:
        if t is not None and (not isinstance(t, torch.Tensor) or t.get_device() != d):
            return False
    return True


def on_device(t, dev: torch.device, home: torch.device):
    """t on dev, for a result on `home`. A result that stays on the device comes
    back while the stream still runs, so the copy of a pinned tensor is waited
    for: its owner may rewrite it after the call. A captured copy cannot be: the
    graph reads the host memory at each replay."""
    if not isinstance(t, torch.Tensor) or t.device == dev:
        return t
    if t.device.type != "cpu" or not t.is_pinned():
        return t.to(dev)
    with torch.cuda.device(dev):
        return t.to(dev, non_blocking=home != dev or torch.cuda.is_current_stream_capturing())


def _refuse_tangents(name: str, *ts) -> None:
    """The kernels see values alone: a dual tensor's tangent would be dropped."""
    for t in ts:
        if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{name}: forward-mode derivatives are not implemented")


def _check_types(name: str, a, b, out_dtype):
    for x in (a, b):
        if not isinstance(x, torch.Tensor) or x.dtype not in DTYPES:
            raise TypeError(f"{name}: operands are bfloat16 or float16 tensors, got {getattr(x, 'dtype', type(x))}")
    dtype = a.dtype
    if dtype != b.dtype:
        _mixed_dtype_error(a, b)
    if out_dtype is None:
        return dtype
    out = out_dtype
    if out not in (dtype, torch.float32):
        raise TypeError(f"{name}: out_dtype is {a.dtype} or float32, got {out_dtype}")
    return out


def check_group_sizes(name: str, sizes, groups: int | None, rows: int) -> None:
    """Shape and dtype of the sizes; their values only where the host holds them."""
    if not isinstance(sizes, torch.Tensor) or sizes.dim() != 1 or sizes.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name}: group_sizes is a 1-D int32 or int64 tensor")
    if groups is not None and sizes.shape[0] != groups:
        raise ValueError(f"{name}: {sizes.shape[0]} group sizes for {groups} matrices")
    if sizes.shape[0] > MAX_GROUPS:
        raise ValueError(f"{name}: at most {MAX_GROUPS} groups, got {sizes.shape[0]}")
    if sizes.device.type == "cpu" and sizes.numel():
        # (each size first: a sum of huge ones wraps around)
        if int(sizes.min()) < 0 or int(sizes.max()) > rows or int(sizes.sum()) > rows:
            raise ValueError(f"{name}: group sizes must not be negative nor sum to more than the {rows} rows")


def _rows_operand(x: torch.Tensor):
    """(tensor, ld) of a rows x cols operand stored row by row."""
    s0, s1 = x.stride()
    rows, cols = x.shape
    if rows == 1 and (s1 == 1 or cols == 1):
        return x, cols  # the stride of a single row says nothing
    if s1 != 1 or s0 < cols:
        return x.contiguous(), cols
    return x, s0


def _weights_operand(B: torch.Tensor, transB: bool):
    """(tensor, ld, stored N x K, matrix stride) of the stack op(B): matrices
    stored by rows or by columns are read where they are; stride 0 is one matrix
    for all groups."""
    G, rows, cols = B.shape
    s0, s1, s2 = B.stride()
    if s2 == 1 and s1 >= cols:
        return B, s1, transB, s0 if G > 1 else 0
    if s1 == 1 and s2 >= rows:
        return B, s2, not transB, s0 if G > 1 else 0
    if G > 1 and s0 == 0:
        return *_weights_operand(B[:1].contiguous(), transB)[:3], 0
    return B.contiguous(), cols, transB, rows * cols


def _c_operand(C, cols: int):
    """(tensor, ld) of a C (..., rows, cols) whose rows are contiguous."""
    if C.stride(-1) == 1 and C.stride(-2) >= cols:
        return C, C.stride(-2)
    return C.contiguous(), cols  # (one row is contiguous whatever its stride says)


def _grouped(alpha, a, B, transB, sizes, beta, C, out_dtype):
    """alpha * a[r] @ op(B[g]) (+ beta * C) on the kernel; C fusable or None."""
    rows, K = a.shape
    G = B.shape[0]
    Nn = B.shape[1] if transB else B.shape[2]
    dev = a.device
    out = empty((rows, Nn), out_dtype, dev)
    if rows == 0 or Nn == 0:
        return out
    at, lda, bt, ldb, tb, sb = a, K, B, Nn, False, 0
    if K and G:
        at, lda = _rows_operand(a)
        bt, ldb, tb, sb = _weights_operand(B, transB)
    c_arg, ldc = _c_operand(C, Nn) if C is not None else (None, 0)
    if not sizes.is_contiguous():
        sizes = sizes.contiguous()
    ap, bp, ws, ws_bytes = at.data_ptr(), bt.data_ptr(), None, 0
    if (lda | ldb | sb) & 7 or (ap | bp) & 15:  # TMA needs copies
        ws_bytes = N.lib().trnblas_grouped_gemm_workspace_size(rows, G, Nn, K, ap, lda, bp, ldb, sb, tb)
        ws = empty((ws_bytes,), torch.uint8, dev)
    rc = call_on(
        dev, N.lib().trnblas_grouped_gemm, N.dtype_code(a.dtype), N.dtype_code(out_dtype), rows, G, Nn, K, float(alpha),
        ap, lda, bp, ldb, sb, tb, sizes.data_ptr(), sizes.dtype == torch.int64,
        float(beta) if C is not None else 0.0, N.ptr(c_arg), ldc, out.data_ptr(), Nn, N.ptr(ws), ws_bytes)
    if rc:
        N.check(rc, "trnblas_grouped_gemm")
    N.count_launches(2 if ws_bytes else 1)
    return out


def _wgrad(alpha, a, b, sizes, beta, C, out_dtype):
    """alpha * a_g^T @ b_g (+ beta * C[g]) on the kernel; C fusable or None."""
    rows, M = a.shape
    Nn = b.shape[1]
    G = sizes.shape[0]
    dev = a.device
    out = torch.empty_strided((G, M, Nn), (M * Nn, Nn, 1), dtype=out_dtype, device=dev)
    if out.numel() == 0:
        return out
    (at, lda), (bt, ldb) = (_rows_operand(a), _rows_operand(b)) if rows else ((a, M), (b, Nn))
    c_arg, ldc, sc = None, 0, 0
    if C is not None:
        c_arg, ldc = _c_operand(C, Nn)
        sc = c_arg.stride(0)
    if not sizes.is_contiguous():
        sizes = sizes.contiguous()
    ap, bp, ws, ws_bytes = at.data_ptr(), bt.data_ptr(), None, 0
    if (lda | ldb) & 7 or (ap | bp) & 15:  # TMA needs copies
        ws_bytes = N.lib().trnblas_grouped_gemm_wgrad_workspace_size(rows, M, Nn, ap, lda, bp, ldb)
        ws = empty((ws_bytes,), torch.uint8, dev)
    rc = call_on(
        dev, N.lib().trnblas_grouped_gemm_wgrad, N.dtype_code(a.dtype), N.dtype_code(out_dtype), rows, G, M, Nn, float(alpha),
        ap, lda, bp, ldb, sizes.data_ptr(), sizes.dtype == torch.int64,
        float(beta) if C is not None else 0.0, N.ptr(c_arg), ldc, sc, out.data_ptr(), Nn, M * Nn, N.ptr(ws), ws_bytes)
    if rc:
        N.check(rc, "trnblas_grouped_gemm_wgrad")
    N.count_launches(2 if ws_bytes else 1)
    return out


class _GroupedGemm(torch.autograd.Function):
    """D[r] = alpha A[r] op(B[g]) + beta C[r] with its gradients:
    dA[r] = alpha dD[r] op(B[g])^T, dB[g] = alpha A_g^T dD_g (or its transpose),
    dC = beta dD."""

    @staticmethod
    def forward(ctx, args, a, B, sizes, C):
        alpha, transB, beta, out_dtype = ctx.args = args
        ctx.save_for_backward(a, B, sizes)
        return _grouped(alpha, a, B, transB, sizes, beta, C, out_dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dD):
        a, B, sizes = ctx.saved_tensors
        alpha, transB, beta, _ = ctx.args
        _, need_a, need_B, _, need_C = ctx.needs_input_grad
        if forward_ad._current_level >= 0 and (need_a or need_B):
            _refuse_tangents("gradient of grouped_gemm", dD)
        y = dD if dD.dtype == a.dtype else dD.to(a.dtype)
        da = dB = dC = None
        if need_a:
            da = _grouped(alpha, y, B, not transB, sizes, 0.0, None, a.dtype)
        if need_B:
            l, r = (y, a) if transB else (a, y)
            dB = _wgrad(alpha, l, r, sizes, 0.0, None, B.dtype)
        if need_C:
            dC = beta * dD
        return None, da, dB, None, dC


def grouped_gemm(
    alpha: float,
    A: torch.Tensor,
    B: torch.Tensor,
    group_sizes: torch.Tensor,
    beta: float = 0.0,
    C: torch.Tensor | None = None,
    transB: bool = False,
    out_dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """D[r] = alpha * A[r] @ op(B[g]) + beta * C[r] for the rows r of group g.

    A is (rows, K); its first group_sizes[0] rows belong to group 0, the next
    group_sizes[1] to group 1, and so on. B is (G, K, N), or (G, N, K) with
    transB; it may be expanded (one matrix for all groups). Rows behind the last
    group are an empty product: beta * C[r], or zero. group_sizes is int32 or
    int64 on any device; on the host its values are checked (ValueError), on
    the device negative sizes count as zero, sizes beyond the rows are cut
    off, and `device_status` then returns 8. At most 1024 groups. bfloat16 or
    float16 with fp32 accumulation; the result (rows, N) has the operands'
    dtype or float32 (out_dtype). alpha, beta and a same-shape C of the result's
    dtype are fused; another C is added afterwards with torch semantics.

    Differentiable in A, B and C (once, in reverse mode; tensors with forward-mode
    tangents raise NotImplementedError): the gradients run on the same kernels,
    rounded once to their operand's dtype; an incoming float32 gradient is
    rounded to the operands' dtype first. Inside a CUDA graph capture, call
    `grouped_gemm` (transB flipped) and `grouped_gemm_wgrad` for them directly,
    or capture forward and backward together on leaves used on no other stream.
    """
    name = "grouped_gemm"
    if transB is not False and transB is not True:
        transB = trans_flag(transB, "transB")
    out_dtype = _check_types(name, A, B, out_dtype)
    if A.dim() != 2 or B.dim() != 3:
        raise ValueError(f"{name}: A is 2-D and B 3-D, got {tuple(A.shape)} and {tuple(B.shape)}")
    if A.shape[1] != B.shape[2 if transB else 1]:
        raise ValueError(f"{name}: inner dimensions differ: A {tuple(A.shape)}, B {tuple(B.shape)}, transB={transB}")
    check_group_sizes(name, group_sizes, B.shape[0], A.shape[0])
    if forward_ad._current_level >= 0:  # inside a dual level (torch adds a C that is not fused)
        D = (A.shape[0], B.shape[1 if transB else 2])
        fused = isinstance(C, torch.Tensor) and _fuse_c(C, beta, D, out_dtype, C.device)
        _refuse_tangents(name, A, B, C if fused else None)
    grad = (A.requires_grad or B.requires_grad) and torch.is_grad_enabled()
    if C is None and _same_cuda_device(A, B, group_sizes):
        if grad:
            return _GroupedGemm.apply((alpha, transB, 0.0, out_dtype), A, B, group_sizes, None)
        return _grouped(alpha, A, B, transB, group_sizes, 0.0, None, out_dtype)
    home = A.device
    dev = _cuda_device(A, B, C, group_sizes)
    a, b, sizes, Cd = (on_device(t, dev, home) for t in (A, B, group_sizes, C))
    fuse = _fuse_c(Cd, beta, (a.shape[0], b.shape[1] if transB else b.shape[2]), out_dtype, dev)
    c_arg = Cd if fuse else None
    if grad or (torch.is_grad_enabled() and fuse and Cd.requires_grad):
        r = _GroupedGemm.apply((alpha, transB, beta, out_dtype), a, b, sizes, c_arg)
        if not fuse:
            r = _add_c(r, beta, Cd)
        return r if home == dev else r.to(home)
    r = _grouped(alpha, a, b, transB, sizes, beta, c_arg, out_dtype)
    if not fuse:
        r = _add_c(r, beta, Cd)
    return _home(r, home, dev)


def grouped_gemm_wgrad(
    alpha: float,
    A: torch.Tensor,
    B: torch.Tensor,
    group_sizes: torch.Tensor,
    beta: float = 0.0,
    C: torch.Tensor | None = None,
    out_dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """D[g] = alpha * A_g^T @ B_g + beta * C[g], the contraction over the rows
    of group g: for A the operand and B the result's gradient of `grouped_gemm`,
    the gradient of its (G, K, N) weights; with A and B exchanged that of
    (G, N, K) weights. C (G, M, N) of the result's dtype adds to a running
    gradient (beta = 1, out_dtype = float32 keeps it in 32 bits). A group
    without rows gives beta * C[g]. Rows behind the last group are not part of
    any sum. group_sizes and dtypes as for `grouped_gemm`; not differentiable.
    """
    name = "grouped_gemm_wgrad"
    out_dtype = _check_types(name, A, B, out_dtype)
    if A.dim() != 2 or B.dim() != 2 or A.shape[0] != B.shape[0]:
        raise ValueError(f"{name}: A and B are 2-D with the same rows, got {tuple(A.shape)} and {tuple(B.shape)}")
    check_group_sizes(name, group_sizes, None, A.shape[0])
    if C is None and _same_cuda_device(A, B, group_sizes):
        return _wgrad(alpha, A, B, group_sizes, 0.0, None, out_dtype)
    home = A.device
    dev = _cuda_device(A, B, C, group_sizes)
    C = C.detach() if isinstance(C, torch.Tensor) else C
    a, b, sizes, Cd = (on_device(t, dev, home) for t in (A.detach(), B.detach(), group_sizes, C))
    fuse = _fuse_c(Cd, beta, (sizes.shape[0], a.shape[1], b.shape[1]), out_dtype, dev)
    r = _wgrad(alpha, a, b, sizes, beta, Cd if fuse else None, out_dtype)
    if not fuse:
        r = _add_c(r, beta, Cd)
    return _home(r, home, dev)
