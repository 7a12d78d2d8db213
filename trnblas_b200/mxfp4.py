"""Microscaled 4-bit floating point (OCP MX, MXFP4) on the block-scaled tensor
cores: `quantize_mxfp4`, `dequantize_mxfp4`, and the products of quantised
operands, `gemm_mxfp4` and `grouped_gemm_mxfp4`.

Blocks of 32 neighbouring values along the last dimension share a power of two
(E8M0) and hold E2M1 values: 0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives. A
product takes both operands with their blocks along the contraction, so B is
stored as (N, K) (what `gemm` calls transB). The reference has no counterpart.
"""

from __future__ import annotations

import math

import torch

from . import _native as N
from .experts import _c_operand, _same_cuda_device, call_on, check_group_sizes, empty, on_device
from .level3 import _add_c, _cuda_device, _fuse_c, _home, _to

BLOCK = 32
_OUT = (torch.bfloat16, torch.float16, torch.float32)


class MXFP4Tensor:
    """A quantised (..., rows, K) operand.

    data    uint8 (..., rows, round_up(K, 32) / 2): two values a byte, the even
            one in the low half, zero behind K;
    scales  uint8 (matrices, ceil(rows / 128), ceil(K / 128), 512), matrices the
            product of the leading dimensions: the E8M0 bytes of 128 rows x 128
            values, the four of row r at 16 * (r % 32) + 4 * (r / 32 % 4), as the
            tensor cores take them; zero behind the rows and behind K;
    shape   the logical shape.
    """

    __slots__ = ("data", "scales", "shape")

    def __init__(self, data: torch.Tensor, scales: torch.Tensor, shape):
        self.data, self.scales, self.shape = data, scales, torch.Size(shape)
        if len(self.shape) < 2 or min(self.shape) < 0:
            raise ValueError(f"MXFP4Tensor: a shape (..., rows, K), got {tuple(shape)}")
        *lead, K = self.shape
        want = (*lead, _round_up(K, BLOCK) // 2)
        if data.dtype != torch.uint8 or tuple(data.shape) != want or not data.is_contiguous():
            raise ValueError(f"MXFP4Tensor: data must be contiguous uint8 {want}, got {data.dtype} {tuple(data.shape)}")
        want = _scale_shape(self.shape)
        if scales.dtype != torch.uint8 or tuple(scales.shape) != want or not scales.is_contiguous():
            raise ValueError(
                f"MXFP4Tensor: scales must be contiguous uint8 {want}, got {scales.dtype} {tuple(scales.shape)}")
        if data.device != scales.device:
            raise ValueError("MXFP4Tensor: data and scales on different devices")

    @property
    def device(self) -> torch.device:
        return self.data.device

    def dim(self) -> int:
        return len(self.shape)

    def to(self, device) -> "MXFP4Tensor":
        """The same operand on another device."""
        return MXFP4Tensor(self.data.to(device), self.scales.to(device), self.shape)

    @classmethod
    def from_parts(cls, codes: torch.Tensor, scales: torch.Tensor, K: int) -> "MXFP4Tensor":
        """From codes (..., rows, at least ceil(K / 2) bytes) and scales
        (..., rows, ceil(K / 32) E8M0 bytes), both in row order, as checkpoints
        hold them. What stands behind K is ignored."""
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError(f"MXFP4Tensor.from_parts: uint8 codes and scales, got {codes.dtype} and {scales.dtype}")
        nb, kb = -(-K // BLOCK), -(-K // 2)
        if (codes.dim() < 2 or codes.shape[:-1] != scales.shape[:-1] or scales.shape[-1] != nb
                or codes.shape[-1] < kb or K < 0):
            raise ValueError(
                f"MXFP4Tensor.from_parts: K = {K} takes codes (..., rows, >= {kb}) and scales (..., rows, {nb}), "
                f"got {tuple(codes.shape)} and {tuple(scales.shape)}")
        lead = codes.shape[:-1]
        data = codes.new_zeros((*lead, _round_up(K, BLOCK) // 2))
        data[..., :kb] = codes[..., :kb]
        if K % 2:
            data[..., kb - 1] &= 0x0F
        mats, rb, kw, _ = _scale_shape((*lead, K))
        rows = lead[-1]
        words = scales.new_zeros((mats, rb * 128, 4 * kw))
        words[:, :rows, :nb] = scales.reshape(mats, rows, nb)
        # (block, row / 32, row % 32, K block, byte) -> (block, K block, row % 32, row / 32, byte)
        blocks = words.view(mats, rb, 4, 32, kw, 4).permute(0, 1, 4, 3, 2, 5)
        return cls(data, blocks.reshape(mats, rb, kw, 512), (*lead, K))

    def parts(self) -> tuple[torch.Tensor, torch.Tensor]:
        """(codes, scales) in row order, as `from_parts` takes them."""
        *lead, K = self.shape
        mats, rb, kw, _ = self.scales.shape
        words = self.scales.view(mats, rb, kw, 32, 4, 4).permute(0, 1, 4, 3, 2, 5).reshape(mats, rb * 128, 4 * kw)
        nb = -(-K // BLOCK)
        return self.data.clone(), words[:, : lead[-1], :nb].reshape(*lead, nb).clone()

    def __repr__(self) -> str:
        return f"MXFP4Tensor(shape={tuple(self.shape)}, device={self.device})"


def _round_up(a: int, b: int) -> int:
    return -(-a // b) * b


def _scale_shape(shape):
    """Shape of the scale blocks of a (..., rows, K) operand."""
    return math.prod(shape[:-2]), -(-shape[-2] // 128), -(-shape[-1] // 128), 512


def _rows2d(x: torch.Tensor):
    """(tensor, ldx, rows, K) of x (..., rows, K): values along K contiguous."""
    K = x.shape[-1]
    if x.dim() != 2:
        x = x.reshape(math.prod(x.shape[:-1]), K)
    rows = x.shape[0]
    s0, s1 = x.stride()
    if (s1 != 1 and K > 1) or (rows > 1 and s0 < K):
        x, s0 = x.contiguous(), K
    return x, max(s0, K), rows, K


def _unchecked(data, scales, shape) -> MXFP4Tensor:
    """An MXFP4Tensor of this module's own making."""
    q = object.__new__(MXFP4Tensor)
    q.data, q.scales, q.shape = data, scales, shape
    return q


def _quantize(x: torch.Tensor) -> MXFP4Tensor:
    """x (..., rows, K) on a CUDA device."""
    x2, ldx, rows, K = _rows2d(x)
    lead = x.shape[:-1]
    ldq = _round_up(K, BLOCK) // 2
    dev = x.device
    data = empty((rows, ldq), torch.uint8, dev)
    if x.dim() != 2:
        data = data.view(*lead, ldq)
    sshape = _scale_shape(x.shape)
    _, rb, kw, _ = sshape
    scales = torch.empty_strided(sshape, (rb * kw * 512, kw * 512, 512, 1), dtype=torch.uint8, device=dev)
    if rows and K:
        rc = call_on(dev, N.lib().trnblas_mxfp4_quantize, N.dtype_code(x.dtype), sshape[0], x.shape[-2], K,
                     x2.data_ptr(), ldx, data.data_ptr(), ldq, scales.data_ptr())
        if rc:
            N.check(rc, "trnblas_mxfp4_quantize")
        N.count_launches(1)
    return _unchecked(data, scales, x.shape)


def quantize_mxfp4(x: torch.Tensor) -> MXFP4Tensor:
    """x (..., rows, K) in blocks of 32 along the last dimension.

    A block's scale is the largest power of two not above its largest
    magnitude, divided by 4 (at least 2^-127); values round to the nearest E2M1
    value, ties to the even mantissa, and what lies above 6 of the scale becomes
    6. A block that holds an infinity or a NaN becomes NaN. float32, bfloat16
    or float16; the result is on x's device. Not differentiable.
    """
    if not isinstance(x, torch.Tensor) or x.dtype not in _OUT:
        raise TypeError(f"quantize_mxfp4: a float32, bfloat16 or float16 tensor, got {getattr(x, 'dtype', type(x))}")
    if x.dim() < 2:
        raise ValueError(f"quantize_mxfp4: a tensor (..., rows, K), got {tuple(x.shape)}")
    if x.is_cuda:
        return _quantize(x)
    dev = _cuda_device(x)
    q = _quantize(_to(x, dev))
    return q if x.device == dev else q.to(x.device)


def dequantize_mxfp4(q: MXFP4Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values of a quantised operand, exact in float32 and bfloat16 for
    what `quantize_mxfp4` makes (float16 rounds and overflows where it must)."""
    if not isinstance(q, MXFP4Tensor):
        raise TypeError(f"dequantize_mxfp4: an MXFP4Tensor, got {type(q)}")
    if dtype not in _OUT:
        raise TypeError(f"dequantize_mxfp4: dtype is float32, bfloat16 or float16, got {dtype}")
    home = dev = q.device
    if not q.data.is_cuda:
        dev = _cuda_device(q.data)
        q = q.to(dev)
    K = q.shape[-1]
    shape = q.shape
    out = empty(shape, dtype, dev) if len(shape) == 2 else torch.empty(tuple(shape), dtype=dtype, device=dev)
    if out.numel():
        rc = call_on(dev, N.lib().trnblas_mxfp4_dequantize, N.dtype_code(dtype), q.scales.shape[0], q.shape[-2], K,
                     q.data.data_ptr(), q.data.shape[-1], q.scales.data_ptr(), out.data_ptr(), K)
        if rc:
            N.check(rc, "trnblas_mxfp4_dequantize")
        N.count_launches(1)
    return out if home == dev else _home(out, home, dev)


def _operands(name, A, B, b_dim, out_dtype):
    if not isinstance(B, MXFP4Tensor):
        raise TypeError(f"{name}: B is an MXFP4Tensor (quantize_mxfp4), got {type(B)}")
    if not isinstance(A, MXFP4Tensor) and not (isinstance(A, torch.Tensor) and A.dtype in _OUT):
        raise TypeError(f"{name}: A is an MXFP4Tensor or a float32, bfloat16 or float16 tensor")
    if out_dtype not in _OUT:
        raise TypeError(f"{name}: out_dtype is float32, bfloat16 or float16, got {out_dtype}")
    if A.dim() != 2 or B.dim() != b_dim:
        raise ValueError(f"{name}: A is 2-D and B {b_dim}-D, got {tuple(A.shape)} and {tuple(B.shape)}")
    if A.shape[1] != B.shape[-1]:
        raise ValueError(f"{name}: inner dimensions differ: A {tuple(A.shape)}, B {tuple(B.shape)}")


def _product(name, alpha, A, B, sizes, beta, C, out_dtype):
    quantised = isinstance(A, MXFP4Tensor)
    a = A.data if quantised else A
    if _same_cuda_device(a, B.data, sizes, C):
        home = dev = a.device
    else:
        home = A.device
        dev = _cuda_device(a, B.data, C, sizes)
        if B.device != dev:
            B = B.to(dev)
        if A.device != dev:
            A = A.to(dev)
        sizes, C = on_device(sizes, dev, home), on_device(C, dev, home)
    rows, K = A.shape
    Nn = B.shape[-2]
    G = B.shape[0] if sizes is not None else 1
    out = empty((rows, Nn), out_dtype, dev)
    fuse = C is not None and _fuse_c(C, beta, out.shape, out_dtype, dev)
    if rows and Nn:
        c_arg, ldc = _c_operand(C, Nn) if fuse else (None, 0)
        if sizes is not None and not sizes.is_contiguous():
            sizes = sizes.contiguous()
        tail = (B.data.data_ptr(), B.data.shape[-1], B.scales.data_ptr(), N.ptr(sizes),
                sizes is not None and sizes.dtype == torch.int64, float(beta) if fuse else 0.0, N.ptr(c_arg), ldc,
                out.data_ptr(), Nn)
        ws = None
        if quantised:
            ws_bytes = 0
            if sizes is not None:
                ws_bytes = N.lib().trnblas_mxfp4_gemm_workspace_size(rows, G, K, True)
                ws = empty((ws_bytes,), torch.uint8, dev) if ws_bytes else None
            rc = call_on(dev, N.lib().trnblas_mxfp4_gemm, N.dtype_code(out_dtype), rows, G, Nn, K, float(alpha),
                         A.data.data_ptr(), A.data.shape[-1], A.scales.data_ptr(), *tail, N.ptr(ws), ws_bytes)
        else:
            x, ldx, _, _ = _rows2d(A)
            ws_bytes = N.lib().trnblas_mxfp4_gemm_x_workspace_size(rows, G, K, sizes is not None)
            ws = empty((ws_bytes,), torch.uint8, dev) if ws_bytes else None
            rc = call_on(dev, N.lib().trnblas_mxfp4_gemm_x, N.dtype_code(x.dtype), N.dtype_code(out_dtype), rows, G, Nn,
                         K, float(alpha), x.data_ptr(), ldx, *tail, N.ptr(ws), ws_bytes)
        if rc:
            N.check(rc, name)
        # (quantiser or regrouping +) the product; a few rows quantise in the product
        N.count_launches(2 if ws is not None else 1)
    if C is not None and not fuse:
        out = _add_c(out, beta, C.detach() if isinstance(C, torch.Tensor) else C)
    return out if home == dev else _home(out, home, dev)


def gemm_mxfp4(
    alpha: float,
    A,
    B: MXFP4Tensor,
    beta: float = 0.0,
    C: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.bfloat16,
) -> torch.Tensor:
    """alpha * A @ B^T + beta * C on the block-scaled 4-bit tensor cores.

    B is a quantised (N, K) operand (weights, quantised once). A is a quantised
    (M, K) operand, or a float32, bfloat16 or float16 matrix, which is quantised
    on the way. Products of the 4-bit values are exact and accumulate in
    fp32; the result (M, N) has out_dtype. A C of the result's shape and dtype
    is fused, another is added afterwards. Not differentiable.
    """
    _operands("gemm_mxfp4", A, B, 2, out_dtype)
    return _product("gemm_mxfp4", alpha, A, B, None, beta, C, out_dtype)


def grouped_gemm_mxfp4(
    alpha: float,
    A,
    B: MXFP4Tensor,
    group_sizes: torch.Tensor,
    beta: float = 0.0,
    C: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.bfloat16,
) -> torch.Tensor:
    """D[r] = alpha * A[r] @ B[g]^T + beta * C[r] for the rows r of group g:
    `grouped_gemm` on 4-bit operands. B is a quantised (G, N, K) operand, A as
    for `gemm_mxfp4`, group_sizes and the rows behind the last group as for
    `grouped_gemm`. Not differentiable.
    """
    name = "grouped_gemm_mxfp4"
    _operands(name, A, B, 3, out_dtype)
    check_group_sizes(name, group_sizes, B.shape[0], A.shape[0])
    return _product(name, alpha, A, B, group_sizes, beta, C, out_dtype)
