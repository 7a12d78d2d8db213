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
from .experts import _c_operand, _on, check_group_sizes
from .level3 import _add_c, _cuda_device, _fuse_c, _home, _to

BLOCK = 32
_OUT = (torch.bfloat16, torch.float16, torch.float32)


class MXFP4Tensor:
    """A quantised (..., rows, K) operand.

    data    uint8 (..., rows, round_up(K, 32) / 2): two values a byte, the even
            one in the low half, zero behind K;
    scales  uint8 (ceil(K / 128), all rows, 4): the E8M0 bytes of a row's four
            blocks in 128 values; what a tensor-core tile reads is contiguous
            whatever row it starts at;
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
        want = (-(-K // 128), math.prod(lead), 4)
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
        kw = -(-K // 128)
        rows = math.prod(lead)
        words = scales.new_zeros((rows, 4 * kw))
        words[:, :nb] = scales.reshape(rows, nb)
        return cls(data, words.view(rows, kw, 4).transpose(0, 1).contiguous(), (*lead, K))

    def parts(self) -> tuple[torch.Tensor, torch.Tensor]:
        """(codes, scales) in row order, as `from_parts` takes them."""
        *lead, K = self.shape
        rows, nb = math.prod(lead), -(-K // BLOCK)
        s = self.scales.transpose(0, 1).reshape(rows, -1)[:, :nb]
        return self.data.clone(), s.reshape(*lead, nb).clone()

    def __repr__(self) -> str:
        return f"MXFP4Tensor(shape={tuple(self.shape)}, device={self.device})"


def _round_up(a: int, b: int) -> int:
    return -(-a // b) * b


def _quantize(x: torch.Tensor) -> MXFP4Tensor:
    """x (..., rows, K) on a CUDA device."""
    *lead, K = x.shape
    rows = math.prod(lead)
    x2 = x.detach().reshape(rows, K)
    if K and x2.stride(1) != 1 and K > 1 or (rows > 1 and x2.stride(0) < K):
        x2 = x2.contiguous()
    ldq = _round_up(K, BLOCK) // 2
    data = torch.empty((*lead, ldq), dtype=torch.uint8, device=x.device)
    scales = torch.empty((-(-K // 128), rows, 4), dtype=torch.uint8, device=x.device)
    if rows and K:
        with _on(x.device):
            rc = N.lib().trnblas_mxfp4_quantize(
                N.dtype_code(x.dtype), rows, K, N.ptr(x2), max(x2.stride(0), K), N.ptr(data), ldq, N.ptr(scales),
                N.stream_ptr(x.device))
        N.check(rc, "trnblas_mxfp4_quantize")
        N.count_launches(1)
    return MXFP4Tensor(data, scales, x.shape)


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
    home = q.device
    dev = _cuda_device(q.data)
    if home != dev:
        q = q.to(dev)
    *lead, K = q.shape
    rows = math.prod(lead)
    out = torch.empty(tuple(q.shape), dtype=dtype, device=dev)
    if out.numel():
        with _on(dev):
            rc = N.lib().trnblas_mxfp4_dequantize(
                N.dtype_code(dtype), rows, K, N.ptr(q.data), q.data.shape[-1], N.ptr(q.scales), N.ptr(out), K,
                N.stream_ptr(dev))
        N.check(rc, "trnblas_mxfp4_dequantize")
        N.count_launches(1)
    return _home(out, home, dev)


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
    home = A.device
    dev = _cuda_device(A if isinstance(A, torch.Tensor) else A.data, B.data, C, sizes)
    if B.device != dev:
        B = B.to(dev)
    if isinstance(A, MXFP4Tensor):
        qa = A if A.device == dev else A.to(dev)
    else:
        qa = _quantize(_to(A, dev))
    sizes, Cd = _to(sizes, dev), _to(C, dev)
    rows, K = A.shape
    Nn = B.shape[-2]
    G = B.shape[0] if sizes is not None else 1
    out = torch.empty((rows, Nn), dtype=out_dtype, device=dev)
    fuse = _fuse_c(Cd, beta, out.shape, out_dtype, dev)
    if out.numel():
        c_arg, ldc = _c_operand(Cd.detach(), Nn) if fuse else (None, 0)
        if sizes is not None:
            sizes = sizes.contiguous()
        with _on(dev):
            rc = N.lib().trnblas_mxfp4_gemm(
                N.dtype_code(out_dtype), rows, G, Nn, K, float(alpha), N.ptr(qa.data), qa.data.shape[-1],
                N.ptr(qa.scales), N.ptr(B.data), B.data.shape[-1], N.ptr(B.scales), N.ptr(sizes),
                int(sizes is not None and sizes.dtype == torch.int64), float(beta) if fuse else 0.0, N.ptr(c_arg),
                ldc, N.ptr(out), Nn, N.stream_ptr(dev))
        N.check(rc, name)
        N.count_launches(1)
    if not fuse:
        out = _add_c(out, beta, Cd.detach() if isinstance(Cd, torch.Tensor) else Cd)
    return _home(out, home, dev)


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
