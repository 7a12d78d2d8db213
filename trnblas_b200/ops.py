"""The kernel boundary as functional torch ops: `torch.ops.trnblas.*`.

The analogue of the reference's op table (trnblas/nki/_native.py:49-259:
every kernel registered with `nki_op("trnblas::<name>", mutates_args={},
fake_fn=...)`, collected in `OPS` at :243-259 and wrapped by `_dtype_checked`
at :262-280). Here each op is a `torch.library.custom_op` whose CUDA
implementation calls the C ABI of include/trnblas_b200.h on the operands'
device and current stream, with a fake (meta) implementation that gives the
output's shape and dtype without touching data, so the ops trace under
FakeTensorMode and torch.compile. They are functional: inputs are read,
outputs are fresh.

    gemm(a, b, alpha, beta, c, ta, tb)            alpha op(a) op(b) + beta c  (2-D)
    batched_gemm(a, b, alpha, beta, c, ta, tb)    the same over a leading batch dim
    syrk(a, alpha, beta, c, lower_c, trans)       alpha a a^T + beta sym(c), full n x n
    ozaki_split(x, k) -> (digits, exps)           k int8 digit planes, per-row exponents
    ozaki_gemm(a, b, k) -> float64                fp64-class a @ b on the int8 pipe
    pair_energy(B, eo, ev, p0, p1) -> float64 0-d the pair-range DF-MP2 energy

    grouped_gemm(a, b, group_sizes, alpha, tb, out_dtype)       rows by expert (with autograd)
    grouped_gemm_wgrad(a, b, group_sizes, alpha, out_dtype)     its weights' gradient
    quantize_mxfp4(x) -> (data, scales)           and dequantize_mxfp4(data, scales, k, dtype)
    gemm_mxfp4(x, b_data, b_scales, alpha, out_dtype, k)        and grouped_gemm_mxfp4 (+ group_sizes);
                                                  k (the weights' K) where it is no multiple of 32

`OPS[name](*args)` calls the op after the reference's operand dtype check:
a tensor of a dtype the kernel does not take raises TypeError naming the op.
"""

from __future__ import annotations

import torch

from . import _native as N
from . import experts as _ex
from . import level3 as _l3
from . import mxfp4 as _mx

_F16 = (torch.float32, torch.bfloat16, torch.float16)


def _check_2d(name, *xs):
    for x in xs:
        if x.dim() != 2:
            raise ValueError(f"trnblas::{name}: expected 2-D operands, got shape {tuple(x.shape)}")


def _gemm_shape(a, b, ta, tb):
    M = a.shape[1] if ta else a.shape[0]
    K = a.shape[0] if ta else a.shape[1]
    K2 = b.shape[1] if tb else b.shape[0]
    Nn = b.shape[0] if tb else b.shape[1]
    return M, K, K2, Nn


# ── GEMM ────────────────────────────────────────────────────────────────────


@torch.library.custom_op("trnblas::gemm", mutates_args=(), device_types="cuda")
def gemm(a: torch.Tensor, b: torch.Tensor, alpha: float = 1.0, beta: float = 0.0,
         c: torch.Tensor | None = None, ta: bool = False, tb: bool = False) -> torch.Tensor:
    _check_2d("gemm", a, b)
    if a.dtype != b.dtype:
        raise RuntimeError(f"trnblas::gemm: operand dtypes differ ({a.dtype}, {b.dtype})")
    M, K, K2, Nn = _gemm_shape(a, b, ta, tb)
    if K != K2:
        raise ValueError(f"trnblas::gemm: inner dimensions differ ({K}, {K2})")
    fuse = c is not None and beta != 0.0
    if fuse and (tuple(c.shape) != (M, Nn) or c.dtype != a.dtype):
        raise ValueError(f"trnblas::gemm: c must be ({M}, {Nn}) {a.dtype}, got {tuple(c.shape)} {c.dtype}")
    return _l3._gemm2d(a.mT if ta else a, b.mT if tb else b, alpha, beta if fuse else 0.0, c if fuse else None)


@gemm.register_fake
def _(a, b, alpha=1.0, beta=0.0, c=None, ta=False, tb=False):
    M, K, K2, Nn = _gemm_shape(a, b, ta, tb)
    torch._check(K == K2, lambda: "trnblas::gemm: inner dimensions differ")
    return a.new_empty((M, Nn))


@torch.library.custom_op("trnblas::batched_gemm", mutates_args=(), device_types="cuda")
def batched_gemm(a: torch.Tensor, b: torch.Tensor, alpha: float = 1.0, beta: float = 0.0,
                 c: torch.Tensor | None = None, ta: bool = False, tb: bool = False) -> torch.Tensor:
    if a.dim() != 3 or b.dim() != 3:
        raise ValueError("trnblas::batched_gemm: expected 3-D (batch, rows, cols) operands")
    r = _l3._batched(alpha, a.mT if ta else a, b.mT if tb else b, beta, c)
    return r if r.data_ptr() not in (a.data_ptr(), b.data_ptr()) else r.clone()


@batched_gemm.register_fake
def _(a, b, alpha=1.0, beta=0.0, c=None, ta=False, tb=False):
    M = a.shape[2] if ta else a.shape[1]
    Nn = b.shape[1] if tb else b.shape[2]
    batch = torch.broadcast_shapes(a.shape[:1], b.shape[:1])
    return a.new_empty((*batch, M, Nn))


@torch.library.custom_op("trnblas::syrk", mutates_args=(), device_types="cuda")
def syrk(a: torch.Tensor, alpha: float = 1.0, beta: float = 0.0, c: torch.Tensor | None = None,
         lower_c: bool = True, trans: bool = False) -> torch.Tensor:
    _check_2d("syrk", a)
    a_eff = a.mT if trans else a
    n = a_eff.shape[0]
    if c is not None and beta != 0.0:
        if tuple(c.shape) != (n, n) or c.dtype != a.dtype:
            raise ValueError(f"trnblas::syrk: c must be ({n}, {n}) {a.dtype}")
        return _l3._syrk_kernel(a_eff, alpha, beta, c, 1 if lower_c else 2)
    return _l3._syrk_kernel(a_eff, alpha, 0.0, None, 0)


@syrk.register_fake
def _(a, alpha=1.0, beta=0.0, c=None, lower_c=True, trans=False):
    n = a.shape[1] if trans else a.shape[0]
    return a.new_empty((n, n))


# ── fp64-class GEMM (Ozaki on the int8 tensor cores) ────────────────────────


@torch.library.custom_op("trnblas::ozaki_split", mutates_args=(), device_types="cuda")
def ozaki_split(x: torch.Tensor, k: int) -> tuple[torch.Tensor, torch.Tensor]:
    _check_2d("ozaki_split", x)
    k = _l3.check_slices(k)
    R, K = x.shape
    dig = torch.empty((k, R, K), dtype=torch.int8, device=x.device)
    ex = torch.empty((R,), dtype=torch.int32, device=x.device)
    if R == 0 or K == 0:
        return dig, ex.zero_()
    xd = x.to(torch.float64)
    ws = N.workspace(8 * R + 256, x.device)
    N.check(N.lib().trnblas_ozaki_split(R, K, N.ptr(xd), xd.stride(0), xd.stride(1), k, N.ptr(dig), K,
                                        N.ptr(ex), N.ptr(ws), 8 * R + 256, N.stream_ptr(x.device)),
            "trnblas_ozaki_split")
    return dig, ex


@ozaki_split.register_fake
def _(x, k):
    R, K = x.shape
    return x.new_empty((k, R, K), dtype=torch.int8), x.new_empty((R,), dtype=torch.int32)


@torch.library.custom_op("trnblas::ozaki_gemm", mutates_args=(), device_types="cuda")
def ozaki_gemm(a: torch.Tensor, b: torch.Tensor, k: int = 8) -> torch.Tensor:
    _check_2d("ozaki_gemm", a, b)
    if a.shape[1] != b.shape[0]:
        raise ValueError("trnblas::ozaki_gemm: inner dimensions differ")
    k = _l3.check_slices(k)
    a64, b64 = a.to(torch.float64), b.to(torch.float64)
    if a.shape[1] == 0:
        return torch.zeros((a.shape[0], b.shape[1]), dtype=torch.float64, device=a.device)
    if not _l3._all_finite(a64, b64):
        return torch.matmul(a64, b64)
    return _l3._gemm_fp64_device(a64, b64, k)


@ozaki_gemm.register_fake
def _(a, b, k=8):
    return a.new_empty((a.shape[0], b.shape[1]), dtype=torch.float64)


# ── DF-MP2 pair energy ──────────────────────────────────────────────────────


@torch.library.custom_op("trnblas::pair_energy", mutates_args=(), device_types="cuda")
def pair_energy(B: torch.Tensor, eo: torch.Tensor, ev: torch.Tensor, pair_begin: int,
                pair_end: int) -> torch.Tensor:
    from .energy import pair_range_energy

    return pair_range_energy(B, eo, ev, pair_begin, pair_end)


@pair_energy.register_fake
def _(B, eo, ev, pair_begin, pair_end):
    return B.new_empty((), dtype=torch.float64)


# ── the op table with the reference's operand dtype check ───────────────────

# operand dtypes each kernel takes (trnblas/nki/dispatch.py:1259-1293,
# `_KERNEL_DTYPES`): the floating point tensors among an op's arguments
KERNEL_DTYPES = {
    "gemm": _F16,
    "batched_gemm": _F16,
    "syrk": _F16,
    "ozaki_split": (torch.float64, torch.float32),
    "ozaki_gemm": (torch.float64, torch.float32),
    "pair_energy": (torch.float32, torch.float64),
}

_RAW = {"gemm": gemm, "batched_gemm": batched_gemm, "syrk": syrk, "ozaki_split": ozaki_split,
        "ozaki_gemm": ozaki_gemm, "pair_energy": pair_energy}


def check_kernel_operands(name: str, *args) -> None:
    """TypeError when a tensor argument of op `name` has a dtype its kernel
    does not take (trnblas/nki/dispatch.py:1259-1293, `_check_kernel_operands`)."""
    ok = KERNEL_DTYPES[name]
    bad = [t.dtype for t in args if isinstance(t, torch.Tensor) and t.dtype not in ok]
    if bad:
        raise TypeError(f"trnblas::{name} takes {[str(d) for d in ok]} operands, got {[str(d) for d in bad]}")


def _dtype_checked(name, op):
    def checked(*args, **kwargs):
        check_kernel_operands(name, *args, *kwargs.values())
        return op(*args, **kwargs)

    checked.__name__ = name
    checked.op = op
    return checked


OPS = {name: _dtype_checked(name, op) for name, op in _RAW.items()}

__all__ = ["OPS", "KERNEL_DTYPES", "check_kernel_operands", "gemm", "batched_gemm", "syrk",
           "ozaki_split", "ozaki_gemm", "pair_energy"]


# ── products grouped by expert and in 4 bits ────────────────────────────────
# No counterparts in the reference, so they stand in a table of their own.
# The 4-bit operands are the (data, scales) pairs of `MXFP4Tensor`, which do not
# hold the logical K: `k` is that, checked against the other operand. Without
# it a product's weights are as wide as their data, whole blocks of 32.


@torch.library.custom_op("trnblas::grouped_gemm", mutates_args=(), device_types="cuda")
def grouped_gemm(a: torch.Tensor, b: torch.Tensor, group_sizes: torch.Tensor, alpha: float = 1.0,
                 tb: bool = False, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    with torch.no_grad():
        return _ex.grouped_gemm(alpha, a, b, group_sizes, transB=tb, out_dtype=out_dtype)


@grouped_gemm.register_fake
def _(a, b, group_sizes, alpha=1.0, tb=False, out_dtype=None):
    torch._check(a.shape[1] == b.shape[2 if tb else 1], lambda: "trnblas::grouped_gemm: inner dimensions differ")
    return a.new_empty((a.shape[0], b.shape[1 if tb else 2]), dtype=out_dtype or a.dtype)


def _grouped_setup(ctx, inputs, output):
    a, b, sizes, alpha, tb, _ = inputs
    ctx.save_for_backward(a, b, sizes)
    ctx.alpha, ctx.tb = alpha, tb


def _grouped_backward(ctx, d):
    a, b, sizes = ctx.saved_tensors
    y = d.to(a.dtype)
    da = db = None
    if ctx.needs_input_grad[0]:
        da = torch.ops.trnblas.grouped_gemm(y, b, sizes, ctx.alpha, not ctx.tb, None)
    if ctx.needs_input_grad[1]:
        l, r = (y, a) if ctx.tb else (a, y)
        db = torch.ops.trnblas.grouped_gemm_wgrad(l, r, sizes, ctx.alpha, None)
    return da, db, None, None, None, None


grouped_gemm.register_autograd(_grouped_backward, setup_context=_grouped_setup)


@torch.library.custom_op("trnblas::grouped_gemm_wgrad", mutates_args=(), device_types="cuda")
def grouped_gemm_wgrad(a: torch.Tensor, b: torch.Tensor, group_sizes: torch.Tensor, alpha: float = 1.0,
                       out_dtype: torch.dtype | None = None) -> torch.Tensor:
    return _ex.grouped_gemm_wgrad(alpha, a, b, group_sizes, out_dtype=out_dtype)


@grouped_gemm_wgrad.register_fake
def _(a, b, group_sizes, alpha=1.0, out_dtype=None):
    return a.new_empty((group_sizes.shape[0], a.shape[1], b.shape[1]), dtype=out_dtype or a.dtype)


@torch.library.custom_op("trnblas::quantize_mxfp4", mutates_args=(), device_types="cuda")
def quantize_mxfp4(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    q = _mx.quantize_mxfp4(x)
    return q.data, q.scales


@quantize_mxfp4.register_fake
def _(x):
    return (x.new_empty((*x.shape[:-1], (x.shape[-1] + 31) // 32 * 16), dtype=torch.uint8),
            x.new_empty(_mx._scale_shape(x.shape), dtype=torch.uint8))


@torch.library.custom_op("trnblas::dequantize_mxfp4", mutates_args=(), device_types="cuda")
def dequantize_mxfp4(data: torch.Tensor, scales: torch.Tensor, k: int, dtype: torch.dtype) -> torch.Tensor:
    return _mx.dequantize_mxfp4(_mx.MXFP4Tensor(data, scales, (*data.shape[:-1], k)), dtype)


@dequantize_mxfp4.register_fake
def _(data, scales, k, dtype):
    return data.new_empty((*data.shape[:-1], k), dtype=dtype)


def _weights4(data, scales, k):
    return _mx.MXFP4Tensor(data, scales, (*data.shape[:-1], 2 * data.shape[-1] if k is None else k))


def _check_k(name, x, data, k):
    torch._check((x.shape[1] + 31) // 32 * 16 == data.shape[-1] and k in (None, x.shape[1]),
                 lambda: f"trnblas::{name}: inner dimensions differ")


@torch.library.custom_op("trnblas::gemm_mxfp4", mutates_args=(), device_types="cuda")
def gemm_mxfp4(x: torch.Tensor, b_data: torch.Tensor, b_scales: torch.Tensor, alpha: float = 1.0,
               out_dtype: torch.dtype = torch.bfloat16, k: int | None = None) -> torch.Tensor:
    return _mx.gemm_mxfp4(alpha, x, _weights4(b_data, b_scales, k), out_dtype=out_dtype)


@gemm_mxfp4.register_fake
def _(x, b_data, b_scales, alpha=1.0, out_dtype=torch.bfloat16, k=None):
    _check_k("gemm_mxfp4", x, b_data, k)
    return x.new_empty((x.shape[0], b_data.shape[0]), dtype=out_dtype)


@torch.library.custom_op("trnblas::grouped_gemm_mxfp4", mutates_args=(), device_types="cuda")
def grouped_gemm_mxfp4(x: torch.Tensor, b_data: torch.Tensor, b_scales: torch.Tensor, group_sizes: torch.Tensor,
                       alpha: float = 1.0, out_dtype: torch.dtype = torch.bfloat16, k: int | None = None) -> torch.Tensor:
    return _mx.grouped_gemm_mxfp4(alpha, x, _weights4(b_data, b_scales, k), group_sizes, out_dtype=out_dtype)


@grouped_gemm_mxfp4.register_fake
def _(x, b_data, b_scales, group_sizes, alpha=1.0, out_dtype=torch.bfloat16, k=None):
    _check_k("grouped_gemm_mxfp4", x, b_data, k)
    return x.new_empty((x.shape[0], b_data.shape[1]), dtype=out_dtype)


EXPERT_OPS = {"grouped_gemm": grouped_gemm, "grouped_gemm_wgrad": grouped_gemm_wgrad,
              "quantize_mxfp4": quantize_mxfp4, "dequantize_mxfp4": dequantize_mxfp4, "gemm_mxfp4": gemm_mxfp4,
              "grouped_gemm_mxfp4": grouped_gemm_mxfp4}

__all__ += ["EXPERT_OPS", *EXPERT_OPS]
