"""Plain 64-bit restatement of the products grouped by expert and of MXFP4.

Torch in float64 on the operands' device, one group at a time, written from
the definitions; the tolerances are derived here, beside the arithmetic.
"""

from __future__ import annotations

import torch

VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def ranges(sizes):
    """(group, first row, end row) of each group."""
    r = 0
    for g, m in enumerate(sizes):
        yield g, r, r + m
        r += m


def grouped_gemm(alpha, A, B, sizes, beta=0.0, C=None, transB=False):
    """(result, sum of the products' magnitudes), both float64."""
    b = (B.mT if transB else B).double()
    a = A.double()
    D = torch.zeros(a.shape[0], b.shape[2], dtype=torch.float64, device=a.device)
    S = torch.zeros_like(D)
    for g, r0, r1 in ranges(sizes):
        D[r0:r1] = alpha * (a[r0:r1] @ b[g])
        S[r0:r1] = abs(alpha) * (a[r0:r1].abs() @ b[g].abs())
    if C is not None and beta != 0.0:
        D = D + beta * C.double()
    return D, S


def wgrad(alpha, A, B, sizes, beta=0.0, C=None):
    a, b = A.double(), B.double()
    D = torch.zeros(len(sizes), a.shape[1], b.shape[1], dtype=torch.float64, device=a.device)
    S = torch.zeros_like(D)
    for g, r0, r1 in ranges(sizes):
        D[g] = alpha * (a[r0:r1].T @ b[r0:r1])
        S[g] = abs(alpha) * (a[r0:r1].abs().T @ b[r0:r1].abs())
    if C is not None and beta != 0.0:
        D = D + beta * C.double()
    return D, S


def tolerance(ref, mags, terms, out_dtype, beta_c=None):
    """What the kernels' arithmetic may be off, element by element.

    Products of 16-bit (or 4-bit, scaled) values are exact in fp32. Each of the
    `terms` additions into an fp32 sum truncates by less than 2^-23 of a partial
    sum, and no partial sum exceeds the sum of the magnitudes; alpha's product
    rounds by 2^-24. With a C: beta * C and the sum round in fp32. The result
    rounds once to its type: half a step, eps / 2 of the value, or half the
    smallest subnormal step.
    """
    fp32 = (terms + 1) * 2.0 ** -23 * mags + 2.0 ** -23 * ref.abs()
    if beta_c is not None:
        fp32 = fp32 + 2.0 ** -23 * beta_c.double().abs()
    half = torch.finfo(out_dtype).eps / 2
    step = torch.finfo(out_dtype).smallest_normal * torch.finfo(out_dtype).eps / 2
    return fp32 * (1 + half) + half * ref.abs() + step


def check(out, ref, tol, what=""):
    """out within tol of ref. A value above the type's largest by half a step
    or more rounds to an infinity of its sign (fp16 from 65520 on), so there
    the infinity is the right answer, and only there."""
    top = torch.finfo(out.dtype).max
    inf = out.isinf()
    assert not out.isnan().any(), f"{what}: NaN"
    assert (ref.abs() + tol >= top)[inf].all() and (torch.sign(out.double()) == torch.sign(ref))[inf].all(), (
        f"{what}: infinities where the values are in range")
    # (half a step above the largest value is below top * (1 + eps / 2))
    assert inf[ref.abs() - tol > top * (1 + torch.finfo(out.dtype).eps / 2)].all(), f"{what}: an overflow is not infinite"
    err = torch.where(inf, 0.0, (out.double() - ref).abs())
    worst = (err - tol).max() if err.numel() else torch.tensor(0.0)
    assert (err <= tol).all(), f"{what}: {(err > tol).sum().item()} elements off by up to {worst.item():.3g} above the bound"


def quantize(x):
    """(values as multiples of the block's unit, unit exponents, whole blocks'
    NaN mask) of x (rows, K) by the definition, in float64."""
    rows, K = x.shape
    nb = -(-K // 32)
    xp = torch.zeros(rows, nb * 32, dtype=torch.float64, device=x.device)
    xp[:, :K] = x.double()
    xp = xp.view(rows, nb, 32)
    amax = xp.abs().amax(-1)
    bad = ~torch.isfinite(amax)
    amax = torch.where(bad, torch.zeros_like(amax), amax)
    e = torch.full(amax.shape, -127, dtype=torch.int64, device=x.device)
    for k in range(-124, 126):  # e = k where 2^(k + 2) <= amax
        e = torch.where(amax >= 2.0 ** (k + 2), k, e)
    e = torch.where(amax >= 2.0 ** -124, e, -127)
    for k in (-126, -125):
        e = torch.where((amax >= 2.0 ** (k + 2)) & (amax < 2.0 ** (k + 3)), k, e)
    t = xp / torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double().cpu()).to(x.device).unsqueeze(-1)
    vals = torch.tensor(VALUES, dtype=torch.float64, device=x.device)
    d = (t.abs().unsqueeze(-1) - vals).abs()
    best = d.amin(-1, keepdim=True)
    near = d == best
    # two neighbours at the same distance: the one with the even code (mantissa bit 0)
    even = torch.tensor([i % 2 == 0 for i in range(8)], device=x.device)
    both = near.sum(-1, keepdim=True) > 1
    code = torch.where(both, near & even, near).double().argmax(-1)
    q = torch.copysign(vals[code], t)
    return q, e, bad


def dequantize(q, e, bad, K):
    """float64 values (rows, K) of `quantize`'s result."""
    unit = torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double().cpu()).to(q.device).unsqueeze(-1)
    v = q * unit
    v = torch.where(bad.unsqueeze(-1), torch.full_like(v, float("nan")), v)
    return v.reshape(q.shape[0], -1)[:, :K]
