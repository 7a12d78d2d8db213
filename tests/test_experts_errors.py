"""Refusals of the grouped and 4-bit products, before any device work, and the
host side of the packed format (CPU)."""

from __future__ import annotations

import pytest
import torch

import trnblas_b200 as tb
from oracle import experts as X
from trnblas_b200 import _native as N

BF = torch.bfloat16
A, B, S = torch.zeros(6, 8, dtype=BF), torch.zeros(2, 8, 4, dtype=BF), torch.tensor([3, 3])


def _mx(*shape):
    *lead, K = shape
    rows = 1
    for n in lead:
        rows *= n
    return tb.MXFP4Tensor(torch.zeros(*lead, -(-K // 32) * 16, dtype=torch.uint8),
                          torch.zeros(rows // lead[-1], -(-lead[-1] // 128), -(-K // 128), 512, dtype=torch.uint8), shape)


@pytest.mark.parametrize("call,exc", [
    (lambda: tb.grouped_gemm(1.0, A.float(), B.float(), S), TypeError),
    (lambda: tb.grouped_gemm(1.0, A, B.half(), S), RuntimeError),
    (lambda: tb.grouped_gemm(1.0, A, B, S, out_dtype=torch.float16), TypeError),
    (lambda: tb.grouped_gemm(1.0, A[0], B, S), ValueError),
    (lambda: tb.grouped_gemm(1.0, A, B[0], S), ValueError),
    (lambda: tb.grouped_gemm(1.0, A, B, S, transB=True), ValueError),
    (lambda: tb.grouped_gemm(1.0, A, B, S, transB="C"), ValueError),
    (lambda: tb.grouped_gemm(1.0, A, B, [3, 3]), ValueError),
    (lambda: tb.grouped_gemm(1.0, A, B, S.float()), ValueError),
    (lambda: tb.grouped_gemm(1.0, A, B, S.view(1, 2)), ValueError),
    (lambda: tb.grouped_gemm(1.0, A, B, torch.tensor([3, 2, 1])), ValueError),
    (lambda: tb.grouped_gemm(1.0, A, B, torch.tensor([3, 4])), ValueError),
    (lambda: tb.grouped_gemm(1.0, A, B, torch.tensor([-1, 4])), ValueError),
    (lambda: tb.grouped_gemm(1.0, A, B[:1].expand(1025, 8, 4), torch.zeros(1025, dtype=torch.int32)), ValueError),
    (lambda: tb.grouped_gemm_wgrad(1.0, A, A[:5], S), ValueError),
    (lambda: tb.grouped_gemm_wgrad(1.0, A, A.half(), S), RuntimeError),
    (lambda: tb.grouped_gemm_wgrad(1.0, A, A, torch.tensor([3, 4])), ValueError),
    (lambda: tb.grouped_gemm_wgrad(1.0, A, A, torch.zeros(1025, dtype=torch.int64)), ValueError),
    (lambda: tb.quantize_mxfp4(A.double()), TypeError),
    (lambda: tb.quantize_mxfp4(A[0]), ValueError),
    (lambda: tb.dequantize_mxfp4(A), TypeError),
    (lambda: tb.dequantize_mxfp4(_mx(3, 64), torch.float64), TypeError),
    (lambda: tb.gemm_mxfp4(1.0, A, A), TypeError),
    (lambda: tb.gemm_mxfp4(1.0, A.double(), _mx(3, 8)), TypeError),
    (lambda: tb.gemm_mxfp4(1.0, A, _mx(3, 9)), ValueError),
    (lambda: tb.gemm_mxfp4(1.0, A, _mx(2, 3, 8)), ValueError),
    (lambda: tb.gemm_mxfp4(1.0, A, _mx(3, 8), out_dtype=torch.float64), TypeError),
    (lambda: tb.grouped_gemm_mxfp4(1.0, A, _mx(3, 8), S), ValueError),
    (lambda: tb.grouped_gemm_mxfp4(1.0, A, _mx(2, 3, 8), torch.tensor([6, 1])), ValueError),
    (lambda: tb.grouped_gemm_mxfp4(1.0, A, _mx(2, 3, 8), torch.tensor([6])), ValueError),
    (lambda: tb.MXFP4Tensor(torch.zeros(3, 16, dtype=torch.uint8), torch.zeros(1, 1, 1, 512, dtype=torch.uint8), (3, 33)), ValueError),
    (lambda: tb.MXFP4Tensor(torch.zeros(3, 16), torch.zeros(1, 1, 1, 512, dtype=torch.uint8), (3, 32)), ValueError),
    (lambda: tb.MXFP4Tensor(torch.zeros(3, 16, dtype=torch.uint8), torch.zeros(1, 1, 2, 512, dtype=torch.uint8), (3, 32)), ValueError),
    (lambda: tb.MXFP4Tensor.from_parts(torch.zeros(3, 16), torch.zeros(3, 1, dtype=torch.uint8), 32), TypeError),
    (lambda: tb.MXFP4Tensor.from_parts(torch.zeros(3, 15, dtype=torch.uint8), torch.zeros(3, 1, dtype=torch.uint8), 32), ValueError),
    (lambda: tb.MXFP4Tensor.from_parts(torch.zeros(3, 16, dtype=torch.uint8), torch.zeros(3, 2, dtype=torch.uint8), 32), ValueError),
])
def test_refused_before_device_work(call, exc):
    with pytest.raises(exc):
        call()


FAKE = 1 << 20  # a non-NULL address that the argument checks reject before any use


def test_c_entry_points_check_their_arguments():
    L = N.lib()
    ok = dict(dt=N.BF16, od=N.BF16, rows=4, G=2, n=8, k=8, a=FAKE, lda=8, b=FAKE, ldb=8, sb=64, tb=0, s=FAKE, c=None,
              ldc=0, d=FAKE, ldd=8)

    def grouped(**kw):
        v = {**ok, **kw}
        return L.trnblas_grouped_gemm(v["dt"], v["od"], v["rows"], v["G"], v["n"], v["k"], 1.0, v["a"], v["lda"], v["b"],
                                      v["ldb"], v["sb"], v["tb"], v["s"], 0, 1.0, v["c"], v["ldc"], v["d"], v["ldd"],
                                      None, 0, None)

    for bad in (dict(dt=N.F32), dict(od=N.F16), dict(rows=-1), dict(G=1025), dict(s=None), dict(d=None), dict(ldd=7),
                dict(a=None), dict(lda=7), dict(ldb=7), dict(sb=-8), dict(c=FAKE, ldc=7), dict(rows=1 << 31), dict(tb=1, k=16)):
        assert grouped(**bad) == N.ERR_ARG, bad
    assert grouped(rows=0) == 0 and grouped(n=0) == 0

    def wgrad(**kw):
        v = {**ok, **kw}
        return L.trnblas_grouped_gemm_wgrad(v["dt"], v["od"], v["rows"], v["G"], v["k"], v["n"], 1.0, v["a"], v["lda"],
                                            v["b"], v["ldb"], v["s"], 0, 1.0, v["c"], v["ldc"], 64, v["d"], v["ldd"],
                                            v["sb"], None, 0, None)

    for bad in (dict(dt=N.F64), dict(od=N.F16), dict(G=-1), dict(s=None), dict(d=None), dict(ldd=7), dict(a=None),
                dict(lda=7), dict(ldb=7), dict(sb=63), dict(c=FAKE, ldc=7)):
        assert wgrad(**bad) == N.ERR_ARG, bad
    assert wgrad(G=0) == 0
    # operands off 16 bytes need a workspace for their copies
    for bad in (dict(a=FAKE + 2), dict(lda=9), dict(b=FAKE + 8), dict(ldb=12), dict(sb=68)):
        assert grouped(**bad) == N.ERR_WORKSPACE, bad
    for bad in (dict(a=FAKE + 2), dict(lda=9), dict(ldb=12)):
        assert wgrad(**bad) == N.ERR_WORKSPACE, bad
    size = L.trnblas_grouped_gemm_workspace_size
    assert size(4, 2, 8, 8, FAKE, 8, FAKE, 8, 64, 0) == 0
    assert size(4, 2, 8, 8, FAKE + 2, 8, FAKE, 8, 64, 0) == 256
    assert size(100, 3, 8, 30, FAKE, 30, FAKE, 8, 240, 0) == 6400
    assert size(100, 3, 9, 64, FAKE, 64, FAKE, 9, 576, 0) == 3 * 64 * 16 * 2
    assert size(100, 3, 9, 64, FAKE, 64, FAKE, 9, 0, 0) == 64 * 16 * 2  # one matrix for all
    assert L.trnblas_grouped_gemm_wgrad_workspace_size(100, 30, 8, FAKE, 30, FAKE, 8) == 6400

    q = L.trnblas_mxfp4_quantize
    for args in ((N.F64, 4, 8, FAKE, 8, FAKE, 16, FAKE), (N.F32, -1, 8, FAKE, 8, FAKE, 16, FAKE),
                 (N.F32, 4, 8, FAKE, 7, FAKE, 16, FAKE), (N.F32, 4, 8, FAKE, 8, FAKE, 8, FAKE),
                 (N.F32, 4, 33, FAKE, 33, FAKE, 16, FAKE), (N.F32, 4, 8, None, 8, FAKE, 16, FAKE),
                 (N.F32, 4, 8, FAKE, 8, FAKE + 8, 16, FAKE), (N.F32, 4, 8, FAKE, 8, FAKE, 16, FAKE + 2)):
        assert q(args[0], 1, *args[1:], None) == N.ERR_ARG, args
    assert q(N.F32, -1, 4, 8, FAKE, 8, FAKE, 16, FAKE, None) == N.ERR_ARG
    assert q(N.F32, 1, 1, (1 << 30) + 1, FAKE, 1 << 31, FAKE, 1 << 30, FAKE, None) == N.ERR_ARG
    dq = L.trnblas_mxfp4_dequantize
    for args in ((N.F64, 4, 8, FAKE, 16, FAKE, FAKE, 8), (N.F32, 4, 8, FAKE, 16, FAKE, FAKE, 7),
                 (N.F32, 4, 8, FAKE, 15, FAKE, FAKE, 8), (N.F32, 4, 8, FAKE, 16, None, FAKE, 8)):
        assert dq(args[0], 1, *args[1:], None) == N.ERR_ARG, args

    def mx(od=N.BF16, rows=4, G=1, n=8, k=64, a=FAKE, lda=32, sa=FAKE, b=FAKE, ldb=32, sb=FAKE, s=None, c=None, ldc=0,
           d=FAKE, ldd=8):
        return L.trnblas_mxfp4_gemm(od, rows, G, n, k, 1.0, a, lda, sa, b, ldb, sb, s, 0, 1.0, c, ldc, d, ldd, None, 0, None)

    for bad in (dict(od=N.F64), dict(rows=-1), dict(G=2), dict(G=1025, s=FAKE), dict(d=None), dict(ldd=7), dict(lda=16),
                dict(ldb=31), dict(a=None), dict(sa=FAKE + 1), dict(sb=None), dict(c=FAKE, ldc=7)):
        assert mx(**bad) == N.ERR_ARG, bad
    assert mx(rows=0) == 0
    assert mx(s=FAKE) == N.ERR_WORKSPACE  # grouped: the scale blocks need a workspace
    assert L.trnblas_mxfp4_gemm_workspace_size(300, 2, 200, 1) == (3 + 2) * 2 * 512
    assert L.trnblas_mxfp4_gemm_workspace_size(300, 1, 200, 0) == 0
    assert L.trnblas_mxfp4_gemm_x_workspace_size(300, 2, 200, 1) == 300 * 112 + 5 * 2 * 512

    def gx(dt=N.BF16, ws=FAKE, n=1 << 20, x=FAKE, ldx=64, rows=40):
        return L.trnblas_mxfp4_gemm_x(dt, N.BF16, rows, 1, 8, 64, 1.0, x, ldx, FAKE, 32, FAKE, None, 0, 0.0, None, 0, FAKE, 8,
                                      ws, n, None)

    assert L.trnblas_mxfp4_gemm_x_workspace_size(16, 1, 1 << 14, 0) == 0  # a few rows quantise in the product
    for bad in (dict(dt=N.F64), dict(x=None), dict(ldx=63), dict(rows=4, x=None), dict(rows=4, ldx=63)):
        assert gx(**bad) == N.ERR_ARG, bad
    for bad in (dict(ws=None), dict(ws=FAKE + 8), dict(n=40 * 32 + 511)):
        assert gx(**bad) == N.ERR_WORKSPACE, bad


@pytest.mark.parametrize("K", [1, 2, 31, 32, 33, 64, 127, 128, 129, 300])
def test_parts_round_trip(K):
    g = torch.Generator().manual_seed(K)
    nb = -(-K // 32)
    codes = torch.randint(0, 256, (2, 5, -(-K // 2)), dtype=torch.uint8, generator=g)
    scales = torch.randint(0, 256, (2, 5, nb), dtype=torch.uint8, generator=g)
    q = tb.MXFP4Tensor.from_parts(codes, scales, K)
    assert q.shape == (2, 5, K) and q.dim() == 3
    c, s = q.parts()
    assert torch.equal(s, scales)
    want = codes.clone()
    if K % 2:
        want[..., -1] &= 0x0F
    assert torch.equal(c[..., : want.shape[-1]], want) and (c[..., want.shape[-1]:] == 0).all()
    # byte [matrix][row / 128][k / 128][16 (r % 32) + 4 (r / 32 % 4) + block % 4]
    f = q.scales
    seen = torch.zeros_like(f, dtype=torch.bool)
    for m in range(2):
        for r in range(5):
            for b in range(nb):
                at = (m, r // 128, b // 4, 16 * (r % 32) + 4 * (r // 32 % 4) + b % 4)
                assert f[at] == scales[m, r, b]
                seen[at] = True
    assert (f[~seen] == 0).all()


def test_parts_of_many_rows():
    g = torch.Generator().manual_seed(3)
    codes = torch.randint(0, 256, (300, 80), dtype=torch.uint8, generator=g)
    scales = torch.randint(0, 256, (300, 5), dtype=torch.uint8, generator=g)
    q = tb.MXFP4Tensor.from_parts(codes, scales, 160)
    assert q.scales.shape == (1, 3, 2, 512)
    for r in (0, 31, 32, 127, 128, 200, 299):
        for b in range(5):
            assert q.scales[0, r // 128, b // 4, 16 * (r % 32) + 4 * (r // 32 % 4) + b % 4] == scales[r, b]
    c, s = q.parts()
    assert torch.equal(c, codes) and torch.equal(s, scales)
    assert tb.MXFP4Tensor.from_parts(codes[:0], scales[:0], 160).parts()[1].shape == (0, 5)


def test_oracle_quantiser_by_hand():
    x = torch.zeros(1, 64)
    x[0, :9] = torch.tensor([4.0, 0.25, -0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9])
    x[0, 32:35] = torch.tensor([2.0 ** -140, -(2.0 ** -128), 0.0])
    v = X.dequantize(*X.quantize(x), 64)
    assert v[0, :9].tolist() == [4.0, 0.0, -1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0]
    assert v[0, 32:35].tolist() == [0.0, -(2.0 ** -128), 0.0]


def test_row_stride_of_a_c_of_one_row():
    from trnblas_b200.experts import _c_operand

    for C in (torch.zeros(40, 1).mT, torch.zeros(3, 40, 1).mT, torch.zeros(40).as_strided((1, 40), (1, 1)),
              torch.zeros(1, 40), torch.zeros(1).expand(1, 40)):
        t, ld = _c_operand(C, 40)
        assert ld >= 40 and t.stride(-1) == 1 and torch.equal(t, C)
    t, ld = _c_operand(torch.zeros(7, 50)[:, 3:43], 40)
    assert ld == 50 and t.storage_offset() == 3


@pytest.mark.parametrize("dual", ["A", "B", "C"])
def test_forward_mode_is_refused(dual):
    """A tangent is never dropped: refused before any device work, with or
    without reverse-mode gradients and under no_grad."""
    import torch.autograd.forward_ad as fwd

    ops = {"A": A, "B": B, "C": torch.zeros(6, 4, dtype=BF)}
    with fwd.dual_level():
        for grad in (False, True):
            t = ops[dual].clone().requires_grad_(grad)
            args = {**ops, dual: fwd.make_dual(t, torch.ones_like(t))}
            for ctx in (torch.enable_grad(), torch.no_grad()):
                with ctx, pytest.raises(NotImplementedError, match="forward-mode"):
                    tb.grouped_gemm(1.0, args["A"], args["B"], S, 1.0, args["C"])


@pytest.mark.parametrize("sizes", [[2 ** 62, 2 ** 62], [2 ** 63 - 1, 2 ** 63 - 1], [7, 0], [6, 1]])
def test_host_sizes_whose_sum_wraps_around(sizes):
    for call in (lambda s: tb.grouped_gemm(1.0, A, B, s), lambda s: tb.grouped_gemm_wgrad(1.0, A, A, s),
                 lambda s: tb.grouped_gemm_mxfp4(1.0, A, _mx(2, 3, 8), s)):
        with pytest.raises(ValueError, match="group sizes"):
            call(torch.tensor(sizes))


@pytest.mark.parametrize("code,words", [(8, "group sizes"), (3, "bounded wait"), (0, None)])
def test_status_message_names_the_cause(monkeypatch, code, words):
    monkeypatch.setattr(N, "device_status", lambda device=None: code)
    if words is None:
        N.raise_on_device_status(0)
    else:
        with pytest.raises(RuntimeError, match=words):
            N.raise_on_device_status(0)
