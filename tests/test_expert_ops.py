"""The grouped and 4-bit products as torch ops: fake shapes without a GPU, and
on a B200 `torch.library.opcheck` and the public functions' results."""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import trnblas_b200 as tb
from trnblas_b200 import ops

T = torch.ops.trnblas
BF, U8 = torch.bfloat16, torch.uint8


def test_fake_shapes_without_gpu():
    with FakeTensorMode():
        a = torch.empty(50, 64, device="cuda", dtype=BF)
        b = torch.empty(3, 64, 40, device="cuda", dtype=BF)
        s = torch.empty(3, device="cuda", dtype=torch.int32)
        d = T.grouped_gemm(a, b, s)
        assert d.shape == (50, 40) and d.dtype == BF
        assert T.grouped_gemm(a, b.mT.contiguous(), s, 1.0, True, torch.float32).dtype == torch.float32
        assert T.grouped_gemm_wgrad(a, d, s).shape == (3, 64, 40)
        data, scales = T.quantize_mxfp4(torch.empty(3, 200, 100, device="cuda"))
        assert data.shape == (3, 200, 64) and scales.shape == (3, 2, 1, 512) and data.dtype == scales.dtype == U8
        assert T.dequantize_mxfp4(data, scales, 100, BF).shape == (3, 200, 100)
        x = torch.empty(7, 100, device="cuda", dtype=BF)
        assert T.grouped_gemm_mxfp4(x, data, scales, s).shape == (7, 200)
        d2, s2 = T.quantize_mxfp4(torch.empty(200, 100, device="cuda"))
        assert T.gemm_mxfp4(x, d2, s2, 1.0, torch.float32).shape == (7, 200)


def test_schemas_are_functional():
    for name in ops.EXPERT_OPS:
        schema = getattr(T, name).default._schema
        assert not any(a.alias_info is not None and a.alias_info.is_write for a in schema.arguments), name


@pytest.mark.gpu
def test_opcheck_and_parity_on_gpu():
    g = torch.Generator(device="cuda").manual_seed(3)
    a = torch.randn(50, 64, device="cuda", generator=g).to(BF)
    b = torch.randn(3, 64, 40, device="cuda", generator=g).to(BF)
    s = torch.tensor([20, 0, 25], device="cuda")
    d = torch.randn(50, 40, device="cuda", generator=g).to(BF)
    ag, bg = a.clone().requires_grad_(), b.clone().requires_grad_()
    torch.library.opcheck(T.grouped_gemm, (ag, bg, s, 0.5, False, None),
                          test_utils=("test_schema", "test_autograd_registration", "test_faketensor"))
    torch.library.opcheck(T.grouped_gemm_wgrad, (a, d, s, 1.0, torch.float32))
    out = T.grouped_gemm(ag, bg, s)
    assert torch.equal(out, tb.grouped_gemm(1.0, a, b, s))
    da, db = torch.autograd.grad(out, (ag, bg), d)
    assert torch.equal(da, tb.grouped_gemm(1.0, d, b, s, transB=True))
    assert torch.equal(db, tb.grouped_gemm_wgrad(1.0, a, d, s))
    w = torch.randn(3, 72, 64, device="cuda", generator=g)
    torch.library.opcheck(T.quantize_mxfp4, (w,))
    data, scales = T.quantize_mxfp4(w)
    q = tb.quantize_mxfp4(w)
    assert torch.equal(data, q.data) and torch.equal(scales, q.scales)
    torch.library.opcheck(T.dequantize_mxfp4, (data, scales, 64, BF))
    torch.library.opcheck(T.grouped_gemm_mxfp4, (a, data, scales, s, 1.0, BF))
    assert torch.equal(T.grouped_gemm_mxfp4(a, data, scales, s), tb.grouped_gemm_mxfp4(1.0, a, q, s))
    d0, s0 = data[0].contiguous(), scales[:1].contiguous()
    torch.library.opcheck(T.gemm_mxfp4, (a, d0, s0, 1.0, BF))
    assert torch.equal(T.gemm_mxfp4(a, d0, s0), tb.gemm_mxfp4(1.0, a, tb.quantize_mxfp4(w[0])))
    assert tb.device_status(0) == 0


def test_fake_products_check_the_inner_dimension():
    with FakeTensorMode():
        s = torch.empty(3, device="cuda", dtype=torch.int32)
        data, scales = T.quantize_mxfp4(torch.empty(3, 200, 100, device="cuda"))
        d2, s2 = T.quantize_mxfp4(torch.empty(200, 100, device="cuda"))
        x = torch.empty(7, 100, device="cuda", dtype=BF)
        assert T.gemm_mxfp4(x, d2, s2, 1.0, BF, 100).shape == T.grouped_gemm_mxfp4(x, data, scales, s, k=100).shape == (7, 200)
        for k, width in ((99, 100), (100, 99), (None, 96), (None, 129)):
            y = torch.empty(7, width, device="cuda", dtype=BF)
            for call in (lambda: T.gemm_mxfp4(y, d2, s2, k=k), lambda: T.grouped_gemm_mxfp4(y, data, scales, s, k=k)):
                with pytest.raises(RuntimeError, match="inner dimensions"):
                    call()


@pytest.mark.gpu
def test_products_check_the_weights_k():
    """Rows of 40 values against weights of K = 64 (or the other way round) are
    refused as the public functions refuse them; k names a K inside a block."""
    g = torch.Generator(device="cuda").manual_seed(4)
    s = torch.tensor([3, 4], device="cuda")
    for K in (64, 40):
        w = torch.randn(2, 72, K, device="cuda", generator=g)
        q = tb.quantize_mxfp4(w)
        q0 = tb.quantize_mxfp4(w[0])
        x = torch.randn(7, K, device="cuda", generator=g).to(BF)
        k = None if K == 64 else K
        torch.library.opcheck(T.gemm_mxfp4, (x, q0.data, q0.scales, 1.0, BF, K))
        assert torch.equal(T.gemm_mxfp4(x, q0.data, q0.scales, k=k), tb.gemm_mxfp4(1.0, x, q0))
        assert torch.equal(T.grouped_gemm_mxfp4(x, q.data, q.scales, s, k=k), tb.grouped_gemm_mxfp4(1.0, x, q, s))
        for y, kk in ((torch.zeros(7, 104 - K, device="cuda", dtype=BF), K), (torch.zeros(7, 40, device="cuda", dtype=BF), None),
                      (x, 33), (x, 65)):
            with pytest.raises(ValueError):
                T.gemm_mxfp4(y, q0.data, q0.scales, k=kk)
            with pytest.raises(ValueError):
                T.grouped_gemm_mxfp4(y, q.data, q.scales, s, k=kk)
    assert tb.device_status(0) == 0
