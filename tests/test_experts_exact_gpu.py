"""The grouped and 4-bit products at sizes where the kernels' pipelines wrap and
a CTA takes several tiles, on small whole numbers (or halves and quarters): no
partial sum leaves 24 bits, so whatever the order of a sum it is exact in fp32
and a lost, doubled or stale block shows as an unequal result."""

from __future__ import annotations

import threading

import pytest
import torch

import trnblas_b200 as tb
from oracle import experts as X

pytestmark = pytest.mark.gpu
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
DEV = "cuda"


def _gen(*key):
    seed = 7
    for k in key:
        seed = (seed * 1000003 + int(k)) % (1 << 31)
    return torch.Generator(device=DEV).manual_seed(seed)


def _whole(*shape, dt=BF, seed=0):
    """-8 .. 8: exact in 16 bits, and K of them times as many below 64 K."""
    return torch.randint(-8, 9, shape, device=DEV, generator=_gen(seed, *shape)).to(dt)


def _sizes(s):
    return torch.tensor(s, dtype=torch.int32, device=DEV)


def _mx(*shape, seed=0):
    """Every code with units of 1 and 2: multiples of 1/2 up to 12, so a
    product of two is a multiple of 1/4 up to 144 (144 K < 2^22 for K < 29000)."""
    *lead, K = shape
    g = _gen(seed, *shape)
    codes = torch.randint(0, 256, (*lead, -(-K // 2)), dtype=torch.uint8, device=DEV, generator=g)
    scales = torch.randint(127, 129, (*lead, -(-K // 32)), dtype=torch.uint8, device=DEV, generator=g)
    return tb.MXFP4Tensor.from_parts(codes, scales, K)


def _values(q):
    return tb.dequantize_mxfp4(q).double()


# one CTA's tiles of 64 rows, pairs (two operand layouts, whole and ragged 64-column
# blocks), and one CTA's tiles of 256 rows, each with more K blocks than stages
FORWARD = [([40, 0, 17, 64], 1032, 264), ([513, 64, 0, 255, 256, 257], 520, 2304), ([513, 64, 0, 255, 256, 257], 1024, 4096),
           ([1, 0, 1290, 3], 1032, 4100), ([2000, 3, 0, 1900], 1040, 4160), ([40000, 0, 30001, 17, 9000], 1032, 128),
           ([30000, 20011, 0, 31000], 712, 100)]


@pytest.mark.parametrize("sizes,K,Nn", FORWARD, ids=lambda v: str(v) if isinstance(v, int) else f"{len(v)}x{max(v)}")
@pytest.mark.parametrize("transB", [False, True])
def test_grouped_gemm(sizes, K, Nn, transB):
    rows = sum(sizes) + 37
    dt = FP if K % 16 else BF
    A, B = _whole(rows, K, dt=dt), _whole(len(sizes), *((Nn, K) if transB else (K, Nn)), dt=dt)
    D = tb.grouped_gemm(1.0, A, B, _sizes(sizes), transB=transB, out_dtype=F32)
    for g, r0, r1 in X.ranges(sizes):
        b = (B[g].mT if transB else B[g]).double()
        assert torch.equal(D[r0:r1].double(), A[r0:r1].double() @ b), g
    assert (D[sum(sizes):] == 0).all()
    assert torch.equal(D, tb.grouped_gemm(1.0, A, B, _sizes(sizes), transB=transB, out_dtype=F32))
    assert tb.device_status(0) == 0


@pytest.mark.parametrize("sizes", [[513, 64, 0, 255, 256, 257], [1, 0, 1290, 3], [5000, 0, 33, 700, 31, 15, 17] * 3],
                         ids=lambda s: f"{len(s)}x{max(s)}")
@pytest.mark.parametrize("M,Nn", [(256, 512), (192, 320), (1024, 2048), (520, 328), (72, 1000), (1000, 128)])
def test_wgrad(sizes, M, Nn):
    """CTA pairs with the one-copy map (whole 64-column blocks on both sides) and
    without, and single CTAs; stores by TMA and, with a C, by lanes."""
    rows = sum(sizes) + 21
    A, B = _whole(rows, M), _whole(rows, Nn, seed=1)
    s = _sizes(sizes)
    ref, mags = X.wgrad(1.0, A, B, sizes)
    D = tb.grouped_gemm_wgrad(1.0, A, B, s, out_dtype=F32)
    assert torch.equal(D.double(), ref)
    C = _whole(len(sizes), M, Nn, dt=F32, seed=2)
    assert torch.equal(tb.grouped_gemm_wgrad(1.0, A, B, s, 1.0, C, out_dtype=F32).double(), ref + C)
    # 16-bit results, and a 16-bit C: the exact sum rounded once
    assert torch.equal(tb.grouped_gemm_wgrad(1.0, A, B, s), ref.to(F32).to(BF))
    assert torch.equal(tb.grouped_gemm_wgrad(1.0, A, B, s, 2.0, C.to(BF)), (ref + 2.0 * C).to(F32).to(BF))
    assert torch.equal(tb.grouped_gemm_wgrad(1.0, A.to(FP), B.to(FP), s, -1.0, C.to(FP)), (ref - C).to(F32).to(FP))
    assert tb.device_status(0) == 0


@pytest.mark.parametrize("M,Nn,K", [(192, 256, 4096), (777, 4096, 4010), (500, 9000, 2000), (2000, 4096, 4096), (9700, 128, 4096),
                                    (30000, 100, 1300), (1100, 3333, 7777)])
def test_gemm_mxfp4(M, Nn, K):
    """Rows quantised before, and 16-bit rows of the same values (whose blocks
    quantise exactly: with a smaller unit where the largest value is smaller)."""
    qa, qb = _mx(M, K, seed=1), _mx(Nn, K, seed=2)
    ref = _values(qa) @ _values(qb).T
    assert torch.equal(tb.gemm_mxfp4(1.0, qa, qb, out_dtype=F32).double(), ref)
    x = tb.dequantize_mxfp4(qa, BF)
    for _ in range(2):
        assert torch.equal(tb.gemm_mxfp4(1.0, x, qb, out_dtype=F32).double(), ref)
    assert tb.device_status(0) == 0


@pytest.mark.parametrize("sizes", [[40, 0, 17, 64], [513, 64, 0, 255, 256, 257], [3000, 0, 5001, 17, 900]],
                         ids=lambda s: f"{len(s)}x{max(s)}")
@pytest.mark.parametrize("K,Nn", [(4096, 2304), (4010, 1000), (2600, 128)])
def test_grouped_gemm_mxfp4(sizes, K, Nn):
    rows = sum(sizes) + 53
    qa, qb, s = _mx(rows, K, seed=4), _mx(len(sizes), Nn, K, seed=5), _sizes(sizes)
    a, b = _values(qa), _values(qb)
    D = tb.grouped_gemm_mxfp4(1.0, qa, qb, s, out_dtype=F32)
    for g, r0, r1 in X.ranges(sizes):
        assert torch.equal(D[r0:r1].double(), a[r0:r1] @ b[g].T), g
    assert (D[sum(sizes):] == 0).all()
    assert torch.equal(D, tb.grouped_gemm_mxfp4(1.0, tb.dequantize_mxfp4(qa, BF), qb, s, out_dtype=F32))
    assert tb.device_status(0) == 0


@pytest.mark.parametrize("M", [1, 16])
@pytest.mark.parametrize("Nn,K", [(130, 33), (64, 8200), (136, 45056), (64, 44000), (128, 50000), (2048, 4000)])
def test_few_rows(M, Nn, K):
    """Rows of 0, 1/2, 1, 2, 4 and their negatives, which E2M1 holds in any
    block's unit, times multiples of 1/2 up to 12: multiples of 1/4 of a
    magnitude up to 48, whose 50000 stay below 2^22. One row is zero in front of
    K's last block of 32, one in front of its last 256 values."""
    g = _gen(M, Nn, K)
    x = torch.tensor([0.0, 0.5, 1.0, 2.0, 4.0, -0.5, -1.0, -2.0, -4.0], device=DEV)[
        torch.randint(0, 9, (M, K), device=DEV, generator=g)]
    for at, row in ((32, 1), (256, 2)):
        if row < M:
            x[row, : (K - 1) // at * at] = 0
            x[row, K - 1] = 4.0
    qb = _mx(Nn, K, seed=3)
    ref = x.double() @ _values(qb).T
    for dt in (BF, FP, F32):
        assert torch.equal(tb.gemm_mxfp4(1.0, x.to(dt), qb, out_dtype=F32).double(), ref), dt
    assert tb.device_status(0) == 0


@pytest.mark.parametrize("op", ["dense", "grouped"])
def test_4_bit_products_from_two_threads_on_one_stream(op):
    """A product is launched beside the kernel in front of it, which here may be
    the other thread's: its quantiser, its product or an elementwise kernel."""
    M, Nn, K = 300, 1000, 1024
    qb = _mx(3, Nn, K) if op == "grouped" else _mx(Nn, K)
    xs = [tb.dequantize_mxfp4(_mx(M, K, seed=i), BF) for i in range(4)]
    s = _sizes([100, 0, 180])

    def product(x):
        return tb.grouped_gemm_mxfp4(1.0, x, qb, s) if op == "grouped" else tb.gemm_mxfp4(1.0, x, qb)

    want = [product(x) for x in xs]
    torch.cuda.synchronize()
    bad, start = [], threading.Barrier(2)

    def work(t):
        start.wait()
        for i in range(60):
            j = 2 * t + i % 2
            x = xs[j] * 2.0  # a kernel of torch's, and a row operand of its own
            d = product(x)
            bad.append((d * 0.5 != want[j]).sum())

    threads = [threading.Thread(target=work, args=(t,)) for t in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(bad) == 120 and sum(int(b) for b in bad) == 0
    assert tb.device_status(0) == 0


def test_large_products_repeat_themselves():
    """Random operands at a large layer's sizes: the same bits at every call."""
    g = _gen(1)
    sizes = [int(v) for v in (512 + torch.randint(-20, 21, (32,), generator=torch.Generator().manual_seed(1)))]
    rows, K, Nn = sum(sizes), 2048, 4096
    A, B = torch.randn(rows, K, device=DEV, generator=g).to(BF), torch.randn(32, K, Nn, device=DEV, generator=g).to(BF)
    dD, s = torch.randn(rows, Nn, device=DEV, generator=g).to(BF), _sizes(sizes)
    calls = (lambda: tb.grouped_gemm(1.0, A, B, s), lambda: tb.grouped_gemm(1.0, dD, B, s, transB=True),
             lambda: tb.grouped_gemm_wgrad(1.0, A, dD, s))
    for call in calls:
        first = call()
        for _ in range(4):
            assert torch.equal(call(), first)
