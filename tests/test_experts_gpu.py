"""Products grouped by expert on a B200 against a plain 64-bit form: lengths
from no row to many tiles, odd sizes, both layouts of the weights, the rows
behind the last group, gradients, streams and captured graphs. The tolerance
is derived in oracle/experts.py."""

from __future__ import annotations

import pytest
import torch

import trnblas_b200 as tb
from oracle import experts as X

pytestmark = pytest.mark.gpu
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
DEV = "cuda"


def _rand(*shape, dt=BF, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + 17 * len(shape) + sum(shape))
    return torch.randn(*shape, device=DEV, generator=g).to(dt)


def _sizes(s, dt=torch.int32):
    return torch.tensor(s, dtype=dt, device=DEV)


SIZES = [
    [0],
    [1],
    [0, 0, 5, 0],
    [300, 0, 1, 17],
    [64, 65, 63, 1, 0, 128],
    [513, 64, 0, 255, 256, 257],
    [2] * 37,
]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
@pytest.mark.parametrize("transB", [False, True])
@pytest.mark.parametrize("K,Nn", [(64, 128), (200, 264), (1032, 72), (65, 129), (1, 8), (8, 1), (7, 3)])
def test_grouped_gemm(sizes, transB, K, Nn):
    dt = BF if K % 2 == 0 else FP
    rows = sum(sizes) + (K % 3) * 29
    if rows == 0:
        rows = 3
    A = _rand(rows, K, dt=dt)
    B = _rand(len(sizes), *((Nn, K) if transB else (K, Nn)), dt=dt)
    for out in (dt, F32):
        D = tb.grouped_gemm(1.0, A, B, _sizes(sizes), transB=transB, out_dtype=out)
        ref, mags = X.grouped_gemm(1.0, A, B, sizes, transB=transB)
        assert D.dtype == out and D.shape == ref.shape
        X.check(D, ref, X.tolerance(ref, mags, K, out), f"{sizes} {K} {Nn} {out}")
    assert tb.device_status(0) == 0


PAIRED = [[513, 64, 0, 255, 256, 257], [1, 0, 1290, 3], [700, 300, 129, 31, 0, 40]]


@pytest.mark.parametrize("sizes", PAIRED, ids=lambda s: f"{len(s)}x{max(s)}")
@pytest.mark.parametrize("transB", [False, True])
@pytest.mark.parametrize("K,Nn", [(200, 2056), (64, 2304), (1032, 4100), (65, 2049), (7, 3000)])
def test_grouped_gemm_on_pairs(sizes, transB, K, Nn):
    """Enough tiles for the CTA pairs, which smaller products do not reach."""
    dt = BF if K % 2 == 0 else FP
    rows = sum(sizes) + (K % 3) * 150
    A, B = _rand(rows, K, dt=dt), _rand(len(sizes), *((Nn, K) if transB else (K, Nn)), dt=dt)
    ref, mags = X.grouped_gemm(0.5, A, B, sizes, transB=transB)
    for out in (dt, F32):
        D = tb.grouped_gemm(0.5, A, B, _sizes(sizes), transB=transB, out_dtype=out)
        X.check(D, ref, X.tolerance(ref, mags, K, out), f"{sizes} {K} {Nn} {out}")
        C = _rand(rows, Nn, dt=out, seed=9)
        D = tb.grouped_gemm(0.5, A, B, _sizes(sizes), 2.0, C, transB=transB, out_dtype=out)
        X.check(D, ref + 2.0 * C.double(), X.tolerance(ref + 2.0 * C.double(), mags, K, out, 2.0 * C))
    assert tb.device_status(0) == 0


@pytest.mark.parametrize("K,Nn", [(64, 128), (200, 100), (33, 9)])
def test_long_groups_of_few_columns(K, Nn):
    """One CTA's long row tiles: many rows, no second block of columns."""
    sizes = [9000, 0, 5001, 17, 6300]
    A, B = _rand(sum(sizes) + 300, K), _rand(5, K, Nn)
    ref, mags = X.grouped_gemm(1.0, A, B, sizes)
    X.check(tb.grouped_gemm(1.0, A, B, _sizes(sizes)), ref, X.tolerance(ref, mags, K, BF))


def test_whole_numbers_are_exact():
    """Small whole numbers: every partial sum is a whole number below 2^24, so
    any association gives the same result, whatever the tiling."""
    sizes = [700, 3, 0, 129, 31]
    g = torch.Generator(device=DEV).manual_seed(5)
    A = torch.randint(-8, 9, (sum(sizes), 520), device=DEV, generator=g).to(BF)
    B = torch.randint(-8, 9, (5, 520, 328), device=DEV, generator=g).to(BF)
    ref, _ = X.grouped_gemm(1.0, A, B, sizes)
    assert torch.equal(tb.grouped_gemm(1.0, A, B, _sizes(sizes), out_dtype=F32).double(), ref)
    dD = torch.randint(-8, 9, (sum(sizes), 328), device=DEV, generator=g).to(BF)
    wref, _ = X.wgrad(1.0, A, dD, sizes)
    assert torch.equal(tb.grouped_gemm_wgrad(1.0, A, dD, _sizes(sizes), out_dtype=F32).double(), wref)


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("out", ["same", "fp32"])
@pytest.mark.parametrize("Nn", [256, 250])
def test_alpha_beta_c(dt, out, Nn):
    out = dt if out == "same" else F32
    sizes, K = [40, 0, 333, 7], 136
    rows = sum(sizes) + 21
    A, B = _rand(rows, K, dt=dt), _rand(4, K, Nn, dt=dt)
    C = _rand(rows, Nn, dt=out, seed=9)
    ref, mags = X.grouped_gemm(-0.75, A, B, sizes, 0.5, C)
    D = tb.grouped_gemm(-0.75, A, B, _sizes(sizes), 0.5, C)
    if out != dt:
        D = tb.grouped_gemm(-0.75, A, B, _sizes(sizes), 0.5, C, out_dtype=out)
    tol = X.tolerance(ref, mags, K, out, C)
    if D.dtype == out:
        X.check(D, ref, tol)
    # the rows behind the last group: beta * C, one rounding
    X.check(D[-21:], 0.5 * C[-21:].double(), X.tolerance(ref, mags, 0, D.dtype, C)[-21:])
    # beta = 0 reads no C
    bad = torch.full_like(C, float("nan"))
    assert torch.equal(tb.grouped_gemm(1.0, A, B, _sizes(sizes), 0.0, bad, out_dtype=out),
                       tb.grouped_gemm(1.0, A, B, _sizes(sizes), out_dtype=out))
    # strided C, and one that broadcasts (added after the product's rounding)
    wide = _rand(rows, 2 * Nn, dt=out, seed=4)
    r2, m2 = X.grouped_gemm(1.0, A, B, sizes, 2.0, wide[:, Nn:])
    D2 = tb.grouped_gemm(1.0, A, B, _sizes(sizes), 2.0, wide[:, Nn:], out_dtype=out)
    X.check(D2, r2, X.tolerance(r2, m2, K, out, 2.0 * wide[:, Nn:]))


def test_strides_and_expanded_weights():
    sizes, K, Nn = [9, 130, 0, 61], 96, 160
    rows = sum(sizes)
    big = _rand(rows, 3 * K)
    A = big[:, K:2 * K]  # row stride 3K
    At = _rand(K, rows).mT  # columns contiguous
    one = _rand(1, K, Nn)
    B = one.expand(4, K, Nn)
    for a in (A, At, big[:, 1:K + 1]):  # the last one off 16 bytes
        ref, mags = X.grouped_gemm(1.0, a, B, sizes)
        X.check(tb.grouped_gemm(1.0, a, B, _sizes(sizes)), ref, X.tolerance(ref, mags, K, BF))
    Bs = _rand(8, K, Nn)[::2]  # matrices two apart
    ref, mags = X.grouped_gemm(1.0, A, Bs, sizes)
    X.check(tb.grouped_gemm(1.0, A, Bs, _sizes(sizes)), ref, X.tolerance(ref, mags, K, BF))
    w = tb.grouped_gemm_wgrad(1.0, At, big[:, 3:3 + K], _sizes(sizes))
    ref, mags = X.wgrad(1.0, At, big[:, 3:3 + K], sizes)
    X.check(w, ref, X.tolerance(ref, mags, max(sizes), BF))


@pytest.mark.parametrize("off,step", [(0, 1), (1, 1), (2, 2), (4, 4), (3, 7)])
def test_operands_off_16_bytes(off, step):
    """Bases and row, matrix strides of every alignment: copied, in the widest
    pieces they allow, before the product."""
    sizes, K, Nn = [5, 0, 70, 140], 93 + step, 61 + step
    rows = sum(sizes) + 3
    flat = _rand(9 * (K + 9) * (Nn + 9) + 2 * rows * (K + Nn))

    def at(o, shape, strides):
        return flat.as_strided(shape, strides, o)

    A = at(off, (rows, K), (K + step, 1))
    dD = at(off + 2, (rows, Nn), (Nn + step, 1))
    for B, tB in ((at(off, (4, K, Nn), (K * (Nn + step) + step, Nn + step, 1)), False),
                  (at(off, (4, Nn, K), (Nn * (K + step), K + step, 1)), True),
                  (at(off, (4, K, Nn), (Nn * (K + step) + step, 1, K + step)), False),  # stored by columns
                  (at(off, (1, K, Nn), (1, Nn + step, 1)).expand(4, K, Nn), False),
                  (at(off, (4, K, Nn), (2 * K * Nn, 2 * Nn, 2)), False)):
        ref, mags = X.grouped_gemm(1.0, A, B, sizes, transB=tB)
        X.check(tb.grouped_gemm(1.0, A, B, _sizes(sizes), transB=tB), ref, X.tolerance(ref, mags, K, BF))
    ref, mags = X.wgrad(1.0, A, dD, sizes)
    X.check(tb.grouped_gemm_wgrad(1.0, A, dD, _sizes(sizes)), ref, X.tolerance(ref, mags, max(sizes), BF))
    a, b = A.clone().requires_grad_(), _rand(4, K, Nn).requires_grad_()
    da, db = torch.autograd.grad(tb.grouped_gemm(1.0, a, b, _sizes(sizes)), (a, b), dD)
    ref, mags = X.grouped_gemm(1.0, dD, b.detach(), sizes, transB=True)
    X.check(da, ref, X.tolerance(ref, mags, Nn, BF))
    ref, mags = X.wgrad(1.0, A, dD, sizes)
    X.check(db, ref, X.tolerance(ref, mags, max(sizes), BF))


def test_single_rows_and_columns_of_any_stride():
    flat, B = _rand(1 << 20), _rand(2, 72, 40)
    for a in (flat.as_strided((1, 72), (1, 1)), flat.as_strided((1, 72), (1 << 19, 1)), flat.as_strided((1, 72), (9, 3)),
              flat.as_strided((7, 72), (0, 1)), flat.as_strided((7, 72), (1, 7))):
        sizes = [0, a.shape[0]]
        ref, mags = X.grouped_gemm(1.0, a, B, sizes)
        X.check(tb.grouped_gemm(1.0, a, B, _sizes(sizes)), ref, X.tolerance(ref, mags, 72, BF))
        ref, mags = X.wgrad(1.0, a, a, sizes)
        X.check(tb.grouped_gemm_wgrad(1.0, a, a, _sizes(sizes)), ref, X.tolerance(ref, mags, 7, BF))
    col = flat.as_strided((9, 1), (5, 77))
    ref, mags = X.grouped_gemm(1.0, col, _rand(1, 1, 24), [9])
    X.check(tb.grouped_gemm(1.0, col, _rand(1, 1, 24), _sizes([9])), ref, X.tolerance(ref, mags, 1, BF))


def test_sizes_on_host_64_bit_and_strided():
    sizes = [5, 0, 90]
    A, B = _rand(95, 64), _rand(3, 64, 64)
    want = tb.grouped_gemm(1.0, A, B, _sizes(sizes))
    assert torch.equal(want, tb.grouped_gemm(1.0, A, B, _sizes(sizes, torch.int64)))
    assert torch.equal(want, tb.grouped_gemm(1.0, A, B, torch.tensor(sizes)))
    pairs = torch.tensor([[5, 1], [0, 2], [90, 3]], device=DEV)
    assert torch.equal(want, tb.grouped_gemm(1.0, A, B, pairs[:, 0]))
    host = tb.grouped_gemm(1.0, A.cpu(), B.cpu(), torch.tensor(sizes))
    assert host.device.type == "cpu" and torch.equal(host, want.cpu())


def test_sizes_out_of_range_are_cut_off_and_reported():
    A, B = _rand(100, 64), _rand(3, 64, 136)
    assert tb.device_status(0) == 0
    D = tb.grouped_gemm(1.0, A, B, _sizes([40, -7, 1 << 30]))
    assert tb.device_status(0) == 8 and tb.device_status(0) == 0
    assert torch.equal(D, tb.grouped_gemm(1.0, A, B, _sizes([40, 0, 60])))
    W = tb.grouped_gemm_wgrad(1.0, A, A, _sizes([1 << 62, -(1 << 62), 1 << 62], torch.int64))
    assert tb.device_status(0) == 8
    assert torch.equal(W, tb.grouped_gemm_wgrad(1.0, A, A, _sizes([100, 0, 0])))
    assert tb.device_status(0) == 0


@pytest.mark.parametrize("Nn", [200, 9000])
def test_nan_and_infinity_stay_in_their_rows_and_groups(Nn):
    sizes, K = [50, 0, 83, 20], 192
    if Nn == 9000:  # CTA pairs
        sizes = [50, 0, 383, 20]
    rows = sum(sizes) + 40
    A, B = _rand(rows, K), _rand(4, K, Nn)
    clean = tb.grouped_gemm(1.0, A, B, _sizes(sizes))
    A2, B2 = A.clone(), B.clone()
    A2[-40:] = float("nan")      # behind the last group
    end = 50 + sizes[2]
    A2[60] = float("inf")        # one row of group 2
    B2[1] = float("nan")         # a group without rows
    B2[3] = float("inf")         # group 3
    D = tb.grouped_gemm(1.0, A2, B2, _sizes(sizes))
    keep = torch.ones(rows, dtype=torch.bool, device=DEV)
    keep[60] = False
    keep[end:end + 20] = False
    assert torch.equal(D[keep], clean[keep])
    assert not D[60].isfinite().any() and not D[end:end + 20].isfinite().any()
    assert (D[-40:] == 0).all()
    # the gradient of the weights: neighbours' rows are not even multiplied by zero
    dD = _rand(rows, Nn, seed=3)
    w = tb.grouped_gemm_wgrad(1.0, A, dD, _sizes(sizes))
    A3, d3 = A.clone(), dD.clone()
    A3[50:end], d3[50:end] = float("inf"), float("nan")  # group 2
    A3[-40:], d3[-40:] = float("nan"), float("inf")
    w3 = tb.grouped_gemm_wgrad(1.0, A3, d3, _sizes(sizes))
    for g in (0, 1, 3):
        assert torch.equal(w3[g], w[g]), g
    assert w3[2].isnan().all() and (w3[1] == 0).all()


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
@pytest.mark.parametrize("M,Nn", [(64, 128), (200, 264), (136, 1000), (65, 129), (1, 1)])
def test_wgrad(sizes, M, Nn):
    dt = FP if M % 2 else BF
    rows = sum(sizes) + (M % 3) * 13
    A, B = _rand(rows, M, dt=dt), _rand(rows, Nn, dt=dt, seed=2)
    for out in (dt, F32):
        D = tb.grouped_gemm_wgrad(0.5, A, B, _sizes(sizes), out_dtype=out)
        ref, mags = X.wgrad(0.5, A, B, sizes)
        assert D.dtype == out and D.shape == ref.shape
        X.check(D, ref, X.tolerance(ref, mags, max(sizes), out), f"{sizes} {M} {Nn} {out}")
    C = _rand(len(sizes), M, Nn, dt=F32, seed=7)
    ref, mags = X.wgrad(1.0, A, B, sizes, 1.0, C)
    D = tb.grouped_gemm_wgrad(1.0, A, B, _sizes(sizes), 1.0, C, out_dtype=F32)
    X.check(D, ref, X.tolerance(ref, mags, max(sizes), F32, C))
    for g, m in enumerate(sizes):
        if m == 0:
            assert torch.equal(D[g], C[g])


def test_no_rows_no_groups():
    B = _rand(3, 64, 32)
    assert tb.grouped_gemm(1.0, _rand(0, 64), B, _sizes([0, 0, 0])).shape == (0, 32)
    assert (tb.grouped_gemm(1.0, _rand(7, 64), _rand(0, 64, 32), _sizes([])) == 0).all()
    C = _rand(7, 32)
    assert torch.equal(tb.grouped_gemm(1.0, _rand(7, 0), _rand(3, 0, 32), _sizes([7, 0, 0]), 1.0, C), C)
    C3 = _rand(3, 8, 16)
    assert torch.equal(tb.grouped_gemm_wgrad(1.0, _rand(0, 8), _rand(0, 16), _sizes([0, 0, 0]), 1.0, C3), C3)
    assert tb.grouped_gemm_wgrad(1.0, _rand(5, 8), _rand(5, 16), _sizes([])).shape == (0, 8, 16)


@pytest.mark.parametrize("transB", [False, True])
@pytest.mark.parametrize("shared", [False, True])
def test_gradients_against_the_formula(transB, shared):
    sizes, K, Nn = [70, 0, 130, 9], 128, 96
    rows = sum(sizes) + 5
    shape = (Nn, K) if transB else (K, Nn)
    A = _rand(rows, K).requires_grad_()
    W = (_rand(1, *shape) if shared else _rand(4, *shape)).requires_grad_()
    B = W.expand(4, *shape)
    C = _rand(rows, Nn, seed=5).requires_grad_()
    dD = _rand(rows, Nn, seed=6)
    D = tb.grouped_gemm(0.5, A, B, _sizes(sizes), 2.0, C, transB=transB)
    assert torch.equal(D.detach(), tb.grouped_gemm(0.5, A.detach(), B.detach(), _sizes(sizes), 2.0, C.detach(),
                                                  transB=transB))
    dA, dW, dC = torch.autograd.grad(D, (A, W, C), dD)
    ra, ma = X.grouped_gemm(0.5, dD, B.detach(), sizes, transB=not transB)
    X.check(dA, ra, X.tolerance(ra, ma, Nn, BF))
    l, r = (dD, A.detach()) if transB else (A.detach(), dD)
    rw, mw = X.wgrad(0.5, l, r, sizes)
    assert dW.shape == W.shape
    if shared:  # the groups' gradients, each rounded to bf16, summed by torch in bf16 with fp32 sums
        tol = X.tolerance(rw, mw, max(sizes), BF).sum(0, keepdim=True)
        rw = rw.sum(0, keepdim=True)
        X.check(dW, rw, tol + 2.0 ** -8 * (rw.abs() + tol))
    else:
        X.check(dW, rw, X.tolerance(rw, mw, max(sizes), BF))
    assert torch.equal(dC, 2.0 * dD)


def test_gradients_against_differences():
    """The product is linear in each operand: with whole numbers the
    difference over a unit step is exact in fp32 and is the gradient."""
    sizes, K, Nn = [33, 0, 20], 40, 24
    rows = sum(sizes) + 4
    g = torch.Generator(device=DEV).manual_seed(1)
    A = torch.randint(-4, 5, (rows, K), device=DEV, generator=g).to(BF).requires_grad_()
    B = torch.randint(-4, 5, (3, K, Nn), device=DEV, generator=g).to(BF).requires_grad_()
    w = torch.randint(-3, 4, (rows, Nn), device=DEV, generator=g).to(F32)
    s = _sizes(sizes)

    def loss(a, b):
        return (tb.grouped_gemm(1.0, a, b, s, out_dtype=F32).double() * w).sum()

    dA, dB = torch.autograd.grad(loss(A, B), (A, B))
    base = loss(A.detach(), B.detach())
    for r, k in [(0, 0), (32, 39), (33, 5), (52, 17), (53, 3), (56, 39)]:
        a = A.detach().clone()
        a[r, k] += 1
        assert loss(a, B.detach()) - base == dA[r, k].double(), (r, k)
    for e, k, n in [(0, 0, 0), (0, 39, 23), (1, 4, 4), (2, 7, 11)]:
        b = B.detach().clone()
        b[e, k, n] += 1
        assert loss(A.detach(), b) - base == dB[e, k, n].double(), (e, k, n)


def test_layer_forward_and_backward():
    """The operators as a layer uses them: tokens sorted by expert, two grouped
    products with a gate between them, gradients through both. Every product is
    checked against 64 bits on the very operands it got."""
    tokens, dim, hidden, G = 301, 128, 192, 6
    g = torch.Generator(device=DEV).manual_seed(2)
    x = torch.randn(tokens, dim, device=DEV, generator=g).to(BF).requires_grad_()
    w1 = (torch.randn(G, hidden, dim, device=DEV, generator=g) * dim ** -0.5).to(BF).requires_grad_()
    w2 = (torch.randn(G, dim, hidden, device=DEV, generator=g) * hidden ** -0.5).to(BF).requires_grad_()
    expert = torch.randint(0, G - 1, (tokens,), device=DEV, generator=g)  # the last one gets none
    order = torch.argsort(expert, stable=True)
    sizes = torch.bincount(expert, minlength=G)
    xs = x[order]
    h = tb.grouped_gemm(1.0, xs, w1, sizes, transB=True)
    a = torch.relu(h)
    y = tb.grouped_gemm(1.0, a, w2, sizes, transB=True)
    dy = torch.randn(tokens, dim, device=DEV, generator=g).to(BF)
    gx, g1, g2, gh = torch.autograd.grad(y, (x, w1, w2, h), dy)
    sz = sizes.tolist()
    for out, ops, terms in (
        (h, (xs.detach(), w1.detach(), True), dim),
        (y, (a.detach(), w2.detach(), True), hidden),
    ):
        ref, mags = X.grouped_gemm(1.0, ops[0], ops[1], sz, transB=ops[2])
        X.check(out.detach(), ref, X.tolerance(ref, mags, terms, BF))
    ref, mags = X.wgrad(1.0, dy, a.detach(), sz)
    X.check(g2, ref, X.tolerance(ref, mags, max(sz), BF))
    ref, mags = X.grouped_gemm(1.0, dy, w2.detach(), sz)
    ok = h.detach() > 0
    X.check(torch.where(ok, gh, 0), torch.where(ok, ref, 0), X.tolerance(ref, mags, dim, BF))
    ref, mags = X.wgrad(1.0, gh, xs.detach(), sz)
    X.check(g1, ref, X.tolerance(ref, mags, max(sz), BF))
    ref, mags = X.grouped_gemm(1.0, gh, w1.detach(), sz)
    inv = torch.empty_like(order)
    inv[order] = torch.arange(tokens, device=DEV)
    X.check(gx, ref[inv], X.tolerance(ref, mags, hidden, BF)[inv])
    assert (g1[G - 1] == 0).all() and (g2[G - 1] == 0).all()


def test_captured_graph_follows_the_sizes():
    sizes = _sizes([10, 50, 4, 0])
    A, B = _rand(90, 128), _rand(4, 128, 136)
    dD = _rand(90, 136, seed=1)
    tb.grouped_gemm(1.0, A, B, sizes)
    tb.grouped_gemm_wgrad(1.0, A, dD, sizes)
    torch.cuda.synchronize()
    graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        D = tb.grouped_gemm(1.0, A, B, sizes)
        dA = tb.grouped_gemm(1.0, dD, B, sizes, transB=True)
        W = tb.grouped_gemm_wgrad(1.0, A, dD, sizes)
    with torch.cuda.graph(graph2):
        D2 = tb.grouped_gemm(2.0, A, B, sizes)
    for s in ([10, 50, 4, 0], [0, 0, 0, 90], [0, 0, 0, 0], [1, 88, 0, 1]):
        sizes.copy_(torch.tensor(s, dtype=torch.int32))
        A.copy_(_rand(90, 128, seed=s[1]))
        graph.replay()
        graph2.replay()
        torch.cuda.synchronize()
        assert torch.equal(D, tb.grouped_gemm(1.0, A, B, _sizes(s)))
        assert torch.equal(D2, tb.grouped_gemm(2.0, A, B, _sizes(s)))
        assert torch.equal(dA, tb.grouped_gemm(1.0, dD, B, _sizes(s), transB=True))
        assert torch.equal(W, tb.grouped_gemm_wgrad(1.0, A, dD, _sizes(s)))
    assert tb.device_status(0) == 0


def test_captured_training_step():
    """Forward and gradients in one captured graph, on leaves of its own."""
    s = _sizes([30, 0, 50])
    A, B = _rand(90, 128).requires_grad_(), _rand(3, 128, 136).requires_grad_()
    dD = _rand(90, 136, seed=1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(tb.grouped_gemm(1.0, A, B, s), (A, B), dD)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        D = tb.grouped_gemm(1.0, A, B, s)
        dA, dB = torch.autograd.grad(D, (A, B), dD)
    for sizes in ([30, 0, 50], [0, 90, 0], [1, 2, 3]):
        s.copy_(torch.tensor(sizes, dtype=torch.int32))
        with torch.no_grad():
            A.copy_(_rand(90, 128, seed=sizes[0]))
        graph.replay()
        torch.cuda.synchronize()
        a, b = A.detach(), B.detach()
        assert torch.equal(D.detach(), tb.grouped_gemm(1.0, a, b, s))
        assert torch.equal(dA, tb.grouped_gemm(1.0, dD, b, s, transB=True))
        assert torch.equal(dB, tb.grouped_gemm_wgrad(1.0, a, dD, s))


@pytest.mark.parametrize("Nn", [640, 4096])
def test_two_streams_and_the_same_result_twice(Nn):
    sizes = [700, 0, 33, 290]
    A, B, s = _rand(1023, 512), _rand(4, 512, Nn), _sizes(sizes)
    dD = _rand(1023, Nn)
    want, wantw = tb.grouped_gemm(1.0, A, B, s), tb.grouped_gemm_wgrad(1.0, A, dD, s)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(4):
        for st in streams:
            with torch.cuda.stream(st):
                outs.append((tb.grouped_gemm(1.0, A, B, s), tb.grouped_gemm_wgrad(1.0, A, dD, s)))
    torch.cuda.synchronize()
    for d, w in outs:
        assert torch.equal(d, want) and torch.equal(w, wantw)


def test_calls_from_two_threads():
    import threading

    sizes = [300, 0, 90]
    A, B, s = _rand(390, 256), _rand(3, 256, 2304), _sizes(sizes)
    want, wantw = tb.grouped_gemm(1.0, A, B, s), tb.grouped_gemm_wgrad(1.0, A, A, s)
    torch.cuda.synchronize()
    bad = []

    def work():
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(20):
                d, w = tb.grouped_gemm(1.0, A, B, s), tb.grouped_gemm_wgrad(1.0, A, A, s)
            st.synchronize()
        if not (torch.equal(d, want) and torch.equal(w, wantw)):
            bad.append(1)

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad and tb.device_status(0) == 0


def test_offsets_past_32_bits():
    """A result of 2.3 G elements: the last rows sit behind 2^31 elements."""
    rows, K, Nn = 71000, 64, 32768
    A, B = _rand(rows, K), _rand(2, K, Nn)
    sizes = [70000, 900]
    D = tb.grouped_gemm(1.0, A, B, _sizes(sizes))
    for r0, r1, g in ((0, 40, 0), (69960, 70000, 0), (70000, 70040, 1), (70860, 70900, 1)):
        ref, mags = X.grouped_gemm(1.0, A[r0:r1], B[g:g + 1], [r1 - r0])
        X.check(D[r0:r1], ref, X.tolerance(ref, mags, K, BF))
    assert (D[70900:] == 0).all()
    del D
    W = tb.grouped_gemm_wgrad(1.0, A[:256], _rand(256, 2 * Nn), _sizes([100, 156] + [0] * 1000 + [0]), out_dtype=BF)
    assert (W[2:] == 0).all()


def test_many_groups():
    G = 1024
    sizes = [(i * 7) % 5 for i in range(G)]
    A, B = _rand(sum(sizes), 64), _rand(G, 64, 40)
    ref, mags = X.grouped_gemm(1.0, A, B, sizes)
    X.check(tb.grouped_gemm(1.0, A, B, _sizes(sizes)), ref, X.tolerance(ref, mags, 64, BF))
    dD = _rand(sum(sizes), 40)
    ref, mags = X.wgrad(1.0, A, dD, sizes)
    X.check(tb.grouped_gemm_wgrad(1.0, A, dD, _sizes(sizes)), ref, X.tolerance(ref, mags, 5, BF))


def test_c_of_one_row_of_any_stride():
    """A C of one row whose row stride says nothing (a transposed column), a
    column of any stride, and stacks of them; in all four products."""
    A, B = _rand(1, 64), _rand(2, 64, 40)
    w, w3 = tb.quantize_mxfp4(_rand(40, 64)), tb.quantize_mxfp4(_rand(2, 40, 64))
    s = _sizes([0, 1])
    flat = _rand(4096)
    for C in (flat[:40].view(40, 1).mT, flat.as_strided((1, 40), (3, 1)), flat.as_strided((1, 40), (1, 5))):
        dense = C.clone(memory_format=torch.contiguous_format).reshape(40).view(1, 40)
        assert dense.stride(0) == 40
        assert torch.equal(tb.grouped_gemm(1.0, A, B, s, 2.0, C), tb.grouped_gemm(1.0, A, B, s, 2.0, dense))
        assert torch.equal(tb.gemm_mxfp4(1.0, A, w, 2.0, C), tb.gemm_mxfp4(1.0, A, w, 2.0, dense))
        assert torch.equal(tb.grouped_gemm_mxfp4(1.0, A, w3, s, 2.0, C), tb.grouped_gemm_mxfp4(1.0, A, w3, s, 2.0, dense))
        ref, mags = X.grouped_gemm(1.0, A, B, [0, 1], 2.0, C)
        X.check(tb.grouped_gemm(1.0, A, B, s, 2.0, C), ref, X.tolerance(ref, mags, 64, BF, 2.0 * C))
    sizes = [5, 0, 2]
    a, b = _rand(7, 1), _rand(7, 40)
    for C in (flat[:120].view(3, 40, 1).mT, flat.as_strided((3, 1, 40), (50, 7, 1)), flat.as_strided((3, 1, 40), (0, 1, 2)),
              flat.as_strided((3, 1, 40), (0, 1, 1))):
        ref, mags = X.wgrad(1.0, a, b, sizes, 0.5, C)
        X.check(tb.grouped_gemm_wgrad(1.0, a, b, _sizes(sizes), 0.5, C), ref, X.tolerance(ref, mags, 5, BF, 0.5 * C))
    col = flat.as_strided((7, 1), (9, 5))
    ref, mags = X.grouped_gemm(1.0, b, _rand(3, 40, 1), sizes, 1.0, col)
    X.check(tb.grouped_gemm(1.0, b, _rand(3, 40, 1), _sizes(sizes), 1.0, col), ref, X.tolerance(ref, mags, 40, BF, col))


def test_forward_mode_is_refused():
    """On the device, through the public function and the torch op; a level
    without dual operands changes nothing."""
    import torch.autograd.forward_ad as fwd

    A, B, s = _rand(6, 64), _rand(2, 64, 32), _sizes([3, 3])
    want = tb.grouped_gemm(1.0, A, B, s)
    with fwd.dual_level():
        assert torch.equal(tb.grouped_gemm(1.0, A, B, s), want)
        for a, b in ((fwd.make_dual(A, A), B), (A, fwd.make_dual(B, B))):
            for call in (lambda: tb.grouped_gemm(1.0, a, b, s), lambda: torch.ops.trnblas.grouped_gemm(a, b, s)):
                with pytest.raises(NotImplementedError):
                    call()
        # forward over reverse: the incoming gradient carries the tangent
        a = A.clone().requires_grad_()
        D = tb.grouped_gemm(1.0, a, B, s)
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(D, a, fwd.make_dual(torch.ones_like(want), want))


def test_pinned_host_operands_may_be_rewritten_after_the_call():
    """Sizes, weights, C in pinned host memory beside rows on the device: the
    call has read them when it returns, whatever the stream is still busy with."""
    A, s = _rand(90, 64), [40, 0, 50]
    B, C, C3 = _rand(3, 64, 136), _rand(90, 136, seed=2), _rand(3, 64, 136, seed=3)
    dD, w3 = _rand(90, 136, seed=4), tb.quantize_mxfp4(_rand(3, 72, 64))
    Cm = _rand(90, 72, seed=5)
    for sizes, b, c, c3, cm in ((torch.tensor(s), B, C, C3, Cm), (_sizes(s), B.cpu(), C.cpu(), C3.cpu(), Cm.cpu())):
        host = [t.pin_memory() if t.device.type == "cpu" else t for t in (sizes, b, c, c3, cm)]
        calls = (lambda z, b, c, c3, cm: tb.grouped_gemm(1.0, A, b, z, 2.0, c),
                 lambda z, b, c, c3, cm: tb.grouped_gemm_wgrad(1.0, A, dD, z, 2.0, c3),
                 lambda z, b, c, c3, cm: tb.grouped_gemm_mxfp4(1.0, A, w3, z, 2.0, cm),
                 lambda z, b, c, c3, cm: tb.grouped_gemm(1.0, A.clone().requires_grad_(), b, z, 2.0, c).detach())
        want = [f(*(t.to(DEV) for t in host)) for f in calls]
        for f, ref in zip(calls, want):
            now = [t.clone().pin_memory() if t.device.type == "cpu" else t for t in host]
            torch.cuda.synchronize()
            torch.cuda._sleep(200_000_000)  # about 0.1 s in front of the call's copies
            got = f(*now)
            for t in now:
                if t.device.type == "cpu":
                    t.zero_()
            torch.cuda.synchronize()
            assert torch.equal(got, ref)


def test_captured_graph_reads_pinned_sizes_at_each_replay():
    A, B = _rand(90, 64), _rand(3, 64, 136)
    s = torch.tensor([40, 0, 50]).pin_memory()
    tb.grouped_gemm(1.0, A, B, s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        D = tb.grouped_gemm(1.0, A, B, s)
    for z in ([40, 0, 50], [0, 90, 0], [1, 2, 3]):
        s.copy_(torch.tensor(z))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(D, tb.grouped_gemm(1.0, A, B, _sizes(z)))


def test_unfused_c_with_and_without_gradients():
    """A C that broadcasts or has another type is added to the rounded product;
    whether gradients are recorded changes no value."""
    sizes, Nn = [40, 0, 50], 136
    A, B, s = _rand(95, 64), _rand(3, 64, Nn), _sizes(sizes)
    dD = _rand(95, Nn, seed=1)
    P = tb.grouped_gemm(0.7, A, B, s)
    for C in (_rand(Nn, seed=2), _rand(95, 1, seed=3), _rand(95, Nn, dt=F32, seed=4), _rand(1, Nn, dt=F32, seed=5)):
        want = tb.grouped_gemm(0.7, A, B, s, 0.3, C)
        # one rounding behind the product's (a sum with an fp32 C rounds twice in fp32)
        ref = P.double() + 0.3 * C.double()
        tol = torch.finfo(want.dtype).eps / 2 * (ref.abs() + 0.3 * C.double().abs()) + 2.0 ** -22 * (P.double().abs() + C.double().abs())
        assert want.dtype == torch.promote_types(BF, C.dtype) and ((want.double() - ref).abs() <= tol).all()
        for need in ((True, False, False), (False, True, True), (False, False, True)):
            a, b, c = (t.clone().requires_grad_(n) for t, n in zip((A, B, C), need))
            D = tb.grouped_gemm(0.7, a, b, s, 0.3, c)
            assert torch.equal(D.detach(), want), need
            leaves = [t for t in (a, b, c) if t.requires_grad]
            grads = dict(zip([i for i in range(3) if need[i]], torch.autograd.grad(D, leaves, dD.to(D.dtype))))
            if 0 in grads:
                assert torch.equal(grads[0], tb.grouped_gemm(0.7, dD, B, s, transB=True))
            if 1 in grads:
                assert torch.equal(grads[1], tb.grouped_gemm_wgrad(0.7, A, dD, s))
            if 2 in grads:
                x = 0.3 * dD.double()
                ref2 = x.sum_to_size(C.shape)
                mag = x.abs().sum_to_size(C.shape)
                # beta * dD rounds to its type, the sum over up to 136 of them once more (fp32 inside)
                eps = torch.finfo(C.dtype).eps
                assert grads[2].shape == C.shape and grads[2].dtype == C.dtype
                assert ((grads[2].double() - ref2).abs() <= (eps + 140 * 2.0 ** -24) * mag).all()


def test_forward_mode_of_a_c_that_torch_adds():
    """Where the kernels take no part, torch's own derivative stands: a C that
    broadcasts, a C that beta = 0 does not read, and C's gradient alone."""
    import torch.autograd.forward_ad as fwd

    A, B, s = _rand(6, 64), _rand(2, 64, 32), _sizes([3, 3])
    C, full = _rand(1, 32, seed=1), _rand(6, 32, seed=2)
    want = tb.grouped_gemm(1.0, A, B, s, 2.0, C)
    with fwd.dual_level():
        for a in (A, A.clone().requires_grad_()):
            D = tb.grouped_gemm(1.0, a, B, s, 2.0, fwd.make_dual(C, C))
            v, t = fwd.unpack_dual(D)
            assert torch.equal(v.detach(), want) and torch.equal(t.detach(), (2.0 * C).expand(6, 32))
        D = tb.grouped_gemm(1.0, A, B, s, 0.0, fwd.make_dual(full, full))
        assert torch.equal(D, tb.grouped_gemm(1.0, A, B, s)) and fwd.unpack_dual(D).tangent is None
        with pytest.raises(NotImplementedError):
            tb.grouped_gemm(1.0, A, B, s, 2.0, fwd.make_dual(full, full))
        c = full.clone().requires_grad_()
        (g,) = torch.autograd.grad(tb.grouped_gemm(1.0, A, B, s, 2.0, c), c, fwd.make_dual(want, full))
        assert torch.equal(fwd.unpack_dual(g).primal, 2.0 * want) and torch.equal(fwd.unpack_dual(g).tangent, 2.0 * full)
