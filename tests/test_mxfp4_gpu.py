"""MXFP4 on a B200: the quantiser bit for bit against the definition, its
inverse, and the dense and grouped products against 64 bits on the values that
the 4-bit operands stand for (tolerance derived in oracle/experts.py)."""

from __future__ import annotations

import pytest
import torch

import trnblas_b200 as tb
from oracle import experts as X

pytestmark = pytest.mark.gpu
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
DEV = "cuda"


def _gen(*key):
    return torch.Generator(device=DEV).manual_seed(hash(key) % (1 << 31))


def _rand(*shape, dt=BF, seed=0):
    return torch.randn(*shape, device=DEV, generator=_gen(seed, *shape)).to(dt)


def _rand_mx(*shape, seed=0, lo=117, hi=138):
    """Every code, and scales of different magnitude in every block."""
    *lead, K = shape
    g = _gen(seed, *shape)
    codes = torch.randint(0, 256, (*lead, -(-K // 2)), dtype=torch.uint8, device=DEV, generator=g)
    scales = torch.randint(lo, hi, (*lead, -(-K // 32)), dtype=torch.uint8, device=DEV, generator=g)
    return tb.MXFP4Tensor.from_parts(codes, scales, K)


def _values(q):
    """float64 values of a quantised operand, from its parts."""
    codes, scales = q.parts()
    K = q.shape[-1]
    lut = torch.tensor([*X.VALUES, *(-v for v in X.VALUES)], dtype=torch.float64, device=codes.device)
    v = torch.stack((lut[(codes & 15).long()], lut[(codes >> 4).long()]), -1).reshape(*codes.shape[:-1], -1, 32)
    pow2 = torch.tensor([2.0 ** (s - 127) for s in range(255)] + [float("nan")], dtype=torch.float64, device=codes.device)
    return (v * pow2[scales.long()].unsqueeze(-1)).reshape(*codes.shape[:-1], -1)[..., :K]


@pytest.mark.parametrize("dt", [BF, FP, F32])
@pytest.mark.parametrize("rows,K", [(1, 1), (1, 32), (3, 33), (5, 128), (31, 200), (33, 256), (70, 1000), (257, 4096), (2, 70001)])
def test_quantise_bit_for_bit(dt, rows, K):
    x = (_rand(rows, K, dt=F32) * torch.exp2(torch.randint(-12, 8, (rows, K), device=DEV, generator=_gen(rows, K)).float())).to(dt)
    q = tb.quantize_mxfp4(x)
    v, e, bad = X.quantize(x)
    codes, scales = q.parts()
    assert torch.equal(scales.long(), e + 127)
    ref = X.dequantize(v, e, bad, K)
    assert torch.equal(_values(q), ref)
    assert torch.equal(torch.signbit(_values(q)), torch.signbit(ref))
    assert torch.equal(tb.dequantize_mxfp4(q).double(), ref)
    assert torch.equal(tb.dequantize_mxfp4(q, BF).double(), ref)
    assert torch.equal(tb.dequantize_mxfp4(q, FP), ref.to(F32).to(FP))
    again = tb.MXFP4Tensor.from_parts(codes, scales, K)  # zeros behind the rows and behind K
    assert torch.equal(again.scales, q.scales) and torch.equal(again.data, q.data)


def test_every_float_of_a_grid_and_the_extremes():
    """All bf16 magnitudes against a block maximum, ties included; subnormals,
    the largest values, signed zeros, blocks with an infinity or a NaN."""
    bits = torch.arange(0, 1 << 15, device=DEV, dtype=torch.int32)
    vals = (bits << 16).view(F32)
    vals = vals[vals.isfinite()]
    n = vals.numel() // 16 * 16
    x = torch.zeros(n // 16, 32, device=DEV)
    x[:, ::2], x[:, 1::2] = vals[:n].view(-1, 16), -vals[:n].view(-1, 16)
    for dt in (BF, F32):
        q = tb.quantize_mxfp4(x.to(dt))
        ref = X.dequantize(*X.quantize(x), 32)
        assert torch.equal(_values(q), ref)
        assert torch.equal(tb.dequantize_mxfp4(q, BF).double(), ref)
    y = torch.zeros(6, 64, device=DEV)
    y[0, 3], y[1, 40], y[2, 0] = float("inf"), float("nan"), float("-inf")
    y[3, :2] = torch.tensor([2.0 ** -149, -(2.0 ** -127)])
    y[4, :3] = torch.tensor([3.4e38, -1e38, 1.0])
    y[5] = -0.0
    q = tb.quantize_mxfp4(y)
    _, s = q.parts()
    assert s.tolist()[:3] == [[255, 0], [0, 255], [255, 0]]
    v = tb.dequantize_mxfp4(q)
    assert v[0, :32].isnan().all() and (v[0, 32:] == 0).all() and v[1, 32:].isnan().all()
    assert torch.equal(v[3:].double(), X.dequantize(*X.quantize(y[3:]), 64))
    assert torch.signbit(v[5]).all()


def test_quantise_layouts():
    x = _rand(40, 3 * 96)
    part = x[:, 96:192]
    want = tb.quantize_mxfp4(part.contiguous())
    for t in (part, part.mT.contiguous().mT, x[:, 95:191].roll(0)):
        got = tb.quantize_mxfp4(t)
        ref = tb.quantize_mxfp4(t.contiguous())
        assert torch.equal(got.data, ref.data) and torch.equal(got.scales, ref.scales)
    assert torch.equal(tb.quantize_mxfp4(part).data, want.data)
    y = _rand(3, 7, 160)
    q3, q2 = tb.quantize_mxfp4(y), tb.quantize_mxfp4(y.reshape(21, 160))
    assert q3.shape == (3, 7, 160) and torch.equal(q3.data.view(21, -1), q2.data)
    assert torch.equal(q3.parts()[1].view(21, -1), q2.parts()[1])
    qc = tb.quantize_mxfp4(y.cpu())
    assert qc.device.type == "cpu" and torch.equal(qc.data, q3.data.cpu())
    assert torch.equal(tb.dequantize_mxfp4(qc), tb.dequantize_mxfp4(q3).cpu())
    assert torch.equal(tb.quantize_mxfp4(_rand(1, 64).expand(5, 64)).data[4], tb.quantize_mxfp4(_rand(1, 64)).data[0])


DENSE = [(1, 128, 64), (1, 8, 32), (3, 130, 33), (17, 257, 256), (64, 128, 1000), (65, 384, 128), (200, 100, 520),
         (192, 256, 256), (385, 200, 4096), (1000, 640, 776), (448, 129, 288), (321, 300, 640),
         (777, 4096, 520), (500, 9000, 264), (1500, 4104, 300), (400, 4100, 1000), (130, 9000, 96),
         (9700, 128, 300), (9601, 100, 64)]


@pytest.mark.parametrize("M,Nn,K", DENSE)
def test_gemm_mxfp4(M, Nn, K):
    qa, qb = _rand_mx(M, K, seed=1), _rand_mx(Nn, K, seed=2)
    a, b = _values(qa), _values(qb)
    ref, mags = a @ b.T, a.abs() @ b.abs().T
    for out in (BF, FP, F32):
        D = tb.gemm_mxfp4(2.0 ** -7, qa, qb, out_dtype=out)
        assert D.dtype == out and D.shape == (M, Nn)
        X.check(D, ref * 2.0 ** -7, X.tolerance(ref * 2.0 ** -7, mags * 2.0 ** -7, K, out), f"{M} {Nn} {K} {out}")
    assert tb.device_status(0) == 0


def test_whole_numbers_are_exact():
    """Scales of 1 and 2 and whole halves: sums below 2^22 quarters are exact."""
    qa, qb = _rand_mx(333, 544, lo=127, hi=129), _rand_mx(210, 544, seed=5, lo=126, hi=129)
    assert torch.equal(tb.gemm_mxfp4(1.0, qa, qb, out_dtype=F32).double(), _values(qa) @ _values(qb).T)


@pytest.mark.parametrize("dt", [BF, FP, F32])
@pytest.mark.parametrize("M", [1, 9, 300])
def test_operand_quantised_on_the_way(dt, M):
    x, qb = _rand(M, 200, dt=dt), tb.quantize_mxfp4(_rand(72, 200, seed=3))
    D = tb.gemm_mxfp4(1.0, x, qb)
    if M > 16:  # (a few rows split K over CTAs: another order of the same sum)
        assert torch.equal(D, tb.gemm_mxfp4(1.0, tb.quantize_mxfp4(x), qb))
    a = X.dequantize(*X.quantize(x), 200)
    b = _values(qb)
    ref = a @ b.T
    X.check(D, ref, X.tolerance(ref, a.abs() @ b.abs().T, 200, BF))


@pytest.mark.parametrize("M", [1, 2, 7, 16])
@pytest.mark.parametrize("Nn,K", [(8, 32), (128, 256), (130, 1000), (520, 4096), (200, 33), (64, 8200), (2048, 700),
                                  (136, 45056), (64, 44000), (128, 50000)])
def test_few_rows(M, Nn, K):
    """Rows quantised inside the product, K split over a cluster: as many
    splits as fit, blocks that end inside a rank's share, and ranks with none."""
    dt = (BF, FP, F32)[M % 3]
    x, qb = _rand(M, K, dt=dt), _rand_mx(Nn, K, seed=3)
    a, b = X.dequantize(*X.quantize(x), K), _values(qb)
    ref, mags = a @ b.T, a.abs() @ b.abs().T
    C = _rand(M, Nn, dt=F32)
    X.check(tb.gemm_mxfp4(1.0, x, qb), ref, X.tolerance(ref, mags, K, BF))
    ref2 = 0.5 * ref - 2.0 * C.double()
    D = tb.gemm_mxfp4(0.5, x, qb, -2.0, C, out_dtype=F32)
    X.check(D, ref2, X.tolerance(ref2, mags, K, F32, 2.0 * C))
    assert torch.equal(D, tb.gemm_mxfp4(0.5, x, qb, -2.0, C, out_dtype=F32))
    big = torch.zeros(M, 2 * K + 8, dtype=dt, device=DEV)  # rows off 16 bytes and far apart
    big[:, 1:K + 1] = x
    assert torch.equal(tb.gemm_mxfp4(1.0, big[:, 1:K + 1], qb), tb.gemm_mxfp4(1.0, x, qb))
    assert tb.device_status(0) == 0


def test_few_rows_with_nan_and_infinity():
    x, qb = _rand(5, 600), tb.quantize_mxfp4(_rand(72, 600))
    clean = tb.gemm_mxfp4(1.0, x, qb)
    x[1, 599], x[3, 0] = float("inf"), float("nan")
    D = tb.gemm_mxfp4(1.0, x, qb)
    assert torch.equal(D[[0, 2, 4]], clean[[0, 2, 4]]) and D[[1, 3]].isnan().all()
    s = torch.randint(100, 140, (72, 19), dtype=torch.uint8, device=DEV, generator=_gen(2))
    s[11, 18] = 255  # a NaN block among the weights
    D = tb.gemm_mxfp4(1.0, x[:1], tb.MXFP4Tensor.from_parts(qb.parts()[0], s, 600))
    assert D[0, 11].isnan() and D.isnan().sum() == 1


def test_alpha_beta_c_and_nan_scales():
    qa, qb = tb.quantize_mxfp4(_rand(130, 320)), tb.quantize_mxfp4(_rand(264, 320, seed=1))
    a, b = _values(qa), _values(qb)
    for out in (BF, F32):
        C = _rand(130, 264, dt=out)
        ref, mags = -1.5 * (a @ b.T) + 0.25 * C.double(), 1.5 * (a.abs() @ b.abs().T)
        X.check(tb.gemm_mxfp4(-1.5, qa, qb, 0.25, C, out_dtype=out), ref, X.tolerance(ref, mags, 320, out, C))
        nan = torch.full_like(C, float("nan"))
        assert torch.equal(tb.gemm_mxfp4(1.0, qa, qb, 0.0, nan, out_dtype=out), tb.gemm_mxfp4(1.0, qa, qb, out_dtype=out))
    x = _rand(130, 320)
    clean = tb.gemm_mxfp4(1.0, x, qb)
    x[7, 100] = float("nan")
    x[129, 319] = float("inf")
    D = tb.gemm_mxfp4(1.0, x, qb)
    keep = [r for r in range(130) if r not in (7, 129)]
    assert D[7].isnan().all() and D[129].isnan().all() and torch.equal(D[keep], clean[keep])
    assert (tb.gemm_mxfp4(1.0, _rand(5, 0), tb.quantize_mxfp4(_rand(7, 0))) == 0).all()
    assert tb.gemm_mxfp4(1.0, _rand(0, 64), tb.quantize_mxfp4(_rand(7, 64))).shape == (0, 7)


SIZES = [[0], [1], [0, 0, 5, 0], [300, 0, 1, 17], [64, 65, 63, 1, 0, 128], [193, 192, 191, 400], [2] * 37, [130, 257, 0, 385, 63]]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
@pytest.mark.parametrize("K,Nn", [(256, 128), (96, 72), (1000, 200), (33, 129)])
def test_grouped_gemm_mxfp4(sizes, K, Nn):
    rows = sum(sizes) + (K % 3) * 23 + (1 if sizes == [0] else 0)
    qa, qb = _rand_mx(rows, K, seed=4), _rand_mx(len(sizes), Nn, K, seed=5)
    s = torch.tensor(sizes, dtype=torch.int32, device=DEV)
    ref, mags = X.grouped_gemm(1.0, _values(qa), _values(qb), sizes, transB=True)
    for out in (BF, F32):
        D = tb.grouped_gemm_mxfp4(1.0, qa, qb, s, out_dtype=out)
        X.check(D, ref, X.tolerance(ref, mags, K, out), f"{sizes} {K} {Nn} {out}")
    C = _rand(rows, Nn, dt=F32)
    ref2 = 0.5 * ref + 2.0 * C.double()
    D = tb.grouped_gemm_mxfp4(0.5, qa, qb, s.long(), 2.0, C, out_dtype=F32)
    X.check(D, ref2, X.tolerance(ref2, mags, K, F32, 2.0 * C))
    assert tb.device_status(0) == 0


@pytest.mark.parametrize("sizes", [[513, 64, 0, 255, 256, 257], [1, 0, 1290, 3], [9000, 0, 5001, 17]],
                         ids=lambda s: f"{len(s)}x{max(s)}")
@pytest.mark.parametrize("K,Nn", [(256, 2056), (1000, 4100), (33, 2304), (96, 128)])
def test_grouped_gemm_mxfp4_many_tiles(sizes, K, Nn):
    """Enough tiles for the CTA pairs (or, with few columns, one CTA's long ones)."""
    rows = sum(sizes) + (K % 3) * 150
    x, qb = _rand(rows, K, seed=4), _rand_mx(len(sizes), Nn, K, seed=5)
    s = torch.tensor(sizes, dtype=torch.int32, device=DEV)
    a = X.dequantize(*X.quantize(x), K)
    ref, mags = X.grouped_gemm(1.0, a, _values(qb), sizes, transB=True)
    D = tb.grouped_gemm_mxfp4(1.0, x, qb, s)
    X.check(D, ref, X.tolerance(ref, mags, K, BF))
    # rows quantised before: their scales are regrouped, the product is the same
    assert torch.equal(D, tb.grouped_gemm_mxfp4(1.0, tb.quantize_mxfp4(x), qb, s))
    assert torch.equal(D, tb.grouped_gemm_mxfp4(1.0, x, qb, s))
    assert tb.device_status(0) == 0


@pytest.mark.parametrize("Nn", [136, 9000])
def test_grouped_nan_stays_in_its_rows(Nn):
    sizes, K = [50, 0, 83, 20], 352
    s = torch.tensor(sizes, device=DEV)
    x, qb = _rand(193, K), tb.quantize_mxfp4(_rand(4, Nn, K))
    clean = tb.grouped_gemm_mxfp4(1.0, x, qb, s)
    x2 = x.clone()
    x2[153:] = float("nan")
    x2[51] = float("inf")
    D = tb.grouped_gemm_mxfp4(1.0, x2, qb, s)
    assert (D[153:] == 0).all() and D[51].isnan().all()
    keep = [r for r in range(153) if r != 51]
    assert torch.equal(D[keep], clean[keep])


def test_layer_in_4_bits():
    """Quantised experts as a serving layer uses them: sorted tokens, two
    grouped products, each checked on the operands it got; a single token too."""
    G, dim, hidden = 5, 256, 384
    w1, w2 = tb.quantize_mxfp4(_rand(G, hidden, dim) * dim ** -0.5), tb.quantize_mxfp4(_rand(G, dim, hidden) * hidden ** -0.5)
    for tokens in (1, 77):
        x = _rand(tokens, dim, seed=tokens)
        expert = torch.randint(0, G, (tokens,), device=DEV, generator=_gen(tokens)).sort().values
        sizes = torch.bincount(expert, minlength=G)
        h = tb.grouped_gemm_mxfp4(1.0, x, w1, sizes)
        a = torch.relu(h)
        y = tb.grouped_gemm_mxfp4(1.0, a, w2, sizes)
        for inp, w, out, K in ((x, w1, h, dim), (a, w2, y, hidden)):
            v = X.dequantize(*X.quantize(inp), K)
            ref, mags = X.grouped_gemm(1.0, v, _values(w), sizes.tolist(), transB=True)
            X.check(out, ref, X.tolerance(ref, mags, K, BF))


def test_captured_graph_and_streams():
    x, qb = _rand(40, 512), tb.quantize_mxfp4(_rand(3, 256, 512))
    s = torch.tensor([10, 5, 20], dtype=torch.int32, device=DEV)
    w = tb.quantize_mxfp4(_rand(256, 512))
    tb.grouped_gemm_mxfp4(1.0, x, qb, s)
    tb.gemm_mxfp4(1.0, x, w)
    torch.cuda.synchronize()
    graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        D = tb.grouped_gemm_mxfp4(1.0, x, qb, s)
    with torch.cuda.graph(graph2):
        E = tb.gemm_mxfp4(1.0, x, w)
    for sizes in ([10, 5, 20], [0, 40, 0], [0, 0, 0]):
        s.copy_(torch.tensor(sizes, dtype=torch.int32))
        x.copy_(_rand(40, 512, seed=sizes[1]))
        graph.replay()
        graph2.replay()
        torch.cuda.synchronize()
        assert torch.equal(D, tb.grouped_gemm_mxfp4(1.0, x, qb, s))
        assert torch.equal(E, tb.gemm_mxfp4(1.0, x, w))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        outs = [tb.gemm_mxfp4(1.0, x, w) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, E) for o in outs)


def test_offsets_past_32_bits():
    rows, K, Nn = 66000, 64, 33000
    x, w = _rand(rows, K), tb.quantize_mxfp4(_rand(Nn, K))
    D = tb.gemm_mxfp4(1.0, x, w)
    a, b = X.dequantize(*X.quantize(x[-50:]), K), _values(w)
    ref = a @ b.T
    X.check(D[-50:], ref, X.tolerance(ref, a.abs() @ b.abs().T, K, BF))


@pytest.mark.parametrize("K,ldq", [(64, 64), (33, 128), (8, 32), (300, 320), (256, 256), (1000, 512), (64, 32)])
def test_row_strides_longer_than_the_rows(K, ldq):
    """Through the C ABI: a stack whose packed rows lie further apart than they
    are long. What lies between them, behind the last one and in a neighbour's
    columns keeps its bytes; the inverse and the product read the same rows."""
    from trnblas_b200 import _native as N

    mats, rows, w = 2, 131, -(-K // 32) * 16
    x = _rand(mats, rows, K, dt=BF)
    want = tb.quantize_mxfp4(x)
    buf = torch.full((mats * rows * ldq + 512,), 0xA5, dtype=torch.uint8, device=DEV)
    scales = torch.empty_like(want.scales)
    st = torch.cuda.current_stream().cuda_stream
    rc = N.lib().trnblas_mxfp4_quantize(N.BF16, mats, rows, K, x.data_ptr(), K, buf.data_ptr(), ldq, scales.data_ptr(), st)
    assert rc == 0 and torch.equal(scales, want.scales)
    got = buf[: mats * rows * ldq].view(mats, rows, ldq)
    assert torch.equal(got[..., :w], want.data)
    assert (got[..., w:] == 0xA5).all() and (buf[mats * rows * ldq:] == 0xA5).all()
    y = torch.full((mats, rows, K), 7.0, dtype=F32, device=DEV)
    rc = N.lib().trnblas_mxfp4_dequantize(N.F32, mats, rows, K, buf.data_ptr(), ldq, scales.data_ptr(), y.data_ptr(), K, st)
    assert rc == 0 and torch.equal(y, tb.dequantize_mxfp4(want))
    # the second matrix as the weights of products of one and of many rows
    q2 = tb.MXFP4Tensor(want.data[1].contiguous(), want.scales[1:].contiguous(), (rows, K))
    for m in (1, 40):
        a = x[0, :m].contiguous()
        ws = torch.empty(max(1, N.lib().trnblas_mxfp4_gemm_x_workspace_size(m, 1, K, 0)), dtype=torch.uint8, device=DEV)
        d = torch.empty(m, rows, dtype=BF, device=DEV)
        rc = N.lib().trnblas_mxfp4_gemm_x(N.BF16, N.BF16, m, 1, rows, K, 1.0, a.data_ptr(), K, buf.data_ptr() + rows * ldq, ldq,
                                          scales[1].data_ptr(), None, 0, 0.0, None, 0, d.data_ptr(), rows, ws.data_ptr(),
                                          ws.numel(), st)
        assert rc == 0 and torch.equal(d, tb.gemm_mxfp4(1.0, a, q2))
