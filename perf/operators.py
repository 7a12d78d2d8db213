"""Products grouped by expert and microscaled 4-bit floating point: the
operators' plain forms, their definitions in 64 bits, and the calls a program
makes of them, over the sizes they are used at.

Operators (`op` of a case):

  forward    D[r] = A[r] @ op(B[g]) for the rows r of group g; the rows behind
             the last group are an empty product (zero)
  training   the forward product, and for an incoming gradient dD the
             gradients dA[r] = dD[r] @ op(B[g])^T and dB[g] = A_g^T dD_g (of
             the same layout as B)
  quantise   rows cut into blocks of 32 values, each block as 32 E2M1 values
             and one power of two: the largest power of two not above the
             block's largest magnitude, divided by 4 (values above 6 of the
             block's unit become 6, ties go to the even mantissa)
  product    D = Q(x) @ W^T for x in 16 or 32 bits, quantised on the way, and
             W already held in 4 bits
  experts    the same grouped by expert: D[r] = Q(x)[r] @ W[g]^T

A case holds sizes, types and how the rows spread over the groups; the group
sizes follow from the case alone, the values from the seed.
"""

import math
import random

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BLOCK = 32


# ── cases ────────────────────────────────────────────────────────────────────


def listed():
    return [
        # one decoding step of a small batch, each token sent to a few of 16
        # experts: some get none, most one or two rows
        {"name": "forward-decode", "op": "forward", "T": 24, "pad": 0, "G": 16, "K": 2048, "N": 1536,
         "dt": "bf16", "transB": False, "spread": "skewed"},
        # a ragged prefill in fp16 with a buffer longer than the rows in use
        {"name": "forward-prefill", "op": "forward", "T": 4133, "pad": 91, "G": 8, "K": 1024, "N": 2816,
         "dt": "fp16", "transB": True, "spread": "skewed"},
        # a large batch over many experts
        {"name": "forward-large", "op": "forward", "T": 16384, "pad": 0, "G": 32, "K": 2048, "N": 4096,
         "dt": "bf16", "transB": False, "spread": "even"},
        # a training step of a small model: few rows an expert
        {"name": "training-small", "op": "training", "T": 515, "pad": 0, "G": 8, "K": 512, "N": 1024,
         "dt": "bf16", "transB": False, "spread": "skewed"},
        # a training step's expert layer at full size
        {"name": "training-large", "op": "training", "T": 16384, "pad": 0, "G": 16, "K": 4096, "N": 2048,
         "dt": "bf16", "transB": True, "spread": "skewed"},
        # the activations of a decoding step
        {"name": "quantise-few", "op": "quantise", "M": 8, "K": 4096, "dt": "bf16"},
        # a layer's weights or a long prefill's activations
        {"name": "quantise-large", "op": "quantise", "M": 16384, "K": 8192, "dt": "bf16"},
        # one token through a 4-bit layer
        {"name": "product-token", "op": "product", "M": 1, "N": 8192, "K": 8192, "dt": "bf16"},
        # an odd number of rows and a length that ends inside a block
        {"name": "product-ragged", "op": "product", "M": 777, "N": 4096, "K": 4010, "dt": "fp16"},
        # a large product
        {"name": "product-large", "op": "product", "M": 8192, "N": 8192, "K": 8192, "dt": "bf16"},
        # a decoding batch over 4-bit experts
        {"name": "experts-decode", "op": "experts", "T": 64, "pad": 0, "G": 32, "K": 4096, "N": 2048,
         "dt": "bf16", "spread": "skewed"},
        # a prefill over 4-bit experts
        {"name": "experts-large", "op": "experts", "T": 16384, "pad": 0, "G": 16, "K": 4096, "N": 4096,
         "dt": "bf16", "spread": "even"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["forward", "training", "quantise", "product", "experts"])
    dt = rng.choice(["bf16", "fp16"])
    if op == "quantise":
        M, K = _log(rng, 1, 16384), _log(rng, 32, 8192)
        return {"op": op, "M": M, "K": K, "dt": rng.choice(["bf16", "fp16", "fp32"])}
    if op == "product":
        M, N, K = _log(rng, 1, 8192), _log(rng, 64, 8192), _log(rng, 64, 8192)
        return {"op": op, "M": M, "N": N, "K": K, "dt": rng.choice(["bf16", "fp16", "fp32"])}
    T, G = _log(rng, 1, 16384), _log(rng, 1, 64)
    K, N = _log(rng, 64, 4096), _log(rng, 64, 4096)
    while G * K * N > 16 * 4096 * 4096:
        G = max(1, G // 2)
    if op == "training":
        K = min(K, 2048)
    # 16-bit rows that start on 16 bytes half the time, any length otherwise
    if rng.random() < 0.5:
        K, N = max(64, K // 8 * 8), max(64, N // 8 * 8)
    case = {"op": op, "T": T, "pad": rng.choice([0, 0, rng.randint(1, 200)]), "G": G, "K": K, "N": N, "dt": dt,
            "spread": rng.choice(["even", "skewed"])}
    if op != "experts":
        case["transB"] = rng.random() < 0.5
    return case


def _group_sizes(case):
    """Rows of each group: even, or skewed with about a quarter of the groups
    empty (the expert that most rows go to gets a few times the mean)."""
    T, G = case["T"], case["G"]
    rng = random.Random(f"{T}/{G}/{case['K']}/{case['N']}/{case['spread']}")
    if case["spread"] == "even":
        w = [1.0 + 0.1 * rng.random() for _ in range(G)]
    else:
        w = [rng.expovariate(1.0) if rng.random() > 0.25 else 0.0 for _ in range(G)]
        if not any(w):
            w[rng.randrange(G)] = 1.0
    total, acc, ends = sum(w), 0.0, []
    for x in w:
        acc += x
        ends.append(int(round(T * acc / total)))
    ends[-1] = T
    return [e - b for b, e in zip([0] + ends[:-1], ends)]


# ── inputs ───────────────────────────────────────────────────────────────────


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    dt, op, K = _DT[case["dt"]], case["op"], case["K"]
    st = {"case": case, "dt": dt}
    if op == "quantise":
        # rows of different magnitudes, as a layer's activations have
        st["x"] = (randn(case["M"], K) * torch.exp(randn(case["M"], 1))).to(dt)
        return st
    if op == "product":
        st["x"] = randn(case["M"], K).to(dt)
        st["w"] = _weights4(g, case["N"], K)
        if own:
            import trnblas_b200 as tb

            st["wq"] = tb.MXFP4Tensor.from_parts(*st["w"], K)
        return st
    T, G, N = case["T"], case["G"], case["N"]
    st["sizes"] = _group_sizes(case)
    st["group_sizes"] = torch.tensor(st["sizes"], dtype=torch.int32, device="cuda")
    st["a"] = randn(T + case["pad"], K).to(dt)
    if op == "experts":
        parts = [_weights4(g, N, K) for _ in range(G)]
        st["w"] = tuple(torch.stack(p) for p in zip(*parts))
        if own:
            import trnblas_b200 as tb

            st["wq"] = tb.MXFP4Tensor.from_parts(*st["w"], K)
        return st
    b = torch.empty(G, *((N, K) if case["transB"] else (K, N)), dtype=dt, device="cuda")
    for i in range(G):
        b[i] = (randn(*b.shape[1:]) * K ** -0.5).to(dt)
    st["b"] = b
    if op == "training":
        st["dd"] = randn(T + case["pad"], N).to(dt)
        st["a"].requires_grad_()
        st["b"].requires_grad_()
    return st


def _weights4(g, rows, K):
    """(codes, scales): rows of K weights in blocks of 32, two 4-bit codes a
    byte (the earlier one in the low half) and one biased exponent a block."""
    w = torch.randn(rows, K, device="cuda", generator=g) * K ** -0.5
    q, e = _quantise(w)
    mag = q.abs()
    codes = torch.zeros_like(q, dtype=torch.uint8)
    for c, v in enumerate((0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)):
        codes[mag == v] = c
    codes += torch.signbit(q).to(torch.uint8) * 8
    codes = codes.reshape(rows, -1)
    return codes[:, 0::2] | (codes[:, 1::2] << 4), (e + 127).to(torch.uint8)


# ── plain forms ──────────────────────────────────────────────────────────────


def _quantise(x):
    """(values in the block's unit (rows, blocks, 32), exponents (rows, blocks))."""
    rows, K = x.shape
    xf = torch.nn.functional.pad(x.float(), (0, -K % _BLOCK)).reshape(rows, -1, _BLOCK)
    amax = xf.abs().amax(-1)
    e = torch.frexp(amax).exponent - 3
    e = torch.where(amax == 0, -127, e).clamp(-127, 125)
    u = torch.ldexp(xf, -e.unsqueeze(-1))
    m = u.abs()
    step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0))
    r = (torch.round(m / step) * step).clamp(max=6.0)
    return torch.copysign(r, u), e


def _quantised(x):
    q, e = _quantise(x)
    return torch.ldexp(q, e.unsqueeze(-1)).reshape(x.shape[0], -1)[:, : x.shape[1]]


def _expand(codes, scales, K, dtype=torch.float32):
    """The values that 4-bit codes and their blocks' exponents stand for."""
    lut = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0],
                       dtype=dtype, device=codes.device)
    v = torch.stack((lut[(codes & 15).long()], lut[(codes >> 4).long()]), -1)
    v = v.reshape(*codes.shape[:-1], -1, _BLOCK)
    v = torch.ldexp(v, scales.int().unsqueeze(-1) - 127)
    return v.reshape(*codes.shape[:-1], -1)[..., :K]


def _ranges(sizes):
    r0 = 0
    for i, m in enumerate(sizes):
        yield i, slice(r0, r0 + m)
        r0 += m


def _plain(st):
    case, op, dt = st["case"], st["case"]["op"], st["dt"]
    if op == "quantise":
        return _quantised(st["x"]).to(torch.bfloat16)
    if op == "product":
        return (_quantised(st["x"]) @ _expand(*st["w"], case["K"]).T).to(torch.bfloat16)
    a = st["a"].detach()
    rows, K, N = a.shape[0], case["K"], case["N"]
    if op == "experts":
        x = _quantised(a)
        d = torch.zeros(rows, N, dtype=torch.bfloat16, device=a.device)
        for i, s in _ranges(st["sizes"]):
            d[s] = (x[s] @ _expand(st["w"][0][i], st["w"][1][i], K).T).to(torch.bfloat16)
        return d
    b = st["b"].detach()
    d = torch.zeros(rows, N, dtype=dt, device=a.device)
    train = op == "training"
    if train:
        dd = st["dd"]
        da, db = torch.zeros_like(a), torch.empty_like(b)
    for i, s in _ranges(st["sizes"]):
        w = b[i].float().T if case["transB"] else b[i].float()
        x = a[s].float()
        d[s] = (x @ w).to(dt)
        if train:
            y = dd[s].float()
            da[s] = (y @ w.T).to(dt)
            db[i] = (y.T @ x if case["transB"] else x.T @ y).to(dt)
    return (d, da, db) if train else d


def run(state):
    if not own:
        return _plain(state)
    import trnblas_b200 as tb

    case, op = state["case"], state["case"]["op"]
    if op == "quantise":
        return tb.dequantize_mxfp4(tb.quantize_mxfp4(state["x"]), torch.bfloat16)
    if op == "product":
        return tb.gemm_mxfp4(1.0, state["x"], state["wq"], out_dtype=torch.bfloat16)
    if op == "experts":
        return tb.grouped_gemm_mxfp4(1.0, state["a"], state["wq"], state["group_sizes"], out_dtype=torch.bfloat16)
    d = tb.grouped_gemm(1.0, state["a"], state["b"], state["group_sizes"], transB=case["transB"])
    if op == "forward":
        return d
    da, db = torch.autograd.grad(d, (state["a"], state["b"]), state["dd"])
    return d.detach(), da, db


# ── the definition in 64 bits ────────────────────────────────────────────────


def _exact_quantised(x):
    """The quantised values from the nearest of the eight magnitudes."""
    x = x.double()
    rows, K = x.shape
    nb = -(-K // _BLOCK)
    xp = torch.zeros(rows, nb * _BLOCK, dtype=torch.float64, device=x.device)
    xp[:, :K] = x
    xp = xp.view(rows, nb, _BLOCK)
    top = xp.abs().max(-1, keepdim=True).values
    # the logarithm may be off by a rounding next to a power of two: the borders decide
    unit = torch.where(top > 0, torch.exp2(torch.floor(torch.log2(top)) - 2), torch.zeros_like(top))
    unit = torch.where(top >= 8 * unit, 2 * unit, torch.where(top < 4 * unit, unit / 2, unit))
    unit = unit.clamp(min=2.0 ** -127)
    t = xp.abs() / unit
    out = torch.zeros_like(t)
    # a magnitude is taken from its lower border on; a border itself goes to
    # the neighbour with the even mantissa
    for border, up, value in ((0.25, False, 0.5), (0.75, True, 1.0), (1.25, False, 1.5), (1.75, True, 2.0),
                              (2.5, False, 3.0), (3.5, True, 4.0), (5.0, False, 6.0)):
        out = torch.where(t >= border if up else t > border, value, out)
    return (torch.sign(xp) * out * unit).view(rows, -1)[:, :K]


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "quantise":
        return _exact_quantised(st["x"])
    if op == "product":
        return torch.matmul(_exact_quantised(st["x"]), _expand(*st["w"], case["K"], torch.float64).mT)
    a = st["a"].detach()
    rows = torch.arange(a.shape[0], device=a.device)
    ends = torch.cumsum(st["group_sizes"].long(), 0)
    owner = torch.bucketize(rows, ends, right=True)  # G behind the last group
    out = torch.zeros(a.shape[0], case["N"], dtype=torch.float64, device=a.device)
    x = _exact_quantised(a) if op == "experts" else a.double()
    grads = op == "training"
    if grads:
        dd = st["dd"].double()
        ga = torch.zeros_like(x)
        gb = torch.zeros(st["b"].shape, dtype=torch.float64, device=a.device)
    for i in range(case["G"]):
        idx = (owner == i).nonzero().squeeze(1)
        if op == "experts":
            w = _expand(st["w"][0][i], st["w"][1][i], case["K"], torch.float64)
        else:
            w = st["b"][i].detach().double()
            if not case["transB"]:
                w = w.mT
        xi = x.index_select(0, idx)
        out.index_copy_(0, idx, torch.einsum("tk,nk->tn", xi, w))
        if grads:
            di = dd.index_select(0, idx)
            ga.index_copy_(0, idx, torch.einsum("tn,nk->tk", di, w))
            gw = torch.einsum("tn,tk->nk", di, xi)
            gb[i] = gw if case["transB"] else gw.mT
    return (out, ga, gb) if grads else out


# ── what a pass cannot do without ────────────────────────────────────────────


def work(case):
    op, es = case["op"], 4 if case["dt"] == "fp32" else 2
    K = case["K"]
    if op == "quantise":
        n = case["M"] * K
        return {"bytes": n * es + n * 2, "flops": 2 * n}
    q4 = (K + 1) // 2 + -(-K // _BLOCK)  # bytes of K values in 4 bits with their scales
    if op == "product":
        M, N = case["M"], case["N"]
        return {"bytes": M * K * es + N * q4 + M * N * 2, "flops": 2 * M * N * K}
    T, N = case["T"], case["N"]
    used = sum(1 for m in _group_sizes(case) if m)
    rows = T + case["pad"]
    if op == "experts":
        return {"bytes": T * K * es + used * N * q4 + rows * N * 2, "flops": 2 * T * N * K}
    fwd = T * K * es + used * N * K * es + rows * N * es
    if op == "forward":
        return {"bytes": fwd, "flops": 2 * T * N * K}
    # read A, B, dD once; write D, dA, dB once
    back = T * N * es + rows * K * es + case["G"] * N * K * es
    return {"bytes": fwd + back, "flops": 6 * T * N * K}
