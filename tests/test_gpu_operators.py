"""GPU checks of the epilogue linears, the extended routing and the sampling against plain implementations in 64 bits, one
operator at a time and as the run of a decode step that they are used in."""
import math

import numpy as np
import pytest

from tests import gen

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}  # a rounding, relative


def _gu():
    from tests import gpu_util
    return gpu_util


def _ops():
    from inferd_amd import ops
    return ops


# ---- routing ---------------------------------------------------------------------------------------------------------
def plain_route(logits, E, k, score, bias, groups, topk_groups, group_top, norm, scale, gate):
    """ifd_moe_route_ex's rule, row by row in 64 bits."""
    idx, wt, sg = [], [], []
    for row in logits.double().cpu().numpy():
        l = np.where(np.isnan(row[:E]), -np.inf, row[:E])
        with np.errstate(all="ignore"):
            if score == "softmax":
                m = l.max()
                s = np.zeros(E) if m == -np.inf else np.where(l == m, 1.0, np.exp(l - m))
                s = s / s.sum() if s.sum() else s
            else:
                s = 0.5 * (1 + np.tanh(l / 2))
                s = np.where(l < -30, np.exp(l), s)
        if bias is None:
            c, v = l.copy(), s if group_top == 2 else l
        else:
            b = bias.double().cpu().numpy()
            c = v = s + np.where(np.isnan(b), -np.inf, b)
        if groups > 1:
            best = np.sort(v.reshape(groups, -1), 1)[:, ::-1][:, :group_top]
            value = np.where((best == -np.inf).any(1), -np.inf, best.sum(1))
            keep = np.argsort(-value, kind="stable")[:topk_groups]
            out = np.repeat(~np.isin(np.arange(groups), keep), E // groups)
        else:
            out = np.zeros(E, bool)
        order = np.lexsort((np.arange(E), -c, out))[:k]
        w = s[order]
        if norm:
            w = w / w.sum() if w.sum() else w
        idx.append(order)
        wt.append(w * np.float64(np.float32(scale)))
        sg.append(1 / (1 + np.exp(-row[E])) if gate else 1.0)
    return np.array(idx), np.array(wt), np.array(sg)


def check_route(logits, E, k, **kw):
    got = [t.cpu().numpy() for t in _ops().moe_route_ex(logits, E, k, **kw)]
    full = dict(score="softmax", bias=None, groups=1, topk_groups=1, group_top=1, norm=True, scale=1.0)
    full.update(kw)
    gate = full.pop("shared_gate", False)
    idx, wt, sg = plain_route(logits, E, k, gate=gate, **full)
    assert np.array_equal(got[0], idx)
    # 64-bit values, rounded once; the 64-bit steps themselves are off by a few 2^-53
    for g, w in ((got[1], wt), (got[2], sg)):
        assert np.all(np.abs(g - w) <= 2.0 ** -24 * (1 + 1e-6) * np.abs(w) + 1e-44)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("T,E,k,groups,keep,top,bias", [
    (1, 1, 1, 1, 1, 1, False), (5, 7, 7, 1, 1, 1, True), (3, 60, 4, 1, 1, 1, False), (65, 64, 6, 8, 3, 1, False),
    (33, 100, 8, 10, 4, 2, True), (70, 128, 16, 2, 1, 2, False), (130, 160, 6, 8, 3, 1, True), (64, 256, 8, 8, 4, 2, True),
    (1000, 256, 8, 8, 4, 2, True), (17, 96, 5, 3, 2, 2, True), (200, 512, 10, 1, 1, 1, False), (99, 512, 16, 64, 9, 2, True),
    (31, 512, 8, 16, 16, 1, True), (40, 510, 12, 5, 3, 2, False), (2, 384, 9, 4, 1, 2, True), (77, 320, 8, 16, 3, 2, True),
])
def test_route(score, bf16, T, E, k, groups, keep, top, bias):
    g = torch.Generator(device="cuda").manual_seed(T * E + k)
    l = 1.5 * torch.randn((T, E + 1), device="cuda", generator=g)
    b = 0.1 * torch.randn((E,), device="cuda", generator=g) if bias else None
    l = l.to(torch.bfloat16) if bf16 else l
    for norm, scale, gate in ((True, 1.0, False), (False, 2.5, True)):
        check_route(l, E, k, score=score, bias=b, groups=groups, topk_groups=keep, group_top=top, norm=norm, scale=scale,
                    shared_gate=gate)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("groups,keep,top", [(1, 1, 1), (8, 4, 1), (8, 4, 2), (5, 2, 2)])
def test_route_edges(score, bias, groups, keep, top):
    """Ties, masked experts, infinities and NaN, rows that a mask leaves empty, all in one batch."""
    E, k = 160, 8
    g = torch.Generator(device="cuda").manual_seed(7)
    l = torch.randn((14, E), device="cuda", generator=g)
    l[0] = 0.0
    l[1] = -math.inf
    l[2, 5:] = -math.inf
    l[3] = torch.finfo(torch.float32).min
    l[4, ::3] = torch.finfo(torch.float32).min
    l[5, 17] = math.inf
    l[6, 100:] = math.nan
    l[7] = math.nan
    l[8] = l[8].round()
    l[9] = torch.where(l[9] > 0, 0.0, -0.0)
    l[10] = 100 * l[10]
    l[11, 50] = l[11, 60] = math.inf
    l[12] = 30 + l[12] * 1e-6
    b = None
    if bias:
        b = (0.1 * torch.randn((E,), device="cuda", generator=g)).round(decimals=1)
        b[3] = -math.inf
        b[4] = math.nan
    check_route(l, E, k, score=score, bias=b, groups=groups, topk_groups=keep, group_top=top)


def test_route_near_ties_are_decided_in_64_bits():
    """Sigmoid scores and biases whose sums differ by less than a rounding of fp32."""
    T, E = 256, 128
    g = torch.Generator(device="cuda").manual_seed(3)
    l = torch.randn((T, E), device="cuda", generator=g)
    s = torch.sigmoid(l[0].double())
    l[:] = l[0] + torch.randint(-2, 3, (T, E), device="cuda", generator=g) * 2.0 ** -23
    check_route(l, E, 16, score="sigmoid", bias=(0.7 - s).float(), norm=True)


def test_route_agrees_with_the_plain_softmax_routing():
    ops = _ops()
    l = torch.randn((300, 513), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    a = ops.moe_route(l, 512, 10, norm=True, shared_gate=True)
    b = ops.moe_route_ex(l, 512, 10, shared_gate=True)
    assert torch.equal(a[0], b[0])
    # fp32 exponentials and sums of 512 terms against 64-bit ones
    assert torch.allclose(a[1], b[1], rtol=2e-6, atol=0) and torch.allclose(a[2], b[2], rtol=1e-6, atol=0)


def test_route_writes_only_its_rows():
    ops = _ops()
    big = torch.randn((9, 400), device="cuda")
    l = big[:, 37:37 + 65]  # a stride and an alignment of their own
    outs = [torch.full((12, 4), -7, dtype=torch.int32, device="cuda"), torch.full((12, 4), -7.0, device="cuda"),
            torch.full((12,), -7.0, device="cuda")]
    ops.moe_route_ex(l, 64, 4, score="sigmoid", shared_gate=True, outs=tuple(t[:9] for t in outs))
    assert all(bool((t[9:] == -7).all()) for t in outs)
    ref = plain_route(l, 64, 4, "sigmoid", None, 1, 1, 1, True, 1.0, True)
    assert np.array_equal(outs[0][:9].cpu().numpy(), ref[0])


# ---- sampling --------------------------------------------------------------------------------------------------------
def plain_sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    """ifd_sample's rule, row by row in 64 bits."""
    tokens, probs = [], []
    at = lambda t, r, off: off if t is None else float(t[r])  # noqa: E731
    u = u.cpu().numpy()
    temperature, top_k, top_p, min_p = (None if t is None else t.cpu().numpy() for t in (temperature, top_k, top_p, min_p))
    for r, l in enumerate(logits.double().cpu().numpy()):
        l = np.where(np.isnan(l), -np.inf, l)
        V, m = len(l), l.max()
        tau = at(temperature, r, 1.0)
        if m == -np.inf or not tau > 0:
            tokens.append(-1 if m == -np.inf else int(l.argmax()))
            probs.append(0.0 if m == -np.inf else 1.0)
            continue
        with np.errstate(all="ignore"):
            w = np.where(l == m, 1.0, np.exp((l - m) / tau))
        w[w <= 2.0 ** -45] = 0.0
        order = np.argsort(-l, kind="stable")
        k = int(at(top_k, r, 0))
        n = k if 0 < k < V else V
        p = at(top_p, r, 1.0)
        if not p >= 1:
            c = np.cumsum(w[order[:n]])
            n = min(n, 1 + int(np.searchsorted(c, (p if p > 0 else 0.0) * c[-1])))
        kept = order[:n]
        mp = at(min_p, r, 0.0)
        kept = np.sort(kept[w[kept] >= min(mp, 1.0)] if mp > 0 else kept)
        c = np.cumsum(w[kept])
        x = min(max(float(u[r]), 0.0) if u[r] == u[r] else 0.0, 1 - 2.0 ** -24)
        t = kept[np.searchsorted(c, x * c[-1], side="right")]
        tokens.append(int(t))
        probs.append(w[t] / c[-1])
    return np.array(tokens), np.array(probs)


def check_sample(logits, u, **kw):
    token, prob = (t.cpu().numpy() for t in _ops().sample(logits, u, **kw))
    want, p = plain_sample(logits, u, **kw)
    bad = np.flatnonzero(token != want)
    assert not len(bad), (bad[:8], token[bad[:8]], want[bad[:8]])
    # a rounding to fp32, and weights rounded to 2^-45 of the largest (their total is at least 1)
    V = logits.shape[1]
    assert np.all(np.abs(prob - p) <= 2.0 ** -24 * (1 + 1e-6) * p + 2.0 ** -44 * (1 + V * p))


def _lm_logits(T, V, seed, bf16=False, std=2.2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    l = std * torch.randn((T, V), device="cuda", generator=g)
    n = min(V, 30)
    l.scatter_(1, torch.randint(0, V, (T, n), device="cuda", generator=g),
               6 + 6 * torch.rand((T, n), device="cuda", generator=g))
    u = torch.rand((T,), device="cuda", generator=g)
    return (l.to(torch.bfloat16) if bf16 else l), u, g


def _col(T, values, dtype=torch.float32):
    return torch.tensor([values[i % len(values)] for i in range(T)], dtype=dtype, device="cuda")


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("T,V", [(1, 1), (3, 2), (4, 63), (5, 1000), (2, 4096), (1, 50021), (17, 50021), (3, 151936),
                                 (1, 248320), (40, 20000), (1, 1 << 19), (130, 3001)])
@pytest.mark.parametrize("kind", ["none", "k", "p", "kp", "min", "all"])
def test_sample(bf16, T, V, kind):
    l, u, _ = _lm_logits(T, V, T + V, bf16)
    kw = dict(temperature=_col(T, [1.0, 0.7, 0.1, 1.5, 0.0, 5.0]))
    if kind in ("k", "kp", "all"):
        kw["top_k"] = _col(T, [40, 1, 0, V, 1000, 5000, 7, -3], torch.int32)
    if kind in ("p", "kp", "all"):
        kw["top_p"] = _col(T, [0.9, 0.5, 1.0, 0.99, 1e-6, 0.999999, 0.0])
    if kind in ("min", "all"):
        kw["min_p"] = _col(T, [0.05, 0.0, 1e-4, 0.5, 1.0])
    for i in range(2):
        check_sample(l, u if i == 0 else 1 - u, **kw)


def test_sample_sizes_are_all_alike_on_ties():
    """Few distinct logits, so that every border falls among equal ones: the lower indices are kept."""
    for V, levels in ((1000, 1), (1000, 3), (30001, 2), (151936, 1), (151936, 17), (248320, 5)):
        T = 24
        g = torch.Generator(device="cuda").manual_seed(V + levels)
        l = torch.randint(0, levels, (T, V), device="cuda", generator=g).float() * 0.37 - 3
        u = torch.rand((T,), device="cuda", generator=g)
        for kw in (dict(top_p=_col(T, [0.5, 0.9, 0.123, 0.999])), dict(top_k=_col(T, [5, 100, 999, 4097], torch.int32)),
                   dict(top_k=_col(T, [900, 333, 50], torch.int32), top_p=_col(T, [0.5, 0.8])), dict()):
            check_sample(l, u, temperature=_col(T, [1.0, 0.3]), **kw)


def test_sample_edges():
    """Masks, infinities, NaN, empty rows, and random numbers at and past the ends."""
    V = 5000
    l, u, g = _lm_logits(24, V, 11)
    l[0] = -math.inf
    l[1] = math.nan
    l[2, 1:] = -math.inf
    l[3, :-1] = -math.inf
    l[4] = torch.finfo(torch.float32).min
    l[5, 10:] = torch.finfo(torch.float32).min
    l[6, 77] = math.inf
    l[7, 77] = l[7, 99] = math.inf
    l[8, ::2] = math.nan
    l[9, 4000:] = -math.inf
    l[10] = 0.0
    l[11] = torch.where(l[11] > 0, 0.0, -0.0)
    l[12] = 1e30 * l[12]
    l[13] = 1e-30 * l[13]
    u[14:20] = torch.tensor([0.0, 1.0, 1 - 2.0 ** -24, 2.0, -1.0, math.nan], device="cuda")
    T = len(l)
    for kw in (dict(), dict(top_k=_col(T, [3], torch.int32)), dict(top_p=_col(T, [0.9])), dict(min_p=_col(T, [0.1])),
               dict(top_k=_col(T, [100], torch.int32), top_p=_col(T, [0.7]), min_p=_col(T, [0.01])),
               dict(top_p=_col(T, [math.nan, -1.0, 2.0])), dict(min_p=_col(T, [math.nan, -1.0, 2.0]))):
        for tau in (None, [1.0], [0.0, -1.0, math.nan], [1e-3], [1e3], [1e-30]):
            check_sample(l, u, temperature=None if tau is None else _col(T, tau), **kw)


def test_sample_frequencies_follow_the_weights():
    """Many random numbers on one row: each token's share is its weight (chi-square, fixed seed)."""
    n, V = 20000, 50
    g = torch.Generator(device="cuda").manual_seed(5)
    l = torch.randn((1, V), device="cuda", generator=g)
    token, prob = _ops().sample(l.expand(n, V).contiguous(), torch.rand((n,), device="cuda", generator=g))
    p = torch.softmax(l[0].double(), 0).cpu().numpy()
    seen = np.bincount(token.cpu().numpy(), minlength=V)
    chi = float(((seen - n * p) ** 2 / (n * p)).sum())
    assert chi < 49 + 6 * math.sqrt(2 * 49)  # six standard deviations of a chi-square with 49 degrees of freedom
    assert np.allclose(prob.cpu().numpy(), p[token.cpu().numpy()], rtol=1e-6)


def test_sample_strides_and_untouched_rows():
    big = torch.randn((6, 3001), device="cuda").to(torch.bfloat16)
    l = big[:, 3:3 + 2500]
    u = torch.rand((6,), device="cuda")
    token, prob = torch.full((9,), -7, dtype=torch.int32, device="cuda"), torch.full((9,), -7.0, device="cuda")
    _ops().sample(l, u, top_p=_col(6, [0.8]), outs=(token[:6], prob[:6]))
    assert bool((token[6:] == -7).all()) and bool((prob[6:] == -7).all())
    assert np.array_equal(token[:6].cpu().numpy(), plain_sample(l, u, top_p=_col(6, [0.8]))[0])


# ---- linears with an epilogue ------------------------------------------------------------------------------------------
def _act64(y, act):
    if act == "relu":
        return torch.where(y < 0, torch.zeros_like(y), y)
    if act == "silu":
        return y / (1 + torch.exp(-y))
    if act == "gelu":
        return y * 0.5 * torch.special.erfc(-y / math.sqrt(2))
    if act == "gelu_tanh":
        return y / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    return y


def _layer(N, K, bits, seed):
    g, ops = _gu(), _ops()
    codes, wq, s, b = gen.qlinear(N, K, seed=seed, bias="free") if bits == 4 else gen.qlinear8(N, K, seed=seed, bias="free")
    W = (ops.pack_t64 if bits == 4 else ops.pack_t64x8)(g.qlinear(wq, s, b, bits=bits))
    return W, torch.from_numpy(gen.dequant_f64(codes, s, b)).cuda()


def _weights_as_used(w, M, N, K, bits):
    """The weights in the arithmetic that the product runs at these sizes."""
    from oracle import oracle as orc
    from tests.test_gpu_t64 import _t64_arith
    exact = M <= 16 and K % 128 == 0 if bits == 8 else _t64_arith(M, N, K) is orc.qmv
    return w if exact else w.to(torch.bfloat16).double()


def check_epi(M, N, K, bits, act, bias, res, fp32=False, inplace=False, seed=0, A=None, W=None):
    ops = _ops()
    g = torch.Generator(device="cuda").manual_seed(seed + M + N)
    layer, w = W or _layer(N, K, bits, seed + 1)
    A = torch.randn((M, K), device="cuda", generator=g).to(torch.bfloat16) if A is None else A
    b = torch.randn((N,), device="cuda", generator=g).to(torch.bfloat16) if bias else None
    r = (2 * torch.randn((M, N), device="cuda", generator=g)).to(torch.bfloat16) if res else None
    w = _weights_as_used(w, M, N, K, bits)
    y = A.double() @ w.T.contiguous()
    # the fp32 sum of K products (and the groups' own steps), through an activation of slope at most 1.13
    tol = 1.13 * (K + 16) * 2.0 ** -24 * (A.double().abs() @ w.abs().T.contiguous())
    y = y if b is None else y + b.double()
    a = _act64(y, act)
    # the activation in fp32: a few roundings of its value, and those of the exponent's argument
    tol = tol + 2.0 ** -20 * (a.abs() + y.abs().clamp(max=8) * 2.0 ** -4 + 2.0 ** -20)
    a = a if r is None else a + r.double()
    C = r if inplace else None
    out = (ops.gemm_t64_epi if bits == 4 else ops.gemm_t64x8_epi)(A, layer, bias=b, act=act, residual=r, C=C, fp32=fp32)
    assert out.dtype == (torch.float32 if fp32 else torch.bfloat16)
    assert not inplace or out.data_ptr() == r.data_ptr()
    err = (out.double() - a).abs() - HALF[out.dtype] * (a.abs() + tol) - tol
    worst = int(err.argmax())
    assert float(err.max()) <= 0, (worst // N, worst % N, float(out.flatten()[worst]), float(a.flatten()[worst]))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("M,N,K", [(1, 256, 512), (16, 1000, 1024), (17, 129, 256), (64, 512, 512), (100, 1024, 512),
                                   (300, 768, 512)])
def test_epilogue_activations(bits, act, M, N, K):
    W = _layer(N, K, bits, 3)
    for bias, res, fp32 in ((True, True, False), (False, False, True), (True, False, True), (False, True, False)):
        check_epi(M, N, K, bits, act, bias, res, fp32=fp32, W=W)


@pytest.mark.parametrize("M", [1, 2, 8, 9, 16, 17, 32, 33, 64, 65, 96, 97, 128, 129, 161, 256, 333, 1000])
@pytest.mark.parametrize("N,K", [(32, 256), (100, 256), (129, 512), (1, 256), (256, 1024), (1000, 768), (5120, 1024)])
def test_epilogue_shapes(M, N, K):
    check_epi(M, N, K, 4, "silu", True, True)


@pytest.mark.parametrize("M", [1, 9, 16, 17, 33, 65, 129, 300])
@pytest.mark.parametrize("N,K", [(32, 64), (100, 128), (129, 320), (1, 256), (1000, 768), (5120, 1024)])
def test_epilogue_shapes_8bit(M, N, K):
    check_epi(M, N, K, 8, "gelu", True, True)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("M,N,K", [(1, 5120, 5120), (8, 5120, 17408), (16, 34816, 5120), (32, 34816, 5120), (128, 5120, 17408),
                                   (777, 5120, 5120), (1300, 5120, 2048)])
def test_epilogue_split_products(M, N, K, bits):
    """Sizes at which K is split among blocks, so that the epilogue runs where the pieces are joined."""
    W = _layer(N, K, bits, 9)
    check_epi(M, N, K, bits, "none", True, True, inplace=True, W=W)
    check_epi(M, N, K, bits, "gelu_tanh", True, False, W=W)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("M", [5, 40, 100, 150, 700])
def test_epilogue_without_any_step_is_the_plain_product(bits, M):
    ops = _ops()
    N, K = 640, 1024
    layer, _ = _layer(N, K, bits, 4)
    A = torch.randn((M, K), device="cuda").to(torch.bfloat16)
    for mode in (0, 1, 2):
        C = torch.randn((M, N), device="cuda").to(torch.bfloat16) if mode == 1 else None
        D = C.clone() if mode == 1 else None
        a = (ops.gemm_t64 if bits == 4 else ops.gemm_t64x8)(A, layer, C, mode=mode)
        b = (ops.gemm_t64_epi if bits == 4 else ops.gemm_t64x8_epi)(A, layer, residual=D, C=D, fp32=mode == 2)
        assert torch.equal(a, b)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("M,N", [(3, 100), (20, 100), (100, 260), (140, 256), (200, 333)])
def test_epilogue_strides(M, N, bits):
    """Rows apart and off alignment in A, C and the residual; what lies between and behind the rows stays."""
    ops = _ops()
    K = 512
    layer, w = _layer(N, K, bits, 5)
    A = torch.randn((M, K + 24), device="cuda").to(torch.bfloat16)[:, 8:8 + K]
    bias = torch.randn((N,), device="cuda").to(torch.bfloat16)
    R = torch.randn((M, N + 13), device="cuda").to(torch.bfloat16)[:, 5:5 + N]
    for dtype in (torch.bfloat16, torch.float32):
        big = torch.full((M + 2, N + 7), 7.0, device="cuda", dtype=dtype)
        out = big[1:M + 1, 3:3 + N]
        (ops.gemm_t64_epi if bits == 4 else ops.gemm_t64x8_epi)(A, layer, bias=bias, act="relu", residual=R, C=out)
        ww = _weights_as_used(w, M, N, K, bits)
        y = A.double() @ ww.T.contiguous()
        ref = torch.relu(y + bias.double()) + R.double()
        tol = (K + 16) * 2.0 ** -24 * (A.double().abs() @ ww.abs().T.contiguous()) + 2.0 ** -20
        assert bool(((out.double() - ref).abs() <= HALF[dtype] * (ref.abs() + tol) + tol).all())
        rest = big.clone()
        rest[1:M + 1, 3:3 + N] = 7.0
        assert bool((rest == 7.0).all())


@pytest.mark.parametrize("M", [2, 24, 100, 140])
def test_epilogue_infinities_and_nan(M):
    """Infinities and NaN in the bias and the residual come out as the formula has them, and nowhere else."""
    ops = _ops()
    N, K = 256, 256
    layer, w = _layer(N, K, 4, 6)
    A = torch.randn((M, K), device="cuda").to(torch.bfloat16)
    bias = torch.zeros((N,), device="cuda", dtype=torch.bfloat16)
    bias[3], bias[5], bias[7] = math.inf, -math.inf, math.nan
    R = torch.zeros((M, N), device="cuda", dtype=torch.bfloat16)
    R[1, 10], R[1, 11], R[0, 12] = math.nan, math.inf, -math.inf
    for act in ("none", "relu", "silu", "gelu", "gelu_tanh"):
        out = ops.gemm_t64_epi(A, layer, bias=bias, act=act, residual=R).double()
        ref = _act64(A.double() @ _weights_as_used(w, M, N, K, 4).T.contiguous() + bias.double(), act) + R.double()
        assert torch.equal(out.isnan(), ref.isnan()), act
        assert torch.equal(out == math.inf, ref == math.inf) and torch.equal(out == -math.inf, ref == -math.inf), act


# ---- empty calls, streams, graphs, and the run of a decode step --------------------------------------------------------
def test_calls_without_rows():
    ops = _ops()
    W, _ = _layer(64, 256, 4, 1)
    z = lambda *s, **k: torch.zeros(s, device="cuda", **k)  # noqa: E731
    assert ops.gemm_t64_epi(z(0, 256, dtype=torch.bfloat16), W, act="relu").shape == (0, 64)
    token, prob = ops.sample(z(0, 1000), z(0))
    assert token.shape == prob.shape == (0,)
    idx, wt, sg = ops.moe_route_ex(z(0, 64), 64, 4)
    assert idx.shape == wt.shape == (0, 4) and sg.shape == (0,)


def _step(T=6, seed=0):
    """The layers and buffers of a small decode step: a projection with bias into the residual stream, experts routed by
    sigmoid scores in groups, a head and its sampling."""
    g, ops = _gu(), _ops()
    H, I, E, k, V = 512, 64, 32, 4, 2000
    gt = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(s, device="cuda", generator=gt)  # noqa: E731

    def scaled(N, K, s):  # products of about the inputs' size
        codes, wq, sc, b = gen.qlinear(N, K, seed=s)
        f = np.float32(1 / (0.0125 * 4.6 * math.sqrt(K)))
        sc = gen.f32_to_bf16(gen.bf16_to_f32(sc) * f)
        b = gen.f32_to_bf16(-7.5 * gen.bf16_to_f32(sc))
        return codes, wq, sc, b

    def stack(N, K, s):
        parts = [scaled(N, K, s + e) for e in range(E)]
        wq, sc, b = (np.stack([q[i] for q in parts]) for i in (1, 2, 3))
        dense = torch.from_numpy(np.stack([gen.dequant_f64(q[0], q[2], q[3]) for q in parts])).cuda()
        return ops.pack_t64_stack(g.moew(wq, sc, b)), dense

    def linear(N, K, s):
        codes, wq, sc, b = scaled(N, K, s)
        return ops.pack_t64(g.qlinear(wq, sc, b)), torch.from_numpy(gen.dequant_f64(codes, sc, b)).cuda()

    d = dict(H=H, I=I, E=E, k=k, V=V, T=T, proj=linear(H, H, 1), egu=stack(2 * I, H, 100), edn=stack(H, I, 200),
             head=linear(V, H, 2), bias=rnd(H).to(torch.bfloat16), nw=(1 + 0.1 * rnd(H)).to(torch.bfloat16),
             router=(rnd(E, H) * H ** -0.5).to(torch.bfloat16), balance=0.1 * rnd(E),
             temperature=_col(T, [0.8, 0.0, 1.2]), top_k=_col(T, [50, 0, 5], torch.int32), top_p=_col(T, [0.9, 1.0]),
             min_p=_col(T, [0.0, 0.02]))
    return d


def _run_step(d, a, x, u):
    """The calls of the step: attention output a and residual stream x bf16 [T, H]; returns what each leaves."""
    ops = _ops()
    x1 = ops.gemm_t64_epi(a, d["proj"][0], bias=d["bias"], residual=x)
    xn = ops.rmsnorm(x1, d["nw"], 1e-6)
    logits = ops.moe_router_logits(xn, d["router"], out_bf16=False)
    idx, wt, sg = ops.moe_route_ex(logits, d["E"], d["k"], score="sigmoid", bias=d["balance"], groups=4, topk_groups=2,
                                   group_top=2, scale=2.5)
    x2 = ops.moe_rows_t64(xn, idx, wt, None, d["egu"][0], d["edn"][0], out=x1.clone(), assign=False)
    hn = ops.rmsnorm(x2, d["nw"], 1e-6)
    head = ops.gemm_t64(hn, d["head"][0], mode=2)
    token, prob = ops.sample(head, u, temperature=d["temperature"], top_k=d["top_k"], top_p=d["top_p"], min_p=d["min_p"])
    return dict(x1=x1, xn=xn, logits=logits, idx=idx, wt=wt, sg=sg, x2=x2, hn=hn, head=head, token=token, prob=prob)


def _step_inputs(d, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(s, device="cuda", generator=g).to(torch.bfloat16)  # noqa: E731
    return rnd(d["T"], d["H"]), rnd(d["T"], d["H"]), torch.rand((d["T"],), device="cuda", generator=g)


def test_decode_step():
    """The operators in a run, each against its 64-bit plain form on what the one before it left."""
    d = _step()
    a, x, u = _step_inputs(d, 1)
    r = _run_step(d, a, x, u)
    K, h = d["H"], 2.0 ** -8
    y = a.double() @ d["proj"][1].T.contiguous() + d["bias"].double() + x.double()
    tol = (K + 16) * 2.0 ** -24 * (a.double().abs() @ d["proj"][1].abs().T.contiguous())
    assert bool(((r["x1"].double() - y).abs() <= h * (y.abs() + tol) + tol).all())
    idx, wt, _ = plain_route(r["logits"], d["E"], d["k"], "sigmoid", d["balance"], 4, 2, 2, True, 2.5, False)
    assert np.array_equal(r["idx"].cpu().numpy(), idx)
    assert np.all(np.abs(r["wt"].cpu().numpy() - wt) <= 2.0 ** -24 * (1 + 1e-6) * wt)
    # the experts' products on that routing: gate and up, their SwiGLU (three roundings to bf16), down, the weighted sum
    xn, gu, dn = r["xn"].double(), d["egu"][1], d["edn"][1]
    out, slack = torch.zeros_like(xn), torch.zeros_like(xn)
    for t in range(d["T"]):
        for j in range(d["k"]):
            e, w = int(r["idx"][t, j]), float(r["wt"][t, j])
            v = gu[e] @ xn[t]
            gate, up = v[:d["I"]], v[d["I"]:]
            hid = gate * torch.sigmoid(gate) * up
            # d(hid): gate and up off by a rounding each (slope of x sigmoid(x) at most 1.1), then two more roundings
            off = h * (1.1 * gate.abs() * up.abs() + 3 * hid.abs()) * 1.1
            out[t] += w * (dn[e] @ hid)
            slack[t] += w * (dn[e].abs() @ off)
    ref = r["x1"].double() + out
    # the sum is rounded before it is added, and the result is
    assert bool(((r["x2"].double() - ref).abs() <= 1.01 * slack + 1.01 * h * (out.abs() + ref.abs()) + 1e-3 * slack).all())
    token, prob = plain_sample(r["head"], u, d["temperature"], d["top_k"], d["top_p"], d["min_p"])
    assert np.array_equal(r["token"].cpu().numpy(), token)
    assert np.allclose(r["prob"].cpu().numpy(), prob, rtol=2.0 ** -23, atol=0)


def test_routing_feeds_the_sorted_experts():
    """moe_route_ex -> moe_dispatch: the expert-sorted rows, and the experts' products over them."""
    ops = _ops()
    d = _step(T=40, seed=3)
    _, x, _ = _step_inputs(d, 4)
    logits = ops.moe_router_logits(x, d["router"], out_bf16=False)
    idx, wt, sg = ops.moe_route_ex(logits, d["E"], d["k"], score="sigmoid", bias=d["balance"], groups=8, topk_groups=3)
    rows = ops.moe_rows_t64(x, idx, wt, None, d["egu"][0], d["edn"][0])
    offsets, perm, inv, *_ = ops.moe_dispatch(idx, d["E"])
    e = idx.flatten()[perm.long()]
    assert bool((e[1:] >= e[:-1]).all()) and int(offsets[-1]) == idx.numel()
    out = torch.zeros_like(rows, dtype=torch.float64)
    for q in range(perm.numel()):
        t, j = divmod(int(perm[q]), d["k"])
        v = d["egu"][1][int(idx[t, j])] @ x[t].double()
        hid = v[:d["I"]] * torch.sigmoid(v[:d["I"]]) * v[d["I"]:]
        out[t] += float(wt[t, j]) * (d["edn"][1][int(idx[t, j])] @ hid)
    assert float((rows.double() - out).norm() / out.norm()) < 2.0 ** -7  # a few roundings to bf16 of half a step each


def test_streams_have_their_own_workspaces():
    """The same calls on two streams at once, over and over: each gets the results it gets alone."""
    d = _step(T=9)
    ins = [_step_inputs(d, s) for s in (5, 6)]
    alone = [_run_step(d, *i) for i in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ins]
    for _ in range(5):
        got = []
        for s, i in zip(streams, ins):
            with torch.cuda.stream(s):
                got.append(_run_step(d, *i))
        torch.cuda.synchronize()
        for a, b in zip(alone, got):
            for name in a:
                assert torch.equal(a[name], b[name]), name


def test_two_captured_graphs():
    """Two graphs of the step, replayed with new inputs, eager calls and synchronizations between; every replay gives the
    eager result."""
    d = _step(T=5)
    eager = {s: _run_step(d, *_step_inputs(d, s)) for s in (7, 8, 9)}
    graphs = []
    for _ in range(2):
        ins = _step_inputs(d, 7)
        _run_step(d, *ins)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = _run_step(d, *ins)
        graphs.append((graph, ins, outs))
    for round_, s in enumerate((8, 9, 7, 8, 8, 9)):
        for k, (graph, ins, outs) in enumerate(graphs):
            for buf, new in zip(ins, _step_inputs(d, s)):
                buf.copy_(new)
            graph.replay()
            if round_ % 2:
                _run_step(d, *_step_inputs(d, 7))
            if round_ % 3 == 0:
                torch.cuda.synchronize()
            for name in outs:
                assert torch.equal(outs[name], eager[s][name]), (round_, k, name)


def test_results_do_not_depend_on_the_batch_or_the_call():
    """A row alone, in a batch, and again: the same token and routing (sums that atomics order would show here)."""
    ops = _ops()
    l, u, _ = _lm_logits(33, 30000, 21)
    kw = dict(temperature=_col(33, [1.1]), top_p=_col(33, [0.93]), min_p=_col(33, [0.001]))
    first = ops.sample(l, u, **kw)
    for _ in range(5):
        again = ops.sample(l, u, **kw)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    for r in (0, 7, 32):
        one = ops.sample(l[r:r + 1], u[r:r + 1], **{n: t[r:r + 1] for n, t in kw.items()})
        assert torch.equal(one[0][0], first[0][r]) and torch.equal(one[1][0], first[1][r])
    q = torch.randn((65, 256), device="cuda")
    whole = ops.moe_route_ex(q, 256, 8, score="sigmoid", groups=8, topk_groups=4, group_top=2)
    for r in (0, 13, 64):
        one = ops.moe_route_ex(q[r:r + 1], 256, 8, score="sigmoid", groups=8, topk_groups=4, group_top=2)
        assert all(torch.equal(a[0], b[r]) for a, b in zip(one, whole))


def test_sample_past_one_launch_of_rows():
    """More rows than one set of launches takes."""
    l, u, _ = _lm_logits(1100, 700, 31, bf16=True)
    check_sample(l, u, top_k=_col(1100, [0, 20], torch.int32), top_p=_col(1100, [0.9, 1.0, 0.5]))


def test_threads_on_one_stream():
    """Two threads that call on the same stream, so that their launches alternate: each gets the results it gets alone."""
    import threading
    d = _step(T=7)
    ins = [_step_inputs(d, s) for s in (11, 12)]
    alone = [_run_step(d, *i) for i in ins]
    torch.cuda.synchronize()
    wrong = []

    def work(k):
        for _ in range(30):
            got = _run_step(d, *ins[k])
            torch.cuda.synchronize()
            wrong.extend(n for n in alone[k] if not torch.equal(got[n], alone[k][n]))

    ts = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not wrong


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("M,N", [(3, 256), (40, 256), (200, 256), (300, 1001)])
@pytest.mark.parametrize("act", ["gelu", "none"])
def test_epilogue_bias_off_alignment(bits, M, N, act):
    """A bias that begins at an odd place of a larger tensor."""
    ops = _ops()
    K = 512
    layer, w = _layer(N, K, bits, 8)
    A = torch.randn((M, K), device="cuda").to(torch.bfloat16)
    bias = torch.randn((N + 3,), device="cuda").to(torch.bfloat16)[1:N + 1]
    call = ops.gemm_t64_epi if bits == 4 else ops.gemm_t64x8_epi
    assert torch.equal(call(A, layer, bias=bias, act=act), call(A, layer, bias=bias.clone(), act=act))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("M,swap", [(1, False), (3, False), (3, True), (40, False), (150, True)])
def test_epilogue_residual_in_other_columns_of_the_same_rows(bits, M, swap):
    ops = _ops()
    layer, _ = _layer(256, 512, bits, 3)
    g = torch.Generator(device="cuda").manual_seed(M)
    A = torch.randn((M, 512), device="cuda", generator=g).to(torch.bfloat16)
    buf = torch.randn((M, 512 + 8), device="cuda", generator=g).to(torch.bfloat16)
    c, r = (264, 0) if swap else (0, 264)
    call = ops.gemm_t64_epi if bits == 4 else ops.gemm_t64x8_epi
    want = call(A, layer, act="silu", residual=buf[:, r:r + 256].clone())
    res = buf[:, r:r + 256].clone()
    call(A, layer, act="silu", residual=buf[:, r:r + 256], C=buf[:, c:c + 256])
    assert torch.equal(buf[:, c:c + 256], want) and torch.equal(buf[:, r:r + 256], res)
    if M > 1:
        with pytest.raises(RuntimeError, match="overlaps"):
            call(A, layer, act="silu", residual=buf[:, 8:264], C=buf[:, :256])


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,k,groups,keep,top", [(256, 8, 8, 4, 2), (96, 16, 1, 1, 1), (512, 10, 4, 3, 1)])
@pytest.mark.parametrize("spread", [1e-2, 1e-4, 1e-6])
def test_route_of_choices_close_together(norm, score, E, k, groups, keep, top, spread):
    """Scores and biases apart by less than fp32 tells, up to all of a token's."""
    g = torch.Generator(device="cuda").manual_seed(E + k)
    l = 0.5 + spread * torch.randn((40, E), device="cuda", generator=g)
    bias = 0.1 * spread * torch.randn((E,), device="cuda", generator=g)
    check_route(l, E, k, score=score, bias=bias, groups=groups, topk_groups=keep, group_top=top, norm=norm)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("M,N,K", [(16, 131201, 1536), (3, 7409, 1536), (12, 1050, 2304), (9, 131071, 1536), (1, 5, 5120)])
def test_epilogue_of_split_rows_of_any_length(bits, M, N, K):
    """Partial sums joined in the GEMV and, past its counters' columns, by a launch: the plain product's fp32 sums bit for bit,
    and what the epilogue makes of them."""
    ops = _ops()
    g = torch.Generator(device="cuda").manual_seed(N)
    wq = torch.randint(-2 ** 31, 2 ** 31 - 1, (N, K * bits // 32), device="cuda", dtype=torch.int32, generator=g)
    s = (0.01 * torch.randn((N, K // 64), device="cuda", generator=g)).to(torch.bfloat16)
    b = (0.01 * torch.randn((N, K // 64), device="cuda", generator=g)).to(torch.bfloat16)
    layer = (ops.pack_t64 if bits == 4 else ops.pack_t64x8)(ops.QLinear(wq, s, b, N, K, False, bits))
    A = torch.randn((M, K), device="cuda", generator=g).to(torch.bfloat16)
    y = (ops.gemm_t64 if bits == 4 else ops.gemm_t64x8)(A, layer, mode=2)
    call = ops.gemm_t64_epi if bits == 4 else ops.gemm_t64x8_epi
    assert torch.equal(call(A, layer, fp32=True), y)
    big = torch.full((M, N + 3), 7.0, device="cuda")  # rows further apart, not 16-byte aligned
    bias = torch.randn((N,), device="cuda", generator=g).to(torch.bfloat16)
    res = torch.randn((M, N), device="cuda", generator=g).to(torch.bfloat16)
    call(A, layer, bias=bias, act="relu", residual=res, C=big[:, :N])
    assert torch.equal(big[:, :N], torch.relu(y + bias.float()) + res.float())
    assert bool((big[:, N:] == 7).all())


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("V", [64, 65, 512, 513, 2047, 4095, 4096, 4097, 6007, 8192, 8193])
def test_sample_of_short_rows(V, bf16):
    """Around the lengths at which a row is its own list: every filter, rows of a few and of all weights."""
    T = 40
    l, u, _ = _lm_logits(T, V, V, bf16)
    l[3:6] *= 1e-3  # flat
    l[6:9] *= 40  # a few tokens have weights
    l[9, V // 3:] = -math.inf
    l[10, 1:] = math.nan
    l[11] = torch.finfo(l.dtype).min
    l[12, 5] = math.inf
    l[13] = -math.inf
    for kw in (dict(), dict(top_k=_col(T, [1, 17, V - 1, V, 2000, 0], torch.int32)), dict(top_p=_col(T, [0.9, 0.1, 0.0, 1.0, 0.9999])),
               dict(min_p=_col(T, [0.1, 1e-9])),
               dict(top_k=_col(T, [60, V // 2, 3], torch.int32), top_p=_col(T, [0.8, 0.95]), min_p=_col(T, [0.0, 0.01]))):
        check_sample(l, u, temperature=_col(T, [1.0, 0.3, 0.0, 2.0]), **kw)
