"""The operators that read what a product leaves, and their speed: a linear with bias, activation and residual in its
epilogue, the routing of tokens to experts, and the sampling of the next token from a head's logits.

Where `own` is false `run` computes them from elementary torch operations (a linear in 32 bits; routing and sampling, whose
choices hang on values next to a border, in 64). Where it is true `run` makes the framework's calls.

The kinds, and what in real use each stands for:

- linear: a quantized linear of a layer on its T64 (4-bit) or T64x8 (8-bit) copy, with what its model puts behind the
  product: a bias, an activation, the residual stream. One row is one agent's decode step, thousands are a prompt.
- route:  the routing of a layer with experts, from the router's logits (fp32 for decode batches, bf16 for prompts, as the
  expert layer here computes them): softmax or sigmoid scores, a balance bias that counts for the choice only, experts in
  groups of which only the best are used, weights renormalised over the picks and scaled.
- sample: the next token of every agent of a decode batch from the head's logits, each with its own temperature, top-k,
  top-p and min-p and a uniform random number. Some rows are greedy, and some are constrained: a grammar has masked most
  of the vocabulary with minus infinity.

The dense sizes are those of a 5120-wide layer with a 17408-wide MLP, the expert counts and the vocabularies (151936 and
248320) those of this repository's bench and tests.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False
DEV = "cuda"


# ---- the cases -----------------------------------------------------------------------------------------------------
def listed():
    return [
        # one agent's output projection, with its bias, added into the residual stream: latency against 15 MB of weights
        dict(name="linear_m1", kind="linear", M=1, N=5120, K=5120, bits=4, act="none", bias=True, res=True, out="bf16"),
        # an 8-bit layer with an activation behind it, a decode batch of a dozen
        dict(name="linear8_m12", kind="linear", M=12, N=17408, K=5120, bits=8, act="silu", bias=True, res=False, out="bf16"),
        # the first linear of an MLP without gate, a decode batch
        dict(name="linear_m32", kind="linear", M=32, N=17408, K=5120, bits=4, act="gelu_tanh", bias=True, res=False, out="bf16"),
        # its second linear for a ragged prompt chunk, added into the residual stream
        dict(name="linear_m777", kind="linear", M=777, N=5120, K=17408, bits=4, act="none", bias=True, res=True, out="bf16"),
        # the first one for a long prompt: the largest call
        dict(name="linear_m4096", kind="linear", M=4096, N=17408, K=5120, bits=4, act="gelu", bias=True, res=False, out="bf16"),
        # routing of one token, and of a decode batch with groups: the smallest calls, latency
        dict(name="route_t1", kind="route", T=1, E=512, k=10, score="softmax", bias=False, groups=1, topk_groups=1,
             group_top=1, norm=True, scale=1.0, gate=True, bf16=False),
        dict(name="route_t16", kind="route", T=16, E=256, k=8, score="sigmoid", bias=True, groups=8, topk_groups=4,
             group_top=2, norm=True, scale=2.5, gate=False, bf16=False),
        # a batch of long prompts
        dict(name="route_t16384", kind="route", T=16384, E=256, k=8, score="sigmoid", bias=True, groups=8, topk_groups=4,
             group_top=2, norm=True, scale=2.5, gate=False, bf16=True),
        # one agent, the usual chat settings
        dict(name="sample_t1", kind="sample", T=1, V=248320, filters="topk_topp", bf16=False),
        # a small batch on a ragged vocabulary in bf16, minimum probability only
        dict(name="sample_t7", kind="sample", T=7, V=50021, filters="minp", bf16=True),
        # a decode batch in which every agent has its own settings
        dict(name="sample_t32", kind="sample", T=32, V=151936, filters="mixed", bf16=False),
        # the largest decode batch, top-p over the whole vocabulary
        dict(name="sample_t128", kind="sample", T=128, V=248320, filters="topp", bf16=False),
    ]


def _log_int(rng, lo, hi, step=1):
    """A multiple of step in [lo, hi], spread over the logarithm."""
    v = lo * (hi / lo) ** rng.random()
    return min(hi, max(lo, int(round(v / step)) * step))


ACTS = ["none", "relu", "silu", "gelu", "gelu_tanh"]


def draw(rng):
    kind = rng.choice(["linear", "linear", "route", "sample"])
    if kind == "linear":
        bits = rng.choice([4, 4, 8])
        M = _log_int(rng, 1, 4096 if bits == 4 else 512)
        # fp32 outputs are those of decode rows, whose weights are not rounded
        return dict(kind=kind, M=M, N=_log_int(rng, 1000, 17408, rng.choice([1, 4, 8, 32, 256])),
                    K=_log_int(rng, 1024, 5120, 256), bits=bits, act=rng.choice(ACTS), bias=rng.random() < 0.8,
                    res=rng.random() < 0.4, out="fp32" if M <= 16 and rng.random() < 0.3 else "bf16")
    if kind == "route":
        groups = rng.choice([1, 1, 2, 4, 8, 16])
        size = _log_int(rng, max(16, 64 // groups), 512 // groups)
        keep = rng.randint((groups + 1) // 2, groups)
        bf16 = rng.random() < 0.4
        return dict(kind=kind, T=_log_int(rng, 1, 16384), E=groups * size, k=rng.randint(1, 16), groups=groups,
                    topk_groups=keep, group_top=rng.choice([1, 2]), score=rng.choice(["softmax", "sigmoid"]),
                    bias=rng.random() < 0.6, norm=rng.random() < 0.8, scale=rng.choice([1.0, 1.0, 2.5]),
                    gate=rng.random() < 0.4, bf16=bf16)
    return dict(kind=kind, T=_log_int(rng, 1, 128), V=_log_int(rng, 1000, 248320), bf16=rng.random() < 0.4,
                filters=rng.choice(["mixed", "mixed", "topk_topp", "topp", "minp", "none"]))


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _codes(wq, bits):
    shift = torch.arange(32 // bits, device=wq.device, dtype=torch.int32) * bits
    return ((wq.unsqueeze(-1) >> shift) & ((1 << bits) - 1)).flatten(-2)


def _packed(wq, s, b, bits):
    """The layer's T64 or T64x8 copy, which the loader makes once: 32-row bands of 64-groups, group-major, codes in the
    order of the matrix instruction's operand, then the rows' (s, b) pairs."""
    N, G = s.shape
    nb = (N + 31) // 32
    q = torch.zeros((nb * 32, 64 * G), dtype=torch.int32, device=DEV) if bits == 4 else torch.full(
        (nb * 32, 64 * G), 128, dtype=torch.int32, device=DEV)
    q[:N] = _codes(wq, bits)
    if bits == 4:
        nibble = torch.tensor([0, 4, 1, 5, 2, 6, 3, 7], device=DEV, dtype=torch.int32) * 4
        words = (q.view(nb, 32, G, 2, 4, 8) << nibble).sum(-1).to(torch.int32)
        tiles = words.permute(2, 0, 3, 1, 4).contiguous().view(torch.uint8).view(G, nb, 1024)
    else:
        tiles = (q ^ 128).to(torch.uint8).view(nb, 32, G, 2, 2, 16).permute(2, 0, 4, 3, 1, 5).reshape(G, nb, 2048)
    sb = torch.zeros((nb * 32, G, 2), dtype=torch.bfloat16, device=DEV)
    sb[:N, :, 0], sb[:N, :, 1] = s, b
    rows = sb.view(nb, 32, G, 2).permute(2, 0, 1, 3).contiguous().view(torch.uint8).view(G, nb, 128)
    return torch.cat([tiles, rows], -1).flatten()


def _linear_inputs(case, seed):
    g = _generator(seed)
    M, N, K, bits = case["M"], case["N"], case["K"], case["bits"]
    levels = 1 << bits
    wq = torch.randint(-2 ** 31, 2 ** 31, (N, K * bits // 32), dtype=torch.int32, device=DEV, generator=g)
    std = levels / 12 ** 0.5 * K ** 0.5  # of a row's product with unit activations
    s = ((0.6 + 0.8 * torch.rand((N, K // 64), device=DEV, generator=g)) / std).to(torch.bfloat16)
    mid = (levels - 1) / 2 * (1 + 0.1 * (torch.rand((N, K // 64), device=DEV, generator=g) - 0.5))
    b = (-mid * s.float()).to(torch.bfloat16)
    x = torch.randn((M, K), device=DEV, generator=g) * (0.5 + 1.5 * torch.rand((M, 1), device=DEV, generator=g))
    bias = (0.5 * torch.randn((N,), device=DEV, generator=g)).to(torch.bfloat16)
    res = (2 * torch.randn((M, N), device=DEV, generator=g)).to(torch.bfloat16)
    return dict(wq=wq, s=s, b=b, x=x.to(torch.bfloat16), bias=bias if case["bias"] else None,
                res=res if case["res"] else None)


def _route_inputs(case, seed):
    g = _generator(seed)
    T, E = case["T"], case["E"]
    E1 = E + (1 if case["gate"] else 0)
    # tokens prefer experts, and experts are preferred: what the balance bias is there for
    logits = 1.2 * torch.randn((T, E1), device=DEV, generator=g) + 0.6 * torch.randn((1, E1), device=DEV, generator=g)
    bias = 0.1 * torch.randn((E,), device=DEV, generator=g)
    return dict(logits=logits.to(torch.bfloat16) if case["bf16"] else logits, bias=bias if case["bias"] else None)


def _sample_inputs(case, seed):
    g = _generator(seed)
    T, V, filters = case["T"], case["V"], case["filters"]
    logits = 2.2 * torch.randn((T, V), device=DEV, generator=g)
    # a few dozen plausible tokens stand out, more or less clearly
    at = torch.randint(0, V, (T, 40), device=DEV, generator=g)
    up = 6 + (2 + 8 * torch.rand((T, 1), device=DEV, generator=g)) * torch.rand((T, 40), device=DEV, generator=g) ** 2
    logits.scatter_(1, at, up.expand(T, 40))
    r = lambda: torch.rand((T,), device=DEV, generator=g)  # noqa: E731
    masked = r() < (0.15 if filters == "mixed" else 0.0)
    allowed = torch.rand((T, V), device=DEV, generator=g) < 0.01
    allowed[:, :2] = True
    logits.masked_fill_(masked[:, None] & ~allowed, -math.inf)
    rows = dict(temperature=0.5 + 0.8 * r(), top_k=None, top_p=None, min_p=None, u=r().clamp_(max=1 - 2 ** -24))
    choice = torch.tensor([0, 1, 20, 40, 100, 1000], device=DEV, dtype=torch.int32)
    if filters == "topk_topp":
        rows["top_k"] = choice[2 + (r() * 3).long().clamp_(max=2)]
        rows["top_p"] = 0.8 + 0.15 * r()
    elif filters == "topp":
        rows["top_p"] = 0.9 + 0.09 * r()
    elif filters == "minp":
        rows["min_p"] = 0.02 + 0.1 * r()
    elif filters == "mixed":
        rows["temperature"] = torch.where(r() < 0.2, torch.zeros((), device=DEV), rows["temperature"])
        rows["top_k"] = choice[(r() * 6).long().clamp_(max=5)]
        rows["top_p"] = torch.where(r() < 0.4, torch.ones((), device=DEV), 0.7 + 0.29 * r())
        rows["min_p"] = torch.where(r() < 0.5, torch.zeros((), device=DEV), 0.1 * r())
    return dict(logits=logits.to(torch.bfloat16) if case["bf16"] else logits, **rows)


INPUTS = dict(linear=_linear_inputs, route=_route_inputs, sample=_sample_inputs)


def prepare(case, seed):
    """What an engine holds before the call: the layer in its checkpoint's form and repacked as the loader does, the rows,
    and the buffers that results go to."""
    st = dict(case=case, **INPUTS[case["kind"]](case, seed))
    empty = lambda shape, dtype: torch.empty(shape, dtype=dtype, device=DEV)  # noqa: E731
    if case["kind"] == "linear":
        st["wt"] = _packed(st["wq"], st["s"], st["b"], case["bits"])
        st["c"] = empty((case["M"], case["N"]), torch.float32 if case["out"] == "fp32" else torch.bfloat16)
    elif case["kind"] == "route":
        T, k = case["T"], case["k"]
        st["outs"] = (empty((T, k), torch.int32), empty((T, k), torch.float32), empty((T,), torch.float32))
    else:
        st["outs"] = (empty((case["T"],), torch.int32), empty((case["T"],), torch.float32))
    return st


# ---- a linear with its epilogue --------------------------------------------------------------------------------------
def _act(y, act):
    if act == "relu":
        return y * (y > 0)
    if act == "silu":
        return y / (1 + torch.exp(-y))
    if act == "gelu":
        return 0.5 * y * (1 + torch.erf(y * 0.5 ** 0.5))
    if act == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh((2 / math.pi) ** 0.5 * (y + 0.044715 * y ** 3)))
    return y


def _run_linear(st):
    case = st["case"]
    if own:
        from inferd_amd import ops
        make, call = (ops.T64Linear, ops.gemm_t64_epi) if case["bits"] == 4 else (ops.T64x8Linear, ops.gemm_t64x8_epi)
        W = make(st["wt"], case["N"], case["K"])
        return call(st["x"], W, bias=st["bias"], act=case["act"], residual=st["res"], C=st["c"])
    q = _codes(st["wq"], case["bits"]).float().view(case["N"], -1, 64)
    w = (q * st["s"].float().unsqueeze(-1) + st["b"].float().unsqueeze(-1)).flatten(1)
    y = st["x"].float() @ w.T
    if st["bias"] is not None:
        y = y + st["bias"].float()
    y = _act(y, case["act"])
    if st["res"] is not None:
        y = y + st["res"].float()
    return y.to(st["c"].dtype)


def _exact_linear(case, seed):
    d = _linear_inputs(case, seed)
    M, N, K = case["M"], case["N"], case["K"]
    out = torch.empty((M, N), dtype=torch.float64, device=DEV)
    step = max(1, (1 << 26) // K)
    for i in range(0, N, step):  # a slice of the outputs at a time
        codes = _codes(d["wq"][i:i + step], case["bits"]).double()
        s, b = (torch.repeat_interleave(d[v][i:i + step].double(), 64, 1) for v in "sb")
        y = torch.mm(d["x"].double(), torch.addcmul(b, s, codes).T.contiguous())
        y = y if d["bias"] is None else y + d["bias"][i:i + step].double()
        if case["act"] == "relu":
            y = y.clamp(min=0)
        elif case["act"] == "silu":
            y = y * torch.sigmoid(y)
        elif case["act"] == "gelu":
            y = y * 0.5 * torch.special.erfc(-y / math.sqrt(2))
        elif case["act"] == "gelu_tanh":
            y = y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y))
        out[:, i:i + step] = y if d["res"] is None else y + d["res"][:, i:i + step].double()
    return out


# ---- routing ---------------------------------------------------------------------------------------------------------
def _run_route(st):
    case = st["case"]
    E, k, groups = case["E"], case["k"], case["groups"]
    if own:
        from inferd_amd import ops
        return ops.moe_route_ex(st["logits"], E, k, score=case["score"], bias=st["bias"], groups=groups,
                                topk_groups=case["topk_groups"], group_top=case["group_top"], norm=case["norm"],
                                scale=case["scale"], shared_gate=case["gate"], outs=st["outs"])
    logits = st["logits"].double()
    l = logits[:, :E]
    if case["score"] == "softmax":
        s = torch.exp(l - l.amax(-1, keepdim=True))
        s = s / s.sum(-1, keepdim=True)
    else:
        s = 1 / (1 + torch.exp(-l))
    # without a bias the order of the scores is the logits' own
    choice = s + st["bias"].double() if st["bias"] is not None else l
    if groups > 1:
        value = choice if case["group_top"] == 1 else (s if st["bias"] is None else choice)
        value = torch.sort(value.view(-1, groups, E // groups), dim=-1, descending=True).values[..., :case["group_top"]].sum(-1)
        best = torch.sort(value, dim=-1, descending=True, stable=True).indices[:, :case["topk_groups"]]
        kept = torch.zeros_like(value, dtype=torch.bool).scatter_(1, best, True)
        choice = choice.masked_fill(~kept.repeat_interleave(E // groups, 1), -math.inf)
    idx = torch.sort(choice, dim=-1, descending=True, stable=True).indices[:, :k]
    w = s.gather(1, idx)
    if case["norm"]:
        w = w / w.sum(-1, keepdim=True)
    sg = 1 / (1 + torch.exp(-logits[:, E])) if case["gate"] else torch.ones_like(l[:, 0])
    return dict(idx=idx.int(), wt=(w * case["scale"]).float(), sg=sg.float())


def _exact_route(case, seed):
    d = _route_inputs(case, seed)
    E, k, groups = case["E"], case["k"], case["groups"]
    logits = d["logits"].double().cpu().numpy()
    l = logits[:, :E]
    if case["score"] == "softmax":
        e = np.exp(l - l.max(1, keepdims=True))
        s = e / e.sum(1, keepdims=True)
    else:
        s = 0.5 + 0.5 * np.tanh(l / 2)
    c = l.copy() if d["bias"] is None else s + d["bias"].double().cpu().numpy()
    rows = np.arange(len(l))
    if groups > 1:
        v = np.partition((s if case["group_top"] == 2 and d["bias"] is None else c).reshape(len(l), groups, -1),
                         -case["group_top"], 2)[:, :, -case["group_top"]:].sum(2)
        out = np.ones(v.shape, bool)
        for _ in range(case["topk_groups"]):
            g = np.where(out, v, -np.inf).argmax(1)
            out[rows, g] = False
        c[np.repeat(out, E // groups, 1)] = -np.inf
    idx = np.empty((len(l), k), np.int32)
    for j in range(k):
        idx[:, j] = c.argmax(1)
        c[rows, idx[:, j]] = -np.inf
    w = np.take_along_axis(s, idx, 1)
    w = case["scale"] * (w / w.sum(1, keepdims=True) if case["norm"] else w)
    sg = 0.5 + 0.5 * np.tanh(logits[:, E] / 2) if case["gate"] else np.ones(len(l))
    return dict(idx=idx, wt=w, sg=sg)


# ---- sampling --------------------------------------------------------------------------------------------------------
def _run_sample(st):
    if own:
        from inferd_amd import ops
        token, prob = ops.sample(st["logits"], st["u"], temperature=st["temperature"], top_k=st["top_k"],
                                 top_p=st["top_p"], min_p=st["min_p"], outs=st["outs"])
        return dict(token=token, prob=prob)
    l = st["logits"].double()
    V = l.shape[1]
    greedy = (st["temperature"] <= 0)[:, None]
    m = l.amax(-1, keepdim=True)
    w = torch.exp((l - m) / torch.where(greedy, torch.ones_like(m), st["temperature"].double()[:, None]))
    order = torch.sort(l, dim=-1, descending=True, stable=True).indices
    w = w.gather(1, order)
    rank = torch.arange(V, device=l.device)
    keep = ~greedy | (rank == 0)
    if st["top_k"] is not None:
        keep &= (rank < st["top_k"][:, None]) | (st["top_k"][:, None] <= 0)
    if st["top_p"] is not None:
        cum = torch.cumsum(w * keep, -1)
        before = cum - w * keep
        keep &= (before < st["top_p"].double()[:, None] * cum[:, -1:]) | (st["top_p"][:, None] >= 1)
    if st["min_p"] is not None:
        keep &= w >= st["min_p"].double()[:, None]
    kept = torch.zeros_like(w).scatter_(1, order, w * keep)
    cum = torch.cumsum(kept, -1)
    total = cum[:, -1:]
    token = torch.searchsorted(cum, st["u"].double()[:, None] * total, right=True)
    return dict(token=token[:, 0].int(), prob=(kept.gather(1, token) / total)[:, 0].float())


def _exact_sample(case, seed):
    d = {n: None if v is None else (v.double() if v.is_floating_point() else v).cpu().numpy()
         for n, v in _sample_inputs(case, seed).items()}
    tokens, probs = [], []
    for r, l in enumerate(d["logits"]):
        if d["temperature"][r] <= 0:
            tokens.append(int(l.argmax()))
            probs.append(1.0)
            continue
        w = np.exp((l - l.max()) / d["temperature"][r])
        n = len(l)
        k = 0 if d["top_k"] is None else int(d["top_k"][r])
        p = 1.0 if d["top_p"] is None else d["top_p"][r]
        mp = 0.0 if d["min_p"] is None else d["min_p"][r]
        at = np.flatnonzero(w > 0)
        if k > 0 or p < 1:
            at = at[np.argsort(-l[at], kind="stable")]
            n = min(len(at), k) if k > 0 else len(at)
            if p < 1:
                c = np.cumsum(w[at[:n]])
                n = int(np.searchsorted(c, p * c[-1])) + 1
            at = np.sort(at[:n])
        at = at[w[at] >= mp]
        c = np.cumsum(w[at])
        t = at[int(np.searchsorted(c, d["u"][r] * c[-1], side="right"))]
        tokens.append(int(t))
        probs.append(float(w[t] / c[-1]))
    return dict(token=np.array(tokens, np.int32), prob=np.array(probs))


# ---- the interface -----------------------------------------------------------------------------------------------------
def run(st):
    kind = st["case"]["kind"]
    if kind == "linear":
        return _run_linear(st)
    if kind == "route":
        out = _run_route(st)
        return out if isinstance(out, dict) else dict(zip(("idx", "wt", "sg"), out))
    return _run_sample(st)


def exact(case, seed):
    return dict(linear=_exact_linear, route=_exact_route, sample=_exact_sample)[case["kind"]](case, seed)


def work(case):
    if case["kind"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        per = 0.5625 if case["bits"] == 4 else 1.0625
        out = (4 if case["out"] == "fp32" else 2) + (2 if case["res"] else 0)
        return {"bytes": N * K * per + M * K * 2 + M * N * out + (2 * N if case["bias"] else 0), "flops": 2.0 * M * N * K}
    if case["kind"] == "route":
        T, E, k = case["T"], case["E"], case["k"]
        row = (E + (1 if case["gate"] else 0)) * (2 if case["bf16"] else 4) + 8 * k + 4
        return {"bytes": T * row + (4 * E if case["bias"] else 0), "flops": 4.0 * T * E}
    T, V = case["T"], case["V"]
    return {"bytes": T * V * (2 if case["bf16"] else 4) + 28.0 * T, "flops": 4.0 * T * V}
