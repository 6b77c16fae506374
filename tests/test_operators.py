"""CPU checks of the epilogue linears, the extended routing and the sampling: what the C ABI and the Python wrappers refuse
before any GPU work."""
import pytest

from inferd_amd import _lib, ops

torch = pytest.importorskip("torch")

P = 4096  # an aligned address that nothing reads


def _refused(rc, status, text):
    assert rc == status
    assert text in _lib.lib().ifd_last_error(), _lib.lib().ifd_last_error()


@pytest.mark.parametrize("kw,text", [
    (dict(E=0), b"routing shape"), (dict(E=513, stride=513), b"routing shape"), (dict(k=0), b"routing shape"),
    (dict(k=17), b"routing shape"), (dict(E=4, k=5), b"routing shape"), (dict(T=-1), b"routing shape"),
    (dict(stride=255), b"stride=255"), (dict(gate=1), b"stride=256"), (dict(score=2), b"score=2"),
    (dict(groups=0), b"groups=0"), (dict(groups=7), b"groups=7"), (dict(groups=128), b"groups=128"),
    (dict(tg=0), b"topk_groups=0"), (dict(groups=8, tg=9), b"topk_groups=9"),
    (dict(groups=64, tg=1), b"cannot give 8 picks"), (dict(gtop=3), b"group_top=3"),
    (dict(E=64, stride=64, groups=64, tg=8, gtop=2), b"group_top=2"), (dict(scale=float("inf")), b"scale"),
    (dict(scale=float("nan")), b"scale"), (dict(logits=None), b"null"), (dict(idx=None), b"null"),
    (dict(wt=None), b"null"), (dict(sg=None), b"null"), (dict(bias=P + 2), b"misaligned"),
    (dict(logits=P + 2), b"misaligned"), (dict(logits=P + 1, bf=1), b"misaligned"),
])
def test_route_ex_refuses(kw, text):
    a = dict(logits=P, bf=0, T=4, E=256, k=8, stride=256, score=1, bias=P, groups=8, tg=4, gtop=2, norm=1, scale=1.0, gate=0,
             idx=P, wt=P, sg=P)
    a.update(kw)
    _refused(_lib.lib().ifd_moe_route_ex(*a.values(), None), _lib.IFD_ERR_ARG, text)


@pytest.mark.parametrize("kw,text", [
    (dict(T=-1), b"bad shape"), (dict(V=0), b"bad shape"), (dict(V=(1 << 19) + 1, ld=1 << 20), b"bad shape"),
    (dict(ld=999), b"ld=999"), (dict(bf=2), b"logits_bf16=2"), (dict(logits=None), b"null"), (dict(u=None), b"null"),
    (dict(token=None), b"null"), (dict(logits=P + 2), b"misaligned"), (dict(temp=P + 1), b"misaligned"),
    (dict(prob=P + 2), b"misaligned"), (dict(ws=P + 8), b"workspace"),
])
def test_sample_refuses(kw, text):
    a = dict(logits=P, bf=0, T=4, V=1000, ld=1000, temp=P, top_k=P, top_p=P, min_p=P, u=P, token=P, prob=P, ws=None,
             ws_bytes=0)
    a.update(kw)
    _refused(_lib.lib().ifd_sample(*a.values(), None), _lib.IFD_ERR_ARG, text)


def test_sample_workspace():
    L = _lib.lib()
    assert L.ifd_sample_workspace(0, 1000) == 0 and L.ifd_sample_workspace(4, (1 << 19) + 1) == 0
    need = L.ifd_sample_workspace(4, 248320)
    if need:
        for ws, size in ((None, 0), (P, need - 1)):
            rc = L.ifd_sample(P, 0, 4, 248320, 248320, P, P, P, P, P, P, P, ws, size, None)
            _refused(rc, _lib.IFD_ERR_WORKSPACE, b"workspace")


@pytest.mark.parametrize("name", ["ifd_gemm_t64_epi", "ifd_gemm_t64x8_epi"])
@pytest.mark.parametrize("kw,text", [
    (dict(K=96, lda=96), b"multiple of"), (dict(M=-1), b"bad shape"), (dict(N=0), b"bad shape"), (dict(act=5), b"act=5"),
    (dict(act=-1), b"act=-1"), (dict(f32=2), b"out_f32=2"), (dict(lda=248), b"lda=248"), (dict(lda=260), b"lda=260"),
    (dict(ldc=99), b"ldc=99"), (dict(ldr=99), b"ldr=99"), (dict(A=None), b"null"), (dict(wt=None), b"null"),
    (dict(C=None), b"null"), (dict(A=P + 8), b"misaligned"), (dict(bias=P + 1), b"misaligned"),
    (dict(C=P + 2, f32=1), b"misaligned"), (dict(res=1 << 20, ldr=104), b"overlaps"),
    (dict(res=(1 << 20) + 100), b"overlaps"), (dict(res=1 << 20, f32=1), b"overlaps"), (dict(ws=P + 8), b"workspace"),
])
def test_epilogue_refuses(name, kw, text):
    a = dict(A=P, lda=256, wt=P, N=100, K=256, bias=P, act=1, res=1 << 24, ldr=100, C=1 << 20, ldc=100, M=4, f32=0, ws=P,
             ws_bytes=1 << 30)
    a.update(kw)
    _refused(getattr(_lib.lib(), name)(*a.values(), None), _lib.IFD_ERR_ARG, text)


@pytest.mark.parametrize("name", ["ifd_gemm_t64_epi", "ifd_gemm_t64x8_epi"])
@pytest.mark.parametrize("M,N,K", [(1, 5120, 5120), (8, 17408, 5120), (64, 5120, 5120), (777, 5120, 17408)])
def test_epilogue_needs_its_workspace(name, M, N, K):
    L = _lib.lib()
    need = getattr(L, name + "_workspace")(M, N, K)
    for ws, size in ((None, 0), (P, need - 1)) if need else ():
        rc = getattr(L, name)(P, K, P, N, K, None, 0, None, 0, 1 << 20, N, M, 0, ws, size, None)
        _refused(rc, _lib.IFD_ERR_WORKSPACE, b"workspace")


def test_empty_calls_do_nothing():
    L = _lib.lib()
    assert L.ifd_moe_route_ex(None, 0, 0, 256, 8, 256, 1, None, 1, 1, 1, 1, 1.0, 0, None, None, None, None) == 0
    assert L.ifd_sample(None, 0, 0, 1000, 1000, None, None, None, None, None, None, None, None, 0, None) == 0
    for name in ("ifd_gemm_t64_epi", "ifd_gemm_t64x8_epi"):
        assert getattr(L, name)(None, 256, None, 100, 256, None, 0, None, 0, None, 100, 0, 0, None, 0, None) == 0


def test_wrappers_refuse():
    z = torch.zeros
    W = ops.T64Linear(z(1, dtype=torch.uint8), 100, 256)
    A = z(4, 256, dtype=torch.bfloat16)
    for call in (
        lambda: ops.gemm_t64_epi(A, W),  # not on a GPU
        lambda: ops.gemm_t64_epi(A.float(), W),
        lambda: ops.gemm_t64_epi(A[:, :128], W),
        lambda: ops.sample(z(4, 100), z(4)),
        lambda: ops.sample(z(100), z(1)),
        lambda: ops.sample(z(4, 100, dtype=torch.float64), z(4)),
        lambda: ops.sample(z(4, 100), z(5)),
        lambda: ops.sample(z(4, 100), z(4), top_k=z(4)),
        lambda: ops.sample(z(4, 100), z(1).expand(4)),
        lambda: ops.sample(z(100, 4).T, z(4)),
        lambda: ops.moe_route_ex(z(4, 64), 64, 8),
        lambda: ops.moe_route_ex(z(4, 64), 65, 8),
        lambda: ops.moe_route_ex(z(4, 64), 64, 8, shared_gate=True),
        lambda: ops.moe_route_ex(z(4, 64), 64, 8, score="relu"),
        lambda: ops.moe_route_ex(z(4, 64), 64, 8, bias=z(63)),
        lambda: ops.moe_route_ex(z(4, 64), 64, 8, outs=(z(4, 8), z(4, 8), z(4))),
    ):
        with pytest.raises(ValueError):
            call()
