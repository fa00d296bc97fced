"""Argument checks of the 8-bit products into fp32, on the CPU: refused before anything is launched."""
import pytest
import torch

from latest_exact_match_attention_amd import _lib, build

P = 1 << 20          # an address that no refused call reads


@pytest.fixture(scope="module")
def L():
    build.ensure_built()
    return _lib.lib()


def test_matmul(L):
    f, size = L.lema_fp8_matmul_f32, L.lema_fp8_matmul_f32_workspace_bytes
    ok = dict(a=P, sa=P, lds=48, w=P, sw=P, w2=None, sw2=None, M=48, N=64, K=64, out=P, ws=None, n=0)

    def call(**kw):
        return f(*{**ok, **kw}.values(), None)
    for kw in (dict(M=-1), dict(N=0), dict(K=0), dict(N=(1 << 20) + 1), dict(K=(1 << 20) + 1), dict(lds=47), dict(lds=50),
               dict(a=None), dict(w=P + 8), dict(out=P + 8), dict(sa=P + 2), dict(w2=P), dict(w2=P, sw2=P, N=60)):
        assert call(**kw) == _lib.BAD_ARG, kw
    assert call(M=0, a=None, sa=None, w=None, sw=None, out=None) == _lib.OK
    n = size(40, 136, 16384, 0)
    assert n > 0 and n % (40 * 136 * 4) == 0 and size(0, 136, 16384, 0) == 0
    assert call(M=40, N=136, K=16384, ws=P, n=n - 1) == _lib.BAD_ARG and b"workspace" in L.lema_last_error()


def test_linear(L):
    f = L.lema_fp8_linear_f32
    assert f(P, 64, P, P, None, None, None, 33, 64, 64, P, None) == _lib.BAD_ARG
    assert f(P, 63, P, P, None, None, None, 4, 64, 64, P, None) == _lib.BAD_ARG
    assert f(P, 64, P, P, P, None, None, 4, 64, 64, P, None) == _lib.BAD_ARG
    assert f(P, 64, P + 4, P, None, None, None, 4, 64, 64, P, None) == _lib.BAD_ARG
    for i in (0, 6, 10):                                        # x, the residual and the result, at half an element
        a = [P, 64, P, P, None, None, None, 4, 64, 64, P, None]
        a[i] = P + 2
        assert f(*a) == _lib.BAD_ARG, i
    assert f(None, 64, None, None, None, None, None, 0, 64, 64, None, None) == _lib.OK


def test_on_the_cpu():
    from latest_exact_match_attention_amd import fp8
    w = fp8.Fp8(torch.zeros(8, 128, dtype=torch.float8_e4m3fn), torch.zeros(1, 1, dtype=torch.float8_e8m0fnu), 64)
    with pytest.raises(TypeError, match="HIP"):
        fp8.linear(torch.randn(4, 64), w)
