"""Argument checks of the decode step's gated launches, on the CPU: refused before anything is launched."""
import pytest

from latest_exact_match_attention_amd import _lib, build


@pytest.fixture(scope="module")
def L():
    build.ensure_built()
    return _lib.lib()


def test_gated(L):
    f = L.lema_skinny_gated_bf16          # x, ldx, wg, wu, ldw, M, N, K, out, stream
    ok = [256, 64, 512, 1024, 64, 4, 64, 64, 1792, None]
    for i, v in ((0, None), (0, 264), (1, 32), (2, None), (3, 520), (4, 68), (5, 33), (5, 0), (6, 0), (7, 40), (8, None)):
        a = list(ok)
        a[i] = v
        assert f(*a) == _lib.BAD_ARG, (i, v)


def test_gated_with_the_norm(L):
    f = L.lema_skinny_norm_gated_bf16     # x, d, nw, eps, x_out, wg, wu, ldw, M, N, K, out, stream
    ok = [256, 512, 768, 1e-5, 1024, 1280, 1536, 64, 4, 64, 64, 1792, None]
    for i, v, what in ((8, 33, b"rows"), (4, 256, b"neither input"), (2, None, b"norm weight"), (5, None, b"weights")):
        a = list(ok)
        a[i] = v
        assert f(*a) == _lib.BAD_ARG and what in L.lema_last_error(), (i, v)
    assert f(256, 512, 768, 1e-5, 1024, 1280, 1536, 2080, 4, 64, 2080, 1792, None) == _lib.BAD_ARG
    assert b"at most 2048" in L.lema_last_error()
    assert f(256, 512, 768, 1e-5, 1024, 1280, 1536, 2048, 32, 64, 2048, 1792, None) == _lib.BAD_ARG
    assert b"LDS" in L.lema_last_error()
