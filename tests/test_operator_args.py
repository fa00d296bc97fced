"""Refusals of the training operators' entry points that need no GPU, and what they do on the CPU."""
import pytest
import torch

from latest_exact_match_attention_amd import _lib, build
from latest_exact_match_attention_amd.loss import policy_loss, preference_loss, token_logprobs
from latest_exact_match_attention_amd.model import embed, layer_norm

P = 4096  # stands for a device pointer; every call below is refused, or empty, before it is used


@pytest.fixture(scope="module")
def L():
    build.ensure_built()
    return _lib.lib()


def test_embedding(L):
    f = L.lema_embedding
    assert f(P, 3, 10, 8, P, 4, 1.0, P, None) == _lib.BAD_ARG            # type
    assert f(P, 0, 0, 8, P, 4, 1.0, P, None) == _lib.BAD_ARG             # no table
    assert f(P, 0, 10, (1 << 20) + 1, P, 4, 1.0, P, None) == _lib.BAD_ARG
    assert f(P + 2, 0, 10, 8, P, 4, 1.0, P, None) == _lib.BAD_ARG        # half an element off
    assert f(None, 0, 10, 8, P, 4, 1.0, P, None) == _lib.BAD_ARG
    assert f(None, 2, 10, 8, None, 0, 1.0, None, None) == _lib.OK
    g, size = L.lema_embedding_grad, L.lema_embedding_grad_workspace_bytes
    n = size(100, 10, 8)
    assert n > 0 and size(-1, 10, 8) == 0 and size(1 << 31, 10, 8) == 0
    assert size(100, (1 << 20) + 1, 8) == 0 and size(100, 0, 8) == 0
    assert g(P, 2, P, 100, 10, 8, 1.0, -1, P, P, n - 1, None) == _lib.BAD_ARG
    assert b"workspace" in L.lema_last_error()
    assert g(P, 2, P, 100, 10, 8, 1.0, -1, P, P + 16, n, None) == _lib.BAD_ARG
    assert g(P, 2, P, 100, (1 << 20) + 1, 8, 1.0, -1, P, P, 1 << 40, None) == _lib.BAD_ARG
    assert g(None, 2, P, 100, 10, 8, 1.0, -1, P, P, n, None) == _lib.BAD_ARG
    assert g(P, 2, P, (1 << 31) - 20000, 1 << 20, 1 << 20, 1.0, -1, P, P, 1 << 62, None) == _lib.BAD_ARG
    assert b"too large" in L.lema_last_error()


def test_norms(L):
    f = L.lema_layer_norm
    assert f(P, None, P, P, 5, 1e-5, 4, 8, None, P, None) == _lib.BAD_ARG
    for D in (0, 16385):
        assert f(P, None, P, P, 2, 1e-5, 4, D, None, P, None) == _lib.BAD_ARG
    assert f(P, P, P, P, 2, 1e-5, 4, 8, None, P, None) == _lib.BAD_ARG   # a sum without its output
    assert f(P + 1, None, P, P, 2, 1e-5, 4, 8, None, P, None) == _lib.BAD_ARG
    assert f(P, None, P, P, 2, 1e-5, 1 << 31, 8, None, P, None) == _lib.BAD_ARG
    assert f(None, None, None, None, 2, 1e-5, 0, 8, None, None, None) == _lib.OK
    g, n = L.lema_norm_grad, L.lema_norm_grad_workspace_bytes(4, 8)
    assert n > 0 and L.lema_norm_grad_workspace_bytes(0, 8) == 0
    assert g(P, P, P, None, 2, 1, 1e-5, 4, 8, P, P, P, P, n - 1, None) == _lib.BAD_ARG
    assert g(P, P, P, None, 2, 1, 1e-5, 4, 8, P, P, P, None, n, None) == _lib.BAD_ARG
    assert g(P, P, P, None, 2, 0, 1e-5, 4, 8, P, P, P, P, n, None) == _lib.BAD_ARG
    assert b"no bias" in L.lema_last_error()
    assert g(P, P, None, None, 2, 1, 1e-5, 4, 8, P, P, P, P, n, None) == _lib.BAD_ARG
    assert g(None, None, None, None, 2, 1, 1e-5, 0, 8, None, None, None, None, 0, None) == _lib.OK
    s = L.lema_swiglu_grad_bf16
    assert s(P, P, P, P, P, 12, None) == _lib.BAD_ARG and s(P, P, P, P, P + 8, 16, None) == _lib.BAD_ARG
    assert s(None, None, None, None, None, 0, None) == _lib.OK


def test_losses(L):
    f = L.lema_token_logprobs
    ok = [P, 2, 4, 4, 8, 0, 8, P, None, 1.0, P, None, P, None]

    def bad(i, v):
        a = list(ok)
        a[i] = v
        assert f(*a) == _lib.BAD_ARG, (i, v)
    for i, v in ((0, None), (0, P + 1), (1, 7), (2, -1), (2, 1 << 31), (3, 0), (4, 0), (5, -8), (6, -1),
                 (7, None), (9, 0.0), (9, -1.0), (9, float("inf")), (9, float("nan")), (9, 1e-40), (10, None),
                 (11, P + 4), (12, P + 4)):
        bad(i, v)
    assert f(None, 2, 0, 1, 8, 0, 8, None, None, 1.0, None, None, None, None) == _lib.OK
    g = L.lema_token_logprobs_grad
    assert g(P, 2, 4, 4, 8, 0, 8, P, None, 1.0, None, P, 1, None, None, 0, P, None) == _lib.BAD_ARG
    assert g(P, 2, 4, 4, 8, 0, 8, P, None, 1.0, P, P, 0, None, None, 0, P, None) == _lib.BAD_ARG
    assert g(P, 2, 4, 4, 8, 0, 8, P, None, 1.0, P, P, 1, None, None, 1, P, None) == _lib.BAD_ARG
    p = L.lema_policy_loss
    args = [P, 2, 4, 4, 8, 0, 8, P, None, 1.0, P, P, None, 0.2, 0.2, 0.0, 1.0, P, P, P, P, P, P, None, None]
    for i, v in ((10, None), (11, None), (13, -0.1), (14, float("nan")), (17, None), (18, None), (18, P + 4),
                 (19, None), (20, None), (21, None), (22, None), (23, P + 1)):
        a = list(args)
        a[i] = v
        assert p(*a) == _lib.BAD_ARG, (i, v)
    r = L.lema_preference_loss
    args = [P, P, None, 2, 3, 0.1, 0.0, P, P, P, None]
    for i, v in ((0, None), (0, P + 4), (1, None), (3, 0), (4, -1), (6, 1.5), (6, float("nan")), (7, None),
                 (8, None), (9, None)):
        a = list(args)
        a[i] = v
        assert r(*a) == _lib.BAD_ARG, (i, v)


def test_on_the_cpu():
    """The model's functions keep torch's operations there; the losses are the device's."""
    x, d = torch.randn(3, 12, dtype=torch.float64), torch.randn(3, 12, dtype=torch.float64)
    norm = torch.nn.LayerNorm(12, dtype=torch.float64)
    h, s = layer_norm(x, norm, d)
    assert torch.equal(s, x + d) and torch.equal(h, norm(x + d))
    emb = torch.nn.Embedding(9, 4)
    ids = torch.tensor([[1, 8]])
    assert torch.equal(embed(emb, ids, 2.0), emb(ids) * 2.0)
    t = torch.zeros(2, 3, dtype=torch.long)
    z = torch.zeros(2, 3)
    for call in (lambda: token_logprobs(torch.zeros(2, 3, 5), t), lambda: policy_loss(torch.zeros(2, 3, 5), t, z, z),
                 lambda: preference_loss(torch.zeros(2, 3, 5), t, z)):
        with pytest.raises(TypeError, match="HIP"):
            call()
    with pytest.raises(ValueError, match="addend"):
        layer_norm(x, norm, d[:2])
