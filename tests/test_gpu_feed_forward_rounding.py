"""A token's gated product is the same in a decode step, a chunk and a prompt: both products in fp32,
silu(g) * u rounded once, however many rows a call has."""
import pytest
import torch

from latest_exact_match_attention_amd.model import SwiGLU, rms_norm

pytestmark = pytest.mark.gpu


def block(dev, K, seed=0):
    """A block whose output is the gated product itself: the down projection is the identity."""
    torch.manual_seed(seed)
    mlp = SwiGLU(K, K).to(dev)
    with torch.no_grad():
        mlp.gate.weight.normal_(0, 2 * K ** -0.5)
        mlp.up.weight.normal_(0, K ** -0.5)
        mlp.down.weight.copy_(torch.eye(K, device=dev))
    return mlp.bfloat16()


def check(got, x, mlp):
    """Against 64 bits: one rounding, half a step, and what comes before it in fp32. K exact products added up in
    fp32 are off by at most K 2^-23 of their sizes' sum, silu' <= 1.1, e^-g is off by 2 ulp (|g| + 2). A
    rounding of g, u or silu(g) to bf16 is 2^-9 more of the result in half of the elements."""
    x, wg, wu = (t.detach().double() for t in (x, mlp.gate.weight, mlp.up.weight))
    g, u = x @ wg.t(), x @ wu.t()
    eg, eu = (x.shape[-1] * 2.0 ** -23 * (x.abs() @ w.abs().t()) for w in (wg, wu))
    act = g * torch.sigmoid(g)
    slack = 1.1 * eg * (u.abs() + eu) + act.abs() * eu + 8 * 2.0 ** -24 * (g.abs() + 4) * (act * u).abs()
    want = act * u
    bad = (got.double() - want).abs() > 2.0 ** -8 * (want.abs() + slack) + slack + 2.0 ** -133
    assert not bool(bad.any()), (int(bad.sum()), bad.numel())


@pytest.mark.parametrize("K", [64, 256, 1536])
@pytest.mark.parametrize("rows", [1, 7, 16, 17, 32, 33, 70])
def test_one_rounding(dev, rows, K):
    mlp = block(dev, K)
    x = torch.randn(rows, K, device=dev).bfloat16()
    with torch.no_grad():
        check(mlp(x), x, mlp)
    y = mlp(x)                                     # where its gradient is wanted, too
    assert y.requires_grad
    check(y.detach(), x, mlp)


def test_a_prompt_in_pieces(dev):
    """The same rows at once, in chunks and one by one differ in few last bits: those that lie so near a
    border that the fp32 sums' order tells (2^-14 of the elements or so), where another rounding on the
    way changes about a third."""
    mlp = block(dev, 256, 1)
    x = torch.randn(96, 256, device=dev).bfloat16()
    with torch.no_grad():
        whole = mlp(x)
        for n in (1, 8, 32, 33):
            parts = torch.cat([mlp(x[a:a + n]) for a in range(0, 96, n)])
            assert float((parts != whole).double().mean()) < 2.0 ** -8, n


def test_the_norm_inside(dev):
    """The launch with the norm in it is the norm and the block."""
    mlp = block(dev, 256, 2)
    norm = torch.nn.RMSNorm(256, eps=1e-5).to(dev, torch.bfloat16)
    x, d = (torch.randn(5, 1, 256, device=dev).bfloat16() for _ in range(2))
    with torch.no_grad():
        got = mlp.forward_normed(x, d, norm)
        h, s = rms_norm(x, norm, d)
        a = mlp(h)
        assert torch.equal(got, s + a)
        check(a, h, mlp)


@pytest.mark.parametrize("rows", [9, 40])
def test_gradients_of_few_rows(dev, rows):
    """Against the formula in 64 bits. dg and du are rounded to bf16 (2^-9 in the root mean square at most, half
    a step 2^-8 in size), their derivatives kept to 2^-12, and the result once more."""
    K = 256
    mlp = block(dev, K, 3)
    x = torch.randn(rows, K, device=dev).bfloat16().requires_grad_(True)
    gy = torch.randn(rows, K, device=dev).bfloat16()
    got = torch.autograd.grad(mlp(x), [x, mlp.gate.weight, mlp.up.weight], gy)
    xd, wg, wu = (t.detach().double().requires_grad_(True) for t in (x, mlp.gate.weight, mlp.up.weight))
    want = torch.autograd.grad(torch.nn.functional.silu(xd @ wg.t()) * (xd @ wu.t()), [xd, wg, wu], gy.double())
    for a, b in zip(got, want):
        assert float((a.double() - b).norm() / b.norm()) < 2 * 2.0 ** -8


def test_other_widths(dev):
    """Widths that are no multiple of 8 keep torch's roundings at every number of rows."""
    mlp = SwiGLU(64, 132).to(dev).bfloat16()
    x = torch.randn(48, 64, device=dev).bfloat16()
    with torch.no_grad():
        whole = mlp(x)
        parts = torch.cat([mlp(x[:16]), mlp(x[16:48])])
        g, u = x.float() @ mlp.gate.weight.float().t(), x.float() @ mlp.up.weight.float().t()
        assert float((whole != parts).double().mean()) < 2.0 ** -5
        a = torch.nn.functional.silu(g) * u
        assert float((whole.float() - a @ mlp.down.weight.float().t()).norm() / whole.float().norm()) < 2.0 ** -6
