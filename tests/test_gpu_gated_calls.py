"""The feed-forward block under what torch wraps around a call: forward mode, gradients of gradients, batched
gradients, vmap, tracing, weights of another tensor class."""
import pytest
import torch
import torch.nn.functional as F
from torch import nn
from torch.autograd import forward_ad

from latest_exact_match_attention_amd.model import SwiGLU, gated_linear, swiglu

pytestmark = pytest.mark.gpu

# A handful of 16-bit roundings, each of half a step 2^-11, one after another and in sums: 16 of them in a row
BOUND = 16 * 2.0 ** -11


def make(dev, rows=48, K=64, N=136, dtype=torch.float16):
    torch.manual_seed(0)
    gate, up = (nn.Linear(K, N, bias=False, device=dev, dtype=dtype) for _ in range(2))
    return torch.randn(rows, K, device=dev).to(dtype), gate, up, torch.randn(rows, N, device=dev).to(dtype)


def plain(x, wg, wu):
    return F.silu(x @ wg.t()) * (x @ wu.t())


def doubles(*ts):
    return tuple(t.detach().double().requires_grad_(True) for t in ts)


def close(a, b):
    assert float((a.double() - b.double()).norm() / b.double().norm()) < BOUND


@pytest.mark.parametrize("rows", [5, 48])
def test_forward_mode(dev, rows):
    x, gate, up, _ = make(dev, rows)
    t = torch.randn_like(x)
    with forward_ad.dual_level():
        y = gated_linear(forward_ad.make_dual(x, t), gate, up)
        value, tangent = forward_ad.unpack_dual(y)
    d = doubles(x, gate.weight, up.weight)
    want, slope = torch.func.jvp(lambda v: plain(v, d[1].detach(), d[2].detach()), (d[0].detach(),), (t.double(),))
    close(value, want)
    close(tangent, slope)
    mlp = block_of(gate, up, dev)
    _, slope2 = torch.func.jvp(mlp, (x,), (t,))
    close(slope2, slope @ mlp.down.weight.detach().double().t())


def block_of(gate, up, dev):
    mlp = SwiGLU(gate.in_features, gate.out_features).to(dev).to(gate.weight.dtype)
    mlp.gate, mlp.up = gate, up
    return mlp


@pytest.mark.parametrize("rows", [5, 48])
def test_gradients_of_gradients(dev, rows):
    x, gate, up, gy = make(dev, rows)
    x.requires_grad_(True)
    leaves = [x, gate.weight, up.weight]
    first = torch.autograd.grad(gated_linear(x, gate, up), leaves, gy, create_graph=True)
    v = [torch.randn_like(t) / t.numel() ** 0.5 for t in leaves]
    second = torch.autograd.grad(sum((a * b).sum() for a, b in zip(first, v)), leaves)
    d = doubles(*leaves)
    one = torch.autograd.grad(plain(*d), d, gy.double(), create_graph=True)
    two = torch.autograd.grad(sum((a * b.double()).sum() for a, b in zip(one, v)), d)
    for a, b in zip((*first, *second), (*one, *two)):
        close(a.detach(), b.detach())


def test_gradient_of_the_output_gradient(dev):
    """The first gradient is linear in gy: a gradient by gy is the product's forward mode."""
    x, gate, up, gy = make(dev)
    x.requires_grad_(True)
    gy.requires_grad_(True)
    (gx,) = torch.autograd.grad(gated_linear(x, gate, up), [x], gy, create_graph=True)
    t = torch.randn_like(x)
    (got,) = torch.autograd.grad((gx * t).sum(), [gy])
    d = doubles(x, gate.weight, up.weight)
    _, want = torch.func.jvp(lambda v: plain(v, d[1].detach(), d[2].detach()), (d[0].detach(),), (t.double(),))
    close(got, want)


def test_batched_gradients(dev):
    x, gate, up, gy = make(dev)
    x.requires_grad_(True)
    leaves = [x, gate.weight, up.weight]
    gys = torch.stack([gy, -2 * gy, gy.flip(0)])
    got = torch.autograd.grad(gated_linear(x, gate, up), leaves, gys, is_grads_batched=True)
    d = doubles(*leaves)
    for i in range(3):
        want = torch.autograd.grad(plain(*d), d, gys[i].double())
        for a, b in zip(got, want):
            close(a[i], b)


def test_functional_transforms(dev):
    x, gate, up, gy = make(dev)
    wg, wu = gate.weight.detach(), up.weight.detach()
    with torch.no_grad():
        stacked = torch.stack([x, 2 * x])
        got = torch.vmap(lambda v: gated_linear(v, gate, up))(stacked)
        for i in range(2):
            close(got[i], plain(stacked[i].double(), wg.double(), wu.double()))
    mlp = block_of(gate, up, dev)
    params = {k: v.detach() for k, v in mlp.named_parameters()}
    grads = torch.func.grad(lambda p: (torch.func.functional_call(mlp, p, (x,)).float().square()).mean())(params)
    d = {k: v.double().requires_grad_(True) for k, v in params.items()}
    y = plain(x.double(), d["gate.weight"], d["up.weight"]) @ d["down.weight"].t()
    for (k, v), w in zip(d.items(), torch.autograd.grad(y.square().mean(), list(d.values()))):
        close(grads[k], w)
    both = {k: torch.stack([v, -v]) for k, v in params.items()}     # an ensemble: the weights are batched
    ys = torch.vmap(lambda p: torch.func.functional_call(mlp, p, (x,)))(both)
    close(ys[0], y.detach())


def test_tracing(dev):
    x, gate, up, _ = make(dev)
    mlp = block_of(gate, up, dev).requires_grad_(False)
    other = torch.randn_like(x)
    traced = torch.jit.trace(mlp, (x,))
    close(traced(other), mlp(other))
    from torch.fx.experimental.proxy_tensor import make_fx
    close(make_fx(mlp)(x)(other), mlp(other))
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        assert mlp(mode.from_tensor(x)).shape == x.shape


def test_compiled(dev):
    """The block is one graph for torch.compile, gradients and all."""
    x, gate, up, _ = make(dev)
    mlp = block_of(gate, up, dev)
    x.requires_grad_(True)
    y = torch.compile(mlp, backend="aot_eager", fullgraph=True)(x)
    want = mlp(x)
    close(y.detach(), want.detach())
    gy = torch.randn_like(y)
    leaves = [x, *mlp.parameters()]
    for a, b in zip(torch.autograd.grad(y, leaves, gy), torch.autograd.grad(want, leaves, gy)):
        close(a, b)


class Held(torch.Tensor):
    """A tensor that holds another one, itself without memory."""

    @staticmethod
    def __new__(cls, t):
        r = torch.Tensor._make_wrapper_subclass(cls, t.shape, dtype=t.dtype, device=t.device, requires_grad=False)
        r.held = t
        return r

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        def bare(v):
            return v.held if isinstance(v, Held) else v
        r = func(*torch.utils._pytree.tree_map(bare, args), **torch.utils._pytree.tree_map(bare, kwargs or {}))
        return Held(r) if func is torch.ops.aten.detach.default else r


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("which", ["gate", "up", "both"])
def test_weights_of_another_class(dev, which, dtype):
    x, gate, up, _ = make(dev, dtype=dtype)
    want = swiglu(F.linear(x, gate.weight), F.linear(x, up.weight)).detach()
    for name, lin in (("gate", gate), ("up", up)):
        if which in (name, "both"):
            lin.weight = nn.Parameter(Held(lin.weight.detach()), requires_grad=False)
        else:
            lin.weight.requires_grad_(False)
    with torch.no_grad():
        assert torch.equal(gated_linear(x, gate, up), want)
    assert torch.equal(gated_linear(x, gate, up), want)
