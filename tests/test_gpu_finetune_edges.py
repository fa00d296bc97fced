"""The model's functions in fine-tuning where a call leaves the ordinary: gradients and saved tensors at
any address."""
import pytest
import torch

from latest_exact_match_attention_amd.model import swiglu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("start", [1, 4, 8])
def test_swiglu_gradient_at_any_address(dev, start):
    """An upstream gradient, or a saved tensor that a hook brings back, that is a slice of a larger
    tensor: the same gradients as from tensors of their own."""
    torch.manual_seed(start)
    g, u, gy = (torch.randn(6, 40, device=dev).bfloat16() for _ in range(3))
    g.requires_grad_(True), u.requires_grad_(True)

    def moved(t):
        flat = torch.empty(t.numel() + start, device=dev, dtype=t.dtype)
        flat[start:] = t.detach().reshape(-1)
        return flat[start:].view(t.shape)
    want = torch.autograd.grad(swiglu(g, u), [g, u], gy)
    got = torch.autograd.grad(swiglu(g, u), [g, u], moved(gy))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    head = torch.zeros(start, device=dev, dtype=torch.bfloat16, requires_grad=True)
    joined = torch.cat([head, swiglu(g, u).reshape(-1)])
    got = torch.autograd.grad(joined, [g, u], torch.cat([head, gy.reshape(-1)]).detach())
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.autograd.graph.saved_tensors_hooks(moved, lambda t: t):
        y = swiglu(g, u)
    got = torch.autograd.grad(y, [g, u], gy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
