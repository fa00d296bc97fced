"""Layer norm and the gradients of layer norm and RMS norm against 64-bit formulas."""
import pytest
import torch

from latest_exact_match_attention_amd.model import layer_norm, rms_norm

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
E = 2.0 ** -24
# Sums over a row go through at most 32 elements of a lane, 6 steps of a wavefront and 16
# wavefronts, so 54 additions and two roundings of each product, and a handful for rsqrt and scaling
K = 80


def make(dev, shape, dtype, center, seed=0, affine=True):
    g = torch.Generator(device=dev).manual_seed(seed)
    D = shape[-1]
    kw = dict(eps=1e-5, elementwise_affine=affine, device=dev, dtype=dtype)
    norm = torch.nn.LayerNorm(D, **kw) if center else torch.nn.RMSNorm(D, **kw)
    rand = lambda *s: torch.randn(s, device=dev, generator=g)  # noqa: E731
    with torch.no_grad():
        for p in norm.parameters():
            p.copy_(rand(D) * 0.5 + 0.5)
    x, d, gh, gs = (rand(*shape).to(dtype) for _ in range(4))
    x = (x.float() * 1.5 + 0.7).to(dtype)
    return norm, x, d, gh, gs


def close(got, want, slack):
    u = torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
    bad = (got.double() - want).abs() > u * (want.abs() + slack) + slack + tiny
    assert not bool(bad.any()), int(bad.sum())


def check(norm, center, s, gh, gs, h=None, gx=None, gw=None, gb=None):
    """Each output against the definition; the slack follows the errors of the mean (m), the
    factor (r) and the normalised row (z) through the formulas, K roundings each."""
    D = s.shape[-1]
    s, gh = s.double().view(-1, D), gh.double().view(-1, D)
    w = norm.weight.detach().double() if norm.weight is not None else torch.ones(D, device=s.device).double()
    m = s.mean(-1, keepdim=True) if center else 0.0
    r = torch.rsqrt((s - m).square().mean(-1, keepdim=True) + norm.eps)
    z = (s - m) * r
    amp = r * s.abs().mean(-1, keepdim=True) if center else 0.0
    dz = z.abs() + amp                                   # z's error, in units of K E
    if h is not None:
        b = norm.bias.detach().double() if center and norm.bias is not None else 0.0 * w
        close(h.view(-1, D), z * w + b, K * E * (dz * w.abs() + b.abs()))
    a = gh * w
    if gx is not None:
        c1 = a.mean(-1, keepdim=True) if center else 0.0
        c2 = (a * z).mean(-1, keepdim=True)
        want = r * (a - c1 - z * c2)
        mean_a = a.abs().mean(-1, keepdim=True)
        slack = 2 * K * E * r * (a.abs() + mean_a + dz * (a * z).abs().mean(-1, keepdim=True)
                                 + z.abs() * (a.abs() * dz).mean(-1, keepdim=True))
        if gs is not None:
            want = want + gs.double().view(-1, D)
            slack = slack + E * (gs.double().view(-1, D).abs() + want.abs())
        close(gx.view(-1, D), want, slack)
    rows = s.shape[0]
    if gw is not None:
        close(gw, (gh * z).sum(0), E * (K * (gh.abs() * dz).sum(0) + (rows + 64) * (gh * z).abs().sum(0)))
    if gb is not None:
        close(gb, gh.sum(0), E * (rows + 64) * gh.abs().sum(0))


# widths of every number of wavefronts and steps, their ends, and odd ones
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [1, 3, 8, 65, 512, 513, 1000, 1024, 1536, 1537, 2048, 2049, 4096, 4104,
                               8191, 8192, 8200, 16384])
def test_layer_norm(dev, dtype, D):
    norm, x, d, gh, gs = make(dev, (5, 7, D), dtype, True, seed=D)
    x.requires_grad_(True), d.requires_grad_(True)
    h, s = layer_norm(x, norm, d)
    assert torch.equal(s, x + d)
    gx, gd, gw, gb = torch.autograd.grad([h, s], [x, d, norm.weight, norm.bias], [gh, gs])
    assert torch.equal(gx, gd)
    check(norm, True, s.detach(), gh, gs, h.detach(), gx, gw, gb)
    h, same = layer_norm(x, norm)
    assert same is x
    gx, gw, gb = torch.autograd.grad(h, [x, norm.weight, norm.bias], gh)
    check(norm, True, x.detach(), gh, None, h.detach(), gx, gw, gb)


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 63, 4097, 9000])
@pytest.mark.parametrize("D", [24, 1544, 2056])
def test_row_counts(dev, rows, D):
    """From one row to more than the workgroups take in one turn."""
    norm, x, d, gh, gs = make(dev, (rows, D), torch.bfloat16, True, seed=rows)
    x.requires_grad_(True), d.requires_grad_(True)
    h, s = layer_norm(x, norm, d)
    gx, gw, gb = torch.autograd.grad([h, s], [x, norm.weight, norm.bias], [gh, gs])
    check(norm, True, s.detach(), gh, gs, h.detach(), gx, gw, gb)


@pytest.mark.parametrize("D", [1530, 1528])
@pytest.mark.parametrize("start", [0, 1])
def test_rows_past_the_cache(dev, D, start):
    """Tensors of more than 128 MB, from any element on: every row as in calls of a few."""
    rows = 44001
    norm, x, _, gh, _ = make(dev, (rows * D + 8,), torch.bfloat16, True, seed=D)
    norm, *_ = make(dev, (1, D), torch.bfloat16, True, seed=D)
    x, gh = (t[start:start + rows * D].view(rows, D) for t in (x, gh))
    leaf = x.detach().requires_grad_(True)
    h, _ = layer_norm(leaf, norm)
    (gx,) = torch.autograd.grad(h, [leaf], gh)
    for i in range(0, rows, 11000):
        part = x[i:i + 11000].detach().requires_grad_(True)
        want, _ = layer_norm(part, norm)
        assert torch.equal(h[i:i + 11000], want)
        assert torch.equal(gx[i:i + 11000], torch.autograd.grad(want, [part], gh[i:i + 11000])[0])


def test_more_rows_than_one_grid_dimension(dev):
    """Short rows, 8.4 million of them: every one as in a call of a few."""
    norm, x, _, gh, _ = make(dev, (4099, 8), torch.bfloat16, True, seed=8)
    n = 2047
    small, _ = layer_norm(x, norm)
    xs = x.repeat(n, 1).requires_grad_(True)
    h, _ = layer_norm(xs, norm)
    assert torch.equal(h.detach().view(n, 4099, 8), small.detach().expand(n, -1, -1))
    x.requires_grad_(True)
    (want,) = torch.autograd.grad(layer_norm(x, norm)[0], [x], gh)
    (gx,) = torch.autograd.grad(h, [xs], gh.repeat(n, 1))
    assert torch.equal(gx.view(n, 4099, 8), want.expand(n, -1, -1))


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,D", [(1, 8), (3, 512), (70, 520), (5000, 1536), (33, 2048), (9, 2056),
                                    (600, 4096)])
def test_rms_norm_gradient(dev, residual, rows, D):
    norm, x, d, gh, gs = make(dev, (rows, D), torch.bfloat16, False, seed=rows + D)
    x.requires_grad_(True), d.requires_grad_(True)
    add, gsum = (d, gs) if residual else (None, None)
    h, s = rms_norm(x, norm, add)
    with torch.no_grad():
        h0, s0 = rms_norm(x, norm, add)
    assert torch.equal(h, h0) and torch.equal(s, s0)         # the values of a call without gradients
    gx, gw = torch.autograd.grad([h, s] if residual else h, [x, norm.weight],
                                 [gh, gs] if residual else gh)
    check(norm, False, s.detach(), gh, gsum, None, gx, gw)


def test_no_affine_and_one_output(dev):
    norm, x, d, gh, gs = make(dev, (40, 96), torch.float32, True, affine=False)
    x.requires_grad_(True), d.requires_grad_(True)
    h, s = layer_norm(x, norm, d)
    (gx,) = torch.autograd.grad(h, [x], gh, retain_graph=True)
    check(norm, True, s.detach(), gh, None, h.detach(), gx)
    (gd,) = torch.autograd.grad(s, [d], gs)                  # only the sum is used
    assert torch.equal(gd, gs)
    only_bias = torch.nn.LayerNorm(96, device=dev)
    only_bias.weight = None
    h, _ = layer_norm(x.detach(), only_bias)
    (gb,) = torch.autograd.grad(h, [only_bias.bias], gh)
    check(only_bias, True, x.detach(), gh, None, h.detach(), gb=gb)


def test_layouts(dev):
    """Transposed and odd-offset inputs, an expanded gradient, a norm over two dims, no rows."""
    norm, x, d, gh, gs = make(dev, (30, 40, 72), torch.bfloat16, True)
    xt = x.transpose(0, 1).requires_grad_(True)
    h, s = layer_norm(xt, norm, d.transpose(0, 1))
    gx, gw, gb = torch.autograd.grad(h, [xt, norm.weight, norm.bias], gh.transpose(0, 1))
    t = lambda v: v.transpose(0, 1).contiguous()  # noqa: E731
    check(norm, True, (x + d).transpose(0, 1).contiguous(), t(gh), None, h.detach().contiguous(),
          gx.contiguous(), gw, gb)
    flat = torch.randn(1 + 50 * 72, device=dev).bfloat16()
    off = flat[1:].view(50, 72).requires_grad_(True)         # rows that start 2 bytes off
    h, _ = layer_norm(off, norm)
    gx, gw, gb = torch.autograd.grad(h.sum(), [off, norm.weight, norm.bias])
    check(norm, True, off.detach(), torch.ones(50, 72, device=dev), None, h.detach(), gx, gw, gb)
    two = torch.nn.LayerNorm((6, 12), device=dev, dtype=torch.bfloat16)
    h, _ = layer_norm(flat[1:].view(50, 6, 12), two)
    gw, gb = torch.autograd.grad(h.sum(), [two.weight, two.bias])
    assert gw.shape == gb.shape == (6, 12) and bool((gb == 50).all())
    h, _ = layer_norm(x[:0].requires_grad_(True), norm)
    gx, gw, gb = torch.autograd.grad(h.sum(), [h, norm.weight, norm.bias], allow_unused=True)
    assert not gw.any() and not gb.any()


def test_values_out_of_range(dev):
    """An infinity or NaN stays in its row; a constant row normalises to the bias; a row far from
    zero keeps its variance."""
    norm, x, _, gh, _ = make(dev, (8, 136), torch.float32, True)
    x[1, 5], x[2, 7], x[3] = float("inf"), float("nan"), 3.25
    x[4] = 4096.0 + torch.arange(136, device=dev) / 64       # exact in fp32
    x.requires_grad_(True)
    h, _ = layer_norm(x, norm)
    (gx,) = torch.autograd.grad(h, [x], gh)
    bad = torch.tensor([1, 2], device=dev)
    assert bool(h[bad].isnan().all()) and bool(gx[bad].isnan().all())
    ok = torch.tensor([0, 3, 4, 5, 6, 7], device=dev)
    assert torch.equal(h[3], norm.bias)
    check(norm, True, x.detach()[ok], gh[ok], None, h.detach()[ok], gx[ok])


def test_differences(dev):
    """The gradient along a direction against a central difference of the kernel's own forward in
    fp32: a step of 2^-6 leaves a third-order error of 2^-12 relative to the direction's third
    derivative (at most 8 r^3 |h|...: bounded here by 16), and roundings of 80 E / 2^-6 a term."""
    norm, x, _, gh, _ = make(dev, (6, 200), torch.float32, True)
    v = torch.randn(6, 200, device=dev)
    x.requires_grad_(True)
    h, _ = layer_norm(x, norm)
    (gx,) = torch.autograd.grad(h, [x], gh)
    with torch.no_grad():
        t = 2.0 ** -6
        up, dn = (layer_norm(x + k * t * v, norm)[0].double() for k in (1, -1))
        diff = ((up - dn) / (2 * t) * gh).sum(-1)
        got = (gx.double() * v).sum(-1)
        size = (gh.abs().double() * (norm.weight.abs() + norm.bias.abs() + 1)).sum(-1)
    assert bool(((diff - got).abs() <= size * (16 * t * t + 2 * 80 * E * 4 / t)).all())


def test_hooks_and_retained(dev):
    norm, x, d, gh, gs = make(dev, (300, 264), torch.bfloat16, True)
    x.requires_grad_(True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.double().cpu(), lambda t: t):
        h, s = layer_norm(x, norm, d)
    a = torch.autograd.grad([h, s], [x, norm.weight], [gh, gs], retain_graph=True)
    b = torch.autograd.grad([h, s], [x, norm.weight], [torch._neg_view(-gh), gs])
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_captured_step(dev):
    """Forward and gradients in a graph. No eager graph of the same leaves is alive meanwhile: torch
    would order the captured gradients after that graph's stream, which a capture cannot."""
    norm, x, d, gh, gs = make(dev, (300, 264), torch.bfloat16, True)
    x.requires_grad_(True)

    def step():
        h, s = layer_norm(x, norm, d)
        return torch.autograd.grad([h, s], [x, norm.weight, norm.bias], [gh, gs])
    st = torch.cuda.Stream(dev)
    st.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(st):
        step()
    torch.cuda.current_stream(dev).wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        gh.copy_(torch.randn_like(gh))
        want = step()
        for t in out:
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_refusals(dev):
    x = torch.randn(4, 16, device=dev)
    norm = torch.nn.LayerNorm(16, device=dev)
    with pytest.raises(ValueError, match="addend"):
        layer_norm(x, norm, x[:2])
    with pytest.raises(TypeError, match="addend"):
        layer_norm(x, norm, x.half())
    with pytest.raises(TypeError, match="weight"):
        layer_norm(x.half(), norm)
    with pytest.raises(ValueError, match="shape"):
        layer_norm(x[:, :8], norm)
    with pytest.raises(ValueError, match="16384"):
        layer_norm(torch.randn(1, 16385, device=dev), torch.nn.LayerNorm(16385, device=dev))
    with pytest.raises(ValueError, match="expected"):
        layer_norm(x, torch.nn.LayerNorm(16))
