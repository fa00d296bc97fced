"""The embedding lookup with a scale and its gradient by sorted tokens, against 64-bit sums."""
import pytest
import torch

from latest_exact_match_attention_amd import _lib
from latest_exact_match_attention_amd.model import embed

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def half_step(dtype):
    """A rounding's largest relative error, and fp16's largest absolute one below its normals."""
    return torch.finfo(dtype).eps / 2, (2.0 ** -25 if dtype == torch.float16 else 0.0)


def table(dev, V, D, dtype, seed=0, **kw):
    g = torch.Generator(device=dev).manual_seed(seed)
    w = torch.randn(V, D, device=dev, generator=g).to(dtype)
    return torch.nn.Embedding(V, D, _weight=w, **kw), g


def check_grad(gw, ids, gy, V, scale, padding=None):
    """gw against the definition in 64 bits. A sum of m fp32 terms is off by at most (m - 1) 2^-24
    of the terms' absolute sum whatever its order, the scale and its product by 2 2^-24 more, and
    the last rounding by half a step."""
    D = gy.shape[-1]
    ids, gy = ids.reshape(-1).long(), gy.reshape(-1, D).double()
    keep = (ids >= 0) & (ids < V)
    if padding is not None:
        keep &= ids != padding
    ids, gy = ids[keep], gy[keep]
    # running sums of the rows in the tokens' order (index_add_ in 64 bits takes minutes where
    # millions of positions hold one token: they wait for each other at its row)
    order = torch.argsort(ids, stable=True)
    m = torch.bincount(ids, minlength=V)[:, None]
    ends = m.cumsum(0)[:, 0]

    def sums(rows):
        run = torch.zeros(rows.shape[0] + 1, D, dtype=torch.float64, device=gw.device)
        torch.cumsum(rows[order], 0, out=run[1:])
        return run[ends] - run[ends - m[:, 0]]
    want, size = sums(gy * scale), sums(gy.abs() * abs(scale))
    u, tiny = half_step(gw.dtype)
    tol = u * want.abs() + (m + 3) * 2.0 ** -24 * size + tiny * (m > 0)
    # the running sums themselves are off by less than 2^-50 of all the rows' sum
    tol = tol + 2.0 ** -50 * gy.abs().sum() * abs(scale) / max(1, D)
    assert bool(((gw.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [1, 7, 8, 64, 511, 520, 1536])
def test_rows_and_scale(dev, dtype, D):
    emb, g = table(dev, 100, D, dtype)
    ids = torch.randint(0, 100, (3, 5), device=dev, generator=g)
    with torch.no_grad():
        assert torch.equal(embed(emb, ids), emb.weight[ids])
        got = embed(emb, ids.int(), 5.7)
        want = emb.weight[ids].double() * 5.7
        u, tiny = half_step(dtype)
        # the scale and the product in fp32, then the type's rounding
        assert bool(((got.double() - want).abs() <= (u + 2.0 ** -23) * want.abs() + tiny).all())


def test_rows_keep_their_bits(dev):
    emb, _ = table(dev, 16, 24, torch.bfloat16)
    bits = torch.randint(-2 ** 15, 2 ** 15, (16, 24), device=dev, dtype=torch.int16)
    with torch.no_grad():
        emb.weight.copy_(bits.view(torch.bfloat16))
        ids = torch.arange(16, device=dev)
        assert torch.equal(embed(emb, ids).view(torch.int16), emb.weight.view(torch.int16))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,V,D", [(1, 1, 1), (1, 5, 8), (70, 3, 24), (1000, 50, 33), (1025, 1024, 40),
                                   (1024, 1025, 512), (4097, 3001, 513), (16385, 50304, 64),
                                   (65536, 20000, 40), (70001, 131072, 8)])
def test_gradient(dev, dtype, n, V, D):
    """Tokens of very different frequencies: lists of none, one, up to 32 and far more rows."""
    emb, g = table(dev, V, D, dtype, seed=n)
    u = torch.rand(n, device=dev, generator=g)
    ids = torch.randperm(V, device=dev, generator=g)[((V + 1) ** u).long().clamp_(1, V) - 1]
    gy = torch.randn(n, D, device=dev, generator=g).to(dtype)
    (gw,) = torch.autograd.grad(embed(emb, ids, 1.5), [emb.weight], gy)
    check_grad(gw, ids, gy, V, 1.5)
    (again,) = torch.autograd.grad(embed(emb, ids, 1.5), [emb.weight], gy)
    assert torch.equal(gw, again)


@pytest.mark.parametrize("dtype,n,V,D", [(torch.bfloat16, 3000, 700, 2048), (torch.float32, 2500, 40, 4096),
                                         (torch.float16, 20000, 90, 1541), (torch.bfloat16, 3000, 1 << 20, 8),
                                         (torch.float32, 900, (1 << 20) + 1, 8),
                                         (torch.bfloat16, 1_200_000, 50304, 8),
                                         (torch.float16, 17_000_001, 3000, 8)])
def test_gradient_of_the_largest(dev, dtype, n, V, D):
    """Rows of more slices than a wavefront takes, the largest table (and one past it, which
    nn.Embedding's own gradient takes), and more positions than 64 and than 1024 spans hold."""
    emb, g = table(dev, V, D, dtype, seed=n)
    u = torch.rand(n, device=dev, generator=g, dtype=torch.float64)
    ids = ((V + 1) ** u).long().clamp_(1, V) - 1
    ids[-1] = V - 1
    gy = torch.randn(n, D, device=dev, generator=g).to(dtype)
    (gw,) = torch.autograd.grad(embed(emb, ids), [emb.weight], gy)
    check_grad(gw, ids, gy, V, 1.0)


@pytest.mark.parametrize("n", [1, 33, 1024, 1025, 7167, 7168, 7169])
@pytest.mark.parametrize("V", [1, 700, 50304, 1 << 20])
def test_gradient_lengths_and_tables(dev, n, V):
    """Around the lengths where the order is found another way, with every number of tokens a bucket,
    frequent tokens at both ends of the table, ids outside it and a padding token."""
    emb, g = table(dev, V, 24, torch.float32, seed=n, padding_idx=V // 2)
    u = torch.rand(n, device=dev, generator=g, dtype=torch.float64)
    ids = (V ** u).long().clamp_(1, V) - 1
    ids[::3] = V - 1 - ids[::3]
    ids[5::17] = V
    ids[7::29] = -1
    gy = torch.randn(n, 24, device=dev, generator=g)
    (gw,) = torch.autograd.grad(embed(emb, ids), [emb.weight], gy)
    check_grad(gw, ids, gy, V, 1.0, V // 2)
    assert torch.equal(gw, torch.autograd.grad(embed(emb, ids), [emb.weight], gy)[0])


@pytest.mark.parametrize("half", [520, 515])
def test_rows_past_the_cache(dev, half):
    """Rows and a table of more than 256 MB: the columns as in calls of half of them."""
    n, V, D = 100001, 32003, 2 * half
    emb, g = table(dev, V, D, torch.bfloat16, seed=half)
    ids = (torch.rand(n, device=dev, generator=g) ** 3 * V).long()
    gy = torch.randn(n, D, device=dev, generator=g).to(torch.bfloat16)
    y = embed(emb, ids)
    assert torch.equal(y, emb.weight[ids])
    (gw,) = torch.autograd.grad(y, [emb.weight], gy)
    for cols in (slice(0, half), slice(half, D)):
        part = torch.nn.Embedding(V, half, _weight=emb.weight.detach()[:, cols].contiguous())
        (want,) = torch.autograd.grad(embed(part, ids), [part.weight], gy[:, cols])
        assert torch.equal(gw[:, cols], want)


def test_more_positions_than_one_grid_dimension(dev):
    emb, g = table(dev, 300, 8, torch.bfloat16, seed=5)
    ids = torch.randint(0, 300, ((1 << 23) + 5,), device=dev, generator=g)
    with torch.no_grad():
        assert torch.equal(embed(emb, ids), emb.weight[ids])


@pytest.mark.parametrize("n", [31, 32, 33, 63, 64, 65, 97, 127, 128, 200, 5000, 40000])
def test_gradient_one_token(dev, n):
    """Every position the same token: lists around the longest that one wavefront adds up."""
    emb, g = table(dev, 9, 72, torch.float32)
    gy = torch.randn(n, 72, device=dev, generator=g)
    ids = torch.full((n,), 4, device=dev)
    ids[: n // 3] = 3                 # the long list starts inside a tile
    (gw,) = torch.autograd.grad(embed(emb, ids), [emb.weight], gy)
    check_grad(gw, ids, gy, 9, 1.0)


def test_gradient_padding_and_strangers(dev):
    """The padding token and ids outside the table get and give nothing; no ids at all, too."""
    emb, g = table(dev, 300, 16, torch.bfloat16, padding_idx=7)
    ids = torch.randint(-20, 320, (40, 50), device=dev, generator=g)
    ids[:, 20:] = 7
    gy = torch.randn(40, 50, 16, device=dev, generator=g).bfloat16()
    y = embed(emb, ids)
    assert bool((y[(ids < 0) | (ids >= 300)] == 0).all())
    (gw,) = torch.autograd.grad(y, [emb.weight], gy)
    check_grad(gw, ids, gy, 300, 1.0, padding=7)
    y = embed(emb, ids[:0])
    assert y.shape == (0, 50, 16)
    (gw,) = torch.autograd.grad(y, [emb.weight], torch.empty_like(y))
    assert not gw.any()


def test_gradient_of_a_sum_and_of_differences(dev):
    """An expanded gradient, and the directional derivative as a difference (the lookup is linear
    in the table, so a difference is exact but for rounding: 2 n D roundings of 2^-24 of the
    terms' sum)."""
    emb, g = table(dev, 60, 12, torch.float32)
    ids = torch.randint(0, 60, (500,), device=dev, generator=g)
    (gw,) = torch.autograd.grad(embed(emb, ids, 3.0).sum(), [emb.weight])
    check_grad(gw, ids, torch.ones(500, 12, device=dev), 60, 3.0)
    step = torch.randn(60, 12, device=dev, generator=g)
    with torch.no_grad():
        a = embed(emb, ids, 3.0).double().sum()
        moved = torch.nn.Embedding(60, 12, _weight=(emb.weight + step))
        b = embed(moved, ids, 3.0).double().sum()
        size = 3 * (emb.weight.abs() + step.abs())[ids].double().sum()
    assert abs(float(b - a - (gw.double() * step).sum())) <= float(size) * 500 * 2.0 ** -24


def test_gradient_deterministic_hooks_and_retained(dev):
    emb, g = table(dev, 500, 40, torch.float16)
    ids = torch.randint(0, 500, (3000,), device=dev, generator=g)
    gy = torch.randn(3000, 40, device=dev, generator=g).half()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu().short() if t.dtype == torch.long
                                                  else t, lambda t: t):
        y = embed(emb, ids)
    (a,) = torch.autograd.grad(y, [emb.weight], gy, retain_graph=True)
    (b,) = torch.autograd.grad(y, [emb.weight], torch._neg_view(-gy))
    assert torch.equal(a, b)
    check_grad(a, ids, gy, 500, 1.0)
    with pytest.raises(RuntimeError):
        y = embed(emb, ids)
        (a,) = torch.autograd.grad(y, [emb.weight], gy.clone().requires_grad_(), create_graph=True)
        a.sum().backward()


def test_torch_paths(dev):
    """Tables that nn.Embedding treats specially keep its operations."""
    ids = torch.tensor([1, 1, 2], device=dev)
    for kw in (dict(max_norm=0.5), dict(sparse=True), dict(scale_grad_by_freq=True)):
        emb, _ = table(dev, 10, 8, torch.float32, **kw)
        (gw,) = torch.autograd.grad(embed(emb, ids, 2.0).sum(), [emb.weight])
        w = torch.nn.Embedding(10, 8, _weight=emb.weight.detach().clone(), **kw)
        (want,) = torch.autograd.grad((w(ids) * 2.0).sum(), [w.weight])
        assert gw.is_sparse == want.is_sparse
        assert torch.equal(gw.to_dense() if gw.is_sparse else gw, want.to_dense() if want.is_sparse else want)


def test_captured_step(dev):
    """Lookup and gradient in a graph, replayed with other tokens and other eager work between."""
    emb, g = table(dev, 700, 48, torch.bfloat16)
    draw = lambda: torch.randint(0, 700, (2000,), device=dev, generator=g)  # noqa: E731
    ids, gy = draw(), torch.randn(2000, 48, device=dev, generator=g).bfloat16()
    step = lambda: torch.autograd.grad(embed(emb, ids, 2.0), [emb.weight], gy)[0]  # noqa: E731
    s = torch.cuda.Stream(dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream(dev).wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gw = step()
    for _ in range(4):
        ids.copy_(draw())
        want = step()
        gw.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(gw, want)


def test_workspace_refusals(dev):
    L = _lib.lib()
    x = torch.zeros(64, 8, device=dev)
    ids = torch.zeros(64, dtype=torch.long, device=dev)
    n = L.lema_embedding_grad_workspace_bytes(64, 10, 8)
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    call = lambda w, size: L.lema_embedding_grad(  # noqa: E731
        x.data_ptr(), 0, ids.data_ptr(), 64, 10, 8, 1.0, -1, x.data_ptr(), w, size, None)
    assert call(ws.data_ptr(), n - 1) == _lib.BAD_ARG and call(None, n) == _lib.BAD_ARG
    assert call(ws.data_ptr() + 8, n) == _lib.BAD_ARG
