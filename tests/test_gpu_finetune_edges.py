"""The model's functions in fine-tuning where a call leaves the ordinary: gradients and saved tensors at
any address, caches, shapes, modules that do more than they are named for."""
import pytest
import torch
from test_gpu_finetune import build, loss_of, plain, record_matches

from latest_exact_match_attention_amd.loss import policy_loss, preference_loss, token_logprobs
from latest_exact_match_attention_amd.model import cross_entropy_sum, embed, layer_norm, linear, lm_loss, rms_norm, swiglu

pytestmark = pytest.mark.gpu


def moved(t, start=1):
    """t as a slice of a larger tensor."""
    flat = torch.empty(t.numel() + start, device=t.device, dtype=t.dtype)
    flat[start:] = t.detach().reshape(-1)
    return flat[start:].view(t.shape)


@pytest.mark.parametrize("start", [1, 4, 8])
def test_swiglu_gradient_at_any_address(dev, start):
    """An upstream gradient, or a saved tensor that a hook brings back, that is a slice of a larger
    tensor: the same gradients as from tensors of their own."""
    torch.manual_seed(start)
    g, u, gy = (torch.randn(6, 40, device=dev).bfloat16() for _ in range(3))
    g.requires_grad_(True), u.requires_grad_(True)
    want = torch.autograd.grad(swiglu(g, u), [g, u], gy)
    got = torch.autograd.grad(swiglu(g, u), [g, u], moved(gy, start))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    head = torch.zeros(start, device=dev, dtype=torch.bfloat16, requires_grad=True)
    joined = torch.cat([head, swiglu(g, u).reshape(-1)])
    got = torch.autograd.grad(joined, [g, u], torch.cat([head, gy.reshape(-1)]).detach())
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: moved(t, start), lambda t: t):
        y = swiglu(g, u)
    got = torch.autograd.grad(y, [g, u], gy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_saved_tensors_at_any_address(dev):
    """Every operator's gradients with saved tensors that a hook brings back as slices."""
    torch.manual_seed(3)
    x = torch.randn(4, 3, 64, device=dev).bfloat16().requires_grad_(True)
    t, z = torch.randint(0, 64, (4, 3), device=dev), torch.full((4, 3), -4.0, device=dev)
    mask = torch.rand(4, 3, device=dev) < 0.7
    norm, rms = (n(64, device=dev, dtype=torch.bfloat16) for n in (torch.nn.LayerNorm, torch.nn.RMSNorm))
    emb = torch.nn.Embedding(70, 64, device=dev, dtype=torch.bfloat16)
    cases = {
        "logprobs": (lambda: token_logprobs(x, t, mask).sum(), [x]),
        "policy": (lambda: 2.0 * policy_loss(x, t, z, z + 5, z, mask, kl_weight=0.1).loss, [x]),
        "preference": (lambda: preference_loss(x, t, z, mask).loss, [x]),
        "cross entropy": (lambda: cross_entropy_sum(x, t), [x]),
        "layer norm": (lambda: layer_norm(x, norm)[0].square().sum(), [x, norm.weight, norm.bias]),
        "rms norm": (lambda: rms_norm(x, rms, x * 2)[0].square().sum(), [x, rms.weight]),
        "embed": (lambda: embed(emb, t, 3.0).square().sum(), [emb.weight])}
    for name, (f, leaves) in cases.items():
        want = torch.autograd.grad(f(), leaves)
        with torch.autograd.graph.saved_tensors_hooks(moved, lambda s: s):
            y = f()
        got = torch.autograd.grad(y, leaves)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), name


@pytest.mark.parametrize("T", [1, 9, 40])
def test_cached_logits_have_no_graph(dev, T):
    """With a cache nothing has a gradient: no graph that ends at the final norm and head, whose
    backward would fill two parameters and leave the others out without a word."""
    model, _ = build(dev, 4)
    idx = torch.randint(0, 200, (2, T), device=dev)
    out = []
    for ctx in (torch.no_grad(), torch.enable_grad()):
        with ctx:
            cache = model.new_cache("hbm", max_cache_len=64, batch=2)
            out.append(model(idx, cache=cache))
            assert not out[-1].requires_grad and cache.t == T
    assert torch.equal(*out)
    assert model(idx).requires_grad


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [20, 4104, 64])
@pytest.mark.parametrize("affine", [True, False])
def test_rms_norm_adds_the_addend(dev, dtype, D, affine):
    """Also for rows that the kernel does not take, and without a weight. Both sides round s = x + d
    once; the norm's factors and product in fp32 are 16 roundings off, then its own rounding."""
    torch.manual_seed(D)
    x, d = (torch.randn(5, D, device=dev).to(dtype).requires_grad_(True) for _ in range(2))
    norm = torch.nn.RMSNorm(D, eps=1e-5, elementwise_affine=affine, device=dev, dtype=dtype)
    h, s = rms_norm(x, norm, d)
    assert torch.equal(s, x + d)
    t = s.detach().double()
    want = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-5)
    u = torch.finfo(dtype).eps / 2
    # torch's own norm rounds the normalised row before the weight, too
    assert bool(((h.double() - want).abs() <= (2 * u + 16 * 2.0 ** -24 + D * 2.0 ** -25) * want.abs()).all())
    gx, gd = torch.autograd.grad(h.float().square().sum(), [x, d])
    assert torch.equal(gx, gd) and bool(gx.isfinite().all())


def test_shapes_that_do_not_match(dev):
    """What torch broadcasts is broadcast, and what it refuses is refused: no kernel reads or writes
    by the first argument's size alone."""
    torch.manual_seed(5)
    x = torch.randn(6, 64, device=dev).bfloat16().requires_grad_(True)
    d = torch.randn(64, device=dev).bfloat16().requires_grad_(True)
    norm = torch.nn.RMSNorm(64, device=dev, dtype=torch.bfloat16)
    h, s = rms_norm(x, norm, d)
    assert torch.equal(s, x + d) and torch.equal(h, norm(x + d))
    assert torch.autograd.grad(h.float().square().sum(), [d])[0].shape == d.shape
    wide = torch.nn.RMSNorm((6, 64), device=dev, dtype=torch.bfloat16)
    assert torch.equal(rms_norm(x, wide)[0], wide(x))
    with pytest.raises(RuntimeError):
        rms_norm(x, torch.nn.RMSNorm(32, device=dev, dtype=torch.bfloat16))
    y = swiglu(x, d)
    assert torch.equal(y, torch.nn.functional.silu(x) * d)
    assert torch.autograd.grad(y.float().sum(), [d])[0].shape == d.shape
    with pytest.raises(RuntimeError):
        swiglu(x, d[:32])
    t = torch.zeros(6, dtype=torch.long, device=dev)
    for wrong in (t[:4], torch.cat([t, t])):
        with pytest.raises(ValueError):
            cross_entropy_sum(x, wrong)
    with pytest.raises(RuntimeError):
        cross_entropy_sum(x, t.cpu())
    with pytest.raises(RuntimeError):
        linear(x, torch.nn.Linear(96, 8, bias=False, device=dev, dtype=torch.bfloat16))


class Doubled(torch.nn.Embedding):
    def forward(self, ids):
        return 2 * super().forward(ids)


class Wrapped(torch.nn.Module):
    """An embedding without a table of its own."""

    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    def forward(self, ids):
        return 2 * self.inner(ids)


def doubled_by(kind, emb):
    """emb, or what stands for it, with rows twice as large, and what takes that back."""
    if kind == "subclass":
        return Doubled(*emb.weight.shape, _weight=emb.weight.detach().clone()), lambda: None
    if kind == "wrapper":
        return Wrapped(emb), lambda: None
    if kind == "own forward":
        plain = emb.forward
        emb.forward = lambda ids: 2 * plain(ids)
        return emb, lambda: None
    if kind == "hook":
        return emb, emb.register_forward_hook(lambda m, i, o: 2 * o).remove
    if kind == "pre-hook":                       # the other half of the table holds the doubled rows
        with torch.no_grad():
            emb.weight[128:] = 2 * emb.weight[:128]
        return emb, emb.register_forward_pre_hook(lambda m, i: (i[0] + 128,)).remove
    every = torch.nn.modules.module.register_module_forward_hook
    return emb, every(lambda m, i, o: 2 * o if m is emb else None).remove


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", ["subclass", "wrapper", "own forward", "hook", "pre-hook", "global hook"])
@pytest.mark.parametrize("B,T", [(2, 9), (4, 600)])
def test_embedding_modules_are_called(dev, dtype, kind, B, T):
    """Hooks and forwards of an embedding run in training as they do without gradients, in the
    function and in the model."""
    model, _ = build(dev, 6)
    model.to(dtype)
    idx = torch.randint(0, 128, (B, T), device=dev)
    rows = model.tok_emb.weight.detach()[idx]
    model.tok_emb, undo = doubled_by(kind, model.tok_emb)
    try:
        assert torch.equal(embed(model.tok_emb, idx), 2 * rows)
        assert torch.equal(embed(model.tok_emb, idx, 3.0), 2 * rows * 3.0)
        with torch.no_grad():
            assert torch.equal(embed(model.tok_emb, idx), 2 * rows)
        seen = []
        handle = model.blocks[0].register_forward_pre_hook(lambda m, i: seen.append(i[0].detach()))
        assert model(idx).requires_grad and model.hidden(idx).requires_grad
        handle.remove()
        assert len(seen) == 2 and all(torch.equal(x, 2 * rows) for x in seen)
    finally:
        undo()


def test_backward_hooks_of_an_embedding(dev):
    model, _ = build(dev, 7)
    idx = torch.randint(0, 200, (4, 600), device=dev)
    seen = []
    model.tok_emb.register_full_backward_hook(lambda m, gi, go: seen.append(go[0].shape))
    model(idx).float().square().sum().backward()
    assert seen == [(4, 600, 64)]


def test_embedding_gradients_compose(dev):
    """A graph of the backward of a model in fp32: as from the embedding module's own gradient, which
    a hook that does nothing brings about. The two add a token's rows up in other orders: some 40
    of them, each sum off by 40 2^-24 of its terms, whose sum a cancellation leaves a fifth of."""
    model, _ = build(dev, 8)
    model.float()
    idx = torch.randint(0, 200, (4, 600), device=dev)
    w = model.tok_emb.weight
    v = torch.randn(w.shape, device=dev, generator=torch.Generator(dev).manual_seed(1))

    def products():
        y = model.hidden(idx)
        (g,) = torch.autograd.grad(y.square().sum(-1).sqrt().mean(), [w], create_graph=True)
        (hv,) = torch.autograd.grad((g * v).sum(), [w])
        return g.detach(), hv
    got = products()
    handle = model.tok_emb.register_forward_hook(lambda m, i, o: None)
    want = products()
    handle.remove()
    for a, b in zip(got, want):
        assert float((a - b).norm()) <= 2 * 5 * 40 * 2.0 ** -24 * float(b.norm()) and bool(b.any())


@pytest.mark.parametrize("dtype,scale,pad", [(torch.float32, 1.0, None), (torch.bfloat16, 3.0, 5)])
def test_embedding_gradients_in_batches(dev, dtype, scale, pad):
    """Each as the gradient alone."""
    torch.manual_seed(9)
    ids = torch.randint(-3, 203, (300,), device=dev)
    emb = torch.nn.Embedding(200, 24, padding_idx=pad, device=dev, dtype=dtype)
    y = embed(emb, ids, scale)
    gy = torch.randn(3, *y.shape, device=dev).to(dtype)
    (many,) = torch.autograd.grad(y, [emb.weight], gy, is_grads_batched=True, retain_graph=True)
    m, u = int(torch.bincount(ids.clamp_min(0)).max()), torch.finfo(dtype).eps / 2
    for k in range(3):
        (one,) = torch.autograd.grad(y, [emb.weight], gy[k], retain_graph=True)
        # each side sums up to m products of at most scale max |gy| in fp32, and rounds once
        tol = 2 * m * 2.0 ** -24 * m * scale * float(gy.abs().max())
        assert bool(((many[k].double() - one.double()).abs() <= 2 * u * one.double().abs() + 2 * tol).all())
        assert pad is None or not many[k][pad].any()


@pytest.mark.parametrize("name", ["logprobs", "norm", "swiglu"])
def test_batched_gradients_are_refused(dev, name):
    """The other operators' gradients come one at a time, and say so."""
    x = torch.randn(4, 64, device=dev).bfloat16().requires_grad_(True)
    norm = torch.nn.LayerNorm(64, device=dev, dtype=torch.bfloat16)
    f = {"logprobs": lambda: token_logprobs(x, torch.zeros(4, dtype=torch.long, device=dev)),
         "norm": lambda: layer_norm(x, norm)[0], "swiglu": lambda: swiglu(x, x)}[name]
    y = f()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, [x], torch.ones(2, *y.shape, device=dev, dtype=y.dtype), is_grads_batched=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_short_lookups_keep_torchs_gradient(dev, dtype):
    """A model's lookup with its gradient is not slower than torch's two operations: those are kept
    below 2048 positions, whose gradient the sort makes no faster. Either gives the same rows."""
    model, _ = build(dev, 10)
    model.to(dtype)
    for B, T, sorts in ((1, 1, False), (3, 200, False), (1, 2047, False), (4, 512, True), (2, 1500, True)):
        idx = torch.randint(0, 200, (B, T), device=dev)
        y = model._embed(idx)
        assert ("ModelEmbed" in y.grad_fn.name()) == sorts
        assert torch.equal(y, model.tok_emb.weight[idx])
        with torch.no_grad():
            assert model._embed(idx).grad_fn is None


@pytest.mark.parametrize("kind", ["policy", "preference", "lm"])
def test_step_of_a_batch(dev, kind):
    """A step whose lookup takes the sorted gradient, every parameter's gradient within 7.9% in the
    Frobenius norm: some 100 roundings lie between a weight and the loss, forward and back, each of
    at most 2^-9 in bf16 and independent of the others, so that they add up as 10 2^-9, and four
    times that for the factors (norms, a softmax, random products) that stretch them. A part that is
    lost (a residual, a norm's mean, a factor of SwiGLU) takes 26% and more off one of them."""
    model, cfg = build(dev)
    B, T = 4, 600
    idx = torch.randint(0, 200, (B, T), device=dev, generator=torch.Generator(dev).manual_seed(T))
    targets = (idx * 7 + 3) % 200
    mask = torch.ones(B, T, dtype=torch.bool, device=dev)
    mask[0, : T // 3] = False
    matches = record_matches(model)
    z = torch.full((B, T), -5.0, device=dev)
    if kind == "lm":
        loss = lm_loss(model, idx, targets, chunk=128)
    elif kind == "policy":
        adv = torch.linspace(-1, 1, B * T, device=dev).view(B, T)
        loss = policy_loss(model(idx), targets, z, adv, mask=mask, clip_low=1.0, clip_high=1e9).loss
    else:
        loss = preference_loss(model(idx), targets, z, mask).loss
    names = [n for n, _ in model.named_parameters()]
    grads = torch.autograd.grad(loss, list(model.parameters()), allow_unused=True)
    logits, w = plain(model, idx, matches)
    want = torch.autograd.grad(loss_of(kind, logits, targets, mask), [w[n] for n in names], allow_unused=True)
    for n, g, r in zip(names, grads, want):
        if "q_proj" in n or "k_proj" in n:
            assert g is None and r is None
        else:
            off = float((g.double() - r).norm() / r.norm())
            assert off <= 4 * 10 * 2.0 ** -9, (n, off)


def test_inputs_at_any_address(dev):
    """Activations and weights that are slices of larger tensors, with their gradients: torch's
    operations take what the fused kernels do not."""
    torch.manual_seed(11)
    x, d, u = (moved(torch.randn(40, 64, device=dev).bfloat16()).requires_grad_(True) for _ in range(3))
    norm = torch.nn.RMSNorm(64, device=dev, dtype=torch.bfloat16)
    norm.weight = torch.nn.Parameter(moved(torch.rand(64, device=dev).bfloat16()))
    t = torch.randint(0, 64, (40,), device=dev)
    h, s = rms_norm(x, norm, d)
    assert torch.equal(s, x + d) and torch.equal(h, norm(x + d))
    assert torch.equal(swiglu(x, u), torch.nn.functional.silu(x) * u)
    loss = cross_entropy_sum(x, t)
    assert torch.equal(loss, torch.nn.functional.cross_entropy(x.float(), t, reduction="sum"))
    total = h.float().square().sum() + swiglu(x, u).float().sum() + loss
    assert all(bool(g.isfinite().all()) for g in torch.autograd.grad(total, [x, d, u, norm.weight]))
    # a model whose parameters lie in one flat buffer
    model, _ = build(dev, 12)
    idx = torch.randint(0, 200, (3, 40), device=dev)
    with torch.no_grad():
        want = model(idx)
        flat = torch.empty(1 + sum(p.numel() + 1 for p in model.parameters()), device=dev, dtype=torch.bfloat16)
        at = 1
        for p in model.parameters():
            flat[at:at + p.numel()] = p.reshape(-1)
            p.data = flat[at:at + p.numel()].view(p.shape)
            at += p.numel() + 1
        got = model(idx)
    # other kernels: a few roundings of bf16 a layer, which may turn a code's sign
    assert got.shape == want.shape and bool(got.isfinite().all())
    assert float(torch.autograd.grad(model(idx).float().square().mean(), [model.lm_head.weight])[0].norm()) > 0


@pytest.mark.parametrize("shape", [(5, 3, 20), (4, 24, 24), (20,), (6, 24)])
def test_cross_entropy_over_the_last_dim(dev, shape):
    """Whatever the type, length and address of the rows, the vocabulary is the last dim."""
    torch.manual_seed(13)
    x = torch.randn(*shape, device=dev)
    y = torch.randint(0, shape[-1], shape[:-1], device=dev)
    for t in (x, x.bfloat16(), moved(x.bfloat16())):
        want = -torch.log_softmax(t.double(), -1).gather(-1, y[..., None]).sum()
        got = cross_entropy_sum(t, y)
        # rows of some 3 each, added up in fp32: 40 roundings of at most the sum
        assert abs(float(got) - float(want)) <= 40 * 2.0 ** -24 * float(want)
