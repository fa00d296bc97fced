"""The operators together: a hard-mode model's training step in bf16, from tokens through the
embedding, norms, exact op and MLP to each loss, against the same model in 64 bits with the
forward's own matches."""
import pytest
import torch
import torch.nn.functional as F

from latest_exact_match_attention_amd.attention import latest_prev_match, pack_codes
from latest_exact_match_attention_amd.decode import decoder
from latest_exact_match_attention_amd.loss import policy_loss, preference_loss, token_logprobs
from latest_exact_match_attention_amd.model import ModelConfig, Transformer, lm_loss, swiglu

pytestmark = pytest.mark.gpu

DEPTH, DIM = 2, 64


def build(dev, seed=0):
    torch.manual_seed(seed)
    cfg = ModelConfig(vocab_size=256, depth=DEPTH, dim=DIM, num_heads=4, d_qk=8, d_v=16, dim_ff=128)
    model = Transformer(cfg)
    model.set_hard(True)
    return model.to(dev).to(torch.bfloat16), cfg


def record_matches(model):
    """Each layer's matches in the next forward, from the inputs it has there. (A forward without
    gradients adds the MLP's residual inside its product, with one rounding less, so that its
    later layers' codes may differ.)"""
    matches, handles = {}, []

    def hook(i):
        @torch.no_grad()
        def fn(blk, inp, _out):
            zq, zk, _ = blk.attn.project(blk.pre_attn(inp[0]))
            qc, kc = pack_codes(zq), pack_codes(zk)
            matches[i] = latest_prev_match(qc.flatten(0, 1), kc.flatten(0, 1)).view(qc.shape)
            handles[i].remove()
        return fn
    handles += [blk.register_forward_hook(hook(i)) for i, blk in enumerate(model.blocks)]
    return matches


def plain(model, idx, matches):
    """The logits in 64 bits, and the leaves: each layer's gather goes by the given matches."""
    w = {k: v.detach().double().requires_grad_(True) for k, v in model.state_dict().items()}
    c = model.cfg
    rms = lambda x, k: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + c.norm_eps) * w[k]  # noqa: E731
    x = w["tok_emb.weight"][idx]
    B, T = idx.shape
    for i in range(c.depth):
        b = f"blocks.{i}."
        h = rms(x, b + "norm1.weight")
        v = (h @ w[b + "attn.v_proj.weight"].t()).view(B, T, c.num_heads, c.d_v).transpose(1, 2)
        src = matches[i]
        y = v.gather(2, src.clamp_min(0)[..., None].expand(v.shape)) * (src >= 0)[..., None]
        x = x + y.transpose(1, 2).reshape(B, T, -1) @ w[b + "attn.o_proj.weight"].t()
        h = rms(x, b + "norm2.weight")
        a = F.silu(h @ w[b + "mlp.gate.weight"].t()) * (h @ w[b + "mlp.up.weight"].t())
        x = x + a @ w[b + "mlp.down.weight"].t()
    return rms(x, "norm_f.weight") @ w["lm_head.weight"].t(), w


def loss_of(kind, logits, targets, mask):
    lp = torch.log_softmax(logits, -1).gather(-1, targets[..., None])[..., 0]
    if kind == "policy":
        old, adv = -5.0, torch.linspace(-1, 1, lp.numel(), device=lp.device).view(lp.shape)
        r = torch.exp(lp - old)
        return (-torch.minimum(r * adv, r.clamp(0.0, 1e9) * adv) * mask).sum() / mask.sum()
    if kind == "preference":
        s = ((lp + 5.0) * mask).sum(1)
        n = s.numel() // 2
        return -F.logsigmoid(0.1 * (s[:n] - s[n:])).mean()
    return -lp.mean()


@pytest.mark.parametrize("kind", ["policy", "preference", "lm"])
@pytest.mark.parametrize("B,T", [(4, 40), (2, 9), (2, 1)])
def test_step(dev, kind, B, T):
    """Every parameter's gradient within 100 half steps of bf16 in the Frobenius norm: about fifty
    roundings lie between a weight and the loss, forward and back, and each moves what follows by
    at most half a step of it, through factors (norms, a softmax, products of random weights) that
    keep relative sizes or halve them again. Queries and keys get none: codes are not
    differentiable. B T below 33 rows goes through the decode-shaped products."""
    model, cfg = build(dev)
    idx = torch.randint(0, 200, (B, T), device=dev, generator=torch.Generator(dev).manual_seed(T)) % 17
    targets = (idx * 7 + 3) % 200
    mask = torch.ones(B, T, dtype=torch.bool, device=dev)
    mask[0, : T // 3] = False
    matches = record_matches(model)
    if kind == "lm":
        loss = lm_loss(model, idx, targets, chunk=16)
    else:
        logits = model(idx)
        if kind == "policy":
            adv = torch.linspace(-1, 1, B * T, device=dev).view(B, T)
            loss = policy_loss(logits, targets, torch.full((B, T), -5.0, device=dev), adv, mask=mask,
                               clip_low=1.0, clip_high=1e9).loss
        else:
            loss = preference_loss(logits, targets, torch.full((B, T), -5.0, device=dev), mask).loss
    names = [n for n, _ in model.named_parameters()]
    grads = torch.autograd.grad(loss, list(model.parameters()), allow_unused=True)
    exact_logits, w = plain(model, idx, matches)
    want_loss = loss_of(kind, exact_logits, targets, mask)
    want = torch.autograd.grad(want_loss, [w[n] for n in names], allow_unused=True)
    assert abs(float(loss.detach()) - float(want_loss.detach())) <= 100 * 2.0 ** -9 * max(1.0, abs(float(want_loss.detach())))
    for n, g, r in zip(names, grads, want):
        if "q_proj" in n or "k_proj" in n:
            assert g is None and r is None
            continue
        assert g is not None and g.dtype == torch.bfloat16, n
        assert float((g.double() - r).norm()) <= 100 * 2.0 ** -9 * float(r.norm()) + 1e-12, n


def test_values_of_a_call_without_gradients(dev):
    """The forward with gradients gives the logits of the one without, bit for bit, on decode
    shapes, whose launches it takes apart."""
    model, _ = build(dev, 1)
    for B, T in ((4, 8), (3, 7), (1, 1)):
        idx = torch.randint(0, 200, (B, T), device=dev) % 17
        with torch.no_grad():
            want = model(idx)
        got = model(idx)
        assert got.requires_grad and torch.equal(got, want)


def test_cache_and_decoder_stay_without_gradients(dev):
    """A cached forward and a decoder built outside no_grad run the fused launches, and sample the
    tokens whose log-probabilities the losses then take."""
    model, cfg = build(dev, 2)
    prompt = torch.randint(0, 200, (2, 12), device=dev)
    runs = []
    for ctx in (torch.no_grad(), torch.enable_grad()):
        with ctx:
            cache = model.new_cache("hbm", max_cache_len=64, batch=2)
            model(prompt[:, :-1], cache=cache, return_logits=False)
            dec = decoder(model, cache, tok=prompt[:, -1:])
            runs.append(torch.cat([dec.step().clone() for _ in range(6)], 1))
            assert not dec.logits.requires_grad
    assert torch.equal(*runs)
    full = torch.cat([prompt, runs[0]], 1)
    logits = model(full[:, :-1])[:, 11:]
    lp = token_logprobs(logits, full[:, 12:])
    assert bool((lp <= 0).all())
    (g,) = torch.autograd.grad(lp.sum(), [model.tok_emb.weight])
    assert bool(g[full[0, 0]].any())


def test_gradients_reach_every_parameter(dev):
    """Finite and not zero, through every part of the chain."""
    model, _ = build(dev, 3)
    idx = torch.randint(0, 200, (4, 32), device=dev)
    loss = lm_loss(model, idx, (idx + 1) % 200)
    params = [p for n, p in model.named_parameters() if "q_proj" not in n and "k_proj" not in n
              and "tok_emb" not in n and "norm1" not in n]
    grads = torch.autograd.grad(loss, params)
    assert all(bool(g.isfinite().all()) and bool(g.any()) for g in grads)


def test_swiglu_gradient(dev):
    """gate and up gradients: fp32 with one rounding, of factors that expf and a division leave
    8 roundings off; sig's complement loses 2^-24 absolutely."""
    g = torch.Generator(dev).manual_seed(5)
    a, b, gy = ((torch.randn(33, 200, device=dev, generator=g) * 4).bfloat16() for _ in range(3))
    a.requires_grad_(True), b.requires_grad_(True)
    ga, gb = torch.autograd.grad(swiglu(a, b), [a, b], gy)
    x, u, y = (t.detach().double() for t in (a, b, gy))
    sig = torch.sigmoid(x)
    for got, want, size in ((ga, y * u * sig * (1 + x * (1 - sig)), (y * u * sig).abs() * (1 + x.abs())),
                            (gb, y * x * sig, (y * x * sig).abs())):
        assert bool(((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 16 * 2.0 ** -24 * size + 1e-38).all())


def operators(dev, seed):
    """A call of each operator with its gradients, on inputs of its own: () -> list of tensors."""
    from latest_exact_match_attention_amd.model import embed, layer_norm
    g = torch.Generator(dev).manual_seed(seed)
    emb = torch.nn.Embedding(3000, 264, device=dev, dtype=torch.bfloat16)
    norm = torch.nn.LayerNorm(264, device=dev, dtype=torch.bfloat16)
    head = (torch.randn(1003, 264, device=dev, generator=g) * 0.06).bfloat16().requires_grad_(True)
    ids = torch.randint(0, 3000, (8, 200), device=dev, generator=g)
    targets = torch.randint(0, 1003, (8, 200), device=dev, generator=g)
    adv = torch.randn(8, 1, device=dev, generator=g)
    old = torch.full((8, 200), -6.9, device=dev)
    with torch.no_grad():
        emb.weight.copy_(torch.randn(3000, 264, device=dev, generator=g))

    def run():
        h, _ = layer_norm(embed(emb, ids, 2.0), norm)
        logits = h @ head.t()
        loss = policy_loss(logits, targets, old, adv, old, kl_weight=0.1).loss \
            + preference_loss(logits, targets, old).loss + token_logprobs(logits, targets).mean()
        return [loss.detach(), *torch.autograd.grad(loss, [emb.weight, norm.weight, norm.bias, head])]
    return run


def test_streams_at_once(dev):
    """Two callers on streams of their own, their launches interleaved: the results of each alone."""
    runs = [operators(dev, s) for s in (1, 2)]
    want = [r() for r in runs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in runs]
    got = [[], []]
    for _ in range(6):
        for k, (r, s) in enumerate(zip(runs, streams)):
            with torch.cuda.stream(s):
                got[k].append(r())
    torch.cuda.synchronize()
    for k in range(2):
        for out in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[k]))


def test_offsets_beyond_32_bits(dev):
    """Rows, tables and logits of more than 2^31 elements: what lies at their ends."""
    from latest_exact_match_attention_amd.model import embed, layer_norm
    V, D = 1_000_000, 2200
    emb = torch.nn.Embedding(V, D, _weight=torch.zeros(V, D, device=dev, dtype=torch.bfloat16))
    with torch.no_grad():
        emb.weight[-3:] = 1.5
    ids = torch.tensor([V - 1, 0, V - 1, V - 3, V - 5], device=dev)
    y = embed(emb, ids)
    assert y[:, 0].tolist() == [1.5, 0.0, 1.5, 1.5, 0.0]
    (gw,) = torch.autograd.grad(y, [emb.weight], torch.ones_like(y))
    assert gw[[0, 1, V - 5, V - 4, V - 3, V - 2, V - 1]].float().mean(1).tolist() == [1, 0, 1, 0, 1, 0, 2]
    del emb, y, gw
    R, D = 270_000, 8000
    norm = torch.nn.LayerNorm(D, device=dev, dtype=torch.bfloat16)
    x = torch.zeros(R, D, device=dev, dtype=torch.bfloat16)
    x[-2:] = torch.randn(2, D, device=dev).bfloat16()
    x.requires_grad_(True)
    h, _ = layer_norm(x, norm)
    gh = torch.zeros_like(h)
    gh[-2:] = torch.randn(2, D, device=dev).bfloat16()
    gx, gw = torch.autograd.grad(h, [x, norm.weight], gh)
    t = x.detach()[-2:].clone().requires_grad_(True)
    h2, _ = layer_norm(t, norm)
    gt, gw2 = torch.autograd.grad(h2, [t, norm.weight], gh[-2:])
    assert torch.equal(h[-2:], h2) and torch.equal(gx[-2:], gt) and not gx[:-2:1000].any()
    assert torch.allclose(gw.float(), gw2.float(), rtol=2 ** -7, atol=0)    # one rounding of bf16 each
    del x, h, gh, gx
    n, V = 43_000, 50_304
    logits = torch.zeros(n, V, device=dev, dtype=torch.bfloat16)
    logits[-1] = torch.randn(V, device=dev).bfloat16()
    logits.requires_grad_(True)
    targets = torch.full((n,), 17, device=dev)
    mask = torch.zeros(n, dtype=torch.bool, device=dev)
    mask[-1] = True
    z = torch.full((n,), -9.0, device=dev)
    r = policy_loss(logits, targets, z, z, mask=mask, clip_low=1.0, clip_high=1e9)
    (g,) = torch.autograd.grad(r.loss, [logits])
    one = logits.detach()[-1:].clone().requires_grad_(True)
    s = policy_loss(one, targets[-1:], z[-1:], z[-1:], clip_low=1.0, clip_high=1e9)
    (w,) = torch.autograd.grad(s.loss, [one])
    assert torch.equal(r.loss, s.loss) and torch.equal(g[-1:], w) and not g[:-1:997].any()
    lp = token_logprobs(logits, targets, mask)
    (g,) = torch.autograd.grad(lp.sum(), [logits])
    one_lp = token_logprobs(one, targets[-1:])
    (w,) = torch.autograd.grad(one_lp.sum(), [one])
    assert torch.equal(lp[-1:], one_lp) and torch.equal(g[-1:], w)


def test_forward_mode_is_refused(dev):
    """A tangent is never dropped: the operators have no forward mode and say so."""
    import torch.autograd.forward_ad as fwd
    from latest_exact_match_attention_amd.model import layer_norm, rms_norm
    x = torch.randn(4, 64, device=dev).bfloat16()
    t = torch.zeros(4, dtype=torch.long, device=dev)
    z = torch.zeros(4, device=dev)
    norm, rms = (n(64, device=dev, dtype=torch.bfloat16) for n in (torch.nn.LayerNorm, torch.nn.RMSNorm))
    with torch.no_grad(), fwd.dual_level():
        d = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: layer_norm(d, norm), lambda: rms_norm(d, rms), lambda: swiglu(d, d),
                     lambda: token_logprobs(d, t), lambda: policy_loss(d, t, z, z),
                     lambda: preference_loss(d[:, None], t[:, None], z[:, None])):
            with pytest.raises((RuntimeError, NotImplementedError)):
                call()
