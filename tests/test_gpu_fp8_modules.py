"""8-bit linear layers wherever a model has a linear layer: blocks of both kinds, single projections, parameter
counts, checkpoints."""
import itertools

import pytest
import torch

from latest_exact_match_attention_amd import fp8
from latest_exact_match_attention_amd.decode import decoder
from latest_exact_match_attention_amd.model import ModelConfig, SwiGLU, Transformer, gated_linear, linear, load_trained, rms_norm, swiglu

pytestmark = pytest.mark.gpu

NAMES = ("gate", "up", "down")
SOME = [s for n in (1, 2) for s in itertools.combinations(NAMES, n)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("which", SOME, ids="-".join)
def test_mixed_blocks(dev, which, dtype):
    """One or two of a block's three weights in 8 bits: the products that it is made of."""
    torch.manual_seed(0)
    mlp = SwiGLU(256, 640).to(dev).to(dtype)
    norm = torch.nn.RMSNorm(256, eps=1e-5).to(dev, dtype)
    for name in which:
        setattr(mlp, name, fp8.Fp8Linear.of(getattr(mlp, name)))
    for n in (2, 50):
        x = torch.randn(n, 1, 256, device=dev).to(dtype)
        r = torch.randn(n, 1, 256, device=dev).to(dtype)
        with torch.no_grad():
            if {"gate", "up"} <= set(which):
                a = fp8.gated_linear(x, mlp.gate.weight, mlp.up.weight)
            elif which == ("down",):
                a = gated_linear(x, mlp.gate, mlp.up)
            else:
                a = swiglu(linear(x, mlp.gate), linear(x, mlp.up))
            y = linear(a, mlp.down)
            got = mlp(x)
            # the gated product of few rows in bf16 has a launch of its own, whose fp32 sums go in another order
            assert float((got - y).double().norm() / y.double().norm()) <= (2.0 ** -8 if which == ("down",) else 0)
            assert torch.equal(mlp(x, residual=r.clone()), r + got) or "down" not in which
            # the sum is rounded once: by half a step of r + y, which is what it is large beside (r is of size 1
            # here and y of 0.1, so a bound by y alone would be 10 times too small); y by half a step before it,
            # and the 2^-8 of above
            half = torch.finfo(dtype).eps / 2
            off = (mlp(x, residual=r.clone()).double() - r.double() - y.double()).norm()
            assert float(off) <= half * float((r.double() + y.double()).norm()) + (half + 2.0 ** -8) * float(y.double().norm())
            assert mlp.forward_normed(x, r, norm) is None
            h, s = rms_norm(x, norm, r)
            assert bool(mlp(h, residual=s).isfinite().all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("name", ["attn.q_proj", "attn.k_proj", "attn.v_proj", "attn.o_proj", "mlp.gate", "mlp.up", "mlp.down"])
def test_every_projection(dev, name, dtype):
    """A model with one projection of a block in 8 bits runs uncached, filled and decoding, and near each other."""
    torch.manual_seed(1)
    m = Transformer(ModelConfig(vocab_size=256, depth=2, dim=128, num_heads=8)).to(dev).to(dtype)
    m.set_hard(True)
    owner, leaf = name.split(".")
    at = getattr(m.blocks[1], owner)
    setattr(at, leaf, fp8.Fp8Linear.of(getattr(at, leaf)))
    prompt = torch.randint(0, 256, (3, 70), device=dev)
    with torch.no_grad():
        cache = m.new_cache("hbm", max_cache_len=128, batch=3)
        m(prompt[:, :-1], cache=cache, return_logits=False)
        step = decoder(m, cache, tok=prompt[:, -1:])
        step.step()
        full = m(prompt)[:, -1:]
        assert full.shape == step.logits.shape and bool(step.logits.isfinite().all())
        # a code whose pre-activation lies at 0 may turn where sums go in another order
        assert float((full - step.logits).double().norm() / full.double().norm()) < 0.3


def test_checkpoints(dev, tmp_path):
    """A model's 8-bit weights load into another one that was held so, and by load_trained."""
    torch.manual_seed(2)
    geo = dict(vocab_size=256, depth=2, dim=128, num_heads=8)
    m, other = (Transformer(ModelConfig(**geo)).to(dev) for _ in range(2))
    for t in (m, other):
        t.set_hard(True)
        fp8.quantize_feed_forward(t, head=True)
    other.load_state_dict(m.state_dict())
    torch.save({"config": geo, "state_dict": m.state_dict()}, tmp_path / "model.pt")
    loaded, _ = load_trained(tmp_path, device=dev)
    ids = torch.randint(0, 256, (2, 40), device=dev)
    with torch.no_grad():
        want = m(ids)
        assert torch.equal(other(ids), want) and torch.equal(loaded(ids), want)
    assert loaded.n_params() == m.n_params()
