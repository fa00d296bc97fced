"""8-bit products of 32-bit activations: exact products, sums in fp32, against 64 bits; a model in fp32."""
import pytest
import torch
from torch import nn

from latest_exact_match_attention_amd import fp8
from latest_exact_match_attention_amd.decode import decoder
from latest_exact_match_attention_amd.model import ModelConfig, SwiGLU, Transformer, load_trained
from latest_exact_match_attention_amd.sampling import sample

pytestmark = pytest.mark.gpu


def rand(dev, *shape, seed=0):
    return torch.randn(shape, device=dev, generator=torch.Generator(device=dev).manual_seed(seed))


def slack_of(a, w):
    """Products of two e4m3 values and their scales are exact, and so is bf16 of each; K of them are added up
    in some order, each addition off by at most a whole step, 2^-23 of a sum that is no larger than that of
    the sizes."""
    return a.shape[1] * 2.0 ** -23 * (a.abs() @ w.abs().t())


def near(got, a, w):
    """Each element within the worst case; their norm within that of K roundings of random signs, each off by
    2^-23 of a partial sum, whose norms are at most the products'. (The 16-bit products' instruction, which
    cuts products off, is off by 2^-16.1 of it: more than this up to K = 16,384.)"""
    assert got.dtype is torch.float32
    a, w = fp8.dequantize(a, torch.float64).reshape(-1, a.columns), fp8.dequantize(w, torch.float64)
    want = a @ w.t()
    off = (got.reshape(want.shape).double() - want).abs()
    bad = ~(off <= slack_of(a, w) + 2.0 ** -149)
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[0].tolist())
    norm = float((a.square() @ w.square().t()).sum().sqrt())
    assert float(off.norm()) <= a.shape[1] ** 0.5 * 2.0 ** -23 * norm + 2.0 ** -149 * off.numel() ** 0.5


SHAPES = [(1, 1, 1), (1, 128, 16), (2, 127, 40), (5, 200, 129), (16, 1536, 6144), (17, 1000, 1234), (32, 264, 33000),
          (33, 128, 128), (64, 384, 8), (100, 8200, 24), (129, 300, 264), (777, 1000, 1234), (2500, 1536, 384),
          (4100, 256, 1000), (40, 16384, 136), (70, 130, 2), (65, 128, 131)]


@pytest.mark.parametrize("M,K,N", SHAPES)
def test_products(dev, M, K, N):
    x = rand(dev, M, K, seed=M) * torch.exp(rand(dev, M, 1, seed=2))
    w = fp8.quantize(rand(dev, N, K, seed=N) * torch.exp(rand(dev, N, 1, seed=3)) * K ** -0.5, 128)
    a = fp8.quantize(x)
    y = fp8.linear(x, w)
    assert y.shape == (M, N)
    near(y, a, w)
    near(fp8.matmul(a, w, torch.float32), a, w)
    r = rand(dev, M, N, seed=9)
    assert torch.equal(fp8.linear(x, w, r), r + y)


@pytest.mark.parametrize("M,K,N", [(1, 128, 8), (16, 1536, 6144), (31, 1000, 1240), (9, 256, 17000), (33, 128, 128),
                                   (129, 300, 264), (2500, 1536, 384), (40, 16384, 136)])
def test_gated(dev, M, K, N):
    x = rand(dev, M, K, seed=M)
    g, u = (fp8.quantize(rand(dev, N, K, seed=s) * K ** -0.5, 128) for s in (5, 6))
    got = fp8.gated_linear(x, g, u)
    a = fp8.dequantize(fp8.quantize(x), torch.float64)
    wg, wu = fp8.dequantize(g, torch.float64), fp8.dequantize(u, torch.float64)
    gv, uv = a @ wg.t(), a @ wu.t()
    eg, eu = slack_of(a, wg), slack_of(a, wu)
    act = gv * torch.sigmoid(gv)                               # |silu'| <= 1.1; e^-g is off by 2 E (|g| + 2)
    slack = 1.1 * eg * (uv.abs() + eu) + act.abs() * eu + 8 * 2.0 ** -24 * (gv.abs() + 4) * (act * uv).abs()
    assert got.dtype is torch.float32 and bool(((got.double() - act * uv).abs() <= slack + 2.0 ** -149).all())


@pytest.mark.parametrize("M", [4, 40])
def test_scales_of_every_size(dev, M):
    """Blocks whose scales lie far apart, along the sum too, and at either end of fp32."""
    K, N = 896, 384
    by = torch.tensor([0.0, 30.0, -30.0, 60.0, 1.0, 110.0, -100.0], device=dev)
    x = (rand(dev, M, K).view(M, 7, 128) * torch.exp2(by)[:, None]).view(M, K)
    w = (rand(dev, N, K, seed=4).view(N, 7, 128) * torch.exp2(-by)[:, None]).view(N, K)
    q = fp8.quantize(w, 128)
    near(fp8.linear(x, q), fp8.quantize(x), q)


def test_ends_of_the_range(dev):
    """The largest number is rounded up to 2^128, which is infinite; the smallest ones go to steps of 2^-133."""
    x = torch.zeros(3, 128, device=dev)
    x[0, 5], x[1, 5], x[2, 5] = 3.4028234e38, 2.0 ** -126 * 1.125, 2.0 ** -140
    w = torch.zeros(8, 128, device=dev)
    w[:, 5] = 1.0
    for call in (lambda: fp8.linear(x, fp8.quantize(w, 128)), lambda: fp8.linear(x.repeat(20, 1), fp8.quantize(w, 128))):
        y = call()
        assert bool((y[0] == float("inf")).all()) and bool((y[1] == 2.0 ** -126 * 1.125).all()) and bool((y[2] == 0).all())


def framed(t, fill):
    flat = torch.full((t.numel() + 1024,), fill, device=t.device, dtype=t.dtype)
    flat[512:512 + t.numel()] = t.reshape(-1)
    return flat[512:512 + t.numel()].view(t.shape)


@pytest.mark.parametrize("M,K,N", [(5, 200, 129), (33, 128, 130), (777, 300, 1234), (300, 2000, 264)])
def test_nothing_around_the_tensors_counts(dev, M, K, N):
    x = rand(dev, M, K)
    w = fp8.quantize(rand(dev, N, K, seed=1), 128)
    want = fp8.linear(x, w)
    w2 = fp8.Fp8(framed(w.values.view(torch.uint8), 255).view(torch.float8_e4m3fn),
                 framed(w.scales.view(torch.uint8), 255).view(torch.float8_e8m0fnu), K)
    flat = torch.full((M * K + 1024,), float("nan"), device=dev)
    for start in (512, 513):                                   # at any element's address
        part = flat[start:start + M * K].view(M, K).copy_(x)
        assert torch.equal(fp8.linear(part, w2), want)


@pytest.mark.parametrize("M", [9, 140])
def test_rows_keep_to_themselves(dev, M):
    x, w = rand(dev, M, 300), rand(dev, 200, 300, seed=1)
    want = fp8.linear(x, fp8.quantize(w, 128))
    x[3, 5], x[M - 1, 299] = float("nan"), float("inf")
    w[7, 11] = float("nan")
    got = fp8.linear(x, fp8.quantize(w, 128))
    keep = torch.ones_like(want, dtype=torch.bool)
    keep[3], keep[M - 1], keep[:, 7] = False, False, False
    assert torch.equal(got[keep], want[keep]) and bool(got[~keep].isnan().all())


def test_lead_dims_and_no_rows(dev):
    x = rand(dev, 3, 5, 7, 300)
    w = fp8.quantize(rand(dev, 50, 300, seed=2), 128)
    want = fp8.linear(x.view(105, 300), w)
    assert torch.equal(fp8.linear(x, w).view(105, 50), want)
    t = x.transpose(0, 2).contiguous().transpose(0, 2)
    assert torch.equal(fp8.linear(t, w).view(105, 50), want)
    assert torch.equal(fp8.matmul(fp8.quantize(x), w, torch.float32).view(105, 50), want)
    assert fp8.linear(x[:0], w).shape == (0, 5, 7, 50)
    assert fp8.matmul(fp8.quantize(x[:0]), w, torch.float32).dtype is torch.float32


def test_captured_and_on_two_streams(dev):
    cases = [(rand(dev, M, K), fp8.quantize(rand(dev, N, K, seed=1), 128))
             for M, K, N in ((16, 1536, 6144), (40, 16384, 136))]
    graphs, outs = [], []
    for x, w in cases:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            fp8.linear(x, w)
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(fp8.linear(x, w))
        graphs.append(g)
    for step in range(4):
        for (x, w), g, out in zip(cases, graphs, outs):
            x.mul_(1 + 0.3 * step)
            g.replay()
            assert torch.equal(out, fp8.linear(x, w)), step
            torch.cuda.synchronize()
    want = [fp8.linear(x, w) for x, w in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for _ in range(4):
        for s, (x, w), y in zip(streams, cases, want):
            with torch.cuda.stream(s):
                got.append((fp8.linear(x, w), y))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in got)


def test_offsets_past_32_bits(dev):
    """Results of more than 2^31 elements and 2^33 bytes."""
    M, K, N = 530000, 264, 4200
    x = rand(dev, M, K)
    w = fp8.quantize(rand(dev, N, K, seed=3), 128)
    y = fp8.linear(x, w)
    rows = torch.tensor([0, 255, 256, 262144, 507904, 523776, M - 1], device=dev)
    near(y[rows], fp8.quantize(x[rows]), w)


def test_refusals(dev):
    x = rand(dev, 4, 300)
    w = fp8.quantize(rand(dev, 50, 300), 128)
    for call in (lambda: fp8.linear(x.double(), w), lambda: fp8.gated_linear(x.double(), w, w),
                 lambda: fp8.matmul(fp8.quantize(x), w, torch.float64)):
        with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
            call()
    for dt in (torch.float32, torch.bfloat16):
        v = x.to(dt)
        with pytest.raises(ValueError, match="columns"):
            fp8.linear(v[:, :200], w)
        with pytest.raises(TypeError, match="float8"):
            fp8.linear(v, fp8.Fp8(w.values.float(), w.scales, 300))
        with pytest.raises(ValueError, match="scales"):
            fp8.linear(v, fp8.Fp8(w.values, w.scales[:, :2], 300))
        with pytest.raises(ValueError, match="values"):
            fp8.linear(v, fp8.Fp8(w.values[:, :256], w.scales, 300))
        with pytest.raises(ValueError, match="residual"):
            fp8.linear(v, w, v)
        with pytest.raises(TypeError, match="residual"):
            fp8.linear(v, w, torch.zeros(4, 50, device=dev, dtype=torch.float16))
        with pytest.raises(ValueError, match="multiple of 8"):
            fp8.gated_linear(v, w, w)
        with pytest.raises(ValueError, match="outputs"):
            fp8.gated_linear(v, w, fp8.quantize(rand(dev, 48, 300), 128))
        with pytest.raises(ValueError, match="cpu"):
            fp8.linear(v, fp8.Fp8(w.values.cpu(), w.scales, 300))
        v = v.detach().requires_grad_(True)
        with pytest.raises(RuntimeError, match="no gradient"):
            fp8.linear(v, w)
        with torch.no_grad():
            fp8.linear(v, w)
    with pytest.raises(ValueError, match="rows of 300"):
        fp8.matmul(w, w, torch.float32)
    with pytest.raises(ValueError, match="block_rows"):
        fp8.quantize(x, 2)
    with pytest.raises(ValueError, match="matrix"):
        fp8.quantize(x[None], 128)
    with pytest.raises(TypeError, match="quantize takes"):
        fp8.quantize(x.double())
    with pytest.raises(ValueError, match="columns"):
        fp8.quantize(x[:, :0])
    with pytest.raises(ValueError, match="bias"):
        fp8.Fp8Linear.of(nn.Linear(8, 8, device=dev))


def test_feed_forward_block(dev):
    torch.manual_seed(0)
    mlp = SwiGLU(256, 640).to(dev)
    ws = [fp8.quantize(lin.weight.detach(), 128) for lin in (mlp.gate, mlp.up, mlp.down)]
    x = {n: torch.randn(n, 3, 256, device=dev) for n in (2, 50)}
    with torch.no_grad():
        old = {n: mlp(v, residual=v) for n, v in x.items()}
        for name in ("gate", "up", "down"):
            setattr(mlp, name, fp8.Fp8Linear.of(getattr(mlp, name)))
        for n, v in x.items():
            got = mlp(v, residual=v)
            assert torch.equal(got, v + fp8.linear(fp8.gated_linear(v, ws[0], ws[1]), ws[2]))
            # e4m3 rounds x and each weight by at most 2^-4, a third of that in the root mean square
            assert float((got - old[n]).double().norm() / (old[n] - v).double().norm()) < 4 * 2.0 ** -4


def test_model_as_it_is_made(dev, tmp_path):
    """A model that nobody cast (and one from load_trained) is held in 8 bits, filled, sampled from and
    decoded."""
    torch.manual_seed(1)
    cfg = ModelConfig(vocab_size=256, depth=2, dim=128, num_heads=8)
    model = Transformer(cfg).cuda()
    torch.save({"config": {"vocab_size": 256, "depth": 2, "dim": 128, "num_heads": 8}, "state_dict": model.state_dict()},
               tmp_path / "model.pt")
    for m in (model, load_trained(tmp_path)[0]):
        m.set_hard(True)
        fp8.quantize_feed_forward(m, head=True)
        prompt = torch.randint(0, 256, (3, 70), device=dev)
        with torch.no_grad():
            cache = m.new_cache("hbm", max_cache_len=128, batch=3)
            logits = m(prompt, cache=cache)
            assert logits.dtype is torch.float32
            draw = sample(logits[:, -1], torch.rand(3, device=dev), temperature=0.8, top_k=50, top_p=0.95)
            step = decoder(m, cache, tok=draw.tokens[:, None], temperature=0.8, top_p=0.95, logprobs=True)
            seq = torch.cat([prompt, draw.tokens[:, None]], 1)
            for _ in range(4):
                tok = step.step().clone()
                full = m(seq)[:, -1:]
                assert float((full - step.logits).double().norm() / full.double().norm()) < 0.1
                seq = torch.cat([seq, tok], 1)
