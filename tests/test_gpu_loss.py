"""Token log-probabilities, the policy and the preference loss, and their gradients, against 64-bit
formulas."""
import math

import pytest
import torch

from latest_exact_match_attention_amd import _lib
from latest_exact_match_attention_amd.loss import policy_loss, preference_loss, token_logprobs
from latest_exact_match_attention_amd.model import cross_entropy_sum

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
E = 2.0 ** -24


def make(dev, shape, V, dtype, seed=0, scale=3.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    logits = (torch.randn(*shape, V, device=dev, generator=g) * scale).to(dtype)
    targets = torch.randint(0, V, shape, device=dev, generator=g)
    return logits, targets, g


def exact(logits, targets, temperature):
    """lp and the softmax in 64 bits, and how far an fp32 lp may be off: three roundings of the
    distance to the maximum, and the error of log S: the terms' arguments are off by two
    roundings of themselves (a softmax weighs them by e^-argument: log2 V bits at most), the
    hardware's 2^x by four E, and the sum by its steps, V / 2048 trips of a thread and 30 more."""
    V = logits.shape[-1]
    x = logits.double() / temperature
    p = torch.log_softmax(x, -1)
    lp = p.gather(-1, targets[..., None].clamp(0, V - 1))[..., 0]
    far = (x.amax(-1) - x.gather(-1, targets[..., None].clamp(0, V - 1))[..., 0]).abs()
    sum_err = E * (4 * math.log2(V + 1) + 4 + V / 2048 + 30)
    return lp, p.exp(), 3 * E * far + sum_err + E * lp.abs(), sum_err


def check_grad(grad, p, targets, c, dc, temperature, sum_err, mask=None):
    """grad against c / temperature (onehot - p): p is off by its argument's roundings (2 E of
    it, and it is at most |log p|), its sum's error, the exponential's and the products' roundings."""
    one = torch.zeros_like(p).scatter_(-1, targets[..., None].clamp(0, p.shape[-1] - 1), 1.0)
    c, dc = c[..., None] / temperature, dc[..., None] / temperature
    want = c * (one - p)
    slack = dc * (one + p) + c.abs() * ((16 * E + sum_err) * (p + one)
                                        + 2 * E * p * p.clamp_min(1e-300).log().abs())
    if mask is not None:
        want, slack = want * mask[..., None], slack * mask[..., None]
    u = torch.finfo(grad.dtype).eps / 2
    # below the normals a step is absolute; fp32's exponential flushes there too
    tiny = {torch.float16: 2.0 ** -25}.get(grad.dtype, 2.0 ** -126)
    bad = (grad.double() - want).abs() > u * (want.abs() + slack) + slack + tiny
    assert not bool(bad.any()), int(bad.sum())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 100, 2047, 2056, 4097, 32003, 50304])
@pytest.mark.parametrize("temperature", [1.0, 0.7])
def test_token_logprobs(dev, dtype, V, temperature):
    logits, targets, g = make(dev, (3, 5), V, dtype, seed=V)
    lp, p, tol, sum_err = exact(logits, targets, temperature)
    logits.requires_grad_(True)
    got = token_logprobs(logits, targets, temperature=temperature)
    with torch.no_grad():
        assert torch.equal(token_logprobs(logits, targets.int(), temperature=temperature), got)
    assert got.dtype == torch.float32 and bool(((got.double() - lp).abs() <= tol).all())
    c = torch.randn(3, 5, device=dev, generator=g)
    (grad,) = torch.autograd.grad(got, [logits], c)
    check_grad(grad, p, targets, c.double(), 0 * lp, temperature, sum_err)


def test_more_rows_than_one_grid_dimension(dev):
    """Short rows, 2.1 million of them: every one as in a call of a few. A loss scaled by their
    repetitions has the same factor, 1 / 1031 rounded once, and so the same gradient."""
    n = 2035
    logits, targets, g = make(dev, (1031,), 8, torch.float16, seed=3)
    many, many_t = logits.repeat(n, 1).requires_grad_(True), targets.repeat(n)
    logits.requires_grad_(True)
    c, z = torch.randn(1031, device=dev, generator=g), torch.zeros(1031, device=dev)
    small = token_logprobs(logits, targets)
    got = token_logprobs(many, many_t)
    assert torch.equal(got.view(n, 1031), small.expand(n, -1))
    (want,) = torch.autograd.grad(small, [logits], c)
    (grad,) = torch.autograd.grad(got, [many], c.repeat(n))
    assert torch.equal(grad.view(n, 1031, 8), want.expand(n, -1, -1))
    small = policy_loss(logits, targets, z, c)
    got = policy_loss(many, many_t, z.repeat(n), c.repeat(n), scale=float(n))
    assert torch.equal(got.logprobs.view(n, 1031), small.logprobs.expand(n, -1))
    (want,) = torch.autograd.grad(small.loss, [logits])
    (grad,) = torch.autograd.grad(got.loss, [many])
    assert torch.equal(grad.view(n, 1031, 8), want.expand(n, -1, -1))


@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(dev, dtype):
    """Slices along any dim, odd row starts, expanded rows, a transposed vocabulary."""
    base, _, g = make(dev, (4, 6), 1003, dtype)
    views = [base[:, :-1], base[1:, 2:], base[..., 1:], base[:, ::2, 5:900], base.transpose(0, 1),
             base[:1].expand(4, 6, 1003), base.transpose(1, 2), base[0, 0], base[:0], base[:, :0],
             base.view(2, 2, 6, 1003)[:, :, ::2], base.permute(1, 0, 2)[::2, :, 3:]]
    for v in views:
        targets = torch.randint(0, v.shape[-1], v.shape[:-1], device=dev, generator=g)
        leaf = base.clone().requires_grad_(True)
        x = torch.as_strided(leaf, v.shape, v.stride(), v.storage_offset())
        got = token_logprobs(x, targets)
        if not v.numel():
            assert got.shape == targets.shape
            torch.autograd.grad(got.sum(), [leaf])
            continue
        lp, p, tol, sum_err = exact(v, targets, 1.0)
        assert bool(((got.double() - lp).abs() <= tol).all()), v.shape
        c = torch.randn(targets.shape, device=dev, generator=g)
        (grad,) = torch.autograd.grad(got, [x], c)
        check_grad(grad, p, targets, c.double(), 0 * lp, 1.0, sum_err)


def test_values_at_the_edge(dev):
    """-inf logits add nothing; the types' lowest values make a uniform row; a NaN, +inf or wholly
    -inf row gives NaN, as log_softmax does; so does a target outside the vocabulary."""
    V = 4100
    for dtype in TYPES:
        x = torch.zeros(7, V, device=dev, dtype=dtype)
        x[0, 10:] = -float("inf")
        x[1] = torch.finfo(dtype).min
        x[2, 50] = float("nan")
        x[2, :50], x[2, 51:] = -float("inf"), -float("inf")
        x[3] = -float("inf")
        x[4, 3] = float("inf")
        x[5, 0], x[5, 1:] = torch.finfo(dtype).max, torch.finfo(dtype).min
        t = torch.tensor([3, 5, 0, 0, 0, 0, V], device=dev)
        x.requires_grad_(True)
        lp = token_logprobs(x, t)
        want = torch.log_softmax(x.detach().double(), -1).gather(1, t.clamp(max=V - 1)[:, None])[:, 0]
        assert bool(((lp - want).abs()[[0, 1, 5]] <= 64 * E * want.abs()[[0, 1, 5]]).all())
        assert bool(lp[[2, 3, 4, 6]].isnan().all())
        (g,) = torch.autograd.grad(lp, [x], torch.ones_like(lp))
        assert not g[0, 10:].any() and not g[5].any()
        assert bool(g[2].isnan().all() and g[3].isnan().all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [12, 1001, 50304, 131073])
def test_policy_values_at_the_edge(dev, dtype, V):
    """Rows whose maximum times log2 e leaves fp32's range or is large in it, rows of -inf with one
    logit, and a NaN: the loss and its gradient from the kernel that holds a row (and, at the last size, from the
    ones that do not)."""
    top = torch.finfo(dtype).max
    x = torch.zeros(6, V, device=dev, dtype=dtype)
    big = {torch.float32: 2.0 ** 30, torch.float16: 2.0 ** 15, torch.bfloat16: 2.0 ** 100}[dtype]
    x[5], x[5, 2:] = big, -big
    x[0] = -top
    x[1, 1:], x[1, 0] = -top, top
    x[2], x[2, 3] = -float("inf"), 1.0
    x[3, 7] = float("nan")
    x[4, ::2] = -float("inf")
    t = torch.tensor([5, 0, 3, 1, 1, 1], device=dev)
    z, one = torch.zeros(6, device=dev), torch.ones(6, device=dev)
    x.requires_grad_(True)
    for rows in ([0, 1, 2, 4, 5], [3]):
        mask = torch.zeros(6, dtype=torch.bool, device=dev)
        mask[rows] = True
        r = policy_loss(x, t, torch.where(t == 5, -math.log(V), 0.0), one, mask=mask, clip_high=1e3)
        (g,) = torch.autograd.grad(r.loss, [x])
        if rows == [3]:
            assert bool(r.loss.isnan() and r.logprobs[3].isnan() and g[3].isnan().all())
            assert not g[[0, 1, 2, 4, 5]].any()
            continue
        want = torch.log_softmax(x.detach().double(), -1)
        lp = want.gather(1, t[:, None])[:, 0]
        assert bool(((r.logprobs - lp).abs()[rows] <= 128 * E * lp.abs().clamp_min(1)[rows]).all())
        c = -torch.exp(lp - torch.where(t == 5, -math.log(V), 0.0)).double()[:, None] / 5
        exact_g = c * (torch.nn.functional.one_hot(t, V) - want.exp())
        u = torch.finfo(dtype).eps / 2
        assert bool(((g.double() - exact_g).abs() <= u * exact_g.abs() + 256 * E * c.abs() + 2.0 ** -25)[rows].all())


def policy_case(dev, shape, V, dtype, seed=0):
    logits, targets, g = make(dev, shape, V, dtype, seed)
    lp = torch.log_softmax(logits.double(), -1).gather(-1, targets[..., None])[..., 0]
    # ratios on both sides of both borders, none within 1e-3 of one
    drift = torch.tensor([0.0, 0.1, -0.1, 0.3, -0.3, 0.05, -0.5], device=dev)
    pick = torch.randint(0, 7, shape, device=dev, generator=g)
    old = (lp - drift[pick]).float()
    adv = torch.randn(shape, device=dev, generator=g)
    ref = (lp + 0.3 * torch.randn(shape, device=dev, generator=g)).float()
    mask = torch.rand(shape, device=dev, generator=g) < 0.7
    return logits, targets, old, adv, ref, mask


def check_policy(r, grad, logits, targets, old, adv, ref, mask, low, high, kl, temperature=1.0, up=1.0):
    lp, p, tol, sum_err = exact(logits, targets, temperature)
    keep = torch.ones_like(lp) if mask is None else mask.double()
    lp, old, adv = lp * keep, torch.where(keep > 0, old.double(), 0.0), torch.where(keep > 0, adv.double(), 0.0)
    assert bool(((r.logprobs.double() - lp).abs() <= tol * keep).all())
    n = max(1.0, float(keep.sum()))
    ratio = torch.exp(lp - old)
    term = -torch.minimum(ratio * adv, ratio.clamp(1 - low, 1 + high) * adv)
    live = torch.where(adv >= 0, ratio <= 1 + high, ratio >= 1 - low)
    c = torch.where(live, -ratio * adv, 0.0)
    steep = ratio * adv.abs()                              # |d c / d lp| and |d term / d lp|
    if kl:
        gap = torch.where(keep > 0, ref.double(), 0.0) - lp
        term = term + kl * (torch.expm1(gap) - gap)
        c = c - kl * torch.expm1(gap)
        steep = steep + kl * (torch.exp(gap) + 1)
    # terms and coefficients are rounded to fp32 once, their clip distances and weights once each
    off = steep * tol + 4 * E * (term.abs() + steep)
    loss = float((term * keep).sum()) / n
    assert abs(float(r.loss.detach()) - loss) <= float((off * keep).sum()) / n + 2 * E * abs(loss)
    check_grad(grad, p, targets, up * c * keep / n, abs(up) * keep * (steep * tol + 6 * E * (c.abs() + steep)) / n,
               temperature, sum_err, keep)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,V", [((1,), 8), ((5,), 1000), ((3, 7), 4099), ((2, 300), 520), ((2, 9), 50304)])
def test_policy_loss(dev, dtype, shape, V):
    logits, targets, old, adv, ref, mask = policy_case(dev, shape, V, dtype, seed=V)
    logits.requires_grad_(True)
    for kw in (dict(), dict(mask=mask), dict(ref_logprobs=ref, kl_weight=0.1, mask=mask),
               dict(ref_logprobs=ref, kl_weight=0.2, clip_low=0.15, clip_high=0.28)):
        r = policy_loss(logits, targets, old, adv, **kw)
        (grad,) = torch.autograd.grad(r.loss, [logits])
        check_policy(r, grad, logits.detach(), targets, old, adv, ref, kw.get("mask"), kw.get("clip_low", 0.2),
                     kw.get("clip_high", 0.2), kw.get("kl_weight", 0.0))


def test_policy_temperature_broadcast_and_scale(dev):
    logits, targets, _, _, ref, mask = policy_case(dev, (4, 33), 777, torch.bfloat16)
    logits.requires_grad_(True)
    with torch.no_grad():
        old = token_logprobs(logits, targets, temperature=1.3) - 0.05
    adv = torch.randn(4, 1, device=dev)
    r = policy_loss(logits, targets, old, adv, mask=mask[:, :1], temperature=1.3)
    # the gradient is computed anew where the loss's is not 1, and by every backward but the first
    (a,) = torch.autograd.grad(r.loss, [logits], retain_graph=True)
    (grad,) = torch.autograd.grad(-2.5 * r.loss, [logits], retain_graph=True)
    (b,) = torch.autograd.grad(r.loss, [logits])
    args = (logits.detach(), targets, old, adv.expand(4, 33), ref, mask[:, :1].expand(4, 33), 0.2, 0.2, 0.0, 1.3)
    for g, up in ((a, 1.0), (grad, -2.5), (b, 1.0)):
        check_policy(r, g, *args, up)
    s = policy_loss(logits, targets, old, adv, mask=mask[:, :1], temperature=1.3, scale=0.25)
    assert abs(float(s.loss.detach()) - 0.25 * float(r.loss.detach())) <= 4 * E * abs(float(r.loss.detach()))
    (grad,) = torch.autograd.grad(s.loss, [logits])
    check_policy(r, grad, *args, 0.25)


def test_policy_backward_in_another_graph(dev, monkeypatch):
    """A backward that is recorded into another graph than the forward (or into one, where the
    forward was not) writes a tensor of its own, whatever the loss's gradient: a replay finds no
    forward before it."""
    logits, targets, old, adv, ref, mask = policy_case(dev, (2, 30), 1000, torch.float32)
    logits.requires_grad_(True)
    first = []
    empty = torch.empty
    with monkeypatch.context() as m:
        m.setattr(torch, "empty", lambda *a, **k: first.append(empty(*a, **k)) or first[-1])
        r = policy_loss(logits, targets, old, adv, mask=mask)
    assert [t.shape for t in first] == [logits.shape]        # the forward's gradient
    first[0].fill_(7.0)
    monkeypatch.setattr(_lib.lib(), "lema_capture_id", lambda stream: 5)
    (g,) = torch.autograd.grad(r.loss, [logits])
    assert g.data_ptr() != first[0].data_ptr() and bool((first[0] == 7.0).all())
    check_policy(r, g, logits.detach(), targets, old, adv, ref, mask, 0.2, 0.2, 0.0)


def test_masked_rows_are_not_read(dev):
    """Whatever a left-out position holds: NaN and infinite logits, log-probabilities and
    advantages, targets outside the vocabulary. With nothing counted the loss is 0."""
    logits, targets, old, adv, ref, mask = policy_case(dev, (3, 40), 1001, torch.float32)
    mask[1] = False
    clean = [t.clone() for t in (logits, targets, old, adv, ref)]
    bad = ~mask
    logits[bad], old[bad], adv[bad], ref[bad] = float("nan"), -float("inf"), float("inf"), float("nan")
    targets[bad] = -100

    def both(logits, targets, old, adv, ref, mask):
        x = logits.clone().requires_grad_(True)
        a = policy_loss(x, targets, old, adv, ref, mask, kl_weight=0.1)
        b = preference_loss(x[:2], targets[:2], ref[:2], mask[:2])
        return (a.loss, a.logprobs, *torch.autograd.grad(a.loss, [x]), b.loss, b.margins, b.logprobs,
                *torch.autograd.grad(b.loss, [x]), token_logprobs(logits, targets, mask))
    got, want = both(logits, targets, old, adv, ref, mask), both(*clean, mask)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    out = both(logits, targets, old, adv, ref, torch.zeros_like(mask))
    assert float(out[0]) == 0.0 and not out[2].any()
    assert abs(float(out[3]) - math.log(2)) <= 2 * E and not out[6].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pairs,T,V", [(1, 1, 8), (3, 5, 1001), (17, 30, 64), (2, 700, 520), (2, 11, 50304)])
def test_preference_loss(dev, dtype, pairs, T, V):
    logits, targets, g = make(dev, (2 * pairs, T), V, dtype, seed=V + T)
    lp, p, tol, sum_err = exact(logits, targets, 1.0)
    ref = (lp + 0.2 * torch.randn(lp.shape, device=dev, generator=g)).float()
    full = torch.rand(lp.shape, device=dev, generator=g) < 0.8
    logits.requires_grad_(True)
    for mask, beta, smooth in ((None, 0.1, 0.0), (full, 0.3, 0.1), (full, -0.2, 1.0)):
        keep = torch.ones_like(lp) if mask is None else mask.double()
        r = preference_loss(logits, targets, ref, mask, beta=beta, label_smoothing=smooth)
        (grad,) = torch.autograd.grad(r.loss, [logits])
        s = ((lp - ref.double()) * keep).sum(1)
        m = beta * (s[:pairs] - s[pairs:])
        dm = abs(beta) * (tol * keep).sum(1).view(2, -1).sum(0) + 4 * E * m.abs()
        assert bool(((r.margins.double() - m).abs() <= dm).all())
        ls = torch.nn.functional.logsigmoid
        loss = float((-(1 - smooth) * ls(m) - smooth * ls(-m)).mean())
        assert abs(float(r.loss.detach()) - loss) <= float(dm.mean()) + 4 * E * (abs(loss) + float(m.abs().mean()))
        cm = (-(1 - smooth) * torch.sigmoid(-m) + smooth * torch.sigmoid(m)) * beta / pairs
        dc = (dm / 4 + 6 * E) * abs(beta) / pairs
        c, dc = torch.cat([cm, -cm])[:, None] * keep, torch.cat([dc, dc])[:, None] * keep
        check_grad(grad, p, targets, c, dc, 1.0, sum_err, keep)


def test_preference_without_tokens(dev):
    x = torch.zeros(4, 0, 9, device=dev, requires_grad=True)
    r = preference_loss(x, torch.zeros(4, 0, dtype=torch.long, device=dev), torch.zeros(4, 0, device=dev))
    assert abs(float(r.loss.detach()) - math.log(2)) <= 2 * E and r.margins.tolist() == [0.0, 0.0]
    (g,) = torch.autograd.grad(r.loss, [x])
    assert g.shape == x.shape
    r = policy_loss(x, torch.zeros(4, 0, dtype=torch.long, device=dev), torch.zeros(4, 0, device=dev),
                    torch.zeros(4, 0, device=dev))
    assert float(r.loss) == 0.0


def test_differences(dev):
    """The loss's gradient along a direction against central differences of the loss in fp32: a
    step of 2^-5 over a direction of norm 1 leaves t^2 times a third derivative below 8, and the
    two losses' roundings, 64 E of at most 4 each, over the step."""
    logits, targets, old, adv, ref, mask = policy_case(dev, (2, 10), 50, torch.float32)
    v = torch.randn_like(logits)
    v /= v.norm()
    t = 2.0 ** -5
    for f in (lambda x: policy_loss(x, targets, old, adv, ref, mask, clip_low=5.0, clip_high=5.0, kl_weight=0.3).loss,
              lambda x: preference_loss(x, targets, ref, mask, beta=0.5, label_smoothing=0.1).loss,
              lambda x: token_logprobs(x, targets).mean()):
        x = logits.clone().requires_grad_(True)
        (g,) = torch.autograd.grad(f(x), [x])
        with torch.no_grad():
            diff = (f(logits + t * v).double() - f(logits - t * v).double()) / (2 * t)
        assert abs(float(diff - (g.double() * v).sum())) <= 8 * t * t + 64 * E * 4 / t


@pytest.mark.parametrize("V", [8, 2056, 50304])
def test_cross_entropy_gradient(dev, V):
    logits, targets, _ = make(dev, (40,), V, torch.bfloat16, seed=V)
    logits[3, : V // 2] = -float("inf")
    targets[3] = V - 1
    plain = cross_entropy_sum(logits, targets)
    _, p, _, sum_err = exact(logits, targets, 1.0)
    x = logits.clone().requires_grad_(True)
    loss = cross_entropy_sum(x, targets)
    assert torch.equal(loss, plain)
    (g,) = torch.autograd.grad(3.0 * loss, [x])
    c = torch.full((40,), -3.0, device=dev, dtype=torch.float64)
    check_grad(g, p, targets, c, 0 * c, 1.0, sum_err)


def test_retained_and_hooks(dev):
    logits, targets, old, adv, ref, mask = policy_case(dev, (2, 30), 1003, torch.bfloat16)
    logits.requires_grad_(True)

    def losses():
        a = policy_loss(logits, targets, old, adv, ref, mask, kl_weight=0.1).loss
        b = preference_loss(logits, targets, ref, mask).loss
        return a + 0.5 * b + token_logprobs(logits, targets, mask).sum()
    (want,) = torch.autograd.grad(losses(), [logits])
    with torch.autograd.graph.saved_tensors_hooks(
            lambda t: t.cpu().long() if t.dtype == torch.bool else t.cpu(), lambda t: t):
        loss = losses()
    (a,) = torch.autograd.grad(loss, [logits], retain_graph=True)
    (b,) = torch.autograd.grad(loss, [logits])
    assert torch.equal(a, want) and torch.equal(b, want)
    with pytest.raises(RuntimeError):
        (a,) = torch.autograd.grad(losses(), [logits], create_graph=True)
        a.sum().backward()


def test_captured_step(dev):
    """Forward and gradient of all three in a graph. No eager graph of the same logits is alive
    meanwhile: torch would order the captured gradient after that graph's stream, which a capture
    cannot."""
    logits, targets, old, adv, ref, mask = policy_case(dev, (2, 30), 1003, torch.bfloat16)
    logits.requires_grad_(True)

    def losses():
        a = policy_loss(logits, targets, old, adv, ref, mask, kl_weight=0.1).loss
        b = preference_loss(logits, targets, ref, mask).loss
        return a + 0.5 * b + token_logprobs(logits, targets, mask).sum()
    step = lambda: torch.autograd.grad(losses(), [logits])[0]  # noqa: E731
    s = torch.cuda.Stream(dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream(dev).wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        mask.copy_(torch.rand_like(old) < 0.5)
        adv.copy_(torch.randn_like(adv))
        want = step()
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_refusals(dev):
    x = torch.randn(4, 3, 20, device=dev)
    t = torch.zeros(4, 3, dtype=torch.long, device=dev)
    z = torch.zeros(4, 3, device=dev)
    for bad in (lambda: token_logprobs(x.double(), t), lambda: token_logprobs(x, z),
                lambda: token_logprobs(x, t, z), lambda: policy_loss(x, t, t, z),
                lambda: token_logprobs(x.cpu(), t), lambda: preference_loss(x, t, z.cpu())):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: token_logprobs(x, t[:3]), lambda: token_logprobs(x, t, temperature=0.0),
                lambda: token_logprobs(x, t, temperature=float("nan")), lambda: token_logprobs(x, t, temperature=1e-40),
                lambda: token_logprobs(x[..., :0], t), lambda: policy_loss(x, t, z[:3], z),
                lambda: policy_loss(x, t, z, z, clip_low=-0.1), lambda: policy_loss(x, t, z, z, kl_weight=0.1),
                lambda: preference_loss(x[:3], t[:3], z[:3]), lambda: preference_loss(x[0], t[0], z[0]),
                lambda: preference_loss(x[:0], t[:0], z[:0]), lambda: preference_loss(x, t, z, label_smoothing=1.5),
                lambda: preference_loss(x, t, z, beta=float("inf")),
                lambda: token_logprobs(x, t, torch.ones(4, 3, dtype=torch.bool))):
        with pytest.raises(ValueError):
            bad()
