"""The losses where logits, targets and margins leave the ordinary: a vocabulary that is partly banned
(-inf logits) at any temperature, against the same logits in 64 bits; targets outside the vocabulary;
answers that cannot occur."""
import pytest
import torch
from test_gpu_loss import E, TYPES, check_grad, exact, make

from latest_exact_match_attention_amd.loss import policy_loss, preference_loss, token_logprobs
from latest_exact_match_attention_amd.model import cross_entropy_sum

pytestmark = pytest.mark.gpu

# log2 e / temperature lies above its nearest float at the first four and below it at the next five; at
# the last it has one, to within fp32's smallest step
TEMPERATURES = [1.0, 1.3, 0.5, 1e-3, 0.7, 0.8, 1.5, 0.1, 1e37, 1e38]


def banned(dev, shape, V, dtype, seed=0):
    """Logits with -inf for a quarter of the words of each row, and for all behind three quarters of
    the vocabulary (its padding); targets among the others."""
    logits, _, g = make(dev, shape, V, dtype, seed)
    ban = torch.rand(logits.shape, device=dev, generator=g) < 0.25
    ban[..., V - V // 4:] = True
    ban[..., 0] = False
    targets = (~ban).float().view(-1, V).multinomial(1, generator=g).view(shape)
    return logits.masked_fill(ban, -float("inf")), targets, ban, g


def check(grad, p, targets, c, dc, temperature, sum_err):
    """check_grad, with no NaN, and with softmax terms below 2^-126 apart: fp32's exponential leaves 0
    of them, so that up to 2^-126 |c / temperature| is lost, where check_grad allows 2^-126. (At a
    temperature of 0.1 a term of 0.36 2^-126 times a factor of 3.8 is 1.4 2^-126.)"""
    assert bool(grad.isfinite().all())
    small = (p < 2.0 ** -126) & (torch.arange(p.shape[-1], device=p.device) != targets[..., None])
    lost = 2.0 ** -126 * (c.abs()[..., None] / temperature + 1)
    assert bool((grad.double().abs() <= lost)[small].all())
    check_grad(grad.masked_fill(small, 0), p.masked_fill(small, 0), targets, c, dc, temperature, sum_err)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [12, 1001, 50304, 131073])
@pytest.mark.parametrize("temperature", TEMPERATURES)
def test_banned_words(dev, dtype, V, temperature):
    """Rows of V above 256 KB take the kernels that do not hold a row."""
    logits, targets, ban, g = banned(dev, (4, 3), V, dtype, seed=V)
    logits.requires_grad_(True)
    lp, p, tol, sum_err = exact(logits.detach(), targets, temperature)
    c = torch.randn(4, 3, device=dev, generator=g)
    got = token_logprobs(logits, targets, temperature=temperature)
    assert bool(((got.double() - lp).abs() <= tol).all())
    (grad,) = torch.autograd.grad(got, [logits], c)
    check(grad, p, targets, c.double(), 0 * lp, temperature, sum_err)
    assert not grad[ban].any()

    r = preference_loss(logits, targets, lp.float(), beta=0.3, temperature=temperature)
    m = 0.3 * (lp - lp.float().double()).view(2, 2, 3).sum(2)
    m, dm = m[0] - m[1], 0.3 * tol.view(2, 2, 3).sum((0, 2)) + 4 * E
    assert bool(((r.margins.double() - m).abs() <= dm).all())
    (grad,) = torch.autograd.grad(r.loss, [logits])
    c = -torch.sigmoid(-m) * 0.3 / 2
    dc = (dm / 4 + 6 * E) * 0.3 / 2
    check(grad, p, targets, torch.cat([c, -c])[:, None].expand(4, 3), torch.cat([dc, dc])[:, None].expand(4, 3),
               temperature, sum_err)

    # the policy loss: the gradient that the forward wrote, one of a scaled loss, and a second one.
    # old = lp: a ratio of 1 but for lp's own error, inside the clip distances
    adv = torch.linspace(-1, 1, 12, device=dev).view(4, 3)
    r = policy_loss(logits, targets, lp.float(), adv, temperature=temperature, clip_low=1.0, clip_high=1e3)
    assert bool(((r.logprobs.double() - lp).abs() <= tol).all())
    ratio = torch.exp(lp - lp.float().double())
    c = -ratio * adv.double() / 12
    for up in (1.0, 2.0, 1.0):
        (grad,) = torch.autograd.grad(up * r.loss, [logits], retain_graph=True)
        check(grad, p, targets, up * c, up * c.abs() * (tol + 8 * E), temperature, sum_err)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temperature", TEMPERATURES)
def test_lowest_values(dev, dtype, temperature):
    """Masks of the type's lowest value; a row of them alone is uniform; a NaN and a row of -inf alone
    give NaN. A distance to the row's maximum that leaves fp32's range counts as infinite (2^129 of
    the widest types' values in row 2, which a temperature of 1e38 alone would bring back to 6.8: the
    row's sum is then 1, not 1 + 2099 e^-6.8)."""
    V = 2100
    low, top = torch.finfo(dtype).min, torch.finfo(dtype).max
    x = torch.zeros(5, V, device=dev, dtype=dtype)
    x[0, 7:] = low
    x[1] = low
    x[2], x[2, 1999] = low, top
    x[3, 5:], x[3, 1000] = -float("inf"), float("nan")
    x[4] = -float("inf")
    t = torch.tensor([3, 5, 1999, 0, 0], device=dev)
    x.requires_grad_(True)
    lp = token_logprobs(x, t, temperature=temperature)
    d = x.detach().double()
    d = d - d.amax(-1, keepdim=True)
    d = d.masked_fill(d < torch.finfo(torch.float32).min, -float("inf"))
    want = torch.log_softmax(d / temperature, -1).gather(1, t[:, None])[:, 0]
    # far from a maximum's own rounding: distances of 0, or of more than the exponential's range
    far = 64 * E * want.abs().clamp_min(1)
    assert bool(((lp.double() - want).abs() <= far)[:3].all()) and bool(lp[3:].isnan().all())
    (g,) = torch.autograd.grad(lp, [x], torch.ones_like(lp))
    assert bool(g[:3].isfinite().all()) and bool(g[3:].isnan().all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [8, 1000, 50304])
def test_targets_outside_the_vocabulary(dev, dtype, V):
    """NaN where the log-probability or the loss is: a wrong target shows in the gradient too, not as
    a descent on the whole row. A gradient of 0 of such a log-probability leaves its row alone."""
    logits, targets, _ = make(dev, (4, 3), V, dtype, seed=V)
    bad = torch.zeros(4, 3, dtype=torch.bool, device=dev)
    bad[0, 1] = bad[1, 0] = bad[3, 2] = True
    targets[0, 1], targets[1, 0], targets[3, 2] = -100, V, 1 << 32
    logits.requires_grad_(True)
    lp = token_logprobs(logits, targets)
    assert torch.equal(lp.isnan(), bad)
    (g,) = torch.autograd.grad(lp, [logits], torch.ones_like(lp), retain_graph=True)
    assert bool(g[bad].isnan().all() and g[~bad].isfinite().all())
    (g,) = torch.autograd.grad(torch.where(bad, 0.0, lp).sum(), [logits])
    assert bool(g.isfinite().all()) and not g[bad].any() and bool(g[~bad].any())
    if dtype == torch.bfloat16:
        loss = cross_entropy_sum(logits.flatten(0, 1), targets)
        (g,) = torch.autograd.grad(loss, [logits])
        assert bool(loss.isnan() and g[bad].isnan().all() and g[~bad].isfinite().all())
    z = torch.zeros(4, 3, device=dev)
    r = policy_loss(logits, targets, z, z + 1, clip_high=1e3)
    for up in (1.0, 2.0):
        (g,) = torch.autograd.grad(up * r.loss, [logits], retain_graph=True)
        assert bool(r.loss.isnan() and g[bad].isnan().all() and g[~bad].isfinite().all())


@pytest.mark.parametrize("pairs", [1, 3, 20])
@pytest.mark.parametrize("smooth", [0.0, 1.0, 0.25])
@pytest.mark.parametrize("side", [0, 1])
def test_infinite_margins(dev, pairs, smooth, side):
    """An answer with a banned word is infinitely unlikely. Its pair costs nothing where the loss
    asks for the other answer (and is infinite where it asks for this one at all), and the other
    pairs keep their gradients."""
    V, T = 40, 5
    logits, targets, _ = make(dev, (2 * pairs, T), V, torch.float32, seed=7)
    lp = torch.log_softmax(logits.double(), -1).gather(-1, targets[..., None])[..., 0]
    row = side * pairs
    logits[row, 2, targets[row, 2]] = -float("inf")
    logits.requires_grad_(True)
    ref = torch.full((2 * pairs, T), -3.0, device=dev)
    r = preference_loss(logits, targets, ref, beta=0.5, label_smoothing=smooth)
    (g,) = torch.autograd.grad(r.loss, [logits])
    m = 0.5 * ((lp[:pairs] + 3).sum(1) - (lp[pairs:] + 3).sum(1))
    m[0] = float("inf") if side else -float("inf")
    ls = torch.nn.functional.logsigmoid
    term = torch.zeros_like(m)
    if smooth < 1:
        term -= (1 - smooth) * ls(m)
    if smooth > 0:
        term -= smooth * ls(-m)
    assert float(r.margins[0]) == float(m[0])
    free = smooth == (0.0 if side else 1.0)
    if free:
        # margins of some tens are off by less than 64 E each, and a term by as much
        assert abs(float(r.loss.detach()) - float(term.mean())) <= 64 * 64 * E
    else:
        assert float(r.loss.detach()) == float("inf")
    assert bool(g.isfinite().all())
    assert bool(g[row].any()) == (not free)
    assert pairs == 1 or bool(g[1].any() and g[pairs + 1].any())
