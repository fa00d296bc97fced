"""The operators of a fine-tuning step around the exact op, as cases that can be timed and checked.

Four kinds, each with its gradient (`grad`) or without:

  embed    token rows of a table times a scale; the gradient adds up the rows of equal tokens
  norm     layer norm or RMS norm of x, or of x + d where a residual branch is added first; the
           gradients of x, d and the weights
  policy   clipped policy loss with a KL term, from logits: loss, log-probabilities, gradient
  pref     paired preference loss, from logits of chosen and rejected sequences

`run` computes them in elementary tensor operations, or through the package where `own` is set.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # a decode step's token embedding, 16 streams, rows scaled by sqrt(dim)
        dict(name="embed_step", kind="embed", n=16, vocab=50304, D=1536, dtype="bf16",
             scale=1536 ** 0.5, pad=0.0, grad=False),
        # the language model's table under a batch of 4 x 16384 tokens
        dict(name="embed_train", kind="embed", n=65536, vocab=50304, D=1536, dtype="bf16",
             scale=1.0, pad=0.0, grad=True),
        # a padded batch of a small fp32 model, odd everywhere
        dict(name="embed_padded", kind="embed", n=5003, vocab=32003, D=771, dtype="f32",
             scale=771 ** 0.5, pad=0.3, grad=True),
        # a decode step's norm with the residual add
        dict(name="layer_norm_step", kind="norm", center=True, rows=16, D=1536, dtype="bf16",
             add=True, grad=False),
        # training, wide rows in half precision
        dict(name="layer_norm_train", kind="norm", center=True, rows=8192, D=4096, dtype="f16",
             add=True, grad=True),
        # odd rows in fp32: nothing is aligned to a vector
        dict(name="layer_norm_odd", kind="norm", center=True, rows=4099, D=1001, dtype="f32",
             add=False, grad=True),
        # the model's pre-norm with its residual add over a batch of 4 x 16384 tokens
        dict(name="rms_norm_train", kind="norm", center=False, rows=65536, D=1536, dtype="bf16",
             add=True, grad=True),
        # one short sequence of a fine-tuning set
        dict(name="rms_norm_short", kind="norm", center=False, rows=200, D=2048, dtype="bf16",
             add=False, grad=True),
        # a handful of short answers
        dict(name="policy_short", kind="policy", seqs=4, T=50, vocab=50304, dtype="bf16",
             temperature=1.0, kl=0.05),
        # a batch of sampled answers, one update's worth of logits
        dict(name="policy_batch", kind="policy", seqs=16, T=1024, vocab=50304, dtype="bf16",
             temperature=0.8, kl=0.05),
        # two short pairs of a small fp32 model with an odd vocabulary
        dict(name="pref_short", kind="pref", seqs=4, T=96, vocab=32003, dtype="f32"),
        # four pairs of answers of up to 1,024 tokens
        dict(name="pref_batch", kind="pref", seqs=8, T=1024, vocab=50304, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    """A whole number spread over [lo, hi] by its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["embed", "norm", "norm", "policy", "pref"])
    if kind == "embed":
        # no more elements of output and table together than embed_train has, bytes counted
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        cap = (65536 + 50304) * 1536 // (2 if dtype == "f32" else 1)
        D = _log(rng, 32, 4096)
        D = D if rng.random() < 0.3 else max(8, D // 8 * 8)
        vocab = min(_log(rng, 1000, 131072), cap // (2 * D))
        n = min(_log(rng, 1, 65536), cap // D - vocab)
        return dict(kind=kind, n=n, vocab=vocab, D=D, dtype=dtype,
                    scale=rng.choice([1.0, D ** 0.5]), pad=rng.choice([0.0, 0.0, 0.4]),
                    grad=rng.random() < 0.8)
    if kind == "norm":
        center = rng.random() < 0.6
        dtype = rng.choice(["bf16", "f16", "f32"]) if center else "bf16"
        # the RMS norm is the model's: bf16 rows of a multiple of 8, at most 4096
        D = _log(rng, 64, 8192 if center else 4096)
        D = D if center and rng.random() < 0.3 else max(8, D // 8 * 8)
        cap = 65536 * 1536 // (2 if dtype == "f32" else 1)
        return dict(kind=kind, center=center, rows=min(_log(rng, 1, 65536), cap // D), D=D,
                    dtype=dtype, add=rng.random() < 0.5, grad=rng.random() < 0.8)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    vocab = _log(rng, 1000, 131072)
    vocab = vocab if rng.random() < 0.3 else max(8, vocab // 8 * 8)
    cap = (16384 if kind == "policy" else 8192) * 50304 // (2 if dtype == "f32" else 1) // vocab
    seqs = min(2 * rng.choice([1, 2, 4, 8]), max(2, cap // 2 * 2))
    T = min(_log(rng, 1, 2048), max(1, cap // seqs))
    if kind == "pref":
        return dict(kind=kind, seqs=seqs, T=T, vocab=vocab, dtype=dtype)
    return dict(kind=kind, seqs=seqs, T=T, vocab=vocab, dtype=dtype,
                temperature=rng.choice([1.0, 0.7, 1.3]), kl=rng.choice([0.0, 0.02, 0.2]))


# ------------------------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _answer(c):
    """[seqs, T] truth values: which positions a loss counts. A sequence opens with a prompt (up
    to a quarter of it) and may end early (its padding); a sequence in seven has no answer left
    when there are that many. The same for every seed: the work of a case is fixed."""
    i = torch.arange(c["seqs"])
    u = (i * 0.618034 + 0.3) % 1.0
    start = (c["T"] * 0.25 * u).long()
    stop = torch.ceil(c["T"] * (0.55 + 0.45 * ((i * 0.754878 + 0.9) % 1.0))).long()
    stop = torch.where(i % 7 == 6, start, stop)
    t = torch.arange(c["T"])
    return (t >= start[:, None]) & (t < stop[:, None])


def _prepare_embed(c, seed):
    g, dt = _gen(seed), DTYPES[c["dtype"]]
    V, D, n = c["vocab"], c["D"], c["n"]
    # tokens of text: Zipf frequencies, frequent tokens anywhere in the table
    p = torch.arange(1, V + 1, dtype=torch.float64, device="cuda") ** -1.05
    cdf = torch.cumsum(p / p.sum(), 0)
    rank = torch.searchsorted(cdf, torch.rand(n, generator=g, device="cuda",
                                              dtype=torch.float64)).clamp_(max=V - 1)
    ids = torch.randperm(V, generator=g, device="cuda")[rank]
    pad = 0 if c["pad"] else None
    if c["pad"]:  # the batch's sequences end in padding
        ids[int(n * (1 - c["pad"])):] = 0
    w = (_randn(g, V, D) * D ** -0.5).to(dt)
    emb = torch.nn.Embedding(V, D, padding_idx=pad, _weight=w)
    s = dict(kind="embed", emb=emb, ids=ids, scale=c["scale"], grad=c["grad"])
    if c["grad"]:
        s["gy"] = (_randn(g, n, D) * 1e-2).to(dt)
    return s


def _prepare_norm(c, seed):
    g, dt = _gen(seed), DTYPES[c["dtype"]]
    R, D = c["rows"], c["D"]
    make = torch.nn.LayerNorm if c["center"] else torch.nn.RMSNorm
    norm = make(D, eps=1e-5, device="cuda", dtype=dt)
    with torch.no_grad():
        norm.weight.copy_(1 + 0.2 * _randn(g, D))
        if c["center"]:
            norm.bias.copy_(0.1 * _randn(g, D))
    # a residual stream: rows of different sizes, a common offset, a few large channels
    x = _randn(g, R, D) * torch.exp(0.5 * _randn(g, R, 1)) + 0.3
    x[:, :: 97] *= 8.0
    s = dict(kind="norm", norm=norm, center=c["center"], x=x.to(dt), grad=c["grad"])
    s["d"] = (0.5 * _randn(g, R, D)).to(dt) if c["add"] else None
    if c["grad"]:
        s["x"].requires_grad_(True)
        s["gh"] = (_randn(g, R, D) * 0.1).to(dt)
        if c["add"]:
            s["d"].requires_grad_(True)
            s["gs"] = (_randn(g, R, D) * 0.1).to(dt)
    return s


def _prepare_loss(c, seed):
    g, dt = _gen(seed), DTYPES[c["dtype"]]
    N, T, V = c["seqs"], c["T"], c["vocab"]
    temp = c.get("temperature", 1.0)
    logits = torch.empty(N, T, V, dtype=dt, device="cuda")
    targets = torch.empty(N, T, dtype=torch.long, device="cuda")
    lp = torch.empty(N, T, device="cuda")
    step = max(1, (1 << 27) // (T * V))
    for a in range(0, N, step):
        # a language model's predictions: a few likely words over a broad tail; the tokens are
        # sampled from them at the temperature
        x = 2.0 * _randn(g, min(step, N - a), T, V)
        top = torch.randint(0, V, x.shape[:2] + (1,), generator=g, device="cuda")
        x.scatter_add_(2, top, 4 + 8 * torch.rand(top.shape, generator=g, device="cuda"))
        logits[a:a + step] = x.to(dt)
        x = logits[a:a + step].float() / temp
        e = torch.empty_like(x).exponential_(generator=g).clamp_min_(1e-20)
        t = (x - e.log()).argmax(-1)
        targets[a:a + step] = t
        lp[a:a + step] = torch.log_softmax(x, -1).gather(-1, t[..., None])[..., 0]
    mask = _answer(c).cuda()
    s = dict(kind=c["kind"], logits=logits.requires_grad_(True), targets=targets, mask=mask,
             temperature=temp)
    if c["kind"] == "policy":
        # the policy has moved since the answers were sampled; the reference is further away.
        # A ratio within 1e-3 of a clip border is moved off it: which side of the border such a
        # row falls on is decided by rounding
        drift = 0.15 * _randn(g, N, T)
        for edge in (math.log(0.8), math.log(1.2)):
            near = (drift - edge).abs() < 1.5e-3
            drift = torch.where(near, torch.full_like(drift, edge + 3e-3), drift)
        s["old"] = torch.where(mask, lp - drift, 0.0)
        s["ref"] = torch.where(mask, lp + 0.3 * _randn(g, N, T), 0.0)
        s["adv"] = _randn(g, N, 1).expand(N, T)          # one advantage for each answer
        s["kl"] = c["kl"]
    else:
        s["ref"] = torch.where(mask, lp + 0.2 * _randn(g, N, T), 0.0)
    return s


def prepare(case, seed):
    if case["kind"] == "embed":
        return _prepare_embed(case, seed)
    if case["kind"] == "norm":
        return _prepare_norm(case, seed)
    return _prepare_loss(case, seed)


# ------------------------------------------------------------------------- the package's calls

def _own_embed(s):
    from latest_exact_match_attention_amd.model import embed
    if not s["grad"]:
        with torch.no_grad():
            return [embed(s["emb"], s["ids"], s["scale"])]
    y = embed(s["emb"], s["ids"], s["scale"])
    return [y.detach(), *torch.autograd.grad(y, [s["emb"].weight], s["gy"])]


def _own_norm(s):
    from latest_exact_match_attention_amd.model import layer_norm, rms_norm
    f, norm, x, d = (layer_norm if s["center"] else rms_norm), s["norm"], s["x"], s["d"]
    if not s["grad"]:
        with torch.no_grad():
            h, r = f(x, norm, d)
        return [h] if d is None else [h, r]
    wrt = [x] + ([d] if d is not None else []) + list(norm.parameters())
    h, r = f(x, norm, d)
    if d is None:
        return [h.detach(), *torch.autograd.grad(h, wrt, s["gh"])]
    return [h.detach(), r.detach(), *torch.autograd.grad([h, r], wrt, [s["gh"], s["gs"]])]


def _own_policy(s):
    from latest_exact_match_attention_amd.loss import policy_loss
    r = policy_loss(s["logits"], s["targets"], s["old"], s["adv"], ref_logprobs=s["ref"],
                    mask=s["mask"], clip_low=0.2, clip_high=0.2, kl_weight=s["kl"],
                    temperature=s["temperature"])
    return [r.loss.detach(), r.logprobs, *torch.autograd.grad(r.loss, [s["logits"]])]


def _own_pref(s):
    from latest_exact_match_attention_amd.loss import preference_loss
    r = preference_loss(s["logits"], s["targets"], s["ref"], mask=s["mask"], beta=0.1,
                        label_smoothing=0.05)
    return [r.loss.detach(), r.margins, r.logprobs, *torch.autograd.grad(r.loss, [s["logits"]])]


# -------------------------------------------------------------------------------- plain forms

def _plain_embed(s):
    w, ids = s["emb"].weight.detach(), s["ids"]
    y = (w[ids].float() * s["scale"]).to(w.dtype)
    if not s["grad"]:
        return [y]
    gw = torch.zeros(w.shape, device=w.device)
    gw.index_add_(0, ids, s["gy"].float())
    gw = gw * s["scale"]
    if s["emb"].padding_idx is not None:
        gw[s["emb"].padding_idx] = 0
    return [y, gw.to(w.dtype)]


def _plain_norm(s):
    dt, norm = s["x"].dtype, s["norm"]
    x, w = s["x"].detach().float(), norm.weight.detach().float()
    if s["d"] is not None:
        r = (x + s["d"].detach().float()).to(dt)
        x = r.float()
    z = x - x.mean(-1, keepdim=True) if s["center"] else x
    rstd = torch.rsqrt((z * z).mean(-1, keepdim=True) + norm.eps)
    z = z * rstd
    h = z * w
    if s["center"]:
        h = h + norm.bias.detach().float()
    out = [h.to(dt)] + ([r] if s["d"] is not None else [])
    if not s["grad"]:
        return out
    gh = s["gh"].float()
    a = gh * w
    gx = a - z * (a * z).mean(-1, keepdim=True)
    if s["center"]:
        gx = gx - a.mean(-1, keepdim=True)
    gx = gx * rstd
    if s["d"] is not None:
        gx = gx + s["gs"].float()
    gx = gx.to(dt)
    out += [gx] + ([gx] if s["d"] is not None else []) + [(gh * z).sum(0).to(dt)]
    return out + ([gh.sum(0).to(dt)] if s["center"] else [])


def _plain_logprobs(s):
    """Per row the softmax's numerators and their sum, and the target's log-probability: in 64
    bits from that sum on, because a preference adds up those of a whole answer."""
    x = s["logits"].detach().float()
    if s["temperature"] != 1.0:
        x = x / s["temperature"]
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    z = e.sum(-1, keepdim=True)
    lp = x.gather(-1, s["targets"][..., None]).double() - top.double() - torch.log(z.double())
    return e, z, torch.where(s["mask"], lp[..., 0], 0.0)


def _plain_grad(s, e, z, c):
    """c (onehot - softmax) / temperature, rounded to the logits' type."""
    c = torch.where(s["mask"], c, 0.0)[..., None] / s["temperature"]
    g = e * (-c / z)
    g.scatter_add_(-1, s["targets"][..., None], c)
    return g.to(s["logits"].dtype)


def _plain_policy(s):
    e, z, lp = _plain_logprobs(s)
    lp = lp.float()
    mask, adv = s["mask"], s["adv"]
    n = mask.sum().clamp_min(1)
    r = torch.exp(lp - s["old"])
    term = -torch.minimum(r * adv, r.clamp(0.8, 1.2) * adv)
    live = torch.where(adv >= 0, r <= 1.2, r >= 0.8)
    c = torch.where(live, -r * adv, 0.0)
    far = torch.exp(s["ref"] - lp)
    term = term + s["kl"] * (far - (s["ref"] - lp) - 1)
    c = c + s["kl"] * (1 - far)
    loss = torch.where(mask, term, 0.0).sum() / n
    return [loss, lp, _plain_grad(s, e, z, c / n)]


def _plain_pref(s):
    e, z, lp = _plain_logprobs(s)
    N = lp.shape[0] // 2
    score = torch.where(s["mask"], lp - s["ref"].double(), 0.0).sum(1)
    m = (0.1 * (score[:N] - score[N:])).float()
    loss = (0.95 * torch.log1p(torch.exp(-m.abs())) + 0.95 * (-m).clamp_min(0)
            + 0.05 * torch.log1p(torch.exp(-m.abs())) + 0.05 * m.clamp_min(0)).mean()
    dm = (-0.95 / (1 + torch.exp(m)) + 0.05 / (1 + torch.exp(-m))) * (0.1 / N)
    c = torch.cat([dm, -dm])[:, None].expand(lp.shape)
    return [loss, m, lp.float(), _plain_grad(s, e, z, c)]


def run(state):
    kind = state["kind"]
    if own:
        return {"embed": _own_embed, "norm": _own_norm, "policy": _own_policy,
                "pref": _own_pref}[kind](state)
    with torch.no_grad():
        return {"embed": _plain_embed, "norm": _plain_norm, "policy": _plain_policy,
                "pref": _plain_pref}[kind](state)


# --------------------------------------------------------------------------------- its work

def work(case):
    size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    if case["kind"] == "embed":
        n, V, D = case["n"], case["vocab"], case["D"]
        b, f = (min(n, V) + n) * D * size + 8 * n, n * D
        if case["grad"]:
            b, f = b + (n + V) * D * size, f + n * D
        return {"bytes": b, "flops": f}
    if case["kind"] == "norm":
        R, D = case["rows"], case["D"]
        passes = 4 if case["add"] else 2       # x (and d) in, h (and the sum) out
        b, f = passes * R * D * size + 2 * D * size, 6 * R * D
        if case["grad"]:                       # gh (and gs) in, the input's gradient out
            b, f = b + (3 if case["add"] else 2) * R * D * size + 2 * D * size, f + 12 * R * D
        return {"bytes": b, "flops": f}
    rows, V = case["seqs"] * case["T"], case["vocab"]
    live = int(_answer(case).sum())
    return {"bytes": (live + rows) * V * size + 28 * rows, "flops": 8 * live * V}


# ---------------------------------------------------------------- definitions in 64 bits

def _exact_embed(s):
    w, ids = s["emb"].weight.detach().double(), s["ids"]
    y = torch.index_select(w, 0, ids) * s["scale"]
    if not s["grad"]:
        return [y]
    keep = torch.ones_like(ids, dtype=torch.bool)
    if s["emb"].padding_idx is not None:
        keep = ids != s["emb"].padding_idx
    ids, gy = ids[keep], s["gy"].double()[keep]
    order = torch.argsort(ids, stable=True)
    ids = ids[order]
    gw = torch.zeros_like(w)
    if ids.numel():
        # runs of equal tokens as differences of running sums, column by column block
        last = torch.cat([ids[1:] != ids[:-1], ids.new_ones(1, dtype=torch.bool)])
        total = torch.cumsum(gy[order], 0)[last]
        total[1:] = total[1:] - total[:-1].clone()
        gw[ids[last]] = total * s["scale"]
    return [y, gw]


def _exact_norm(s):
    dt, norm = s["x"].dtype, s["norm"]
    x = s["x"].detach().double()
    out = []
    if s["d"] is not None:                     # the sum is held in the inputs' type
        x = (x + s["d"].detach().double()).to(dt).double()
        out = [x.clone()]
    x.requires_grad_(True)
    w = norm.weight.detach().double().requires_grad_(True)
    wrt = [x, w]
    if s["center"]:
        b = norm.bias.detach().double().requires_grad_(True)
        wrt.append(b)
        var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
        h = (x - mean) / torch.sqrt(var + norm.eps) * w + b
    else:
        h = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + norm.eps) * w
    out = [h.detach()] + out
    if not s["grad"]:
        return out
    gx, *gw = torch.autograd.grad(h, wrt, s["gh"].double())
    if s["d"] is None:
        return out + [gx] + gw
    gx = gx + s["gs"].double()
    return out + [gx, gx] + gw


def _exact_loss(s):
    """Term by term through automatic differentiation in the log-probabilities; the softmax's
    derivative row by row."""
    logits, t, mask = s["logits"].detach(), s["targets"], s["mask"]
    grad = torch.zeros(logits.shape, dtype=torch.float64, device="cuda")
    lp = torch.zeros(t.shape, dtype=torch.float64, device="cuda")
    for i in range(t.shape[0]):
        x = logits[i].double() / s["temperature"]
        p = torch.log_softmax(x, -1)
        lp[i] = p.gather(1, t[i][:, None])[:, 0]
        grad[i] = -torch.exp(p)
    grad.scatter_add_(2, t[..., None], torch.ones_like(grad[..., :1]))
    lp[~mask] = 0
    leaf = lp.clone().requires_grad_(True)
    ref, live = s["ref"].double(), mask.double()
    if s["kind"] == "policy":
        ratio = torch.exp(leaf - s["old"].double())
        adv = s["adv"].double()
        term = -torch.minimum(ratio * adv, ratio.clamp(0.8, 1.2) * adv)
        gap = ref - leaf
        term = term + s["kl"] * (torch.expm1(gap) - gap)
        loss = (term * live).sum() / max(1.0, float(live.sum()))
        out = [loss.detach(), lp]
    else:
        score = ((leaf - ref) * live).sum(1)
        N = score.numel() // 2
        m = 0.1 * (score[:N] - score[N:])
        ls = torch.nn.functional.logsigmoid
        loss = (-0.95 * ls(m) - 0.05 * ls(-m)).mean()
        out = [loss.detach(), m.detach(), lp]
    (c,) = torch.autograd.grad(loss, [leaf])
    grad *= (c / s["temperature"])[..., None]
    grad[~mask] = 0
    return out + [grad]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "embed":
        return _exact_embed(s)
    if case["kind"] == "norm":
        return _exact_norm(s)
    return _exact_loss(s)
