"""The operators between a hidden state and the next token, as cases that can be timed and checked.

Three kinds:

  gated   the feed-forward block's input: silu(x . Wg^T) * (x . Wu^T); with `grad` the gradients of
          x and both weights
  fp8     x . W^T in 8-bit floating point (e4m3) with power-of-two scales: one for each 128 columns
          of a row of x, one for each 128 x 128 block of W; x comes in 16 or 32 bits
  sample  a token of each row of logits from a given random number, after temperature, top-k, top-p
          and min-p; and its log-probability at that temperature

`run` computes them in elementary tensor operations, or through the package where `own` is set.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # a short prompt of a small model
        dict(name="gated_prompt", kind="gated", rows=48, dim=1024, ff=2816, dtype="bf16", grad=False),
        # a prefill chunk of the language model
        dict(name="gated_prefill", kind="gated", rows=16384, dim=1536, ff=6144, dtype="bf16",
             grad=False),
        # its training batch, 4 x 16384 tokens
        dict(name="gated_train", kind="gated", rows=65536, dim=1536, ff=6144, dtype="bf16", grad=True),
        # fine-tuning on short answers, widths that fill no tile, half precision
        dict(name="gated_odd", kind="gated", rows=1001, dim=776, ff=2072, dtype="f16", grad=True),
        # one stream's decode step through the up projection
        dict(name="fp8_step", kind="fp8", rows=1, K=1536, N=6144, dtype="bf16"),
        # the head of a batch of 16 streams
        dict(name="fp8_head", kind="fp8", rows=16, K=1536, N=50304, dtype="bf16"),
        # a ragged batch, widths that end inside a block
        dict(name="fp8_odd", kind="fp8", rows=777, K=1000, N=1234, dtype="f16"),
        # the down projection of a long prefill
        dict(name="fp8_prefill", kind="fp8", rows=65536, K=6144, N=1536, dtype="bf16"),
        # a decode step of one stream
        dict(name="sample_one", kind="sample", rows=1, vocab=50304, dtype="bf16", temperature=0.8,
             top_k=50, top_p=0.95, min_p=0.0, each=False),
        # a batch whose streams each have settings of their own
        dict(name="sample_batch", kind="sample", rows=64, vocab=50304, dtype="bf16", temperature=1.0,
             top_k=200, top_p=0.9, min_p=0.05, each=True),
        # nucleus alone on fp32 logits of an odd vocabulary
        dict(name="sample_nucleus", kind="sample", rows=13, vocab=32003, dtype="f32", temperature=1.3,
             top_k=0, top_p=0.98, min_p=0.0, each=False),
        # many rollouts over a large vocabulary
        dict(name="sample_rollouts", kind="sample", rows=1024, vocab=131072, dtype="bf16",
             temperature=1.0, top_k=0, top_p=1.0, min_p=0.02, each=False),
    ]


def _log(rng, lo, hi):
    """A whole number spread over [lo, hi] by its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _eights(n):
    return max(8, n // 8 * 8)


def draw(rng):
    kind = rng.choice(["gated", "fp8", "sample"])
    if kind == "gated":
        # the operator's kernels take widths of a multiple of 8 and more rows than a decode step has
        dim, ff = _eights(_log(rng, 128, 4096)), _eights(_log(rng, 256, 16384))
        rows = _log(rng, 33, 65536)
        rows = max(33, min(rows, 65536 * 1536 * 6144 // (dim * ff)))
        return dict(kind=kind, rows=rows, dim=dim, ff=ff, dtype=rng.choice(["bf16", "bf16", "f16"]),
                    grad=rng.random() < 0.6)
    if kind == "fp8":
        K, N = _log(rng, 128, 16384), _log(rng, 128, 65536)
        N = min(N, (1 << 27) // K)
        K, N = (K, N) if rng.random() < 0.3 else (_eights(K), _eights(N))
        rows = max(1, min(_log(rng, 1, 65536), 65536 * 6144 * 1536 // (K * N)))
        return dict(kind=kind, rows=rows, K=K, N=N, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))
    vocab = _log(rng, 1000, 131072)
    vocab = vocab if rng.random() < 0.3 else _eights(vocab)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    cap = 1024 * 131072 // (2 if dtype == "f32" else 1)
    return dict(kind=kind, rows=min(_log(rng, 1, 1024), cap // vocab), vocab=vocab, dtype=dtype,
                temperature=rng.choice([0.6, 0.8, 1.0, 1.3]),
                top_k=rng.choice([0, 0, 1, 20, 50, 1000]),
                top_p=rng.choice([1.0, 0.5, 0.9, 0.95, 0.99]),
                min_p=rng.choice([0.0, 0.0, 0.02, 0.1]), each=rng.random() < 0.3)


# ------------------------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _hidden(g, rows, dim):
    """Normalised hidden states: unit rows, a few channels that stand out."""
    x = _randn(g, rows, dim)
    x[:, :: 61] *= 6.0
    return x


def _prepare_gated(c, seed):
    g, dt = _gen(seed), DTYPES[c["dtype"]]
    R, D, N = c["rows"], c["dim"], c["ff"]
    s = dict(kind="gated", grad=c["grad"], x=_hidden(g, R, D).to(dt))
    for name in ("gate", "up"):
        lin = torch.nn.Linear(D, N, bias=False, device="cuda", dtype=dt)
        with torch.no_grad():
            lin.weight.copy_(_randn(g, N, D) * D ** -0.5)
        s[name] = lin.requires_grad_(c["grad"])
    if c["grad"]:
        s["x"].requires_grad_(True)
        s["gy"] = (_randn(g, R, N) * 0.05).to(dt)
    return s


def _scale_exponents(amax):
    """The least e with amax <= 448 * 2^e (448: e4m3's largest value); 0 for a block of zeros."""
    m, e = torch.frexp(amax)                        # amax = m 2^e, 1/2 <= m < 1; 448 = 0.875 * 2^9
    return torch.where(amax > 0, e - 9 + (m > 0.875).int(), 0).clamp(-127, 127)


def _powers(e):
    """2^e in 64 bits, exactly: from the bits (a device's pow may be off in the last one)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _prepare_fp8(c, seed):
    g, dt = _gen(seed), DTYPES[c["dtype"]]
    R, K, N = c["rows"], c["K"], c["N"]
    Kb, Nb = -(-K // 128), -(-N // 128)
    # weights whose size differs from block to block, held in whole blocks of columns: zeros behind
    # the last
    w = torch.zeros(Nb * 128, Kb * 128, device="cuda")
    w[:N, :K] = _randn(g, N, K) * K ** -0.5
    blocks = w.view(Nb, 128, Kb, 128)
    blocks *= torch.exp(0.5 * _randn(g, Nb, 1, Kb, 1))
    e = _scale_exponents(blocks.abs().amax((1, 3)))
    q = (blocks * _powers(-e).float()[:, None, :, None]).to(torch.float8_e4m3fn)
    x = _hidden(g, R, K) * torch.exp(0.5 * _randn(g, R, 1))
    return dict(kind="fp8", x=x.to(dt), values=q.view(Nb * 128, Kb * 128)[:N].contiguous(),
                scales=(e + 127).to(torch.uint8).view(torch.float8_e8m0fnu))


def _prepare_sample(c, seed):
    g, dt = _gen(seed), DTYPES[c["dtype"]]
    R, V = c["rows"], c["vocab"]
    logits = torch.empty(R, V, dtype=dt, device="cuda")
    step = max(1, (1 << 27) // V)
    for a in range(0, R, step):
        # a language model's predictions: a few likely words over a broad tail
        x = 2.0 * _randn(g, min(step, R - a), V)
        top = torch.randint(0, V, (x.shape[0], 8), generator=g, device="cuda")
        x.scatter_add_(1, top, 3 + 8 * torch.rand(top.shape, generator=g, device="cuda"))
        logits[a:a + step] = x.to(dt)
    s = dict(kind="sample", logits=logits, u=torch.rand(R, generator=g, device="cuda"))
    names = ("temperature", "top_k", "top_p", "min_p")
    if c["each"]:  # settings of each stream around the case's own
        f = 0.7 + 0.6 * torch.rand(4, R, generator=g, device="cuda")
        s.update(temperature=c["temperature"] * f[0], top_k=(c["top_k"] * f[1]).long(),
                 top_p=c["top_p"] ** (2 * f[2]), min_p=c["min_p"] * f[3])
    else:
        s.update({n: c[n] for n in names})
    return s


def prepare(case, seed):
    return {"gated": _prepare_gated, "fp8": _prepare_fp8, "sample": _prepare_sample}[case["kind"]](case, seed)


# ------------------------------------------------------------------------- the package's calls

def _own_gated(s):
    from latest_exact_match_attention_amd.model import gated_linear
    y = gated_linear(s["x"], s["gate"], s["up"])
    if not s["grad"]:
        return [y]
    wrt = [s["x"], s["gate"].weight, s["up"].weight]
    return [y.detach(), *torch.autograd.grad(y, wrt, s["gy"])]


def _own_fp8(s):
    from latest_exact_match_attention_amd import fp8
    return [fp8.linear(s["x"], fp8.Fp8(s["values"], s["scales"], s["x"].shape[-1]))]


def _own_sample(s):
    from latest_exact_match_attention_amd.sampling import sample
    r = sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
               min_p=s["min_p"])
    return [r.tokens, r.logprobs]


# -------------------------------------------------------------------------------- plain forms

def _plain_gated(s):
    dt = s["x"].dtype
    x, wg, wu = (t.detach().float() for t in (s["x"], s["gate"].weight, s["up"].weight))
    g, u = x @ wg.t(), x @ wu.t()
    sig = 1 / (1 + torch.exp(-g))
    a = g * sig
    y = (a * u).to(dt)
    if not s["grad"]:
        return [y]
    gy = s["gy"].float()
    du = gy * a
    dg = gy * u * sig * (1 + g * (1 - sig))
    gx = dg @ wg + du @ wu
    return [y, gx.to(dt), (dg.t() @ x).to(dt), (du.t() @ x).to(dt)]


def _plain_fp8(s):
    x, N = s["x"], s["values"].shape[0]
    R, K = x.shape
    Kb = s["scales"].shape[1]
    xp = torch.zeros(R, Kb * 128, device=x.device)
    xp[:, :K] = x.float()
    xp = xp.view(R, Kb, 128)
    e = _scale_exponents(xp.abs().amax(-1))[..., None]
    xq = (xp * _powers(-e).float()).to(torch.float8_e4m3fn).float() * _powers(e).float()
    sw = _powers(s["scales"].view(torch.uint8).int() - 127).float().repeat_interleave(128, 0)[:N]
    wq = s["values"].float().view(N, Kb, 128) * sw[..., None]
    return [(xq.view(R, -1) @ wq.view(N, -1).t()).to(x.dtype)]


def _column(v, like):
    """A setting as a column in 64 bits; a number is first rounded to the 32 that it is passed in."""
    if not torch.is_tensor(v):
        v = torch.full(like.shape[:1], v, dtype=torch.float32, device=like.device)
    return v.double()[:, None]


def _plain_sample(s):
    """In 64 bits: a drawn number may lie next to the border between two tokens."""
    z = s["logits"].double()
    V = z.shape[1]
    T, k, p, m = (_column(s[n], z) for n in ("temperature", "top_k", "top_p", "min_p"))
    z = (z - z.amax(1, keepdim=True)) / T
    lse = torch.log(torch.exp(z).sum(1))
    down, order = torch.sort(z, dim=1, descending=True, stable=True)
    w = torch.exp(down)
    rank = torch.arange(V, device=z.device)
    w = torch.where((k > 0) & (rank >= k), 0.0, w)
    before = torch.cumsum(w, 1) - w
    w = torch.where((p < 1) & (rank > 0) & (before >= p * w.sum(1, keepdim=True)), 0.0, w)
    w = torch.where((m > 0) & (down < torch.log(m)), 0.0, w)
    kept = torch.zeros_like(w).scatter_(1, order, w)
    total = torch.cumsum(kept, 1)
    tok = (total > s["u"].double()[:, None] * total[:, -1:]).to(torch.uint8).argmax(1)
    return [tok, (z.gather(1, tok[:, None])[:, 0] - lse).float()]


def run(state):
    kind = state["kind"]
    if own:
        return {"gated": _own_gated, "fp8": _own_fp8, "sample": _own_sample}[kind](state)
    with torch.no_grad():
        return {"gated": _plain_gated, "fp8": _plain_fp8, "sample": _plain_sample}[kind](state)


# --------------------------------------------------------------------------------- its work

def work(case):
    size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    R = case["rows"]
    if case["kind"] == "gated":
        D, N = case["dim"], case["ff"]
        b, f = (R * D + 2 * N * D + R * N) * size, 4 * R * D * N
        if case["grad"]:
            b, f = b + (R * N + R * D + 2 * N * D) * size, 3 * f
        return {"bytes": b, "flops": f}
    if case["kind"] == "fp8":
        K, N = case["K"], case["N"]
        return {"bytes": R * (K + N) * size + N * K + -(-N // 128) * -(-K // 128), "flops": 2 * R * K * N}
    return {"bytes": R * case["vocab"] * size + 16 * R, "flops": 8 * R * case["vocab"]}


# ---------------------------------------------------------------- definitions in 64 bits

def _exact_gated(s):
    x, wg, wu = (t.detach().double().requires_grad_(s["grad"])
                 for t in (s["x"], s["gate"].weight, s["up"].weight))
    y = torch.nn.functional.silu(torch.nn.functional.linear(x, wg)) * torch.nn.functional.linear(x, wu)
    if not s["grad"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, [x, wg, wu], s["gy"].double())]


def _e4m3(v):
    """v, at most 448 in size, rounded to the nearest e4m3 value, halves to even."""
    _, e = torch.frexp(v.abs().clamp_min(2.0 ** -6))    # 2^(e - 1) <= |v| < 2^e
    step = _powers(e - 4)
    return torch.round(v / step) * step


def _exact_fp8(s):
    x, (N, Kp) = s["x"].double(), s["values"].shape
    y = torch.zeros(x.shape[0], N, dtype=torch.float64, device=x.device)
    sw = s["scales"].float().double()
    for b in range(Kp // 128):
        part = x[:, 128 * b:128 * b + 128]
        top = part.abs().amax(1, keepdim=True)
        e = torch.ceil(torch.log2(top.clamp_min(2.0 ** -200) / 448)).long()
        e = e + (top > 448 * _powers(e)).long()
        e = e - (top <= 448 * _powers(e - 1)).long()
        scale = _powers(torch.where(top > 0, e.clamp(-127, 127), 0))
        part = _e4m3(part / scale) * scale
        w = s["values"][:, 128 * b:128 * b + part.shape[1]].float().double()
        y.addmm_(part, (w * sw[:, b].repeat_interleave(128)[:N, None]).t())
    return [y]


def _exact_sample(s):
    """Row by row: the tokens in the order of their logits, cut three times, then the draw."""
    tokens, logprobs = [], []
    for r in range(s["logits"].shape[0]):
        T, k, p, m = (float(_column(s[n], s["logits"])[r]) for n in ("temperature", "top_k", "top_p", "min_p"))
        q = torch.softmax(s["logits"][r].double() / T, 0)
        order = torch.argsort(s["logits"][r].double().neg(), stable=True)
        keep = order[:int(k)] if k > 0 else order
        if p < 1:
            cum = torch.cumsum(q[keep], 0) / q[keep].sum()
            keep = keep[:1 + int((cum[:-1] < p).sum())]
        if m > 0:
            keep = keep[q[keep] >= m * q.max()]
        keep = torch.sort(keep).values
        cum = torch.cumsum(q[keep], 0)
        at = torch.searchsorted(cum, s["u"][r].double() * cum[-1], right=True)
        t = keep[at.clamp_max(keep.numel() - 1)]
        tokens.append(t)
        logprobs.append(torch.log(q[t]))
    return [torch.stack(tokens), torch.stack(logprobs)]


def exact(case, seed):
    s = prepare(case, seed)
    return {"gated": _exact_gated, "fp8": _exact_fp8, "sample": _exact_sample}[case["kind"]](s)
