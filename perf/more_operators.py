"""Measured cases of the operators of a gated-recurrence language model: its recurrence, the norms around its
blocks, and the log probabilities that it is scored and trained by.

  prompt    gated_recurrence over whole prompts, in and out of a state:
            a = e^{-c softplus(lam) sigmoid(r)},  h <- a h + sqrt(1 - a^2) sigmoid(i) x,  y = h
  learn     the same and gated_recurrence_backward: gradients of x, r, i, lam and the entering state
  token     gated_recurrence_step: one token of every sequence, state in place
  norms     block_norm: x' = x + scale norm(y) silu(z), n = norm(x')
  teach     the same and block_norm_backward: gradients of x, y, z and of the three weights
  score     token_logprobs: log probability of a given token of each row, entropy, top alternatives
  loss      the same and token_logprobs_backward: gradient of the logits

`run` computes them from elementary torch operations in 32 bits, or, where `own` is true, with the
calls of ssmjs_amd.kernels. `exact` follows the definitions in 64 bits.
"""
import math

import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}
C = 8.0
EPS = 1e-6


# ------------------------------------------------------------------ cases
def listed():
    def rec(name, op, B, L, D, dt, ragged=False, state=False):
        return {"name": name, "op": op, "B": B, "L": L, "D": D, "dtype": dt, "ragged": ragged, "state": state}

    def norms(name, op, T, D, dt, gate=True):
        return {"name": name, "op": op, "T": T, "D": D, "dtype": dt, "gate": gate}

    def logits(name, op, M, N, dt, k=0, masked=False):
        return {"name": name, "op": op, "M": M, "N": N, "dtype": dt, "k": k, "masked": masked}

    return [
        # a batch of equal prompts through a layer 2048 wide
        rec("prompts bf16", "prompt", 8, 4096, 2048, "bf16"),
        # prompts of mixed lengths in one padded batch (none and one token among them), going on
        # from a state, in the model path's own type and an inner width of its 768-wide preset
        rec("ragged prompts f32", "prompt", 5, 1500, 1536, "f32", True, True),
        # one long document
        rec("long prompt bf16", "prompt", 1, 32768, 1024, "bf16", False, True),
        # a training batch of four sequences
        rec("training batch bf16", "learn", 4, 2048, 2048, "bf16"),
        # a single session's next token
        rec("token of one session", "token", 1, 1, 2048, "f32"),
        # the next token of a full batch
        rec("token of 64 sessions", "token", 64, 1, 4096, "bf16"),
        # between two blocks: the tokens of 64 decoded sequences
        norms("norms of 64 tokens", "norms", 64, 2048, "bf16"),
        # the tokens of a batch of prompts, and a training batch of a 768-wide model, without a gate
        norms("norms of prompts", "norms", 16384, 2048, "bf16"),
        norms("norms in training", "teach", 8192, 768, "f32", False),
        # the last position of 64 sequences with 20 alternatives each
        logits("64 tokens, 20 alternatives", "score", 64, 128000, "f32", 20, True),
        # every position of a scored text of 2047 tokens, five alternatives each
        logits("scored text", "score", 2047, 32000, "f32", 5),
        # a training batch's loss over an odd vocabulary: no row but the first is aligned
        logits("loss of 4096 tokens", "loss", 4096, 50257, "bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A width: mostly of whole 64s, at times any."""
    w = _log(rng, lo, hi)
    return w if rng.random() < 0.25 else max(64, w // 64 * 64)


def draw(rng):
    op = rng.choice(["prompt", "prompt", "learn", "learn", "token", "norms", "teach", "score", "loss"])
    dt = rng.choice(["f32", "bf16"])
    if op in ("prompt", "learn", "token"):
        D = _width(rng, 64, 4096)
        B = _log(rng, 1, 64)
        if op == "token":
            return {"op": op, "B": B, "L": 1, "D": D, "dtype": dt, "ragged": False, "state": False}
        size = 1 << ((26 if op == "prompt" else 24) - (dt == "f32"))
        most = min(32768 if op == "prompt" else 4096, size // (B * D))
        return {"op": op, "B": B, "L": _log(rng, 1, most), "D": D, "dtype": dt,
                "ragged": rng.random() < 0.4, "state": rng.random() < 0.5}
    if op in ("norms", "teach"):
        D = _width(rng, 64, 4096)
        most = (1 << (24 if op == "norms" else 23)) // D
        return {"op": op, "T": _log(rng, 1, most), "D": D, "dtype": dt, "gate": rng.random() < 0.7}
    N = _log(rng, 256, 128000)
    most = min(4096, (1 << 27) // N)
    k = rng.choice([0, 1, 5, 20, 50]) if op == "score" else 0
    return {"op": op, "M": _log(rng, 1, most), "N": N, "dtype": dt, "k": k, "masked": rng.random() < 0.3}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    c = dict(case)
    dt = DT[c["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    if c["op"] in ("prompt", "learn", "token"):
        B, L, D = c["B"], c["L"], c["D"]
        c["x"] = normal(B, L, D).to(dt)
        # both gates as one product leaves them, side by side in each row
        rows = (normal(B, L, 2 * D) * 1.5).to(dt)
        c["r"], c["i"] = rows[..., :D], rows[..., D:]
        # decays of a token between 0.9 and 0.999 where the gate is wide open
        keep = 0.9 + 0.099 * torch.rand(D, generator=gen, device=dev, dtype=torch.float64)
        c["lam"] = torch.log(torch.expm1(-torch.log(keep) / C)).float()
        c["lengths"], c["h0"], c["hT"], c["dhT"] = None, None, None, None
        if c["op"] == "token":
            c["x"], c["r"], c["i"] = c["x"][:, 0], c["r"][:, 0], c["i"][:, 0]
            c["h"] = normal(B, D)
            return c
        if c["state"]:
            c["h0"] = normal(B, D)
        if c["ragged"]:
            n = torch.randint(0, L + 1, (B,), generator=gen, device=dev)
            n[0] = L
            n[1:2] = 0
            n[2:3] = min(1, L)
            c["lengths"] = n.to(torch.int32)
        c["hT"] = torch.zeros(B, D, device=dev)
        if c["op"] == "learn":
            c["dy"] = normal(B, L, D).to(dt)
            c["dhT"] = normal(B, D) if c["state"] else None
            c["dh0"] = torch.zeros(B, D, device=dev)
            c["states"] = torch.zeros(B, -(-L // 64), D, device=dev)
    elif c["op"] in ("norms", "teach"):
        T, D = c["T"], c["D"]
        c["x"] = (3 * normal(T, D)).to(dt)     # a residual stream some blocks deep
        c["y"] = normal(T, D).to(dt)
        c["z"] = normal(T, D).to(dt) if c["gate"] else None
        c["post"], c["pre"] = 1 + 0.2 * normal(D), 1 + 0.2 * normal(D)
        c["scale"] = 0.5 + 0.1 * normal(D)
        if c["op"] == "teach":
            c["dx1"], c["dn"] = normal(T, D).to(dt), normal(T, D).to(dt)
    else:
        M, N = c["M"], c["N"]
        # logits of a text: wide rows with some likely tokens, and given tokens that are among them
        x = 2.5 * normal(M, N)
        c["ids"] = torch.randint(0, N, (M,), generator=gen, device=dev)
        x[torch.arange(M, device=dev), c["ids"]] += 8 * torch.rand(M, generator=gen, device=dev)
        if c["masked"]:
            # tokens that a grammar forbids, the given one apart
            off = torch.rand(M, N, generator=gen, device=dev) < 0.4
            off[torch.arange(M, device=dev), c["ids"]] = False
            x.masked_fill_(off, float("-inf"))
        c["x"] = x.to(dt)
        # padding behind the texts has no token
        c["ids"] = torch.where(torch.rand(M, generator=gen, device=dev) < 0.1, -1, c["ids"]).to(torch.int32)
        if c["op"] == "loss":
            c["dlogp"], c["dent"] = normal(M) / M, 0.01 * normal(M) / M
            c["stats"] = torch.zeros(M, 2, device=dev)
    return c


# ------------------------------------------------------------------ one pass
def run(s):
    if own:
        from ssmjs_amd import kernels
        if s["op"] == "prompt":
            y = kernels.gated_recurrence(s["x"], s["r"], s["i"], s["lam"], c=C, lengths=s["lengths"],
                                         h0=s["h0"], hT=s["hT"])
            return y, s["hT"]
        if s["op"] == "learn":
            y = kernels.gated_recurrence(s["x"], s["r"], s["i"], s["lam"], c=C, lengths=s["lengths"],
                                         h0=s["h0"], hT=s["hT"], states=s["states"])
            grads = kernels.gated_recurrence_backward(s["dy"], s["x"], s["r"], s["i"], s["lam"], s["states"], c=C,
                                                      lengths=s["lengths"], dhT=s["dhT"], dh0=s["dh0"])
            return y, s["hT"], *grads, s["dh0"]
        if s["op"] == "token":
            return kernels.gated_recurrence_step(s["x"], s["r"], s["i"], s["lam"], s["h"], c=C), s["h"]
        if s["op"] == "norms":
            return kernels.block_norm(s["x"], s["y"], s["z"], s["post"], s["scale"], s["pre"], eps=EPS)
        if s["op"] == "teach":
            x1, n = kernels.block_norm(s["x"], s["y"], s["z"], s["post"], s["scale"], s["pre"], eps=EPS)
            return x1, n, *kernels.block_norm_backward(s["dx1"], s["dn"], s["x"], s["y"], s["z"], s["post"],
                                                       s["scale"], s["pre"], eps=EPS)
        if s["op"] == "score":
            return kernels.token_logprobs(s["x"], s["ids"], k=s["k"])
        logp, ent, _, _ = kernels.token_logprobs(s["x"], s["ids"], stats=s["stats"])
        return logp, ent, kernels.token_logprobs_backward(s["x"], s["ids"], s["stats"], ent, s["dlogp"], s["dent"])
    return {"prompt": _prompt, "learn": _learn, "token": _token, "norms": _norms, "teach": _teach,
            "score": _score, "loss": _loss}[s["op"]](s)


def _gates(s):
    """log a, a, sqrt(1 - a^2) and the two gates, in 32 bits."""
    r, i = torch.sigmoid(s["r"].float()), torch.sigmoid(s["i"].float())
    soft = torch.log1p(torch.exp(s["lam"].double())).float()
    loga = -C * soft * r
    return loga, torch.exp(loga), torch.sqrt(-torch.expm1(2 * loga)), r, i


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dimension 1 from a zero state: spans of 2, 4, 8 .. steps, in place of
    a loop over all of them."""
    a, h, k = a.clone(), b.clone(), 1
    while k < a.shape[1]:
        h[:, k:] += a[:, k:] * h[:, :-k]
        a[:, k:] *= a[:, :-k].clone()
        k *= 2
    return h


def _inside(s):
    if s["lengths"] is None:
        return None
    return (torch.arange(s["L"], device=s["x"].device) < s["lengths"][:, None])[..., None]


def _forward(s):
    loga, a, beta, r, i = _gates(s)
    x, inside = s["x"].float(), _inside(s)
    b = beta * i * x
    if inside is not None:
        a, b = torch.where(inside, a, 1.0), torch.where(inside, b, 0.0)
    if s["h0"] is not None:
        b[:, 0] += a[:, 0] * s["h0"]
    h = _scan(a, b)
    y = h if inside is None else torch.where(inside, h, 0.0)
    return (loga, a, beta, r, i, x, inside, h), y.to(s["x"].dtype)


def _prompt(s):
    kept, y = _forward(s)
    return y, kept[-1][:, -1].clone()


def _learn(s):
    (loga, a, beta, r, i, x, inside, h), y = _forward(s)
    dt, dy = s["x"].dtype, s["dy"].float()
    if inside is not None:
        dy = torch.where(inside, dy, 0.0)
    # g_t = dy_t + a_{t+1} g_{t+1}, from the last step on
    if s["dhT"] is not None:
        dy[:, -1] += s["dhT"]
    after = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], 1)
    g = _scan(after.flip(1), dy.flip(1)).flip(1)
    dh0 = a[:, 0] * g[:, 0]
    h0 = s["h0"] if s["h0"] is not None else torch.zeros_like(dh0)
    before = torch.cat([h0[:, None], h[:, :-1]], 1)
    if inside is not None:
        g = torch.where(inside, g, 0.0)
    q = g * (before * a * loga - i * x * a * a * (loga / beta))     # dL/dlog a * log a
    dx, di, dr = g * beta * i, g * beta * x * i * (1 - i), q * (1 - r)
    lam = s["lam"].double()
    dlam = (q.double().sum((0, 1)) * torch.sigmoid(lam) / torch.log1p(torch.exp(lam))).float()
    return y, h[:, -1].clone(), dx.to(dt), dr.to(dt), di.to(dt), dlam, dh0


def _token(s):
    _, a, beta, _, i = _gates(s)
    s["h"].mul_(a).add_(beta * i * s["x"].float())
    return s["h"].to(s["x"].dtype), s["h"]


def _block(s):
    x, y = s["x"].float(), s["y"].float()
    ry = torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS)
    u = y * ry * s["post"]
    z = s["z"].float() if s["z"] is not None else None
    v = u * (z * torch.sigmoid(z)) if z is not None else u
    x1 = x + s["scale"] * v
    rx = torch.rsqrt((x1 * x1).mean(-1, keepdim=True) + EPS)
    return y, ry, u, z, v, x1, rx


def _norms(s):
    *_, x1, rx = _block(s)
    return x1.to(s["x"].dtype), (x1 * rx * s["pre"]).to(s["x"].dtype)


def _teach(s):
    y, ry, u, z, v, x1, rx = _block(s)
    dt, dn = s["x"].dtype, s["dn"].float()
    n = x1 * rx
    d = dn * s["pre"]
    g = s["dx1"].float() + rx * (d - n * (d * n).mean(-1, keepdim=True))
    dscale, dpre = (g * v).double().sum(0).float(), (dn * n).double().sum(0).float()
    du, dz = g * s["scale"], None
    if z is not None:
        e = torch.sigmoid(z)
        dz = (du * u * e * (1 + z * (1 - e))).to(dt)
        du = du * (z * e)
    w = y * ry
    dpost = (du * w).double().sum(0).float()
    d = du * s["post"]
    dy = ry * (d - w * (d * w).mean(-1, keepdim=True))
    return x1.to(dt), (n * s["pre"]).to(dt), g.to(dt), dy.to(dt), dz, dpost, dscale, dpre


def _likely(s):
    """Shifted logits, their exponentials, the log of their sum, log p of the given tokens, entropy."""
    x = s["x"].float()
    d = x - x.amax(1, keepdim=True)
    e = torch.exp(d)
    z = e.sum(1, keepdim=True)
    logz = torch.log(z)
    at = s["ids"].long()
    logp = torch.where(at < 0, 0.0, (d.gather(1, at.clamp(min=0)[:, None]) - logz)[:, 0])
    ent = (logz - torch.where(e > 0, e * d, 0.0).sum(1, keepdim=True) / z)[:, 0]
    return d, e, z, logz, logp, ent


def _score(s):
    d, _, _, logz, logp, ent = _likely(s)
    if s["k"] == 0:
        return logp, ent, None, None
    # one whole number for each logit, larger for larger logits and, of equal ones, for the first
    bits = s["x"].float().add(0.0).view(torch.int32).long()
    order = torch.where(bits < 0, -2147483648 - bits, bits)
    key = order * (1 << 20) - torch.arange(s["N"], device=bits.device)
    top = torch.topk(key, s["k"], dim=1).indices
    return logp, ent, top.to(torch.int32), d.gather(1, top) - logz


def _loss(s):
    d, e, z, logz, logp, ent = _likely(s)
    p = e / z
    given = s["ids"].long()
    w = torch.where(given < 0, 0.0, s["dlogp"])
    dx = -p * (w[:, None] + s["dent"][:, None] * torch.where(e > 0, d - logz + ent[:, None], 0.0))
    dx[torch.arange(s["M"], device=dx.device), given.clamp(min=0)] += w
    return logp, ent, dx.to(s["x"].dtype)


# ------------------------------------------------------------------ what a pass cannot do without
def work(c):
    e = SIZE[c["dtype"]]
    if c["op"] in ("prompt", "learn", "token"):
        B, L, D = c["B"], c["L"], c["D"]
        rows = B * L
        if c["ragged"]:
            rows = L + (min(1, L) if B > 2 else 0) + max(0, B - 3) * L // 2     # L, 0, 1 and L / 2 on average
        if c["op"] == "token":
            return {"bytes": B * D * (4 * e + 8) + 4 * D, "flops": 16 * B * D}
        states = 4 * B * D * (2 if c["state"] else 1)
        if c["op"] == "prompt":
            return {"bytes": 4 * rows * D * e + states + 4 * D, "flops": 16 * rows * D}
        return {"bytes": 8 * rows * D * e + 2 * states + 8 * D, "flops": 48 * rows * D}
    if c["op"] in ("norms", "teach"):
        n, gate = c["T"] * c["D"], c["gate"]
        if c["op"] == "norms":
            return {"bytes": (4 + gate) * n * e + 12 * c["D"], "flops": (10 + 5 * gate) * n}
        return {"bytes": (8 + 2 * gate) * n * e + 24 * c["D"], "flops": (30 + 15 * gate) * n}
    M, N = c["M"], c["N"]
    if c["op"] == "score":
        return {"bytes": M * N * e + 12 * M + 8 * M * c["k"], "flops": 6 * M * N}
    return {"bytes": 2 * M * N * e + 24 * M, "flops": 12 * M * N}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] in ("prompt", "learn", "token"):
        return _exact_recurrence(s)
    if s["op"] in ("norms", "teach"):
        return _exact_norms(s)
    x = s["x"].double().requires_grad_(s["op"] == "loss")
    lp = torch.nn.functional.log_softmax(x, 1)
    some = s["ids"] >= 0
    logp = torch.where(some, lp[torch.arange(s["M"], device=lp.device), s["ids"].clamp(min=0).long()], 0.0)
    ent = -(lp.exp() * lp.clamp(min=-1e4)).sum(1)
    if s["op"] == "score":
        if s["k"] == 0:
            return logp, ent, None, None
        at = torch.sort(s["x"].double(), dim=1, descending=True, stable=True).indices
        return logp, ent, None, lp.gather(1, at[:, :s["k"]])
    (logp * s["dlogp"].double() + ent * s["dent"].double()).sum().backward()
    return logp.detach(), ent.detach(), x.grad


def _exact_recurrence(s):
    """Step by step; the gradients by torch's own differentiation of those steps."""
    learn = s["op"] == "learn"
    x, r, i, lam = (s[n].double().requires_grad_(learn) for n in ("x", "r", "i", "lam"))
    loga = -C * torch.nn.functional.softplus(lam, threshold=40) / (1 + torch.exp(-r))
    a = torch.exp(loga)
    b = (-torch.expm1(2 * loga)).sqrt() / (1 + torch.exp(-i)) * x
    if s["op"] == "token":
        h = a * s["h"].double() + b
        return h, h
    B, L, D = s["B"], s["L"], s["D"]
    h = s["h0"].double() if s["h0"] is not None else torch.zeros(B, D, device=x.device, dtype=torch.float64)
    h0 = h.requires_grad_(learn)
    if s["lengths"] is not None:
        on = (torch.arange(L, device=x.device) < s["lengths"][:, None])[..., None]
        a, b = torch.where(on, a, 1.0), torch.where(on, b, 0.0)
    steps = []
    for at, bt in zip(a.unbind(1), b.unbind(1)):
        h = torch.addcmul(bt, at, h)
        steps.append(h)
    y = torch.stack(steps, 1)
    if s["lengths"] is not None:
        y = torch.where(on, y, 0.0)
    if not learn:
        return y, h
    loss = (y * s["dy"].double()).sum()
    if s["dhT"] is not None:
        loss = loss + (h * s["dhT"].double()).sum()
    grads = torch.autograd.grad(loss, (x, r, i, lam, h0))
    return y.detach(), h.detach(), *grads


def _exact_norms(s):
    teach = s["op"] == "teach"
    names = ["x", "y", "z", "post", "scale", "pre"]
    v = {n: s[n].double().requires_grad_(teach) if s[n] is not None else None for n in names}
    u = v["y"] / (v["y"].square().sum(-1, keepdim=True) / s["D"] + EPS).sqrt() * v["post"]
    if v["z"] is not None:
        u = u * v["z"] / (1 + torch.exp(-v["z"]))
    x1 = v["x"] + v["scale"] * u
    n = x1 / (x1.square().sum(-1, keepdim=True) / s["D"] + EPS).sqrt() * v["pre"]
    if not teach:
        return x1, n
    loss = (x1 * s["dx1"].double()).sum() + (n * s["dn"].double()).sum()
    there = [m for m in names if v[m] is not None]
    grads = dict(zip(there, torch.autograd.grad(loss, [v[m] for m in there])))
    return x1.detach(), n.detach(), *(grads.get(m) for m in names)
