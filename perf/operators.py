"""Measured cases of the operators of a linear-attention layer whose projections are held in 8 bits.

  heads     qk_norm_rope: RMS norm of every query and key head, with the position rotation
  prompt    linear_attention: linear attention with a decay for each head, over whole prompts
  token     linear_attention_step: the same for one token of every sequence, state in place
  product   linear_q8: y = x W^T (+ bias) with the rows of x rounded to 8-bit integers on the way
            and the weights held in 8 bits with a scale for each output channel

`run` computes them from elementary torch operations in 32 bits, or, where `own` is true, with the
calls of ssmjs_amd.kernels. `exact` follows the definitions in 64 bits.
"""
import math

import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}


# ------------------------------------------------------------------ cases
def listed():
    def heads(name, B, L, H, G, D, R, pair, dt, far):
        return {"name": name, "op": "heads", "B": B, "L": L, "H": H, "G": G, "D": D, "R": R,
                "pair": pair, "dtype": dt, "far": far}

    def prompt(name, B, L, H, G, K, V, dt, ragged, state):
        return {"name": name, "op": "prompt", "B": B, "L": L, "H": H, "G": G, "K": K, "V": V,
                "dtype": dt, "ragged": ragged, "state": state}

    def token(name, B, H, G, K, V, dt):
        return {"name": name, "op": "token", "B": B, "H": H, "G": G, "K": K, "V": V, "dtype": dt}

    def product(name, M, N, K, dt, bias):
        return {"name": name, "op": "product", "M": M, "N": N, "K": K, "dtype": dt, "bias": bias}

    return [
        # one token of each of 64 decoded sequences, positions deep in a long context
        heads("heads of 64 tokens", 64, 1, 32, 8, 128, 128, "half", "bf16", 200000),
        # prompts of 4096 tokens, rotation of half of each head, pairs side by side
        heads("heads of prompts", 4, 4096, 32, 4, 128, 64, "beside", "bf16", 0),
        # a batch of equal prompts at a large model's width
        prompt("prompts bf16", 8, 4096, 16, 16, 128, 128, "bf16", False, False),
        # prompts of mixed lengths in one padded batch (none and one token among them), keys and
        # values shared by four heads, continuing from a state
        prompt("ragged prompts bf16", 8, 1500, 32, 8, 128, 128, "bf16", True, True),
        # a session's prompt in the model path's own type, 12 heads of 128 (the large preset)
        prompt("prompts f32", 2, 2000, 12, 12, 128, 128, "f32", False, True),
        # one long document with few heads
        prompt("long prompt bf16", 1, 32768, 8, 8, 64, 64, "bf16", False, False),
        # a single session's next token
        token("token of one session", 1, 12, 12, 128, 128, "f32"),
        # the next token of a full batch
        token("token of 64 sessions", 64, 32, 8, 128, 128, "bf16"),
        # a single session's token through the widest projection of the 2048-wide layer
        product("8-bit product of a token", 1, 8512, 2048, "f32", False),
        # a full batch of decoded tokens
        product("8-bit product of 64 tokens", 64, 8512, 2048, "bf16", False),
        # an odd prompt through the 1024-wide model's input projection
        product("8-bit product of 1000 rows", 1000, 4384, 1024, "f32", True),
        # a batch of prompts through the 2048-wide layer's input projection
        product("8-bit product of prompts", 8192, 8512, 2048, "bf16", False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["heads", "prompt", "prompt", "token", "product", "product"])
    dt = rng.choice(["f32", "bf16"])
    G = rng.choice([1, 2, 4, 8, 3])
    H = G * rng.choice([1, 2, 4])
    if op == "heads":
        D = rng.choice([64, 128, 128, 80, 256])
        rows = _log(rng, 1, 16384)
        B = rng.choice([b for b in (1, 2, 5, 64) if b <= rows])
        return {"op": op, "B": B, "L": max(1, rows // B), "H": H, "G": G, "D": D,
                "R": rng.choice([D, D // 2]), "pair": rng.choice(["half", "beside"]), "dtype": dt,
                "far": rng.choice([0, 5000, 1000000])}
    if op == "prompt":
        K, V = rng.choice([(128, 128), (128, 128), (64, 64), (64, 128), (96, 128), (32, 64)])
        B = rng.choice([1, 1, 2, 4, 7])
        most = min(32768, (1 << 26) // (B * H * (K + V)) * (1 if dt == "f32" else 2))
        return {"op": op, "B": B, "L": _log(rng, 1, most), "H": H, "G": G, "K": K, "V": V,
                "dtype": dt, "ragged": rng.random() < 0.4, "state": rng.random() < 0.5}
    if op == "token":
        K, V = rng.choice([(128, 128), (128, 128), (64, 64), (64, 128), (96, 128), (32, 64)])
        return {"op": op, "B": _log(rng, 1, 64), "H": H, "G": G, "K": K, "V": V, "dtype": dt}
    K = rng.choice([256, 768, 1000, 1024, 1536, 2048, 4096])
    N = rng.choice([256, 768, 1000, 2048, 4384, 4096])
    most = min(8192, (1 << 37) // (N * K))
    return {"op": op, "M": _log(rng, 1, most), "N": N, "K": K, "dtype": dt,
            "bias": rng.random() < 0.5}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    c = dict(case)
    dt = DT[c["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    if c["op"] == "heads":
        B, L, H, G, D, R = (c[x] for x in "BLHGDR")
        # the heads as the input projection leaves them: q, k and v side by side in each row
        rows = normal(B, L, (H + 2 * G) * D).to(dt)
        c["q"] = rows[..., :H * D].unflatten(-1, (H, D))
        c["k"] = rows[..., H * D:(H + G) * D].unflatten(-1, (G, D))
        c["wq"] = 1 + 0.2 * normal(D)
        c["wk"] = 1 + 0.2 * normal(D)
        first = torch.randint(0, c["far"] + 1, (B, 1), generator=gen, device=dev)
        c["pos"] = (first + torch.arange(L, device=dev)).to(torch.int32)
        c["freq"] = 10000.0 ** (-torch.arange(R // 2, device=dev, dtype=torch.float64) / (R // 2))
    elif c["op"] in ("prompt", "token"):
        B, H, G, K, V = (c[x] for x in "BHGKV")
        L = c.get("L", 1)
        # heads of unit size, as the norms leave them, and values as a projection does
        c["q"] = normal(B, L, H, K).to(dt)
        c["k"] = normal(B, L, G, K).to(dt)
        c["v"] = normal(B, L, G, V).to(dt)
        c["scale"] = K ** -0.5
        # memories from a token or two to some hundreds of tokens over the heads
        c["g"] = -torch.exp2(-8 * torch.arange(1, H + 1, device=dev, dtype=torch.float32) / H)
        c["lengths"] = None
        if c["op"] == "prompt":
            c["y"] = torch.zeros(B, L, H, V, device=dev, dtype=dt)
            c["h0"] = normal(B, H, V, K) if c["state"] else None
            c["hT"] = torch.zeros(B, H, V, K, device=dev)
            if c["ragged"]:
                n = torch.randint(0, L + 1, (B,), generator=gen, device=dev)
                n[0] = L
                n[1:2] = 0
                n[2:3] = 1
                c["lengths"] = n.to(torch.int32)
        else:
            c["q"], c["k"], c["v"] = c["q"][:, 0], c["k"][:, 0], c["v"][:, 0]
            c["h"] = normal(B, H, V, K)
    else:
        M, N, K = c["M"], c["N"], c["K"]
        # activations with a few large channels, and weights rounded once, as a program keeps them
        size = torch.exp(0.5 * normal(K)) * torch.where(torch.rand(K, generator=gen, device=dev) < 0.01, 10.0, 1.0)
        c["x"] = (normal(M, K) * size).to(dt)
        w = normal(N, K) * K ** -0.5
        c["sw"] = (w.abs().amax(1).double() / 127).float()
        c["wq"] = torch.round(w.double() / c["sw"].double()[:, None]).to(torch.int8)
        c["b"] = normal(N) if c["bias"] else None
    return c


# ------------------------------------------------------------------ one pass
def run(s):
    if own:
        from ssmjs_amd import kernels
        if s["op"] == "heads":
            return kernels.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["pos"], s["freq"],
                                        eps=1e-6, interleaved=s["pair"] == "beside")
        if s["op"] == "prompt":
            y = kernels.linear_attention(s["q"], s["k"], s["v"], s["g"], scale=s["scale"],
                                         lengths=s["lengths"], h0=s["h0"], hT=s["hT"])
            return y, s["hT"]
        if s["op"] == "token":
            return kernels.linear_attention_step(s["q"], s["k"], s["v"], s["g"], s["h"],
                                                 scale=s["scale"]), s["h"]
        return kernels.linear_q8(s["x"], s["wq"], s["sw"], bias=s["b"])
    return {"heads": _heads, "prompt": _prompt, "token": _token, "product": _product}[s["op"]](s)


def _rotate(x, w, s):
    R = s["R"]
    f = x.float()
    f = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + 1e-6) * w
    angle = s["pos"].double()[..., None] * s["freq"]
    cos, sin = (t.float()[:, :, None] for t in (torch.cos(angle), torch.sin(angle)))
    if s["pair"] == "half":
        a, b = f[..., :R // 2], f[..., R // 2:R]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = f[..., 0:R:2], f[..., 1:R:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, f[..., R:]], -1).to(x.dtype)


def _heads(s):
    return _rotate(s["q"], s["wq"], s), _rotate(s["k"], s["wk"], s)


def _power(g, n):
    """exp(g n) in 32 bits; the exponents' product in 64."""
    return torch.exp(g.double() * n.double()).float()


def _prompt(s):
    """Blocks of C tokens: products within each block, and the blocks' states carried by one
    product with the decays between blocks."""
    B, L, H, G, K, V = (s[x] for x in "BLHGKV")
    C = min(128, L)
    n = -(-L // C)
    dev, g = s["q"].device, s["g"]
    q, k, v = (t.float().permute(0, 2, 1, 3) for t in (s["q"], s["k"], s["v"]))
    k, v = (t.repeat_interleave(H // G, 1) for t in (k, v))
    t = torch.arange(L, device=dev)
    length = s["lengths"].long() if s["lengths"] is not None else torch.full((B,), L, device=dev)
    inside = (t < length[:, None])[:, None, :, None]
    k = torch.where(inside, k, 0.0)
    v = torch.where(inside, v, 0.0)
    # the state behind each sequence's last token
    left = (length[:, None] - 1 - t).clamp(min=0)[:, None]
    hT = (v * _power(g[None, :, None], left)[..., None]).transpose(2, 3) @ k
    if s["h0"] is not None:
        hT = hT + _power(g[None], length[:, None])[..., None, None] * s["h0"]
    q, k, v = (torch.nn.functional.pad(x, (0, 0, 0, n * C - L)).reshape(B, H, n, C, -1)
               for x in (q, k, v))
    i = torch.arange(C, device=dev)
    gap = (i[:, None] - i).clamp(min=0)
    near = torch.where(i[:, None] >= i, _power(g[:, None, None], gap), 0.0)
    y = (q @ k.transpose(-1, -2) * near[:, None]) @ v
    own_state = (v * _power(g[:, None], C - 1 - i)[:, None, :, None]).transpose(-1, -2) @ k
    m = torch.arange(n, device=dev)
    apart = C * (m[:, None] - 1 - m).clamp(min=0)
    carry = torch.where(m[:, None] > m, _power(g[:, None, None], apart), 0.0)
    enter = (carry @ own_state.reshape(B, H, n, V * K)).reshape(B, H, n, V, K)
    if s["h0"] is not None:
        enter = enter + _power(g[:, None], C * m)[..., None, None] * s["h0"][:, :, None]
    y = y + (q @ enter.transpose(-1, -2)) * _power(g[:, None], i + 1)[:, None, :, None]
    y = y.reshape(B, H, n * C, V)[:, :, :L] * s["scale"]
    return torch.where(inside, y, 0.0).permute(0, 2, 1, 3).to(s["q"].dtype), hT


def _token(s):
    q, k, v = (s[x].float() for x in "qkv")
    k, v = (t.repeat_interleave(s["H"] // s["G"], 1) for t in (k, v))
    h = s["h"]
    h.mul_(torch.exp(s["g"].double()).float()[:, None, None]).add_(v[..., None] * k[..., None, :])
    return ((h @ q[..., None])[..., 0] * s["scale"]).to(s["q"].dtype), h


def _product(s):
    x = s["x"].float()
    sx = (x.abs().amax(1).double() / 127).float()
    xq = torch.round(x.double() / sx.double()[:, None]).float()
    y = (xq @ s["wq"].float().t()) * sx[:, None] * s["sw"]
    if s["b"] is not None:
        y = y + s["b"]
    return y.to(s["x"].dtype)


# ------------------------------------------------------------------ what a pass cannot do without
def work(c):
    e = SIZE[c["dtype"]]
    if c["op"] == "heads":
        n = c["B"] * c["L"] * (c["H"] + c["G"]) * c["D"]
        return {"bytes": 2 * n * e + 4 * c["B"] * c["L"], "flops": 8 * n}
    if c["op"] == "product":
        M, N, K = c["M"], c["N"], c["K"]
        return {"bytes": (M * K + M * N) * e + N * K + 4 * N * (2 if c["bias"] else 1),
                "flops": 2 * M * N * K}
    B, L, H, G, K, V = c["B"], c.get("L", 1), c["H"], c["G"], c["K"], c["V"]
    states = 2 if c["op"] == "token" or c["state"] else 1
    rows = B * L
    if c.get("ragged"):
        rows = L + min(1, max(0, B - 2)) + max(0, B - 3) * L // 2   # L, 0, 1 and L / 2 on average
    return {"bytes": rows * (H * (K + V) + G * (K + V)) * e + states * 4 * B * H * K * V,
            "flops": 4 * rows * H * K * V}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "heads":
        angle = s["pos"].double()[:, :, None, None] * s["freq"]
        turn = torch.polar(torch.ones_like(angle), angle)
        done = []
        for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
            x = x.double()
            x = x / (x.square().sum(-1, keepdim=True) / s["D"] + 1e-6).sqrt() * w.double()
            half = s["R"] // 2
            at = torch.arange(half, device=x.device)
            re, im = (at, at + half) if s["pair"] == "half" else (2 * at, 2 * at + 1)
            z = torch.complex(x[..., re], x[..., im]) * turn
            x[..., re], x[..., im] = z.real, z.imag
            done.append(x)
        return tuple(done)
    if s["op"] == "product":
        x = s["x"].double()
        sx = (x.abs().max(1).values / 127).float().double()
        y = (x / sx[:, None]).round() @ s["wq"].double().t() * (sx[:, None] * s["sw"].double())
        return y if s["b"] is None else y + s["b"].double()
    group = torch.arange(s["H"], device=s["q"].device) // (s["H"] // s["G"])
    keep = torch.exp(s["g"].double())[:, None, None]
    if s["op"] == "token":
        k, v = s["k"].double()[:, group], s["v"].double()[:, group]
        h = keep * s["h"].double() + v[..., :, None] * k[..., None, :]
        return (h * s["q"].double()[:, :, None]).sum(-1) * s["scale"], h
    B, L, H, K, V = (s[x] for x in "BLHKV")
    h = torch.zeros(B, H, V, K, device="cuda", dtype=torch.float64)
    if s["h0"] is not None:
        h += s["h0"]
    y = torch.zeros(B, L, H, V, device="cuda", dtype=torch.float64)
    for t in range(L):
        q, k, v = s["q"][:, t].double(), s["k"][:, t, group].double(), s["v"][:, t, group].double()
        new = torch.baddbmm((keep * h).flatten(0, 1), v.reshape(-1, V, 1), k.reshape(-1, 1, K))
        new = new.reshape(h.shape)
        out = torch.bmm(new.flatten(0, 1), q.reshape(-1, K, 1)).reshape(B, H, V) * s["scale"]
        if s["lengths"] is None:
            h, y[:, t] = new, out
        else:
            on = (t < s["lengths"])[:, None, None]
            h = torch.where(on[..., None], new, h)
            y[:, t] = torch.where(on, out, 0.0)
    return y, h
