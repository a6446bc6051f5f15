"""A small gated-recurrence model made of gated_recurrence, block_norm and token_logprobs: trained on a padded batch,
then answering token by token, eager and captured, against the same model in 64 bits.

Bounds: an operator's or a product's result is within 100 * 2^-24 of its value and of the magnitudes it adds up (the
operators' own tests hold them to less; products here add up 64 to 97 terms). The model in 64 bits with each such
result moved by that much, the signs drawn, tells what this does to any later value; four times the largest of eight
draws is the bound, over a tensor's largest.
A row's log S, S = sum e^{x - max} >= 1, takes the rounding of S over as 2^-24 in the absolute, however small log S is:
log probabilities and entropies, which add it, are moved by NOISE of 1 + their value."""
import pytest

torch = pytest.importorskip("torch")

import test_gpu_gated_recurrence as recurrence  # noqa: E402

pytestmark = pytest.mark.gpu

V, D, LAYERS, B, L = 97, 64, 2, 3, 200
NOISE = 100 * 2.0 ** -24
EPS, C = 1e-6, 8.0


def model(seed, size=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    f = lambda *s: torch.randn(*s, generator=gen, device="cuda")   # noqa: E731
    p = {"emb": size * f(V, D), "pre0": 1 + 0.1 * f(D)}
    for n in range(LAYERS):
        p |= {f"in{n}": f(D, 4 * D) / 8, f"out{n}": f(D, D) / 8, f"lam{n}": 2 * f(D) - 3, f"post{n}": 1 + 0.1 * f(D),
              f"scale{n}": 0.5 + 0.1 * f(D), f"pre{n + 1}": 1 + 0.1 * f(D)}
    ids = torch.randint(0, V, (B, L), generator=gen, device="cuda")
    lengths = torch.tensor([L, 1, 131], dtype=torch.int32, device="cuda")
    nxt = torch.full((B, L), -1, dtype=torch.int32, device="cuda")
    nxt[:, :-1] = ids[:, 1:].int()
    nxt[torch.arange(L, device="cuda") >= lengths[:, None] - 1] = -1
    return p, ids, lengths, nxt


# ---- in 64 bits
def plain(p, ids, lengths, nxt, jog=lambda t, m=None: t):
    """Logits, logp, entropy and the loss; jog(result, magnitudes) moves a result."""
    p = {k: v.double() for k, v in p.items()}
    on = (torch.arange(L, device="cuda") < lengths[:, None])[..., None]

    def mm(a, b):
        return jog((a.reshape(-1, a.shape[-1]) @ b).view(*a.shape[:-1], -1), a.detach().abs().reshape(-1, a.shape[-1]) @ b.detach().abs())

    def norm(t, w):
        return t / (t.square().mean(-1, keepdim=True) + EPS).sqrt() * w

    x = p["emb"][ids]
    n = jog(norm(x, p["pre0"]))
    for k in range(LAYERS):
        v, r, i, z = mm(n, p[f"in{k}"]).split(D, -1)
        zz = C * torch.nn.functional.softplus(p[f"lam{k}"]) * torch.sigmoid(r)
        a, b = torch.exp(-zz), (-torch.expm1(-2 * zz)).sqrt() * torch.sigmoid(i) * v
        h, hs = torch.zeros(B, D, dtype=torch.float64, device="cuda"), []
        for t in range(L):
            h = a[:, t] * h + b[:, t]
            hs.append(h)
        y = jog(torch.where(on, torch.stack(hs, 1), 0.0))
        x = jog(x + p[f"scale{k}"] * norm(mm(y, p[f"out{k}"]), p[f"post{k}"]) * torch.nn.functional.silu(z))
        n = jog(norm(x, p[f"pre{k + 1}"]))
    lg = mm(n, p["emb"].t())
    ls = torch.log_softmax(lg, -1)
    ls = jog(ls, 1 + ls.detach().abs())
    ent = -(ls.exp() * ls).sum(-1)
    ent = jog(ent, 1 + ent.detach().abs())
    given = nxt >= 0
    logp = torch.where(given, ls.gather(-1, nxt.clamp(min=0).long()[..., None])[..., 0], 0.0)
    return lg, logp, ent, -logp.sum() + 0.1 * torch.where(given, ent, 0.0).sum()


def plain_grads(p, *batch, jog=lambda t, m=None: t):
    leaves = {k: v.double().requires_grad_() for k, v in p.items()}
    lg, logp, ent, loss = plain(leaves, *batch, jog=jog)
    g = torch.autograd.grad(loss, list(leaves.values()))
    return {"logits": lg.detach(), "logp": logp.detach(), "entropy": ent.detach()} | dict(zip(leaves, g))


class _Jog(torch.autograd.Function):
    """Moves a result, and what comes back to it."""
    @staticmethod
    def forward(ctx, t, m, gen):
        ctx.gen = gen
        sign = torch.randint(0, 2, t.shape, generator=gen, device="cuda") * 2 - 1
        return t + NOISE * sign * (t.abs() if m is None else m.reshape(t.shape))

    @staticmethod
    def backward(ctx, g):
        return g * (1 + NOISE * (torch.randint(0, 2, g.shape, generator=ctx.gen, device="cuda") * 2 - 1)), None, None


def bounds(p, *batch):
    ref = plain_grads(p, *batch)
    worst = {k: 0.0 for k in ref}
    for s in range(8):
        gen = torch.Generator(device="cuda").manual_seed(s)
        moved = plain_grads(p, *batch, jog=lambda t, m=None: _Jog.apply(t, m, gen))
        worst = {k: max(w, float((moved[k] - ref[k]).abs().max())) for k, w in worst.items()}
    return ref, {k: 4 * w for k, w in worst.items()}


# ---- with the operators
def run(p, ids, lengths, nxt):
    """A training step: logits, logp, entropy and the gradients of every parameter."""
    from ssmjs_amd import kernels as k
    x = p["emb"][ids]
    zero = torch.zeros_like(x)
    kept = []
    x1, n = k.block_norm(x, zero, pre=p["pre0"], eps=EPS)
    for q in range(LAYERS):
        u = (n.view(-1, D) @ p[f"in{q}"]).view(B, L, 4 * D)
        v, r, i, z = u.split(D, -1)
        st = k.gated_recurrence_states(B, L, D, "cuda")
        y = k.gated_recurrence(v, r, i, p[f"lam{q}"], lengths=lengths, states=st)
        o = (y.view(-1, D) @ p[f"out{q}"]).view(B, L, D)
        kept.append((x1, n, u, st, y, o))
        x1, n = k.block_norm(x1, o, z, p[f"post{q}"], p[f"scale{q}"], p[f"pre{q + 1}"], EPS)
    lg = n.view(-1, D) @ p["emb"].t()
    stats = torch.empty(B * L, 2, device="cuda")
    logp, ent, _, _ = k.token_logprobs(lg, nxt.view(-1), stats=stats)
    given = (nxt.view(-1) >= 0).float()
    g = {}
    dlg = k.token_logprobs_backward(lg, nxt.view(-1), stats, ent, -given, 0.1 * given)
    g["emb"] = dlg.t() @ n.view(-1, D)
    dn, dx1 = (dlg @ p["emb"]).view(B, L, D), None
    for q in reversed(range(LAYERS)):
        x0, n0, u, st, y, o = kept[q]
        v, r, i, z = u.split(D, -1)
        du = torch.empty_like(u)
        dx = torch.empty_like(x0)
        do = torch.empty_like(x0)
        _, _, _, g[f"post{q}"], g[f"scale{q}"], g[f"pre{q + 1}"] = k.block_norm_backward(
            dx1, dn, x0, o, z, p[f"post{q}"], p[f"scale{q}"], p[f"pre{q + 1}"], EPS, out=(dx, do, du[..., 3 * D:]))
        dx1 = dx
        g[f"out{q}"] = y.view(-1, D).t() @ do.view(-1, D)
        dy = (do.view(-1, D) @ p[f"out{q}"].t()).view(B, L, D)
        du[..., :3 * D] = 0      # (rows behind a sequence stay so)
        *_, g[f"lam{q}"] = k.gated_recurrence_backward(dy, v, r, i, p[f"lam{q}"], st, lengths=lengths,
                                                       out=du[..., :3 * D].split(D, -1))
        g[f"in{q}"] = n0.view(-1, D).t() @ du.view(-1, 4 * D)
        dn = (du.view(-1, 4 * D) @ p[f"in{q}"].t()).view(B, L, D)
    dx, _, _, _, _, g["pre0"] = k.block_norm_backward(dx1, dn, x, zero, pre=p["pre0"], eps=EPS)
    g["emb"] = g["emb"].index_add(0, ids.view(-1), dx.view(-1, D)) if not torch.cuda.is_current_stream_capturing() else \
        g["emb"] + torch.nn.functional.one_hot(ids.view(-1), V).float().t() @ dx.view(-1, D)
    return {"logits": lg.view(B, L, V), "logp": logp.view(B, L), "entropy": ent.view(B, L)} | g


@pytest.mark.parametrize("size", [1.0, 0.1])     # rows of a likeliest token, and of many
def test_training_step(size):
    print(f"[case] gated model, training step {size}", flush=True)
    p, *batch = model(1, size)
    ref, bound = bounds(p, *batch)
    got = run(p, *batch)
    torch.cuda.synchronize()
    for k, want in ref.items():
        worst = float((got[k].double() - want).abs().max()) / bound[k]
        print(f"  {k}: worst |err| / bound {worst:.3f}", flush=True)
        assert worst <= 1, k


@pytest.mark.parametrize("size", [1.0, 0.1])
def test_prompt_then_tokens(size):
    """A prompt leaves its states, from which tokens follow one by one, eager and as a captured call."""
    from ssmjs_amd import kernels as k
    print("[case] gated model, prompt then tokens", flush=True)
    p, ids, _, nxt = model(2, size)
    whole = torch.full((B,), L, dtype=torch.int32, device="cuda")
    ref, bound = bounds(p, ids, whole, nxt)
    cut = L - 8

    def trunk(x, recur):
        x1, n = k.block_norm(x, torch.zeros_like(x), pre=p["pre0"], eps=EPS)
        for q in range(LAYERS):
            u = (n.view(-1, D) @ p[f"in{q}"]).view(*x.shape[:-1], 4 * D)
            v, r, i, z = u.split(D, -1)
            o = (recur(q, v, r, i).view(-1, D) @ p[f"out{q}"]).view_as(x)
            x1, n = k.block_norm(x1, o, z, p[f"post{q}"], p[f"scale{q}"], p[f"pre{q + 1}"], EPS)
        return n.view(-1, D) @ p["emb"].t()

    h = torch.zeros(LAYERS, B, D, device="cuda")
    lg = trunk(p["emb"][ids[:, :cut]], lambda q, v, r, i: k.gated_recurrence(v, r, i, p[f"lam{q}"], h0=h[q], hT=h[q]))
    torch.cuda.synchronize()
    assert float((lg.view(B, cut, V).double() - ref["logits"][:, :cut]).abs().max()) <= bound["logits"]
    after = h.clone()
    token = torch.zeros(B, dtype=torch.long, device="cuda")

    def answer():
        lg = trunk(p["emb"][token], lambda q, v, r, i: k.gated_recurrence_step(v, r, i, p[f"lam{q}"], h[q]))
        return [lg, *k.token_logprobs(lg, None, 5)[1:]]

    eager = []
    for t in range(cut, L):
        token.copy_(ids[:, t])
        eager.append(answer())
        torch.cuda.synchronize()
        lg, ent, top, toplp = eager[-1]
        want = ref["logits"][:, t]
        assert float((lg.double() - want).abs().max()) <= bound["logits"]
        assert float((ent.double() - ref["entropy"][:, t]).abs().max()) <= bound["entropy"]
        ls = torch.log_softmax(want, -1)
        # a listed token is as likely as any that is not, but for the bound on either side
        assert float((toplp.double() - ls.gather(1, top.long())).abs().max()) <= bound["logits"] * 2 + bound["entropy"]
        rest = ls.scatter(1, top.long(), -1e9).amax(1)
        assert bool((ls.gather(1, top.long()).amin(1) >= rest - 2 * bound["logits"]).all())
    last = h.clone()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        answer()
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        out = answer()
    for _ in range(2):
        h.copy_(after)
        for n, t in enumerate(range(cut, L)):
            token.copy_(ids[:, t])
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, eager[n]):
                assert torch.equal(a, b)
        assert torch.equal(h, last)


def test_training_step_captured():
    """A captured step beside live eager work gives the eager bits, replay after replay, and so do two streams."""
    print("[case] gated model, captured training step", flush=True)
    p, ids, lengths, nxt = model(3)
    keep = [n for n in ("logits", "logp", "entropy", "lam0", "pre0", "post1", "scale0", "pre2")]
    want = run(p, ids, lengths, nxt)
    torch.cuda.synchronize()
    side, graph = [torch.cuda.Stream(), torch.cuda.Stream()], torch.cuda.CUDAGraph()
    got = []
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(run(p, ids, lengths, nxt))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(g[n], want[n]) for n in keep)
    with torch.cuda.graph(graph):
        out = run(p, ids, lengths, nxt)
    for _ in range(3):
        graph.replay()
        run(p, ids, lengths, nxt)
        torch.cuda.synchronize()
        assert all(torch.equal(out[n], want[n]) for n in keep)


@pytest.mark.parametrize("ragged", [False, True])
def test_states_in_place(ragged):
    """hT in h0's place and dh0 in dhT's, over one segment and several, whole and ragged."""
    from ssmjs_amd import kernels as k
    for b, n, d in ((3, 50, 68), (2, 5000, 64), (3, 3000, 33)):
        print(f"[case] states in place {b} {n} {d} {ragged}", flush=True)
        gen = torch.Generator(device="cuda").manual_seed(n)
        f = lambda *s: torch.randn(*s, generator=gen, device="cuda")   # noqa: E731
        x, r, i, dy, lam, h0, dhT = f(b, n, d), f(b, n, d), f(b, n, d), f(b, n, d), f(d) - 3, f(b, d), f(b, d)
        lengths = torch.tensor([n - 1, 0, 7][:b], dtype=torch.int32, device="cuda") if ragged else None
        st, hT, dh0 = k.gated_recurrence_states(b, n, d, "cuda"), torch.empty_like(h0), torch.empty_like(h0)
        y = k.gated_recurrence(x, r, i, lam, lengths=lengths, h0=h0, hT=hT, states=st)
        grads = k.gated_recurrence_backward(dy, x, r, i, lam, st, lengths=lengths, dhT=dhT, dh0=dh0)
        h, e = h0.clone(), dhT.clone()
        y2 = k.gated_recurrence(x, r, i, lam, lengths=lengths, h0=h, hT=h)
        grads2 = k.gated_recurrence_backward(dy, x, r, i, lam, st, lengths=lengths, dhT=e, dh0=e)
        torch.cuda.synchronize()
        assert torch.equal(y, y2) and torch.equal(h, hT) and torch.equal(e, dh0)
        assert all(torch.equal(a, c) for a, c in zip(grads, grads2))
        if ragged:      # (a sequence of nothing hands its state on)
            assert torch.equal(hT[1], h0[1]) and torch.equal(dh0[1], dhT[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,n,d", [(3, 16, 66), (70, 13, 64), (2, 17, 130), (3, 128, 64), (2, 129, 64), (40, 150, 1024), (17, 512, 2048)])
def test_short_prompts(b, n, d, dtype):
    """Short prompts, few and many, whole and ragged, are what the same tokens one by one give, and their gradients
    those of the same tokens in a longer, padded batch: the steps' order of sums differs, which is worth
    n / 2 + 32 roundings of each of the magnitudes added (here bounded by a walk over magnitudes)."""
    from ssmjs_amd import kernels as k
    print(f"[case] short prompts {b} {n} {d} {dtype}", flush=True)
    gen = torch.Generator(device="cuda").manual_seed(n)
    f = lambda *s: torch.randn(*s, generator=gen, device="cuda")   # noqa: E731
    x, r, i, dy = (f(b, n, d).to(dtype) for _ in range(4))
    lam, h0, dhT = f(d) - 3, f(b, d), f(b, d)
    half = 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -8
    lengths = torch.randint(0, n + 1, (b,), generator=gen, device="cuda").to(torch.int32)
    lengths[0] = n
    for ln in (None, lengths):
        st, hT = k.gated_recurrence_states(b, n, d, "cuda"), torch.empty_like(h0)
        y = k.gated_recurrence(x, r, i, lam, lengths=ln, h0=h0, hT=hT, states=st)
        # (the gates are the same numbers either way; every state adds up |h0| and the steps' inputs, sqrt(n) of |x| <= 6)
        scale = 6 * (n ** 0.5 + 1)
        tol = (n / 2 + 32) * 2.0 ** -24 * scale
        h, end = h0.clone(), h0.clone()
        for t in range(n):
            yt = k.gated_recurrence_step(x[:, t], r[:, t], i[:, t], lam, h)
            on = (torch.ones(b, dtype=torch.bool, device="cuda") if ln is None else t < ln)[:, None]
            want = torch.where(on, yt, 0).double()
            assert bool(((y[:, t].double() - want).abs() <= tol + 2 * half * want.abs()).all()), t
            end = torch.where(on, h, end)
        assert float((hT - end).abs().max()) <= tol
        # the same batch behind more padding: workgroups of another size
        more = 1400
        pad = lambda t: torch.cat([t, torch.full((b, more - n, d), float("nan"), device="cuda", dtype=dtype)], 1)   # noqa: E731
        whole = torch.full((b,), n, dtype=torch.int32, device="cuda") if ln is None else ln
        big = [pad(t) for t in (x, r, i, dy)]
        st2, dh0, dh02 = k.gated_recurrence_states(b, more, d, "cuda"), torch.empty_like(h0), torch.empty_like(h0)
        y2 = k.gated_recurrence(*big[:3], lam, lengths=whole, h0=h0, states=st2)
        assert bool(((y2[:, :n].double() - y.double()).abs() <= tol + 2 * half * y.double().abs()).all()) and bool((y2[:, n:] == 0).all())
        g = k.gated_recurrence_backward(dy, x, r, i, lam, st, lengths=ln, dhT=dhT, dh0=dh0)
        g2 = k.gated_recurrence_backward(big[3], *big[:3], lam, st2, lengths=whole, dhT=dhT, dh0=dh02)
        torch.cuda.synchronize()
        # adjoints add up like states; dr multiplies one by a state (and by at most 1)
        for a, c, m in ((g[0], g2[0], scale), (g[1], g2[1], scale * scale), (g[2], g2[2], 6 * scale), (dh0, dh02, scale)):
            c = c[:, :n] if c.dim() == 3 else c
            far = (a.double() - c.double()).abs()
            assert bool((far <= 4 * (n / 2 + 32) * 2.0 ** -24 * m + 2 * half * c.double().abs()).all())
        assert float((g[3] - g2[3]).abs().max()) <= 4 * (n / 2 + 32) * 2.0 ** -24 * scale * scale * b * n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_nothing_to_do(dtype):
    """Batches of no sequences and of no tokens: states go through, gradients of nothing are zeros."""
    from ssmjs_amd import kernels as k
    print(f"[case] nothing to do {dtype}", flush=True)
    e = lambda *s: torch.empty(*s, device="cuda", dtype=dtype)   # noqa: E731
    lam, w = torch.randn(70, device="cuda"), torch.ones(70, device="cuda")
    for b, n in ((0, 9), (3, 0), (0, 0)):
        x = e(b, n, 70)
        h0 = torch.randn(b, 70, device="cuda")
        hT, dh0 = torch.full_like(h0, 7.0), torch.full_like(h0, 7.0)
        st = k.gated_recurrence_states(b, n, 70, "cuda")
        for ln in (None, torch.zeros(b, dtype=torch.int32, device="cuda")):
            y = k.gated_recurrence(x, x, x, lam, lengths=ln, h0=h0, hT=hT, states=st)
            torch.cuda.synchronize()
            assert y.shape == x.shape and torch.equal(hT, h0)
            if b:
                g = k.gated_recurrence_backward(x, x, x, x, lam, st, lengths=ln, dhT=h0, dh0=dh0)
                torch.cuda.synchronize()
                assert torch.equal(dh0, h0) and bool((g[3] == 0).all())
    h = torch.empty(0, 70, device="cuda")
    assert k.gated_recurrence_step(e(0, 70), e(0, 70), e(0, 70), lam, h).shape == (0, 70)
    x1, n1 = k.block_norm(e(0, 70), e(0, 70), e(0, 70), w, w, w)
    assert x1.shape == n1.shape == (0, 70)
    g = k.block_norm_backward(x1, n1, e(0, 70), e(0, 70), e(0, 70), w, w, w)
    torch.cuda.synchronize()
    assert all(bool((t == 0).all()) and t.shape == (70,) for t in g[3:])
    ids, stats = torch.empty(0, dtype=torch.int32, device="cuda"), torch.empty(0, 2, device="cuda")
    lp, ent, top, _ = k.token_logprobs(e(0, 70), ids, 3, stats)
    assert lp.shape == ent.shape == (0,) and top.shape == (0, 3)
    assert k.token_logprobs_backward(e(0, 70), ids, stats, ent, lp, ent).shape == (0, 70)


def test_far_apart():
    """Rows whose offsets pass 2^31 elements give the bits of rows side by side."""
    from ssmjs_amd import kernels as k
    print("[case] far apart", flush=True)
    room = torch.empty((1 << 33) + (1 << 21), dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(3)
    f = lambda *s: torch.randn(*s, generator=gen, device="cuda").bfloat16()   # noqa: E731
    b, n, d, ld = 5, 3000, 130, (1 << 19) + 1000          # 5 * 3000 rows of 2^19: 2^32.9 elements
    x, r, i, dy = f(b, n, d), f(b, n, d), f(b, n, d), f(b, n, d)
    lam = torch.randn(d, generator=gen, device="cuda") - 3
    far = [room.as_strided((b, n, d), (n * ld, ld, 1), 1000 * j) for j in range(8)]
    for t, v in zip(far, (x, r, i, dy)):
        t.copy_(v)
    st, st2 = k.gated_recurrence_states(b, n, d, "cuda"), k.gated_recurrence_states(b, n, d, "cuda")
    y = k.gated_recurrence(x, r, i, lam, states=st)
    k.gated_recurrence(*far[:3], lam, states=st2, out=far[4])
    g = k.gated_recurrence_backward(dy, x, r, i, lam, st)
    g2 = k.gated_recurrence_backward(far[3], *far[:3], lam, st2, out=far[5:8])
    torch.cuda.synchronize()
    assert torch.equal(y, far[4]) and torch.equal(st, st2) and all(torch.equal(a, c) for a, c in zip(g, g2))
    # norms of the same rows, with x as z, r as x, i as y
    w = [torch.randn(d, generator=gen, device="cuda") for _ in range(3)]
    want = k.block_norm(r, i, x, *w)
    back = k.block_norm_backward(dy, y, r, i, x, *w)
    flat = lambda t: t.as_strided((b * n, d), (ld, 1), t.storage_offset())   # noqa: E731
    fx, fr, fi, fd, fy = (flat(t) for t in far[:5])
    got = k.block_norm(fr, fi, fx, *w, out=(flat(far[5]), flat(far[6])))
    torch.cuda.synchronize()
    assert all(torch.equal(a.view(-1, d), c) for a, c in zip(want, got))
    got = k.block_norm_backward(fd, fy, fr, fi, fx, *w, out=[flat(t) for t in far[5:8]])
    torch.cuda.synchronize()
    assert all(torch.equal(a.view(c.shape), c) for a, c in zip(back, got))
    # logits: nine rows 2^30 - 8 apart, and in place of them their gradient
    m, v = 9, 1001
    lg = f(m, v)
    wide = room.as_strided((m, v), ((1 << 30) - 8, 1), 5)
    wide.copy_(lg)
    ids = torch.arange(m, device="cuda").int() * 100
    stats, stats2 = torch.empty(m, 2, device="cuda"), torch.empty(m, 2, device="cuda")
    want, got = k.token_logprobs(lg, ids, 7, stats), k.token_logprobs(wide, ids, 7, stats2)
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(want, got))
    a = k.token_logprobs_backward(lg, ids, stats, want[1], want[0], want[1])
    k.token_logprobs_backward(wide, ids, stats2, want[1], want[0], want[1], out=wide)
    torch.cuda.synchronize()
    assert torch.equal(a, wide)


@pytest.mark.parametrize("L", [9, 200, 700])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_infinities_at_other_lengths(bad, L):
    """Infinities and NaN in workgroups of one wave and in those of 32 channels."""
    print(f"[case] infinities {L} {bad}", flush=True)
    recurrence.test_an_infinity_stays_where_it_is(bad, L)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", [
    (1, 129, 1, False, True, False, False), (3, 700, 33, True, True, True, False), (2, 256, 34, False, False, True, True),
    (2, 513, 66, True, True, False, True), (5, 1025, 100, True, True, True, False), (4, 900, 2048, False, True, False, False),
    (1, 1024, 68, False, True, False, True), (1, 10, 66, False, True, True, True), (2, 60, 33, True, True, False, True)])
def test_other_groups(case, dtype):
    """The recurrence and its gradients, to the bounds of its own tests, where groups of 32 channels and few waves run."""
    recurrence.test_forward_backward(case, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradient_of_logits_wherever_rows_lie(dtype):
    """Rows at every place in 16 bytes, of lengths around whole eights, gradients beside and in place: the bits of
    contiguous rows, and nothing beside the rows written."""
    from ssmjs_amd import kernels as k
    gen = torch.Generator(device="cuda").manual_seed(4)
    for n in (1, 5, 8, 9, 16, 23, 8184, 8185, 8192, 8199, 16384):
        print(f"[case] logits' gradient, {n} {dtype}", flush=True)
        lg = torch.randn(3, n, generator=gen, device="cuda").to(dtype)
        ids = torch.tensor([0, n // 2, n - 1], dtype=torch.int32, device="cuda")
        stats = torch.empty(3, 2, device="cuda")
        lp, ent, _, _ = k.token_logprobs(lg, ids, stats=stats)
        w, v = torch.randn(3, generator=gen, device="cuda"), torch.randn(3, generator=gen, device="cuda")
        want = k.token_logprobs_backward(lg, ids, stats, ent, w, v)
        for shift in range(9):
            for ld in (n, n + 3, n + 8):
                a = torch.full((3 * ld + 40,), 5.0, dtype=dtype, device="cuda")
                b = torch.full((3 * ld + 40,), 5.0, dtype=dtype, device="cuda")
                xs, out = (t.as_strided((3, n), (ld, 1), 8 + o) for t, o in ((a, shift), (b, (shift * 5 + 3) % 9)))
                xs.copy_(lg)
                k.token_logprobs_backward(xs, ids, stats, ent, w, v, out=out)
                k.token_logprobs_backward(xs, ids, stats, ent, w, v, out=xs)
                torch.cuda.synchronize()
                assert torch.equal(out, want) and torch.equal(xs, want)
                for t, r in ((a, xs), (b, out)):
                    r.fill_(5.0)
                    assert bool((t == 5).all())


@pytest.mark.parametrize("n", [12, 100, 700, 5000])
def test_lengths_out_of_range(n):
    """Lengths below 0 are 0, lengths above L are L."""
    from ssmjs_amd import kernels as k
    print(f"[case] lengths out of range {n}", flush=True)
    gen = torch.Generator(device="cuda").manual_seed(n)
    f = lambda *s: torch.randn(*s, generator=gen, device="cuda")   # noqa: E731
    x, r, i, dy, lam, h0 = f(4, n, 66), f(4, n, 66), f(4, n, 66), f(4, n, 66), f(66) - 3, f(4, 66)
    got = []
    for ln in ([-5, n + 7, 3, 2**31 - 1], [0, n, 3, n]):
        ln = torch.tensor(ln, dtype=torch.int32, device="cuda")
        st, hT, dh0 = k.gated_recurrence_states(4, n, 66, "cuda").zero_(), torch.empty_like(h0), torch.empty_like(h0)
        y = k.gated_recurrence(x, r, i, lam, lengths=ln, h0=h0, hT=hT, states=st)
        got.append([y, hT, st, dh0, *k.gated_recurrence_backward(dy, x, r, i, lam, st, lengths=ln, dhT=h0, dh0=dh0)])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(*got))
