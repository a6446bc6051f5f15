"""The operators of a linear-attention layer together, as a model would call them: 8-bit input
projection, head norms with rotation, linear attention over a padded batch of prompts, 8-bit output
projection onto the residual; then the same for single tokens, with the state going on. Each stage is
held against the 64-bit result of the stage's own inputs (bounds as in the operators' own tests), and
captured runs against eager ones, bit for bit."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

D, H, G, K, V = 256, 4, 2, 64, 64        # width, query and key heads, head sizes
W = (H + G) * K + G * V


class Layer:
    def __init__(self, dtype, seed=0):
        from ssmjs_amd import kernels
        gen = torch.Generator(device="cuda").manual_seed(seed)
        f = lambda *s: torch.randn(*s, generator=gen, device="cuda")   # noqa: E731
        self.k = kernels
        self.dtype = dtype
        self.win, self.sin = kernels.quantize_rows(f(W, D) * D ** -0.5)
        self.wout, self.sout = kernels.quantize_rows(f(D, H * V) * (H * V) ** -0.5)
        self.wq, self.wk = 1 + 0.1 * f(K), 1 + 0.1 * f(K)
        self.freqs = 10000.0 ** (-torch.arange(K // 2, device="cuda", dtype=torch.float64) / (K // 2))
        self.g = -torch.exp2(-8 * torch.arange(1, H + 1, device="cuda") / H).float()

    def heads(self, x, pos):
        """(q, k, v) of rows x (.., D); q and k are normed and turned in place."""
        rows = self.k.linear_q8(x.reshape(-1, D), self.win, self.sin).view(*x.shape[:-1], W)
        q = rows[..., :H * K].unflatten(-1, (H, K))
        k = rows[..., H * K:(H + G) * K].unflatten(-1, (G, K))
        v = rows[..., (H + G) * K:].unflatten(-1, (G, V))
        self.k.qk_norm_rope(q, k, self.wq, self.wk, pos, self.freqs, out=(q, k))
        return q, k, v

    def out(self, y, x):
        return self.k.linear_q8(y.reshape(-1, H * V), self.wout, self.sout, out=x.view(-1, D), beta=1.0).view_as(x)

    def prompt(self, x, pos, lengths, state):
        """The layer over (B,L,D) onto x, state (B,H,V,K) in place."""
        q, k, v = self.heads(x, pos)
        y = torch.zeros(*x.shape[:-1], H, V, dtype=self.dtype, device=x.device)
        self.k.linear_attention(q, k, v, self.g, scale=K ** -0.5, lengths=lengths, h0=state, hT=state, out=y)
        self.out(y, x)
        return q, k, v, y

    def token(self, x, pos, state):
        q, k, v = self.heads(x, pos)
        y = self.k.linear_attention_step(q, k, v, self.g, state, scale=K ** -0.5)
        self.out(y, x)
        return q, k, v, y


def attention64(q, k, v, g, lengths, h):
    """The recurrence in 64 bits: outputs, state, and the sums of magnitudes."""
    q, k, v = q.double(), k.double().repeat_interleave(H // G, 2), v.double().repeat_interleave(H // G, 2)
    keep = torch.exp(g.double())[:, None, None]
    h, a = h.double(), h.double().abs()
    y, ya = torch.zeros(*q.shape[:3], V, dtype=torch.float64, device="cuda"), None
    ya = torch.zeros_like(y)
    for t in range(q.shape[1]):
        on = (t < lengths)[:, None, None, None]
        kv = v[:, t, :, :, None] * k[:, t, :, None]
        h, a = torch.where(on, keep * h + kv, h), torch.where(on, keep * a + kv.abs(), a)
        y[:, t] = torch.where(on[..., 0], (h * q[:, t, :, None]).sum(-1) * K ** -0.5, 0.0)
        ya[:, t] = torch.where(on[..., 0], (a * q[:, t, :, None].abs()).sum(-1) * K ** -0.5, 0.0)
    return y, h, ya, a


def close(got, ref, bound, what):
    worst = float(((got.double() - ref).abs() / bound.clamp(min=1e-300)).max())
    print(f"  {what}: worst |err| / bound {worst:.3f}", flush=True)
    assert torch.isfinite(got).all() and worst <= 1, what


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompt_then_tokens(dtype):
    print(f"[case] linear layer, prompts then tokens {dtype}", flush=True)
    layer = Layer(dtype)
    B, L, T = 3, 90, 4
    gen = torch.Generator(device="cuda").manual_seed(5)
    lengths = torch.tensor([90, 1, 37], dtype=torch.int32, device="cuda")
    x = torch.randn(B, L, D, generator=gen, device="cuda").to(dtype)
    x0 = x.clone()
    pos = torch.arange(L, dtype=torch.int32, device="cuda").expand(B, L).contiguous()
    state = torch.zeros(B, H, V, K, device="cuda")
    q, k, v, y = layer.prompt(x, pos, lengths, state)
    torch.cuda.synchronize()
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    # the projection: integers, four roundings and the output's
    acc, s = layer.k.quantize_rows(x0.view(-1, D))
    p = acc.double() @ layer.win.double().t() * s.double()[:, None] * layer.sin.double()
    close(v, p.view(B, L, W)[..., (H + G) * K:].unflatten(-1, (G, V)),
          (4 * 2.0 ** -24 + half) * p.abs().view(B, L, W)[..., (H + G) * K:].unflatten(-1, (G, V)), "v")
    # the attention, of the q, k and v that it was given
    ry, rh, ya, a = attention64(q, k, v, layer.g, lengths, torch.zeros_like(state))
    units = 2.0 ** -24 * 2 * (K + 64 + 4 * 3)   # (2: the distances' share of the exponents' rounding)
    close(y, ry, units * ya + half * ry.abs() + (2.0 ** -16 * ya if half else 0), "y")
    close(state, rh, units * a, "state")
    # the output projection onto the residual
    acc, s = layer.k.quantize_rows(y.view(-1, H * V))
    p = acc.double() @ layer.wout.double().t() * s.double()[:, None] * layer.sout.double()
    r = p + x0.view(-1, D).double()
    close(x.view(-1, D), r, 2.0 ** -24 * (4 * p.abs() + 2 * r.abs()) + half * r.abs(), "residual")
    # the next tokens, each sequence from its own length on
    for i in range(T):
        x = torch.randn(B, D, generator=gen, device="cuda").to(dtype)
        before = state.clone()
        q, k, v, y = layer.token(x, lengths + i, state)
        torch.cuda.synchronize()
        one = torch.ones(B, dtype=torch.int32, device="cuda")
        ry, rh, ya, a = attention64(q[:, None], k[:, None], v[:, None], layer.g, one, before)
        close(y, ry[:, 0], 2.0 ** -24 * 2 * (K + 4) * ya[:, 0] + half * ry[:, 0].abs(), f"y of token {i}")
        close(state, rh, 2.0 ** -24 * 4 * a, f"state of token {i}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tokens_one_by_one_are_the_prompt(dtype):
    """The recurrent form over a prompt's tokens gives the chunked form's state and outputs."""
    print(f"[case] linear layer, one by one {dtype}", flush=True)
    layer = Layer(dtype, 1)
    B, L = 2, 70
    x = torch.randn(B, L, D, device="cuda").to(dtype)
    pos = torch.arange(100, 100 + L, dtype=torch.int32, device="cuda").expand(B, L).contiguous()
    q, k, v = layer.heads(x, pos)
    whole, each = torch.zeros(B, H, V, K, device="cuda"), torch.zeros(B, H, V, K, device="cuda")
    y = layer.k.linear_attention(q, k, v, layer.g, scale=K ** -0.5, hT=whole)
    ys = []
    for t in range(L):
        qt, kt, vt = layer.heads(x[:, t].contiguous(), pos[:, t].contiguous())
        assert torch.equal(qt, q[:, t]) and torch.equal(kt, k[:, t]) and torch.equal(vt, v[:, t])
        ys.append(layer.k.linear_attention_step(qt, kt, vt, layer.g, each, scale=K ** -0.5))
    torch.cuda.synchronize()
    n = torch.full((B,), L, device="cuda")
    ry, rh, ya, a = attention64(q, k, v, layer.g, n, torch.zeros_like(whole))
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    units = 2.0 ** -24 * 2 * (K + 64 + 12)
    close(y, ry, units * ya + half * ry.abs() + (2.0 ** -16 * ya if half else 0), "y, chunked")
    close(whole, rh, units * a, "state, chunked")
    units = 2.0 ** -24 * (K + 2 * L)
    close(torch.stack(ys, 1), ry, units * ya + half * ry.abs(), "y, one by one")
    close(each, rh, units * a, "state, one by one")


@pytest.mark.parametrize("B,L", [(3, 200), (1, 4500)])   # (segments and their workspace in the second)
def test_captured(B, L):
    """Two graphs, of the prompt and of the token, replayed in turn with other inputs between eager
    work: the eager bits each time."""
    print(f"[case] linear layer captured B={B} L={L}", flush=True)
    layer = Layer(torch.bfloat16, 2)
    x = torch.zeros(B, L, D, device="cuda", dtype=torch.bfloat16)
    xt = torch.zeros(B, D, device="cuda", dtype=torch.bfloat16)
    pos = torch.arange(L, dtype=torch.int32, device="cuda").expand(B, L).contiguous()
    at = torch.full((B,), L, dtype=torch.int32, device="cuda")
    lengths = torch.full((B,), L, dtype=torch.int32, device="cuda")
    state = torch.zeros(B, H, V, K, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.prompt(x, pos, lengths, state)
        layer.token(xt, at, state)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(one):
        y = layer.prompt(x, pos, lengths, state)[3]
    with torch.cuda.graph(two):
        yt = layer.token(xt, at, state)[3]
    for i in range(4):
        gen = torch.Generator(device="cuda").manual_seed(10 + i)
        fx = torch.randn(B, L, D, generator=gen, device="cuda").bfloat16()
        ft = torch.randn(B, D, generator=gen, device="cuda").bfloat16()
        h = torch.randn(B, H, V, K, generator=gen, device="cuda")
        n = torch.randint(1, L + 1, (B,), generator=gen, device="cuda").to(torch.int32)
        x.copy_(fx), xt.copy_(ft), state.copy_(h), lengths.copy_(n)
        one.replay()
        two.replay()
        torch.cuda.synchronize()
        ey = layer.prompt(fx, pos, n, h)[3]
        et = layer.token(ft, at, h)[3]
        torch.cuda.synchronize()
        for b in range(B):
            assert torch.equal(y[b, :n[b]], ey[b, :n[b]])
        for got, want in ((x, fx), (yt, et), (xt, ft), (state, h)):
            assert torch.equal(got, want)


def test_calls_on_two_streams():
    """Calls on two streams at once, each with workspaces of its own: the bits of calls in turn."""
    print("[case] linear layer on two streams", flush=True)
    layer = Layer(torch.bfloat16, 3)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    L = 3000
    pos = torch.arange(L, dtype=torch.int32, device="cuda")[None]
    xs = [torch.randn(1, L, D, device="cuda").bfloat16() for _ in streams]
    n = torch.tensor([L], dtype=torch.int32, device="cuda")
    want = []
    for x in xs:
        x, h = x.clone(), torch.zeros(1, H, V, K, device="cuda")
        want.append((layer.prompt(x, pos, n, h)[3], h, x))
    torch.cuda.synchronize()
    got = []
    for s, x in zip(streams, xs):
        with torch.cuda.stream(s):
            for _ in range(3):
                z, h = x.clone(), torch.zeros(1, H, V, K, device="cuda")
                out = (layer.prompt(z, pos, n, h)[3], h, z)
            got.append(out)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_python_refusals_on_the_device():
    from ssmjs_amd import kernels as k
    z = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt, device="cuda")   # noqa: E731
    q, g = z(2, 8, 4, 64), z(4)
    with pytest.raises(TypeError):
        k.linear_attention(q, z(2, 8, 2, 64, dt=torch.bfloat16), z(2, 8, 2, 64), g)
    with pytest.raises(ValueError, match="shape"):
        k.linear_attention(q, z(2, 7, 2, 64), z(2, 8, 2, 64), g)
    with pytest.raises(ValueError, match="shape"):
        k.linear_attention(q, z(2, 8, 2, 64), z(2, 8, 2, 64), z(3))
    with pytest.raises(ValueError, match="shape"):
        k.linear_attention(q, z(2, 8, 2, 64), z(2, 8, 2, 64), g, hT=z(2, 4, 64, 32))
    with pytest.raises(TypeError):
        k.linear_attention(q, z(2, 8, 2, 64), z(2, 8, 2, 64), g, lengths=z(2, dt=torch.int64))
    with pytest.raises(k._lib.SsmError, match="bad shape"):   # 4 query heads over 3 of keys
        k.linear_attention(q, z(2, 8, 3, 64), z(2, 8, 3, 64), g)
    with pytest.raises(ValueError, match="contiguous"):
        k.linear_attention_step(q[:, 0], z(2, 2, 64), z(2, 2, 64), g, z(2, 4, 64, 128)[..., :64])
    with pytest.raises(ValueError, match="state"):
        k.linear_attention_step(q[:, 0], z(2, 2, 64), z(2, 2, 64), g, None)
    with pytest.raises(ValueError, match="shape"):
        k.qk_norm_rope(q, z(2, 8, 2, 32), None, None, z(2, 8, dt=torch.int32), None)
    with pytest.raises(ValueError, match="shape"):
        k.linear_q8(z(2, 64), z(8, 32, dt=torch.int8), z(8))
    with pytest.raises(TypeError):
        k.linear_q8(z(2, 64), z(8, 64), z(8))
    with pytest.raises(ValueError, match="shape"):
        k.linear_i8(z(2, 64, dt=torch.int8), z(3), z(8, 64, dt=torch.int8), z(8))
