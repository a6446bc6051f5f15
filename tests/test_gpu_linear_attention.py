"""linear_attention and linear_attention_step against the recurrence in 64 bits.

Bounds, with A = the same sums over magnitudes (|q|, |k|, |v|, |h0|, each weight times 1 + |g| times
its distance for the rounding of its exponent): an fp32 sum's error is at most 2^-24 A for every
rounding that a term meets: K for the product with the state, C = 64 within a chunk, and 4 for each
chunk that a state passes through. bfloat16: half a step of the output, 2^-8 |y|; the state and the
products q k enter their products in two parts each, 2^-16 A. States are fp32 sums whatever the inputs'
type."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def recurrence(q, k, v, g, scale, lengths, h0):
    """y, hT, A of y, A of hT."""
    q, k, v, g = (t.double() for t in (q, k, v, g))
    B, L, H, K = q.shape
    r = H // k.shape[2]
    k, v = k.repeat_interleave(r, 2), v.repeat_interleave(r, 2)
    V = v.shape[3]
    z = lambda *s: torch.zeros(*s, dtype=torch.float64, device=q.device)   # noqa: E731
    h = h0.double().clone() if h0 is not None else z(B, H, V, K)
    keep = torch.exp(g)[:, None, None]
    # magnitudes: a, and d the same with each weight times its distance
    a, d = h.abs(), z(B, H, V, K)
    y, ya = z(B, L, H, V), z(B, L, H, V)
    step = torch.where(g.isinf(), 0.0, g.abs())[:, None, None]
    n = lengths.tolist() if lengths is not None else [L] * B
    for t in range(L):
        on = torch.tensor([t < m for m in n], device=q.device)[:, None, None, None]
        kv = v[:, t, :, :, None] * k[:, t, :, None, :]
        h = torch.where(on, keep * h + kv, h)
        d = torch.where(on, keep * (d + step * a), d)
        a = torch.where(on, keep * a + kv.abs(), a)
        on = on[..., 0]
        y[:, t] = torch.where(on, (h @ q[:, t, :, :, None])[..., 0] * scale, 0.0)
        ya[:, t] = torch.where(on, ((a + d) @ q[:, t, :, :, None].abs())[..., 0] * abs(scale), 0.0)
    return y, h, ya, a + d


def make(B, L, H, G, K, V, dtype, seed, fast=False):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    f = lambda *s: torch.randn(*s, generator=gen, device="cuda")   # noqa: E731
    q, k, v = f(B, L, H, K).to(dtype), f(B, L, G, K).to(dtype), f(B, L, G, V).to(dtype)
    g = -torch.exp2(-8 * torch.arange(1, H + 1, device="cuda") / H) * (20 if fast else 1)
    return q, k, v, g.float(), f(B, H, V, K)


def close(got, ref, bound, what):
    got, ref = got.double(), ref.double()
    assert torch.isfinite(got).all(), what
    worst = float(((got - ref).abs() / bound.clamp(min=1e-300)).max()) if got.numel() else 0.0
    print(f"  {what}: worst |err| / bound {worst:.3f}", flush=True)
    assert worst <= 1, what


def bounds(ref, K, L, dtype):
    y, h, ya, ha = ref
    units = 2.0 ** -24 * (K + 64 + 4 * -(-L // 32))
    by = units * ya
    if dtype == torch.bfloat16:
        by = by + 2.0 ** -8 * y.abs() + 2.0 ** -16 * ya
    return by, units * ha


CASES = [   # B, L, H, G, K, V
    (1, 1, 1, 1, 1, 1), (1, 1, 2, 1, 64, 64), (2, 31, 2, 2, 64, 64), (1, 64, 3, 1, 128, 128),
    (1, 65, 2, 1, 128, 128), (2, 130, 4, 2, 128, 64), (1, 96, 2, 2, 64, 128), (1, 200, 2, 1, 96, 96),
    (1, 77, 2, 1, 256, 64), (1, 70, 1, 1, 200, 136), (1, 130, 2, 2, 33, 17), (1, 67, 1, 1, 129, 65),
    (1, 100, 2, 1, 32, 260), (1, 700, 2, 2, 128, 128), (3, 1100, 1, 1, 64, 64), (1, 2050, 2, 1, 128, 128),
    # enough heads for 128 columns a workgroup: whole sequences, segments in a chain, odd widths
    (75, 70, 4, 2, 128, 128), (75, 70, 4, 2, 64, 128), (75, 40, 4, 1, 60, 136), (4, 2050, 16, 4, 128, 128), (5, 1030, 6, 2, 64, 128),
]


@pytest.mark.parametrize("B,L,H,G,K,V", CASES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("state", [False, True])
def test_matches_recurrence(B, L, H, G, K, V, dtype, state):
    print(f"[case] linear_attention B={B} L={L} H={H} G={G} K={K} V={V} {dtype} state {state}", flush=True)
    from ssmjs_amd import kernels
    q, k, v, g, h0 = make(B, L, H, G, K, V, dtype, L + K, fast=state)
    scale = K ** -0.5
    hT = torch.full((B, H, V, K), float("nan"), device="cuda")
    y = kernels.linear_attention(q, k, v, g, scale=scale, h0=h0 if state else None, hT=hT)
    torch.cuda.synchronize()
    ref = recurrence(q, k, v, g, scale, None, h0 if state else None)
    by, bh = bounds(ref, K, L, dtype)
    close(y, ref[0], by, "y")
    close(hT, ref[1], bh, "state")


@pytest.mark.parametrize("K,V,G,H", [(128, 128, 1, 2), (64, 64, 2, 2), (40, 72, 1, 2), (33, 17, 2, 2), (128, 128, 7, 14)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_lengths(K, V, G, H, dtype):
    """Padded batches: what lies behind a sequence is neither used (NaN there) nor written."""
    print(f"[case] linear_attention lengths K={K} V={V} H={H} {dtype}", flush=True)
    from ssmjs_amd import kernels
    n = [0, 1, 63, 64, 65, 255, 256, 257, 600, 2000]
    B, L = len(n), 600
    q, k, v, g, h0 = make(B, L, H, G, K, V, dtype, 3)
    lengths = torch.tensor(n, dtype=torch.int32, device="cuda")
    n = [min(m, L) for m in n]   # held to 0 .. L
    for b, m in enumerate(n):
        for t in (q, k, v):
            t[b, m:] = float("nan")
    y = torch.full((B, L, H, V), 7.0, device="cuda", dtype=dtype)
    state = h0.clone()
    kernels.linear_attention(q, k, v, g, lengths=lengths, h0=state, hT=state, out=y)   # in place
    torch.cuda.synchronize()
    for b, m in enumerate(n):
        assert (y[b, m:] == 7.0).all(), m
    q, k, v = (torch.nan_to_num(t) for t in (q, k, v))
    ref = recurrence(q, k, v, g, 1.0, torch.tensor(n), h0)
    by, bh = bounds(ref, K, L, dtype)
    for b, m in enumerate(n):
        close(y[b, :m], ref[0][b, :m], by[b, :m], f"y of {m}")
    close(state, ref[1], bh, "state")
    assert torch.equal(state[0], h0[0])   # an empty sequence keeps its state
    y0 = kernels.linear_attention(q[:, :0], k[:, :0], v[:, :0], g, h0=h0, hT=state)
    torch.cuda.synchronize()
    assert y0.shape == (B, 0, H, V) and torch.equal(state, h0)
    kernels.linear_attention(q[:, :0], k[:, :0], v[:, :0], g, hT=state)
    torch.cuda.synchronize()
    assert not state.any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_extreme_decays(dtype):
    """No decay, a decay too slow for fp32's e^g, one that ends within a token, and none kept."""
    print(f"[case] linear_attention decays {dtype}", flush=True)
    from ssmjs_amd import kernels
    B, L, K, V = 1, 1500, 64, 64
    q, k, v, _, h0 = make(B, L, 4, 4, K, V, dtype, 9)
    g = torch.tensor([0.0, -1e-6, -90.0, -float("inf")], device="cuda")
    hT = torch.empty_like(h0)
    y = kernels.linear_attention(q, k, v, g, h0=h0, hT=hT)
    hs, ys = h0.clone(), []
    for t in range(L):
        ys.append(kernels.linear_attention_step(q[:, t], k[:, t], v[:, t], g, hs))
    torch.cuda.synchronize()
    ref = recurrence(q, k, v, g, 1.0, None, h0)
    by, bh = bounds(ref, K, L, dtype)
    close(y, ref[0], by, "y")
    close(hT, ref[1], bh, "state")
    # the recurrent form: two roundings a step, and the sum over K
    units = 2.0 ** -24 * (K + 2 * L)
    rb = units * ref[2] + (2.0 ** -8 * ref[0].abs() if dtype == torch.bfloat16 else 0)
    close(torch.stack(ys, 1), ref[0], rb, "y, recurrent")
    close(hs, ref[1], units * ref[3], "state, recurrent")
    assert torch.equal(hs[:, 3], (v[:, -1, 3].float()[..., None] * k[:, -1, 3].float()[:, None]))


@pytest.mark.parametrize("where", ["q", "k", "v"])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B", [1, 150])   # (64 columns a workgroup, and 128)
def test_odd_values_are_causal(where, value, dtype, B):
    """An inf or NaN at token 150 of one head changes no earlier token, and no other head."""
    print(f"[case] linear_attention {value} in {where} {dtype}", flush=True)
    from ssmjs_amd import kernels
    q, k, v, g, _ = make(B, 300, 2, 2, 128, 128, dtype, 4)
    clean = kernels.linear_attention(q, k, v, g)
    {"q": q, "k": k, "v": v}[where][0, 150, 1, 70] = value
    y = kernels.linear_attention(q, k, v, g)
    torch.cuda.synchronize()
    assert torch.equal(y[:, :150], clean[:, :150]) if where != "v" else True
    ok = torch.isfinite(y)
    assert ok[:, :150].all() and ok[:, :, 0].all()
    assert torch.equal(y[:, :, 0], clean[:, :, 0])
    if where == "q":
        assert not ok[0, 150, 1].any() and torch.equal(y[:, 151:], clean[:, 151:])
    elif where == "k":
        assert not ok[0, 150:, 1].any()
    else:   # one column of v
        assert not ok[0, 150:, 1, 70].any()
        near = (y[:, :150, 1, 70].double() - clean[:, :150, 1, 70].double()).abs().max()
        assert near <= 2.0 ** -6 * clean[:, :150, 1, 70].abs().max()
        assert ok[0, 150:, 1, :70].all() and ok[0, 150:, 1, 71:].all()


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_views(dtype, shift):
    """q, k, v as parts of one projection's rows (aligned, and not), outputs into wider rows."""
    print(f"[case] linear_attention views {dtype} shift {shift}", flush=True)
    from ssmjs_amd import kernels
    B, L, H, G, K, V = 2, 150, 4, 2, 64, 32
    W = H * K + G * K + G * V + 8 * (1 - shift) + shift
    gen = torch.Generator(device="cuda").manual_seed(2)
    flat = torch.randn(B * L * W + shift, generator=gen, device="cuda").to(dtype)
    rows = flat[shift:].view(B, L, W)
    q = rows[..., :H * K].unflatten(-1, (H, K))
    k = rows[..., H * K:(H + G) * K].unflatten(-1, (G, K))
    v = rows[..., (H + G) * K:(H + G) * K + G * V].unflatten(-1, (G, V))
    g = -torch.rand(H, generator=gen, device="cuda")
    wide = torch.full((B, L, H * V + 24), 3.0, device="cuda", dtype=dtype)
    out = wide[..., 8:8 + H * V].unflatten(-1, (H, V))
    kernels.linear_attention(q, k, v, g, out=out)
    ref = recurrence(q, k, v, g, 1.0, None, None)
    torch.cuda.synchronize()
    close(out, ref[0], bounds(ref, K, L, dtype)[0], "y")
    assert (wide[..., :8] == 3).all() and (wide[..., 8 + H * V:] == 3).all()


STEPS = [(1, 1, 1, 1, 1), (1, 12, 12, 128, 128), (3, 4, 2, 64, 64), (2, 2, 1, 96, 40), (1, 3, 1, 33, 17),
         (2, 2, 2, 256, 256), (1, 2, 1, 250, 70), (64, 16, 4, 128, 128), (5, 2, 1, 32, 300)]


@pytest.mark.parametrize("B,H,G,K,V", STEPS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_step(B, H, G, K, V, dtype):
    print(f"[case] linear_attention_step B={B} H={H} G={G} K={K} V={V} {dtype}", flush=True)
    from ssmjs_amd import kernels
    q, k, v, g, h = make(B, 1, H, G, K, V, dtype, K + V)
    ref = recurrence(q, k, v, g, 0.5, None, h)
    out = torch.empty(B, H, V + 3, device="cuda", dtype=dtype).view(B, -1)[:, :H * V].unflatten(1, (H, V))
    y = kernels.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, h, scale=0.5, out=out)
    torch.cuda.synchronize()
    units = 2.0 ** -24 * (K + 4)
    b = units * ref[2][:, 0] + (2.0 ** -8 * ref[0][:, 0].abs() if dtype == torch.bfloat16 else 0)
    close(y, ref[0][:, 0], b, "y")
    close(h, ref[1], units * ref[3], "state")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_nan_decay_shows(dtype):
    """A NaN decay makes its own head's results NaN and no other's."""
    print(f"[case] NaN decay {dtype}", flush=True)
    from ssmjs_amd import kernels
    q, k, v, g, h0 = make(2, 70, 3, 1, 64, 64, dtype, 5)
    g[1] = float("nan")
    hT = torch.empty_like(h0)
    y = kernels.linear_attention(q, k, v, g, h0=h0, hT=hT)
    h = h0.clone()
    y1 = kernels.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, h)
    torch.cuda.synchronize()
    for t, heads in ((y, 2), (y1, 1)):
        assert t.select(heads, 1).isnan().all()
        assert torch.isfinite(t.index_select(heads, torch.tensor([0, 2], device="cuda"))).all()
    for s in (hT, h):
        assert s[:, 1].isnan().all() and torch.isfinite(s[:, [0, 2]]).all()


@pytest.mark.parametrize("L,g", [(1, -12.0), (2, -9.0), (5, -1.0), (40, -0.6), (600, -0.05), (2000, -0.02), (700, -1e-6)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_what_a_decay_leaves(L, g, dtype):
    """With no values the state is e^{g L} h0, to within the roundings of each chunk's and segment's decay
    (its exponent's, relative to it, and four of 2^-24: the function's two, a sum, a product)."""
    print(f"[case] linear_attention decay of a state L={L} g={g} {dtype}", flush=True)
    from ssmjs_amd import kernels
    q, k, v, _, h0 = make(1, L, 2, 1, 64, 64, dtype, 1)
    v = torch.zeros_like(v)
    gs = torch.full((2,), g, device="cuda")
    hT = torch.empty_like(h0)
    kernels.linear_attention(q, k, v, gs, h0=h0, hT=hT)
    h = h0.clone()
    kernels.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], gs, h)
    torch.cuda.synchronize()
    g = gs.double()[0]
    for got, n in ((hT, L), (h, 1)):
        ref = h0.double() * torch.exp(g * n)
        units = float(g.abs()) * n + 4 * (-(-n // 32) + 32)   # (at most 32 segments)
        close(got, ref, units * 2.0 ** -24 * ref.abs(), f"state after {n}")
