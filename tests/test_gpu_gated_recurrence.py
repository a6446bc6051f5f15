"""gated_recurrence, its gradients and its step against the recurrence in 64 bits, walked step by step.

Bounds, with u = 2^-24. An open gate sigmoid(v) from one exp2, one sum and one reciprocal is within (|v| + 6) u of
its value, z = c softplus(lam) sigmoid(r) within (|r| + 16) u, so a = e^-z within (8 + z (|r| + 24)) u =: ka (its
rounding, the product over a run, the sum of the series) and b within (|r| + |i| + 40) u =: kb. What that does to the
states is carried along with them: with m_t = a m_{t-1} + |b_t| the sum of the magnitudes of h's terms,
E_t = a E_{t-1} + ka a m_{t-1} + kb |b_t| + u m_t. The adjoint's bound is carried the same way, from the end.
A bfloat16 output adds half a step, 2^-8 of its value. The exp2 instruction gives 0 for results below 2^-126: that
much a is off at most, and a z h_{t-1} g so much times z |h_{t-1}| |g| (`gone`). 1e-37 is 8 * 2^-126.
In dr = g (u a^2 z / beta - a z h) (1 - sigmoid r), the factors u, a^2, z, 1 / beta and 1 - sigmoid r (e^-r times the
open gate) are within |i| + 6, 2 ka, |r| + 16, |r| / 2 + 15 and 2 |r| + 9 units: 4 |r| + |i| + 80 with their products,
and 2 z (|r| + 24) more for a^2."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def gates(x, r, i, lam, c):
    x, r, i, lam = (t.double() for t in (x, r, i, lam))
    z = c * torch.nn.functional.softplus(lam, threshold=1e4) / (1 + torch.exp(-r))
    gi = 1 / (1 + torch.exp(-i))
    a, beta = torch.exp(-z), (-torch.expm1(-2 * z)).sqrt()
    return {"x": x, "z": z, "a": a, "beta": beta, "gi": gi, "b": beta * gi * x, "R": r.abs(), "I": i.abs(),
            "cr": 1 / (1 + torch.exp(r)), "ci": 1 / (1 + torch.exp(i)),
            "ka": (8 + z * (r.abs() + 24)) * U, "kb": (r.abs() + i.abs() + 40) * U}


def walk(g, lengths, h0):
    """h_t, the sums of magnitudes and the bounds, (B, L + 1, D) with the entering state first."""
    B, L, D = g["a"].shape
    h = h0.double() if h0 is not None else torch.zeros(B, D, dtype=torch.float64, device=g["a"].device)
    m, e = h.abs(), torch.zeros_like(h)
    hs, ms, es = [h], [m], [e]
    for t in range(L):
        on = (t < lengths)[:, None]
        a, b = g["a"][:, t], g["b"][:, t]
        e1 = a * e + g["ka"][:, t] * a * m + g["kb"][:, t] * b.abs()
        h1, m1 = a * h + b, a * m + b.abs()
        e1 = e1 + U * m1
        h, m, e = torch.where(on, h1, h), torch.where(on, m1, m), torch.where(on, e1, e)
        hs.append(h), ms.append(m), es.append(e)
    return torch.stack(hs, 1), torch.stack(ms, 1), torch.stack(es, 1)


def adjoint(g, dy, lengths, dhT):
    """g_t of every step, its magnitudes and bounds, and those of dh0."""
    B, L, D = g["a"].shape
    e = dhT.double() if dhT is not None else torch.zeros(B, D, dtype=torch.float64, device=dy.device)
    m, err = e.abs(), torch.zeros_like(e)
    gs, ms, es = [], [], []
    for t in range(L - 1, -1, -1):
        on = (t < lengths)[:, None]
        a, d = g["a"][:, t], dy[:, t].double()
        gt, mt = d + e, d.abs() + m
        et = err + U * mt
        gs.append(torch.where(on, gt, 0.0)), ms.append(torch.where(on, mt, 0.0)), es.append(torch.where(on, et, 0.0))
        e, m = torch.where(on, a * gt, e), torch.where(on, a * mt, m)
        err = torch.where(on, a * et + g["ka"][:, t] * a * mt + U * a * mt, err)
    flip = lambda v: torch.stack(v[::-1], 1) if v else torch.zeros(B, 0, D, dtype=torch.float64, device=dy.device)  # noqa: E731
    return flip(gs), flip(ms), flip(es), e, err


def close(got, ref, bound, what):
    half = 2.0 ** -8 * ref.abs() if got.dtype == torch.bfloat16 else 0
    bound = bound + half + 1e-37
    worst = float(((got.double() - ref).abs() / bound).max()) if got.numel() else 0.0
    print(f"  {what}: worst |err| / bound {worst:.3f}", flush=True)
    assert torch.isfinite(got).all() and worst <= 1, what


def inputs(B, L, D, dtype, seed, strided=False, far=False):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    f = lambda *s: torch.randn(*s, generator=gen, device="cuda")   # noqa: E731
    if strided:
        rows = (2 * f(B, L, 3 * D + 4)).to(dtype)
        x, r, i = (rows[..., k * D:(k + 1) * D] for k in (0, 1, 2))
    else:
        x, r, i = (2 * f(B, L, D)).to(dtype), (2 * f(B, L, D)).to(dtype), (2 * f(B, L, D)).to(dtype)
    # decays next to 1 (c softplus(lam) from 1e-4 on), and, with `far`, down to e^-100
    lam = f(D) * 2 - 5 if not far else f(D) * 6
    return x, r, i, lam, f(B, D), gen


CASES = [   # B, L, D, ragged, state, strided, far
    (1, 1, 1, False, False, False, False), (2, 3, 5, False, True, False, False), (1, 17, 64, False, True, False, True),
    (3, 64, 66, True, True, False, False), (2, 65, 132, False, False, True, False), (1, 255, 68, False, True, True, True),
    (2, 256, 64, False, True, False, False), (2, 257, 100, True, False, False, False), (1, 1000, 37, False, True, False, False),
    (4, 130, 256, True, True, True, False), (1, 5000, 64, False, True, False, False), (5, 3000, 68, True, True, False, True),
    (2, 2100, 33, True, True, True, False),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", CASES)
def test_forward_backward(case, dtype):
    from ssmjs_amd import kernels as k
    B, L, D, ragged, state, strided, far = case
    print(f"[case] gated recurrence {case} {dtype}", flush=True)
    x, r, i, lam, h0, gen = inputs(B, L, D, dtype, 7, strided, far)
    h0 = h0 if state else None
    n = torch.full((B,), L, dtype=torch.int32, device="cuda")
    if ragged:
        n = torch.randint(0, L + 1, (B,), generator=gen, device="cuda").to(torch.int32)
        n[0], n[-1] = L, 0
        if B > 2:
            n[1] = 1
    lengths = n if ragged else None
    g = gates(x, r, i, lam, 8.0)
    hs, ms, es = walk(g, n, h0)
    states, hT = k.gated_recurrence_states(B, L, D, "cuda"), torch.empty(B, D, device="cuda")
    y = k.gated_recurrence(x, r, i, lam, lengths=lengths, h0=h0, hT=hT, states=states)
    torch.cuda.synchronize()
    inside = (torch.arange(L, device="cuda") < n[:, None])[..., None]
    close(torch.where(inside, y, 0.0), torch.where(inside, hs[:, 1:], 0.0), es[:, 1:], "y")
    assert bool((torch.where(inside, 0.0, y.float()) == 0).all())
    close(hT, hs[:, -1], es[:, -1], "hT")
    for s in range(0, L, 64):
        on = (s < n)[:, None]
        close(torch.where(on, states[:, s // 64], 0.0), torch.where(on, hs[:, s], 0.0), es[:, s], f"state {s}")
    # gradients
    dy = torch.randn(B, L, D, generator=gen, device="cuda").to(dtype)
    dhT = torch.randn(B, D, generator=gen, device="cuda") if state else None
    dh0 = torch.empty(B, D, device="cuda")
    dx, dr, di, dlam = k.gated_recurrence_backward(dy, x, r, i, lam, states, lengths=lengths, dhT=dhT, dh0=dh0)
    torch.cuda.synchronize()
    gt, mg, eg, e0, ee0 = adjoint(g, dy, n, dhT)
    k2 = (g["R"] + g["I"] + 60) * U
    bi, bu = g["beta"] * g["gi"], (g["b"] * g["ci"])
    close(dx, gt * bi, bi * (eg + mg * k2), "dx")
    close(di, gt * bu, bu.abs() * (eg + mg * k2), "di")
    p1 = g["gi"] * g["x"] * g["a"] ** 2 * g["z"] / g["beta"].clamp(min=1e-300)
    p2 = g["a"] * g["z"]
    hp, mp, ep = hs[:, :-1], ms[:, :-1], es[:, :-1]
    q = gt * (p1 - p2 * hp)
    k3 = (4 * g["R"] + g["I"] + 80 + 4 * g["z"] * (g["R"] + 24)) * U
    eq = eg * (p1.abs() + p2 * mp) + mg * (p1.abs() * k3 + p2 * (ep + k3 * mp))
    gone = 2.0 ** -126 * (1 + g["z"]) * (1 + mp) * mg      # (a below 2^-126)
    close(dr, q * g["cr"], g["cr"] * (eq + gone), "dr")
    f = torch.sigmoid(lam.double()) / torch.nn.functional.softplus(lam.double(), threshold=1e4)
    # a lane adds up to L / 8 + 16 values one after another
    sums = (eq + gone + (L / 8 + 48) * U * mg * (p1.abs() + p2 * mp)).sum((0, 1))
    close(dlam, f * q.sum((0, 1)), f * sums, "dlam")
    close(dh0, e0, ee0, "dh0")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_against_differences(dtype):
    """The 64-bit gradient formulas of this file against differences of the recurrence in 64 bits, and against
    torch's own differentiation."""
    x, r, i, lam, h0, gen = inputs(2, 9, 4, dtype, 3)
    n = torch.tensor([9, 5], device="cuda")
    dy, dhT = torch.randn(2, 9, 4, generator=gen, device="cuda"), torch.randn(2, 4, generator=gen, device="cuda")

    def loss(x, r, i, lam, h0):
        hs, _, _ = walk(gates(x, r, i, lam, 8.0), n, h0)
        on = (torch.arange(9, device="cuda") < n[:, None])[..., None]
        return (torch.where(on, hs[:, 1:], 0.0) * dy.double()).sum() + (hs[:, -1] * dhT.double()).sum()

    at = [t.double().requires_grad_() for t in (x, r, i, lam, h0)]
    auto = torch.autograd.grad(loss(*at), at)
    g = gates(x, r, i, lam, 8.0)
    hs, _, _ = walk(g, n, h0)
    gt, _, _, e0, _ = adjoint(g, dy, n, dhT)
    q = gt * (g["gi"] * g["x"] * g["a"] ** 2 * g["z"] / g["beta"] - g["a"] * g["z"] * hs[:, :-1])
    f = torch.sigmoid(lam.double()) / torch.nn.functional.softplus(lam.double(), threshold=1e4)
    mine = (gt * g["beta"] * g["gi"], q * g["cr"], gt * g["b"] * g["ci"], f * q.sum((0, 1)), e0)
    for a, m in zip(auto, mine):
        assert float((a - m).abs().max()) <= 1e-12 * float(a.abs().max() + 1)
    for j in range(5):
        d = torch.randn(at[j].shape, generator=gen, device="cuda").double()
        moved = [[t + s * 1e-6 * d if k == j else t for k, t in enumerate(at)] for s in (1, -1)]
        slope = (loss(*moved[0]) - loss(*moved[1])) / 2e-6
        assert abs(float(slope - (mine[j] * d).sum())) <= 1e-7 * (1 + abs(float(slope)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,D,strided", [(1, 1, False), (3, 5, True), (64, 256, True), (2, 4097, False), (7, 1024, False)])
def test_step(B, D, strided, dtype):
    from ssmjs_amd import kernels as k
    print(f"[case] gated recurrence step {B} {D} {dtype}", flush=True)
    x, r, i, lam, h, _ = inputs(B, 1, D, dtype, 11, strided, True)
    x, r, i = x[:, 0], r[:, 0], i[:, 0]
    g = gates(x[:, None], r[:, None], i[:, None], lam, 8.0)
    one = torch.ones(B, device="cuda")
    hs, ms, es = walk(g, one, h)
    y = k.gated_recurrence_step(x, r, i, lam, h)
    torch.cuda.synchronize()
    close(y, hs[:, 1], es[:, 1], "y")
    close(h, hs[:, 1], es[:, 1], "h")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pieces_and_steps_are_the_whole(dtype):
    """A prompt in two calls through a state in place, and its last tokens one by one."""
    from ssmjs_amd import kernels as k
    B, L, D = 2, 2700, 64
    print(f"[case] gated recurrence in pieces {dtype}", flush=True)
    x, r, i, lam, h0, _ = inputs(B, L, D, dtype, 5)
    n = torch.full((B,), L, device="cuda")
    hs, _, es = walk(gates(x, r, i, lam, 8.0), n, h0)
    h = h0.clone()
    cut = 2400
    y0 = k.gated_recurrence(*(t[:, :cut].contiguous() for t in (x, r, i)), lam, h0=h, hT=h)
    y1 = k.gated_recurrence(*(t[:, cut:L - 3].contiguous() for t in (x, r, i)), lam, h0=h, hT=h)
    ys = [k.gated_recurrence_step(x[:, t], r[:, t], i[:, t], lam, h) for t in range(L - 3, L)]
    torch.cuda.synchronize()
    close(torch.cat([y0, y1, torch.stack(ys, 1)], 1), hs[:, 1:], 2 * es[:, 1:], "y")
    close(h, hs[:, -1], 2 * es[:, -1], "h")


def test_rows_behind_a_sequence():
    """Rows of the caller's outputs behind a sequence's end are left as they were, whatever its inputs hold there."""
    from ssmjs_amd import kernels as k
    B, L, D = 3, 700, 68
    x, r, i, lam, h0, gen = inputs(B, L, D, torch.float32, 2)
    n = torch.tensor([700, 0, 333], dtype=torch.int32, device="cuda")
    beyond = (torch.arange(L, device="cuda") >= n[:, None])[..., None].expand(B, L, D)
    st = k.gated_recurrence_states(B, L, D, "cuda")
    clean = k.gated_recurrence(x, r, i, lam, lengths=n, h0=h0, states=st)
    dy = torch.randn(B, L, D, generator=gen, device="cuda")
    grads = k.gated_recurrence_backward(dy, x, r, i, lam, st, lengths=n)
    dirty = [torch.where(beyond, float("nan"), t) for t in (x, r, i, dy)]
    out = torch.full((B, L, D), 5.0, device="cuda")
    st2 = torch.full_like(st, 3.0)
    k.gated_recurrence(*dirty[:3], lam, lengths=n, h0=h0, states=st2, out=out)
    torch.cuda.synchronize()
    assert torch.equal(out, torch.where(beyond, 5.0, clean))
    for s in range(st.shape[1]):
        for b in range(B):
            want = st[b, s] if 64 * s < int(n[b]) else torch.full_like(st[b, s], 3.0)
            assert torch.equal(st2[b, s], want)
    outs = [torch.full((B, L, D), 5.0, device="cuda") for _ in range(3)]
    *_, dlam = k.gated_recurrence_backward(dirty[3], *dirty[:3], lam, st2, lengths=n, out=outs)
    torch.cuda.synchronize()
    for o, w in zip(outs, grads):
        assert torch.equal(o, torch.where(beyond, 5.0, w))
        assert bool((torch.where(beyond, w, 0.0) == 0).all())
    assert torch.equal(dlam, grads[3])


@pytest.mark.parametrize("L", [40, 3000])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_an_infinity_stays_where_it_is(bad, L):
    """No earlier token and no other channel meets an inf or NaN; an infinite state stays infinite through decays
    below fp32's range."""
    from ssmjs_amd import kernels as k
    B, D, at = 2, 68, L // 2
    for far in (False, True):
        x, r, i, lam, h0, _ = inputs(B, L, D, torch.float32, 4, False, far)
        clean = k.gated_recurrence(x, r, i, lam, h0=h0)
        x[1, at, 7] = bad
        hT = torch.empty(B, D, device="cuda")
        y = k.gated_recurrence(x, r, i, lam, h0=h0, hT=hT)
        torch.cuda.synchronize()
        hit = torch.zeros_like(y, dtype=torch.bool)
        hit[1, at:, 7] = True
        assert torch.equal(torch.where(hit, 0.0, y), torch.where(hit, 0.0, clean))
        tail = y[1, at:, 7]
        assert bool(tail.isnan().all()) if bad != bad else bool((tail == bad).all())
        x[1, at, 7] = 0.0
        h0[0, 3] = float("-inf")
        lam[3] = 40.0      # decays of e^-300 and less
        y = k.gated_recurrence(x, r, i, lam, h0=h0, hT=hT)
        torch.cuda.synchronize()
        assert bool((y[0, :, 3] == float("-inf")).all()) and float(hT[0, 3]) == float("-inf")
        h = h0.clone()
        k.gated_recurrence_step(x[:, 0], r[:, 0], i[:, 0], lam, h)
        torch.cuda.synchronize()
        assert float(h[0, 3]) == float("-inf")


def test_gates_shut_and_open():
    """Gates at their ends: a = 1 keeps the state and gives finite gradients, a = 0 drops it."""
    from ssmjs_amd import kernels as k
    B, L, D = 1, 70, 8
    x, r, i, lam, h0, gen = inputs(B, L, D, torch.float32, 6)
    r[..., 0], r[..., 1], r[..., 2] = -200.0, 200.0, float("-inf")
    i[..., 3], i[..., 4] = -200.0, 200.0
    lam[1], lam[5], lam[6] = 60.0, -200.0, -90.0
    n = torch.full((B,), L, device="cuda")
    st = k.gated_recurrence_states(B, L, D, "cuda")
    y = k.gated_recurrence(x, r, i, lam, h0=h0, states=st)
    dy = torch.randn(B, L, D, generator=gen, device="cuda")
    grads = k.gated_recurrence_backward(dy, x, r, i, lam, st)
    torch.cuda.synchronize()
    hs, _, es = walk(gates(x, r.clamp(-200, 200), i, lam, 8.0), n, h0)
    # (sqrt(2 z) of a shut gate: below 2^-63 of x)
    close(y, hs[:, 1:], es[:, 1:] + 2.0 ** -50, "y")
    assert torch.equal(y[0, :, 0], h0[0, 0].expand(L)) and torch.equal(y[0, :, 2], h0[0, 2].expand(L))
    assert all(bool(torch.isfinite(t).all()) for t in grads)


def test_captured_and_on_two_streams():
    """Captured calls and calls on two streams give the eager calls' bits, replay after replay."""
    from ssmjs_amd import kernels as k
    B, L, D = 1, 5000, 64
    x, r, i, lam, h0, gen = inputs(B, L, D, torch.bfloat16, 9)
    dy = torch.randn(B, L, D, generator=gen, device="cuda").to(torch.bfloat16)

    def whole(h0):
        st, hT, dh0 = k.gated_recurrence_states(B, L, D, "cuda"), torch.empty(B, D, device="cuda"), torch.empty(B, D, device="cuda")
        y = k.gated_recurrence(x, r, i, lam, h0=h0, hT=hT, states=st)
        return [y, hT, dh0, *k.gated_recurrence_backward(dy, x, r, i, lam, st, dh0=dh0)]

    want = [whole(h) for h in (h0, h0 + 1)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for s, h in zip(streams, (h0, h0 + 1)):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(whole(h))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for w, g in zip(want, got) for a, b in zip(w, g))
    h, graph = h0.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = whole(h)
    for k_ in (0, 1, 0, 1):
        h.copy_(h0 + k_)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[k_]))
        whole(h0)
