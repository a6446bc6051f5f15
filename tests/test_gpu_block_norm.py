"""block_norm and its gradients against the formulas in 64 bits.

Bounds, with u = 2^-24. A sum over a row is at most 32 terms one after another in a lane, 6 exchanges and 16 waves: 56 u
of the sum of its terms' magnitudes; 1 / sqrt(mean + eps) of squares is within half of that and the instruction's 2 u: 32 u
in all with its products. silu(z) is within (|z| + 8) u. So v is within (|z| + 44) u of its value, and x' within e1 of
its own; what e1 does to the norm of x' is at most |e1| / |x'| over the row (Cauchy). The gradients' bounds follow
their formulas term by term; a column sum adds up to T / 512 + 64 rounded terms in a chain. A bfloat16 output adds half a
step, 2^-8 of its value."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def reference(x, y, z, post, scale, pre, eps, dx1=None, dn=None):
    """{name: (value, bound)} in 64 bits."""
    D = x.shape[-1]
    x, y = x.double(), y.double()
    one = torch.ones(D, dtype=torch.float64, device=x.device)
    post, scale, pre = (w.double() if w is not None else one for w in (post, scale, pre))
    mean = lambda t: t.mean(-1, keepdim=True)   # noqa: E731
    ry = (mean(y * y) + eps).rsqrt()
    w = y * ry
    u = w * post
    if z is not None:
        z = z.double()
        s = torch.sigmoid(z)
        sl, az = z * s, z.abs()
    else:
        s = q = torch.ones_like(x)
        sl, az = torch.ones_like(x), torch.zeros_like(x)
    v = u * sl
    x1 = x + scale * v
    e1 = (az + 46) * U * (scale * v).abs() + U * x1.abs()
    rx = (mean(x1 * x1) + eps).rsqrt()
    rho = 32 * U + e1.norm(dim=-1, keepdim=True) * rx * D ** -0.5
    nh = x1 * rx
    enh = rx * e1 + nh.abs() * (rho + U)
    out = {"x1": (x1, e1), "n": (nh * pre, pre.abs() * (enh + U * nh.abs()))}
    if dn is None:
        return out
    dn = dn.double()
    d = dn * pre
    g0 = dx1.double() if dx1 is not None else torch.zeros_like(x)
    m1 = mean(d * nh)
    em1 = mean(d.abs() * enh) + 62 * U * mean((d * nh).abs())
    inner = d - nh * m1
    g = g0 + rx * inner
    einner = U * d.abs() + enh * m1.abs() + nh.abs() * (em1 + 2 * U * m1.abs()) + U * inner.abs()
    eg = rx * (einner + (d.abs() + (nh * m1).abs()) * (rho + 2 * U)) + U * g.abs()
    t = g * scale
    c = t * sl * post
    ec = (scale * sl * post).abs() * eg + c.abs() * (az + 12) * U
    m2 = mean(c * w)
    em2 = mean(ec * w.abs()) + 98 * U * mean((c * w).abs())
    dy = ry * (c - w * m2)
    edy = ry * (ec + w.abs() * em2 + (c.abs() + (w * m2).abs()) * 72 * U) + U * dy.abs()
    T = x.numel() // D
    rows = lambda val, err: (val.reshape(-1, D).sum(0),   # noqa: E731
                             (err + (T / 512 + 64) * U * val.abs()).reshape(-1, D).sum(0))
    out["dx"], out["dy"] = (g, eg), (dy, edy)
    out["dscale"] = rows(g * v, eg * v.abs() + (g * v).abs() * (az + 46) * U)
    out["dpre"] = rows(dn * nh, dn.abs() * enh + U * (dn * nh).abs())
    out["dpost"] = rows(t * sl * w, (scale * sl * w).abs() * eg + (t * sl * w).abs() * (az + 46) * U)
    if z is not None:
        q = 1 + z * (1 - s)
        out["dz"] = (t * u * s * q, scale.abs() * (eg * (u * s * q).abs() + (g * u * s).abs()
                                                   * (q.abs() * (az + 50) + az * (az + 8)) * U))
    return out


def close(got, ref, what):
    value, bound = ref
    bound = bound + (2.0 ** -8 * value.abs() if got.dtype == torch.bfloat16 else 0) + 1e-37
    worst = float(((got.double() - value).abs() / bound).max())
    print(f"  {what}: worst |err| / bound {worst:.3f}", flush=True)
    assert torch.isfinite(got).all() and worst <= 1, what


def inputs(shape, dtype, seed, strided):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    f = lambda *s: torch.randn(*s, generator=gen, device="cuda")   # noqa: E731
    D = shape[-1]
    if strided:
        wide = f(*shape[:-1], 5 * D + 3).to(dtype)
        x, y, z, dx1, dn = (wide[..., k * D:(k + 1) * D] for k in range(5))
    else:
        x, y, z, dx1, dn = (f(*shape).to(dtype) for _ in range(5))
    return x, y, z, dx1, dn, 1 + 0.3 * f(D), f(D), 1 + 0.3 * f(D)


CASES = [((1, 1), False), ((3, 5), True), ((2, 3, 64), True), ((7, 512), False), ((9, 513), False), ((5, 768), True),
         ((33, 1000), False), ((1, 1024), False), ((6, 1027), True), ((4, 2048), True), ((5, 2049), False),
         ((3, 4096), False), ((3, 4100), True), ((2, 8193), False), ((2, 16384), False), ((2500, 66), False),
         ((1300, 1100), False), ((300, 8200), True), ((520, 16384), False)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,strided", CASES)
def test_forward_backward(shape, strided, dtype):
    from ssmjs_amd import kernels as k
    print(f"[case] block norm {shape} {strided} {dtype}", flush=True)
    x, y, z, dx1, dn, post, scale, pre = inputs(shape, dtype, 1, strided)
    for gate, given in ((True, True), (False, True), (True, False)):
        zz = z if gate else None
        ws = (post, scale, pre) if given else (None, None, None)
        dd = dx1 if given else None
        ref = reference(x, y, zz, *ws, 1e-6, dd, dn)
        x1, n = k.block_norm(x, y, zz, *ws)
        got = dict(zip(("dx", "dy", "dz", "dpost", "dscale", "dpre"), k.block_norm_backward(dd, dn, x, y, zz, *ws)))
        torch.cuda.synchronize()
        got |= {"x1": x1, "n": n}
        for name, t in got.items():
            if t is None:
                assert (name == "dz" and not gate) or (name in ("dpost", "dscale", "dpre") and not given)
            else:
                close(t, ref[name], f"{name} gate {gate} weights {given}")


def test_formulas_against_differentiation():
    """This file's 64-bit gradients against torch's own differentiation and against differences."""
    x, y, z, dx1, dn, post, scale, pre = (t.double() for t in inputs((4, 6), torch.float32, 2, False))

    def loss(x, y, z, post, scale, pre):
        r = reference(x, y, z, post, scale, pre, 1e-6)
        return (r["x1"][0] * dx1).sum() + (r["n"][0] * dn).sum()

    at = [t.clone().requires_grad_() for t in (x, y, z, post, scale, pre)]
    auto = torch.autograd.grad(loss(*at), at)
    ref = reference(x, y, z, post, scale, pre, 1e-6, dx1, dn)
    mine = [ref[k][0] for k in ("dx", "dy", "dz", "dpost", "dscale", "dpre")]
    at = [t.detach() for t in at]
    for j, (a, m) in enumerate(zip(auto, mine)):
        assert float((a - m).abs().max()) <= 1e-12 * float(a.abs().max() + 1)
        d = torch.randn_like(at[j])
        up, down = ([t + s * 1e-6 * d if i == j else t for i, t in enumerate(at)] for s in (1, -1))
        slope = float(loss(*up) - loss(*down)) / 2e-6
        assert abs(slope - float((m * d).sum())) <= 1e-7 * (1 + abs(slope))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [70, 1500, 5000])
def test_in_place(D, dtype):
    """x' in x's place, n in y's, and dx in dx1's give the bits of separate outputs."""
    from ssmjs_amd import kernels as k
    x, y, z, dx1, dn, post, scale, pre = inputs((11, D), dtype, 3, False)
    x1, n = k.block_norm(x, y, z, post, scale, pre)
    grads = k.block_norm_backward(dx1, dn, x, y, z, post, scale, pre)
    a, b, g = x.clone(), y.clone(), dx1.clone()
    k.block_norm(a, b, z, post, scale, pre, out=(a, b))
    dy, dz = torch.empty_like(x), torch.empty_like(x)
    again = k.block_norm_backward(g, dn, x, y, z, post, scale, pre, out=(g, dy, dz))
    torch.cuda.synchronize()
    assert torch.equal(a, x1) and torch.equal(b, n)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))


def test_rows_of_zeros_and_bad_rows():
    """A row of zeros gives zeros (eps holds the root); an inf or NaN stays in its row."""
    from ssmjs_amd import kernels as k
    x, y, z, dx1, dn, post, scale, pre = inputs((9, 200), torch.float32, 4, False)
    x[2], y[2] = 0, 0
    clean = k.block_norm(x, y, z, post, scale, pre)
    grads = k.block_norm_backward(dx1, dn, x, y, z, post, scale, pre)
    torch.cuda.synchronize()
    assert bool((clean[0][2] == 0).all()) and bool((clean[1][2] == 0).all())
    assert all(bool(torch.isfinite(t).all()) for t in grads)
    y[5, 3], x[6, 1] = float("nan"), float("inf")
    dirty = k.block_norm(x, y, z, post, scale, pre)
    dgrads = k.block_norm_backward(dx1, dn, x, y, z, post, scale, pre)
    torch.cuda.synchronize()
    keep = [r for r in range(9) if r not in (5, 6)]
    for a, b in zip([*clean, *grads[:3]], [*dirty, *dgrads[:3]]):
        assert torch.equal(a[keep], b[keep])
    assert bool(dirty[1][5].isnan().all())


def test_captured():
    """A captured pass forwards and back gives the eager bits, replay after replay."""
    from ssmjs_amd import kernels as k
    x, y, z, dx1, dn, post, scale, pre = inputs((700, 768), torch.bfloat16, 5, False)

    def whole():
        return [*k.block_norm(x, y, z, post, scale, pre), *k.block_norm_backward(dx1, dn, x, y, z, post, scale, pre)]

    x0, want = x.clone(), []
    for s in (1, 2):
        x.copy_(x0 * s)
        want.append(whole())
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = whole()
    for s in (0, 1, 0):
        x.copy_(x0 * (s + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[s]))
        whole()
