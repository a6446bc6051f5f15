"""token_logprobs and its gradient against the definitions in 64 bits.

Bounds, with u = 2^-24 and d = x - max, l = log Z. A term e^d of Z is within (4 |d| + 3) u of its value (the difference,
its product with log2 e, the instruction, and the same for the maxima that it was first held against), a chain of
c = ceil(N / 256) + 16 terms a lane and 80 joins adds (1.5 c + 80) u: ez = sum p (4 |d| + 3) u + (1.5 c + 80) u of Z, and as much in l. log p of
one token is then within ez + (|d| + 4 l + |log p| + 4) u, the entropy within that of l and of S / Z, whose terms p |d|
are within (4 |d| + 6) u + (1.5 c + 80) u each. A bfloat16 gradient adds half a step, 2^-8 of its value."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def reference(x, ids, k):
    """Values and bounds in 64 bits: logp, entropy, the order of the likeliest, their log p."""
    M, N = x.shape
    x = x.double()
    m = x.max(1, keepdim=True).values
    none = m == float("-inf")
    d = torch.where(none, 0.0, x - m.clamp(min=-1e300))
    d = torch.where(x == float("-inf"), float("-inf"), d)
    e = torch.exp(d)
    Z = e.sum(1, keepdim=True)
    l = torch.log(Z)   # noqa: E741
    p = torch.where(none, 0.0, e / Z)
    dd = torch.where(e > 0, d, 0.0)
    c = -(-N // 256) + 16
    chain = (1.5 * c + 80) * U
    ez = (p * (4 * dd.abs() + 3)).sum(1, keepdim=True) * U + chain
    lp = torch.where(none, float("-inf"), d - l)
    S = (p * dd).sum(1, keepdim=True)
    H = torch.where(none, 0.0, l - S)[:, 0]
    eH = (ez + (p * dd.abs() * (4 * dd.abs() + 6)).sum(1, keepdim=True) * U + S.abs() * (chain + ez)
          + (4 * l.abs() + 2 * S.abs()) * U)[:, 0]

    def bound(at):
        q, w = lp.gather(1, at), torch.where(d.gather(1, at) > -1e30, d.gather(1, at), 0.0)
        return torch.where(q > -1e30, ez + (w.abs() + 4 * l.abs() + q.abs() + 4) * U, 0.0)

    given = (ids >= 0) & (ids < N)
    at = ids.long().clamp(0, N - 1)[:, None]
    logp = torch.where(given, lp.gather(1, at)[:, 0], 0.0)
    top = torch.sort(x + 0.0, dim=1, descending=True, stable=True).indices[:, :k]
    return {"logp": (logp, torch.where(given, bound(at)[:, 0], 0.0)), "H": (H, eH), "top": top,
            "toplp": (lp.gather(1, top), bound(top)), "lp": lp, "p": p, "ez": ez, "l": l, "d": dd, "given": given,
            "none": none[:, 0]}


def close(got, ref, what):
    value, bound = ref
    same = (got.double() == value)
    off = torch.where(same, 0.0, (got.double() - value).abs())
    bound = bound + (2.0 ** -8 * value.abs() if got.dtype == torch.bfloat16 else 0) + 1e-37
    worst = float((off / bound).max())
    print(f"  {what}: worst |err| / bound {worst:.3f}", flush=True)
    assert not bool(got.isnan().any()) and worst <= 1, what


def check(x, ids, k, grad=True, out=None):
    from ssmjs_amd import kernels
    M, N = x.shape
    stats = torch.empty(M, 2, device="cuda")
    logp, ent, top, toplp = kernels.token_logprobs(x, ids, k=k, stats=stats)
    torch.cuda.synchronize()
    ref = reference(x, ids, max(k, 1))
    close(logp, ref["logp"], "logp")
    close(ent, ref["H"], "entropy")
    if k:
        assert torch.equal(top.long(), ref["top"]), "order"
        close(toplp, ref["toplp"], "top logp")
    if not grad:
        return logp, ent, top, toplp
    gen = torch.Generator(device="cuda").manual_seed(1)
    w, v = torch.randn(M, generator=gen, device="cuda"), torch.randn(M, generator=gen, device="cuda")
    lp, p, H, eH = ref["lp"], ref["p"], ref["H"][0], ref["H"][1]
    at = ids.long().clamp(0, N - 1)[:, None]
    some = p > 0
    llp = torch.where(some, lp, 0.0)
    ep = p * ((4 * llp.abs() + 4 * ref["l"].abs() + 8) * U + ref["ez"])
    for use in ((True, True), (True, False), (False, True)):
        ww = torch.where(ref["given"] & ~ref["none"], w.double(), 0.0) * use[0]
        vv = v.double()[:, None] * use[1]
        term = ww[:, None] + vv * (llp + H[:, None])
        eterm = vv.abs() * (ref["ez"] + eH[:, None] + (2 * llp.abs() + 4 * ref["l"].abs() + 2 * H[:, None].abs() + 4) * U) \
            + U * (ww.abs()[:, None] + term.abs())
        value, bound = -p * term, ep * term.abs() + p * eterm + 2 * U * (p * term).abs()
        value.scatter_add_(1, at, ww[:, None])
        bound.scatter_add_(1, at, U * ww.abs()[:, None])
        # (a row of nothing but -inf: exactly zeros)
        value, bound = (torch.where(ref["none"][:, None], 0.0, t) for t in (value, bound))
        got = kernels.token_logprobs_backward(x, ids, stats, ent, w if use[0] else None, v if use[1] else None)
        torch.cuda.synchronize()
        close(got, (value, bound), f"gradient {use}")
    return logp, ent, top, toplp


def logits(M, N, dtype, seed, strided=False):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = 3 * torch.randn(M, N + (5 if strided else 0), generator=gen, device="cuda")
    ids = torch.randint(0, N, (M,), generator=gen, device="cuda").to(torch.int32)
    ids[M // 2] = -100
    return x.to(dtype)[:, :N], ids


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,N,k,strided", [
    (1, 1, 1, False), (2, 3, 3, False), (3, 7, 0, True), (5, 63, 20, False), (4, 64, 64, True), (3, 100, 64, False),
    (7, 2047, 5, False), (2, 2048, 64, True), (3, 2049, 20, False), (9, 8191, 1, True), (2, 8193, 50, False),
    (3, 20001, 20, True), (1, 128000, 64, False), (300, 5003, 7, False), (2000, 9001, 3, False), (1100, 33, 4, True),
])
def test_against_the_definition(M, N, k, strided, dtype):
    print(f"[case] token logprobs {M} {N} {k} {strided} {dtype}", flush=True)
    check(*logits(M, N, dtype, 5, strided), k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N", [40, 3000, 30000])
def test_masks(N, dtype):
    """Rows whose mask leaves little or nothing, masks of the type's lowest value, equal and ordered logits."""
    print(f"[case] token logprobs, masks {N} {dtype}", flush=True)
    x, ids = logits(12, N, dtype, 8)
    lowest = torch.finfo(dtype).min
    x[0] = float("-inf")
    x[1] = float("-inf")
    x[1, N // 3] = 2.0
    ids[1] = N // 3
    x[2] = lowest
    x[3, ::2] = lowest
    x[4] = 1.5
    x[5] = torch.linspace(-9, 9, N, device="cuda").to(dtype)
    x[6] = torch.linspace(9, -9, N, device="cuda").to(dtype)
    x[7, 1:] = float("-inf")
    ids[7] = N - 1          # a token that cannot be
    x[8] = torch.where(torch.arange(N, device="cuda") % 2 == 0, 0.0, -0.0).to(dtype)
    x[9, 5:] = float("-inf")
    x[10, 3] = 3e38
    ids[10] = 3
    ids[11] = N             # past the end
    logp, ent, top, toplp = check(x, ids, 20)
    assert float(logp[0]) == float("-inf") and float(ent[0]) == 0 and bool((toplp[0] == float("-inf")).all())
    assert top[0].tolist() == list(range(20)) and top[8].tolist() == list(range(20))
    assert float(logp[1]) == 0 and float(logp[7]) == float("-inf") and float(logp[11]) == 0
    assert top[9].tolist()[5:] == list(range(5, 20))


def test_bad_rows():
    """NaN and +inf make their row's probabilities NaN and no other's; NaN comes last in the order."""
    from ssmjs_amd import kernels
    x, ids = logits(6, 30000, torch.float32, 9)
    ids[:] = 17
    clean = kernels.token_logprobs(x, ids, k=8)
    x[1, 20000], x[4, 3] = float("nan"), float("inf")
    stats = torch.empty(6, 2, device="cuda")
    got = kernels.token_logprobs(x, ids, k=8, stats=stats)
    dx = kernels.token_logprobs_backward(x, ids, stats, got[1], torch.ones(6, device="cuda"))
    torch.cuda.synchronize()
    for r in range(6):
        for a, b in zip(clean, got):
            if r in (1, 4):
                assert not a.dtype.is_floating_point or bool(b[r].isnan().all())
            else:
                assert torch.equal(a[r], b[r])
        assert bool(dx[r].isnan().any()) == (r in (1, 4))
    order = torch.sort(torch.where(x[1].isnan(), float("-inf"), x[1]), descending=True, stable=True).indices[:8]
    assert torch.equal(got[2][1].long(), order) and int(got[2][4, 0]) == 3
    x = torch.full((1, 70), float("nan"), device="cuda")
    x[0, 60:] = torch.arange(10.0, device="cuda")
    top = kernels.token_logprobs(x, k=12)[2]
    torch.cuda.synchronize()
    assert top[0].tolist() == [69, 68, 67, 66, 65, 64, 63, 62, 61, 60, 0, 1]


def test_gradient_against_differences():
    """The 64-bit gradient formula of this file against torch's own differentiation and against differences."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(4, 9, generator=gen, device="cuda").double()
    ids, w, v = torch.tensor([1, 8, 0, 3], device="cuda"), x[:, 0] + 1, x[:, 1] - 0.3

    def loss(x):
        lp = x - torch.logsumexp(x, 1, keepdim=True)
        return (lp.gather(1, ids[:, None])[:, 0] * w).sum() - ((lp.exp() * lp).sum(1) * v).sum()

    a = x.clone().requires_grad_()
    auto, = torch.autograd.grad(loss(a), a)
    r = reference(x, ids, 1)
    mine = -r["p"] * (w[:, None] + v[:, None] * (r["lp"] + r["H"][0][:, None]))
    mine.scatter_add_(1, ids[:, None], w[:, None])
    assert float((auto - mine).abs().max()) <= 1e-12
    d = torch.randn(4, 9, generator=gen, device="cuda").double()
    slope = float(loss(x + 1e-6 * d) - loss(x - 1e-6 * d)) / 2e-6
    assert abs(slope - float((mine * d).sum())) <= 1e-7 * (1 + abs(slope))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradient_in_place_and_captured(dtype):
    """The gradient in the logits' own place, and captured passes, give the eager bits, replay after replay."""
    from ssmjs_amd import kernels
    x0, ids = logits(37, 12345, dtype, 4)
    w = torch.randn(37, device="cuda")
    x, stats = x0.clone(), torch.empty(37, 2, device="cuda")

    def whole(out=None):
        got = kernels.token_logprobs(x, ids, k=6, stats=stats)
        return [*got, kernels.token_logprobs_backward(x, ids, stats, got[1], w, w, out=out)]

    want = whole()
    torch.cuda.synchronize()
    here = whole(x)
    torch.cuda.synchronize()
    assert here[4] is x and all(torch.equal(a, b) for a, b in zip(want, here))
    x.copy_(x0)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = whole()
    for _ in range(3):
        stats.zero_()
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, out))
        whole()
