"""How many bits linear attention keeps of its fp32 operands with bfloat16 inputs: sums that cancel, and
terms that stand alone, so that a dropped part of an operand is all that a result would hold.

Bounds: every operand of a product enters whole, so a result differs from the exact one by the roundings
that its few terms meet (counted at each test, 2^-24 of the terms' magnitudes each) and by the output's
own (2^-8 of it)."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def worst(got, ref, bound, what):
    assert torch.isfinite(got).all(), what
    w = float(((got.double() - ref).abs() / bound.clamp(min=1e-300)).max())
    print(f"  {what}: worst |err| / bound {w:.3f}", flush=True)
    assert w <= 1, what


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


@pytest.mark.parametrize("B,K,V", [(1, 64, 64), (1, 128, 128), (200, 128, 128), (2, 200, 72)])
def test_the_state_enters_its_product_whole(B, K, V):
    """Two columns of the state that differ by some 2^-17, and queries that subtract them. A term meets its
    three parts' and the pair's sums: at most eight roundings."""
    print(f"[case] state bits B={B} K={K} V={V}", flush=True)
    from ssmjs_amd import kernels
    H, L = 2, K // 2
    r = gen(K)
    h0 = normal(r, B, H, V, K)
    h0[..., 1::2] = h0[..., 0::2] * (1 + 2.0 ** -17 * normal(r, B, H, V, K // 2))
    q = torch.zeros(B, L, H, K, device="cuda")
    sign = torch.where(normal(r, B, L, H) < 0, -1.0, 1.0)
    t = torch.arange(L, device="cuda")
    q[:, t, :, 2 * t] = sign.transpose(0, 1)
    q[:, t, :, 2 * t + 1] = -sign.transpose(0, 1)
    q = q.bfloat16()
    k, v = normal(r, B, L, H, K).bfloat16(), torch.zeros(B, L, H, V, device="cuda").bfloat16()
    y = kernels.linear_attention(q, k, v, torch.zeros(H, device="cuda"), h0=h0)
    torch.cuda.synchronize()
    pair = h0.double().unflatten(-1, (K // 2, 2))                                  # (B,H,V,L,2)
    ref = ((pair[..., 0] - pair[..., 1]) * sign.double().permute(0, 2, 1)[:, :, None]).permute(0, 3, 1, 2)
    a = pair.abs().sum(-1).permute(0, 3, 1, 2)
    worst(y, ref, 2.0 ** -8 * ref.abs() + 8 * U * a, "y")


@pytest.mark.parametrize("B,K,V", [(8, 64, 64), (200, 128, 128), (4, 256, 40)])
def test_the_weights_enter_their_product_whole(B, K, V):
    """Pairs of tokens whose keys all but agree and whose values are opposite; a pair has three dimensions
    of its own. A weight meets two roundings in its sum and one each by the decay and the scale, a term six
    in the parts' sums: ten."""
    print(f"[case] weight bits B={B} K={K} V={V}", flush=True)
    from ssmjs_amd import kernels
    H, n = 2, min(K // 3, 30)
    L = 2 * n
    r = gen(K + 1)
    q = torch.zeros(B, L, H, K, device="cuda")
    k = torch.zeros(B, L, H, K, device="cuda")
    v = normal(r, B, L, H, V).bfloat16().float()
    for p in range(n):
        a, b, d = 2 * p, 2 * p + 1, 3 * p
        q[:, b, :, d] = 2.0 ** -10
        q[:, b, :, d + 1:d + 3] = normal(r, B, H, 2)
        k[:, a, :, d:d + 3] = 1 + torch.rand(B, H, 3, generator=r, device="cuda")
        k[:, b] = k[:, a]
        k[:, b, :, d] += 2.0 ** -6
        v[:, b] = -v[:, a]
    q, k, v = q.bfloat16(), k.bfloat16(), v.bfloat16()
    y = kernels.linear_attention(q, k, v, torch.zeros(H, device="cuda"))
    torch.cuda.synchronize()
    s = torch.tril(torch.ones(L, L, dtype=torch.float64, device="cuda"))
    qd, kd, vd = (x.double().permute(0, 2, 1, 3).contiguous() for x in (q, k, v))
    kt = kd.transpose(-1, -2).contiguous()
    ref = ((qd @ kt * s) @ vd).permute(0, 2, 1, 3)
    size = ((qd.abs() @ kt.abs() * s) @ vd.abs()).permute(0, 2, 1, 3)
    worst(y, ref, 2.0 ** -8 * ref.abs() + 10 * U * size, "y")


@pytest.mark.parametrize("L,g", [(128, -0.033), (700, -0.004), (192, -0.033), (64, -0.02), (1500, -0.0015)])
@pytest.mark.parametrize("V", [64, 128])
def test_the_decayed_values_enter_the_state_whole(L, g, V):
    """64 tokens with a key dimension each, and nothing behind them: each element of the state is one term,
    e^{g n} v k. Its roundings: three of the exponent of the weight, g d for d < 64 (the constant, g's
    product with it, d's), two of its exponential, one of the weighted value, three of its parts' sums; then
    for each chunk and segment that it passes, its decay's exponent, and four (the exponential's two, a sum,
    a product)."""
    print(f"[case] decayed values L={L} g={g} V={V}", flush=True)
    from ssmjs_amd import kernels
    H, K, n = 2, 64, 64
    r = gen(L)
    k = torch.zeros(1, L, H, K, device="cuda")
    t = torch.arange(n, device="cuda")
    k[:, t, :, t] = 1 + torch.rand(n, 1, H, generator=r, device="cuda")
    v = normal(r, 1, L, H, V)
    v[:, n:] = 0
    q, k, v = normal(r, 1, L, H, K).bfloat16(), k.bfloat16(), v.bfloat16()
    gs = torch.full((H,), g, device="cuda")
    hT = torch.empty(1, H, V, K, device="cuda")
    kernels.linear_attention(q, k, v, gs, hT=hT)
    torch.cuda.synchronize()
    g = float(gs.double()[0])
    far = L - 1 - t.double()
    ref = torch.exp(g * far) * v[0, :n].double().permute(1, 2, 0) * k[0, t, :, t].double().t()[:, None]
    passed = -(-L // 64) + (-(-L // 256) if L > 256 else 0)
    units = 3 * abs(g) * 63 + 6 + abs(g) * L + 4 * (passed - 1)
    worst(hT[0], ref, units * U * ref.abs(), "state")


@pytest.mark.parametrize("B,L", [(1, 130), (200, 70), (1, 3000)])
def test_the_largest_states(B, L):
    """States next to the largest fp32 number, which is above the largest that rounds into bfloat16: their
    products with small queries are numbers."""
    print(f"[case] largest states B={B} L={L}", flush=True)
    from ssmjs_amd import kernels
    H, K, V = 1, 64, 128
    r = gen(L)
    h0 = torch.zeros(B, H, V, K, device="cuda")
    h0[..., 5] = torch.finfo(torch.float32).max * (1 - 2.0 ** -12 * torch.rand(B, H, V, generator=r, device="cuda"))
    q = torch.zeros(B, L, H, K, device="cuda")
    q[..., 5] = 2.0 ** -20 * (1 + torch.rand(B, L, H, generator=r, device="cuda"))
    q, z = q.bfloat16(), torch.zeros(B, L, H, V, device="cuda").bfloat16()
    hT = torch.empty_like(h0)
    y = kernels.linear_attention(q, torch.zeros_like(q), z, torch.zeros(H, device="cuda"), h0=h0, hT=hT)
    torch.cuda.synchronize()
    ref = q[..., 5].double()[..., None] * h0[..., 5].double()[:, None]
    worst(y, ref, (2.0 ** -8 + 4 * U) * ref.abs(), "y")
    assert torch.equal(hT, h0)
