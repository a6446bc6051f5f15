"""Rows as 8-bit integers and their products. The integers are exact (the nearest to the exact
quotient, ties to even), and so are the sums; an output meets four roundings of 2^-24 (the sum, the
product of the scales, their product, the bias), one more with beta, and bfloat16's half step."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def integers(x):
    """(q, scale) in exact arithmetic: the quotient of two fp32 numbers is a tie or at least 2^-25 of
    its size away from one, which 64 bits tell apart."""
    x = x.double().cpu().numpy()
    s = (np.abs(x).max(1) / 127).astype(np.float32)
    with np.errstate(all="ignore"):
        q = np.clip(np.rint(x / s.astype(np.float64)[:, None]), -127, 127)
    q[~(np.isfinite(s) & (s > 0))] = 0
    return q.astype(np.int8), s


def data(M, K, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(M, K, generator=gen, device="cuda") * torch.exp(2 * torch.randn(M, 1, generator=gen, device="cuda"))
    return x.to(dtype)


@pytest.mark.parametrize("M,K", [(1, 1), (1, 2048), (3, 100), (7, 9000), (5, 1023), (1100, 768), (1030, 2048), (2, 131071)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_rows(M, K, dtype):
    print(f"[case] quantize_rows {M} x {K} {dtype}", flush=True)
    from ssmjs_amd import kernels
    x = data(M, K, dtype, K)
    if K >= 8:   # halves of the scale: 127 s is the largest
        x[0, :8] = torch.tensor([127.0, 0.5, 1.5, -2.5, -0.5, 126.5, 0.0, -126.5], device="cuda")
        x[0, 8:] = x[0, 8:].clamp(-100, 100)
    q, s = kernels.quantize_rows(x)
    wide = torch.full((M, K + 5), 99, dtype=torch.int8, device="cuda")
    q2, _ = kernels.quantize_rows(x, out=(wide[:, 3:3 + K], torch.empty_like(s)))
    torch.cuda.synchronize()
    rq, rs = integers(x)
    np.testing.assert_array_equal(s.cpu().numpy(), rs)
    np.testing.assert_array_equal(q.cpu().numpy(), rq)
    np.testing.assert_array_equal(q2.cpu().numpy(), rq)
    assert (wide[:, :3] == 99).all() and (wide[:, 3 + K:] == 99).all()


def test_quantize_odd_rows():
    """Zeros, the smallest and the largest numbers; rows with an inf or NaN make NaN products and
    touch no other row."""
    print("[case] quantize odd rows", flush=True)
    from ssmjs_amd import kernels
    torch.manual_seed(0)
    x = torch.randn(8, 64, device="cuda")
    x[1] = 0
    x[2] *= 1e-43
    x[3] = 1e-45
    x[4] = x[4].sign() * 3e38
    x[5, 9] = float("nan")
    x[6, 10] = -float("inf")
    q, s = kernels.quantize_rows(x)
    W = torch.randint(-127, 128, (32, 64), device="cuda", dtype=torch.int32).to(torch.int8)
    # (row 4: 3e38 / 127 times 64 * 127 * 127 at most is 2.5e42, so the products stay finite at 1e-4)
    sw = torch.rand(32, device="cuda") * 1e-4
    y = kernels.linear_q8(x, W, sw)
    torch.cuda.synchronize()
    rq, rs = integers(torch.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0))
    fine = [0, 1, 2, 3, 4, 7]
    np.testing.assert_array_equal(q.cpu().numpy()[fine], rq[fine])
    np.testing.assert_array_equal(s.cpu().numpy()[fine], rs[fine])
    assert not q[5:7].any() and s[5].isnan() and s[6].isinf()
    assert y[5:7].isnan().all() and torch.isfinite(y[fine]).all() and not y[1].any()


def product(q, s, W, sw, bias, beta, y0):
    """y in 64 bits, and the magnitudes that meet its roundings."""
    acc = q.cpu().double() @ W.cpu().double().t()
    p = acc * s.cpu().double()[:, None] * sw.cpu().double()
    y = p + (bias.cpu().double() if bias is not None else 0)
    size = 3 * p.abs() + y.abs()
    if beta:
        y = y + beta * y0.cpu().double()
        size = size + (beta * y0.cpu().double()).abs() + y.abs()
    return y, size


SHAPES = [   # M, N, K
    (1, 1, 1), (1, 8512, 2048), (2, 17, 64), (16, 100, 256), (17, 33, 300), (33, 4384, 1024), (64, 257, 512),
    (64, 96, 4096), (65, 100, 200), (100, 256, 1000), (127, 513, 768), (200, 130, 999), (300, 1028, 128),
    (1000, 600, 1536), (4200, 4100, 512), (3, 40, 131071), (70, 40, 131071), (9, 4112, 700), (20, 4100, 2600),
    (2, 4200, 5000),
]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_products(M, N, K, dtype):
    print(f"[case] linear_q8 {M} x {N} x {K} {dtype}", flush=True)
    from ssmjs_amd import kernels
    x = data(M, K, dtype, M + N)
    W, sw = kernels.quantize_rows(data(N, K, torch.float32, K) * K ** -0.5)
    bias = torch.randn(N, device="cuda") if N % 2 else None
    beta = 1.0 if M % 2 == 0 else 0.0
    y0 = torch.randn(M, N, device="cuda").to(dtype)
    y = kernels.linear_q8(x, W, sw, bias=bias, out=y0.clone() if beta else torch.full_like(y0, float("nan")),
                          beta=beta)
    q, s = kernels.quantize_rows(x)
    y2 = kernels.linear_i8(q, s, W, sw, bias=bias, out=y0.clone(), beta=beta)
    torch.cuda.synchronize()
    ref, size = product(q, s, W, sw, bias, beta, y0)
    bound = 2.0 ** -24 * size + (2.0 ** -8 * ref.abs() if dtype == torch.bfloat16 else 0)
    worst = float(((y.cpu().double() - ref).abs() / bound.clamp(min=1e-300)).max())
    print(f"  worst |err| / bound {worst:.3f}", flush=True)
    assert torch.isfinite(y).all() and worst <= 1
    assert torch.equal(y, y2)


@pytest.mark.parametrize("M", [3, 40, 150, 2100])
def test_extreme_integers(M):
    """-128 everywhere (weights rounded by another hand): the sums are exact."""
    print(f"[case] linear_i8 extremes {M}", flush=True)
    from ssmjs_amd import kernels
    N, K = 48, 131071 if M < 2000 else 4096
    x = torch.full((M, K), -128, dtype=torch.int8, device="cuda")
    W = torch.full((N, K), -128, dtype=torch.int8, device="cuda")
    W[1::2] = 127
    one = torch.ones(max(M, N), device="cuda")
    y = kernels.linear_i8(x, one[:M], W, one[:N])
    torch.cuda.synchronize()
    want = torch.tensor([128 * 128 * K, -128 * 127 * K], dtype=torch.float64).to(torch.float32).cuda()
    assert (y[:, 0::2] == want[0]).all() and (y[:, 1::2] == want[1]).all()


@pytest.mark.parametrize("M", [5, 64, 130])
def test_views_and_alignment(M):
    """Operands and outputs inside wider rows, at odd places: the bits of contiguous ones."""
    print(f"[case] linear_i8 views {M}", flush=True)
    from ssmjs_amd import kernels
    N, K = 70, 512
    gen = torch.Generator(device="cuda").manual_seed(M)
    big = lambda r, c: torch.randint(-127, 128, (r, c), generator=gen, device="cuda", dtype=torch.int32).to(torch.int8)   # noqa: E731
    xs, ws = big(M, K + 48), big(N, K + 48)
    sx, sw = torch.rand(M, device="cuda"), torch.rand(N, device="cuda")
    xf = torch.randn(M, K + 3, device="cuda", dtype=torch.bfloat16)
    for at in (0, 1, 16, 7):
        x, W = xs[:, at:at + K], ws[:, at:at + K]
        want = kernels.linear_i8(x.contiguous(), sx, W.contiguous(), sw)
        wide = torch.full((M, N + 9), 5.0, device="cuda")
        got = kernels.linear_i8(x, sx, W, sw, out=wide[:, 3:3 + N])
        f = xf[:, at % 3:at % 3 + K]
        assert torch.equal(kernels.linear_q8(f, W, sw), kernels.linear_q8(f.contiguous(), W.contiguous(), sw))
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        assert (wide[:, :3] == 5).all() and (wide[:, 3 + N:] == 5).all()


@pytest.mark.parametrize("M,K", [(1, 1024), (4, 2048), (9, 512), (200, 256)])
def test_output_over_the_input(M, K):
    """y written over x: bit-equal to a call with an output of its own."""
    print(f"[case] linear_q8 in place {M} x {K}", flush=True)
    from ssmjs_amd import kernels
    x = data(M, K, torch.float32, M)
    W, sw = kernels.quantize_rows(data(K, K, torch.float32, M + 1))
    y = kernels.linear_q8(x, W, sw)
    for beta in (0.0, 0.5):
        mine = x.clone()
        ref = x.clone()
        kernels.linear_q8(x, W, sw, out=ref, beta=beta)
        kernels.linear_q8(mine, W, sw, out=mine, beta=beta)
        torch.cuda.synchronize()
        assert torch.equal(mine, ref), beta
    kernels.linear_q8(x, W, sw, out=x)
    torch.cuda.synchronize()
    assert torch.equal(x, y)
