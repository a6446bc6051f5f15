"""The 8-bit products' tiles by the way they are walked: every tile size, output type, beta and bias, several
tiles a workgroup, last turns whole and in quarters, k that ends anywhere in the blocks' groups."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def ints(g, *shape):
    return torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int32).to(torch.int8)


SHAPES = [   # M, N, K
    # 64 rows and 128 channels a workgroup; 128 rows (a tile for every CU)
    (300, 600, 300), (1000, 4384, 1024), (1030, 4384, 130), (2000, 2050, 300),
    # 256 x 256: two and more tiles a workgroup with a last turn in quarters
    (4200, 8200, 300), (8192, 8512, 300), (4200, 8200, 1024),
    # whole last turns: 16, 18 and 12 or 13 tiles over 32 workgroups
    (6144, 4096, 300), (5120, 5113, 130), (5120, 5120, 1000), (4864, 4864, 64),
]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("beta,with_bias", [(0.0, False), (0.0, True), (1.0, False), (0.5, True)])
def test_tiles(M, N, K, dtype, beta, with_bias):
    """Roundings: the integer sum, two scales, the bias; with beta its product and the sum; the output's."""
    print(f"[case] linear_i8 tiles {M} x {N} x {K} {dtype} beta {beta} bias {with_bias}", flush=True)
    from ssmjs_amd import kernels
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    x, W = ints(g, M, K), ints(g, N, K)
    sx = torch.rand(M, generator=g, device="cuda") + 0.5
    sw = torch.rand(N, generator=g, device="cuda") + 0.5
    bias = 100 * torch.randn(N, generator=g, device="cuda") if with_bias else None
    wide = torch.full((M, N + 8), 3.0, device="cuda", dtype=dtype)
    y = wide[:, :N]
    y0 = torch.randn(M, N, generator=g, device="cuda").to(dtype) if beta else None
    y.copy_(y0 if beta else torch.full_like(y, float("nan")))
    kernels.linear_i8(x, sx, W, sw, bias=bias, out=y, beta=beta)
    packed = y0.clone() if beta else torch.empty(M, N, device="cuda", dtype=dtype)
    kernels.linear_i8(x, sx, W, sw, bias=bias, out=packed, beta=beta)
    torch.cuda.synchronize()
    p = (x.double() @ W.double().t()) * sx.double()[:, None] * sw.double()
    ref = p + bias.double() if with_bias else p
    size = 3 * p.abs() + ref.abs()
    if beta:
        ref = ref + beta * y0.double()
        size = size + (beta * y0.double()).abs() + ref.abs()
    bound = U * size + (2.0 ** -8 * ref.abs() if dtype == torch.bfloat16 else 0) + 1e-300
    worst = float(((y.double() - ref).abs() / bound).max())
    print(f"  worst |err| / bound {worst:.3f}", flush=True)
    assert torch.isfinite(y).all() and worst <= 1
    assert torch.equal(y, packed) and (wide[:, N:] == 3).all()
