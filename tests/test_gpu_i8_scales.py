"""The 8-bit products' scales where their own product leaves fp32's range and the results do not."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


# few rows (one launch, two), tiles of 64 and 128 rows, and of 256
SHAPES = [(1, 64, 256), (20, 63, 256), (64, 4200, 256), (130, 300, 256), (300, 601, 256), (1000, 4384, 256),
          (4200, 4100, 256), (4200, 4107, 256)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("beta", [0.0, 1.0])
def test_a_sum_of_zero_is_zero(M, N, K, beta):
    """Scales whose product is above the largest number, and sums that cancel to zero."""
    print(f"[case] scales above the range {M} x {N} x {K}", flush=True)
    from ssmjs_amd import kernels
    x = torch.ones(M, K, device="cuda") * 1e30
    x[:, 1::2] *= -1
    W = torch.full((N, K), 100, dtype=torch.int8, device="cuda")
    sw = torch.full((N,), 1e20, device="cuda")
    y = torch.ones(M, N, device="cuda")
    kernels.linear_q8(x, W, sw, out=y, beta=beta)
    torch.cuda.synchronize()
    assert (y == beta).all()


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_small_scales_keep_their_digits(M, N, K, dtype):
    """Scales of some 2^-80 and 2^-60, sums of 2^21 to 2^22: the results are some 2^-118, their scales'
    product has ten digits. Three roundings of 2^-24, and the output's."""
    print(f"[case] scales below the range {M} x {N} x {K} {dtype}", flush=True)
    from ssmjs_amd import kernels
    g = torch.Generator(device="cuda").manual_seed(M)
    x = torch.randint(90, 128, (M, K), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
    W = torch.randint(90, 128, (N, K), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
    sx = (torch.rand(M, generator=g, device="cuda") + 1) * 2.0 ** -80
    sw = (torch.rand(N, generator=g, device="cuda") + 1) * 2.0 ** -60
    y = kernels.linear_i8(x, sx, W, sw, out_dtype=dtype)
    torch.cuda.synchronize()
    ref = (x.double() @ W.double().t()) * sx.double()[:, None] * sw.double()
    worst = float(((y.double() - ref).abs() / ((3 * 2.0 ** -24 + (2.0 ** -8 if dtype == torch.bfloat16 else 0)) * ref)).max())
    print(f"  worst |err| / bound {worst:.3f}", flush=True)
    assert worst <= 1
