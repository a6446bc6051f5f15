"""Padded batches without an output of the caller's: rows behind a sequence are zeros."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_behind_a_sequence_are_zeros(dtype):
    print(f"[case] padded rows {dtype}", flush=True)
    from ssmjs_amd import kernels
    B, L, H, G, K, V = 4, 300, 4, 2, 64, 64
    g = torch.Generator(device="cuda").manual_seed(0)
    f = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)   # noqa: E731
    q, k, v = f(B, L, H, K), f(B, L, G, K), f(B, L, G, V)
    n = [300, 0, 1, 130]
    decays = -torch.rand(H, generator=g, device="cuda")
    # memory that the call may be given, not zeros
    used = torch.full((B, L, H, V), float("nan"), dtype=dtype, device="cuda")
    del used
    y = kernels.linear_attention(q, k, v, decays, lengths=torch.tensor(n, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    for b, m in enumerate(n):
        one = kernels.linear_attention(q[b:b + 1, :m], k[b:b + 1, :m], v[b:b + 1, :m], decays)
        torch.cuda.synchronize()
        assert not y[b, m:].any() and torch.isfinite(y[b]).all()
        assert (y[b, :m].double() - one[0].double()).abs().max() <= 2.0 ** -6 * one.abs().max() if m else True
