"""An infinite state stays infinite, as in the recurrence, through chunks, segments and single tokens."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

INF = float("inf")


@pytest.mark.parametrize("B,L", [(1, 1), (1, 200), (150, 70), (1, 1500), (1, 6000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("g", [0.0, -1e-6, -0.004, -0.5, -20.0])
def test_an_infinite_state_stays(B, L, dtype, g):
    print(f"[case] infinite state B={B} L={L} {dtype} g={g}", flush=True)
    from ssmjs_amd import kernels
    H, K, V = 2, 64, 128
    r = torch.Generator(device="cuda").manual_seed(1)
    f = lambda *s: torch.randn(*s, generator=r, device="cuda")   # noqa: E731
    q, k, v, h0 = f(B, L, H, K).to(dtype), f(B, L, H, K).to(dtype), f(B, L, H, V).to(dtype), f(B, H, V, K)
    gs = torch.full((H,), g, device="cuda")
    h0[0, 1, 3, 9], h0[0, 1, 70, 20] = INF, -INF
    clean = torch.where(h0.isinf(), 0.0, h0)
    hT, cT = torch.empty_like(h0), torch.empty_like(h0)
    y = kernels.linear_attention(q, k, v, gs, h0=h0, hT=hT)
    cy = kernels.linear_attention(q, k, v, gs, h0=clean, hT=cT)
    h = h0.clone()
    y1 = kernels.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], gs, h)
    torch.cuda.synchronize()
    touched = torch.zeros(B, H, V, dtype=torch.bool, device="cuda")
    touched[0, 1, [3, 70]] = True
    for s in (hT, h):
        assert s[0, 1, 3, 9] == INF and s[0, 1, 70, 20] == -INF
        assert int((~torch.isfinite(s)).sum()) == 2
    assert torch.equal(torch.where(h0.isinf(), 0.0, hT), torch.where(h0.isinf(), 0.0, cT))
    assert torch.equal(torch.isfinite(y), ~touched[:, None].expand(y.shape))
    assert torch.equal(torch.isfinite(y1), ~touched)
    assert torch.equal(torch.where(touched[:, None], 0, y), torch.where(touched[:, None], 0, cy))
    # inf q, to the sign, while no weight is too small for fp32
    n = min(L, int(80 / -g)) if g < 0 else L
    for at, kk, s in ((3, 9, INF), (70, 20, -INF)):
        assert torch.equal(y[0, :n, 1, at].float(), q[0, :n, 1, kk].float() * s)
        assert y1[0, 1, at] == q[0, 0, 1, kk].float() * s
