"""Outputs and states that lie between the rows of other operands, in one buffer, share no memory with them:
the bits of operands of their own."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [3, 70])
def test_a_product_beside_its_weights(M):
    print(f"[case] y beside W, M={M}", flush=True)
    from ssmjs_amd import kernels
    g = torch.Generator(device="cuda").manual_seed(M)
    N, K = 96, 256
    rows = torch.randint(-127, 128, (N, K + 4 * N), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
    W, y = rows[:, :K], rows.view(torch.float32)[:M, K // 4:]
    x, sw = torch.randn(M, K, generator=g, device="cuda"), torch.rand(N, generator=g, device="cuda")
    want = kernels.linear_q8(x, W.contiguous(), sw)
    before = W.clone()
    kernels.linear_q8(x, W, sw, out=y)
    torch.cuda.synchronize()
    assert torch.equal(y, want) and torch.equal(W, before)


def test_a_state_between_the_sequences_rows():
    print("[case] state between rows", flush=True)
    from ssmjs_amd import kernels
    g = torch.Generator(device="cuda").manual_seed(0)
    B, H, G, K, V = 2, 4, 2, 16, 16
    buf = torch.randn(2 * 4096, generator=g, device="cuda")
    q = buf.as_strided((B, H, K), (4096, K, 1))
    h = buf[H * K:H * K + B * H * V * K].view(B, H, V, K)
    k, v = torch.randn(B, G, K, generator=g, device="cuda"), torch.randn(B, G, V, generator=g, device="cuda")
    decays = -torch.rand(H, generator=g, device="cuda")
    mine = h.clone()
    want = kernels.linear_attention_step(q.contiguous(), k, v, decays, mine)
    y = kernels.linear_attention_step(q, k, v, decays, h)
    torch.cuda.synchronize()
    assert torch.equal(y, want) and torch.equal(h, mine)
    # prompts of one token, the state in place again
    want = kernels.linear_attention(q[:, None].contiguous(), k[:, None], v[:, None], decays, h0=mine, hT=mine)
    y = kernels.linear_attention(q[:, None], k[:, None], v[:, None], decays, h0=h, hT=h)
    torch.cuda.synchronize()
    assert torch.equal(y, want) and torch.equal(h, mine)
