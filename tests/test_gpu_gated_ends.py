"""The gated recurrence where its arguments end: batches of no sequences, decays past fp32's range."""
import pytest

torch = pytest.importorskip("torch")

import test_gpu_gated_recurrence as rec  # noqa: E402
from test_gpu_gated_scales import drawn  # noqa: E402

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_of_an_empty_batch(dtype):
    """A batch of no sequences, whose forward call is one, has a gradient too: zeros for lam, nothing else."""
    from ssmjs_amd import kernels as k
    lam = torch.randn(70, device="cuda")
    for n in (9, 0):
        print(f"[case] gradients of an empty batch {n} {dtype}", flush=True)
        x, h = torch.empty(0, n, 70, device="cuda", dtype=dtype), torch.empty(0, 70, device="cuda")
        st = k.gated_recurrence_states(0, n, 70, "cuda")
        outs = [torch.empty_like(x) for _ in range(3)]
        for ln in (None, torch.empty(0, dtype=torch.int32, device="cuda")):
            k.gated_recurrence(x, x, x, lam, lengths=ln, h0=h, hT=h, states=st)
            for out in (None, outs):
                *g, dlam = k.gated_recurrence_backward(x, x, x, x, lam, st, lengths=ln, dhT=h, dh0=h, out=out)
                torch.cuda.synchronize()
                assert all(t.shape == x.shape and t.dtype == dtype for t in g)
                assert dlam.dtype == torch.float32 and torch.equal(dlam, torch.zeros(70, device="cuda"))
        with pytest.raises(ValueError):      # (its operands are looked at all the same)
            k.gated_recurrence_backward(x, x, x, x, lam[:-1], st)
        with pytest.raises(TypeError):
            k.gated_recurrence_backward(x, x, x, x, lam.double(), st)


@pytest.mark.parametrize("L", [5, 100, 3000])
@pytest.mark.parametrize("c,top", [(3e38, 60.0), (8.0, 3e38), (1e20, 3.0)])
def test_products_past_the_range(c, top, L):
    """c softplus(lam) beyond fp32's range, or far up in it: decays are 0 where the gate is open and 1 where it is shut, and
    gradients are finite. The recurrence counts c softplus(lam) up to 2^64. A gate below fp32's range (r = -120) is 0, or, in
    the gradients, 2^-126: z is then 2^-62 and sqrt(1 - a^2) 2^-30.5 at most."""
    from ssmjs_amd import kernels as k
    print(f"[case] products past the range {c} {top} {L}", flush=True)
    B, D = 2, 68
    x, r, i, lam, h0, dy, dhT, _ = drawn(B, L, D, torch.float32, 25)
    lam[::2] = top
    r[..., 0], r[..., 2], r[..., 4], r[..., 6] = -80.0, 80.0, -40.0, -120.0
    g = rec.gates(x, r, i, lam, c)
    z = torch.clamp(c * torch.nn.functional.softplus(lam.double(), threshold=1e4), max=2.0 ** 64) / (1 + torch.exp(-r.double()))
    g["z"], g["a"], g["beta"] = z, torch.exp(-z), (-torch.expm1(-2 * z)).sqrt()
    g["b"] = g["beta"] * g["gi"] * x.double()
    # (a z of more than 2^10 gives a = 0 however it is rounded)
    g["ka"] = (8 + z.clamp(max=1024) * (g["R"] + 24)) * U
    n = torch.full((B,), L, device="cuda")
    hs, _, es = rec.walk(g, n, h0)
    st, hT, dh0 = k.gated_recurrence_states(B, L, D, "cuda"), torch.empty(B, D, device="cuda"), torch.empty(B, D, device="cuda")
    y = k.gated_recurrence(x, r, i, lam, c=c, h0=h0, hT=hT, states=st)
    grads = k.gated_recurrence_backward(dy, x, r, i, lam, st, c=c, dhT=dhT, dh0=dh0)
    h = h0.clone()
    y1 = k.gated_recurrence_step(x[:, 0], r[:, 0], i[:, 0], lam, h, c=c)
    torch.cuda.synchronize()
    assert all(bool(torch.isfinite(t).all()) for t in (y, hT, y1, h, *grads, dh0))
    rec.close(y, hs[:, 1:], es[:, 1:], "y")
    rec.close(hT, hs[:, -1], es[:, -1], "hT")
    rec.close(y1, hs[:, 1], es[:, 1], "step")
    gt, mg, eg, e0, ee0 = rec.adjoint(g, dy, n, dhT)
    k2 = (g["R"] + g["I"] + 60) * U
    bi = g["beta"] * g["gi"]
    rec.close(grads[0], gt * bi, bi * (eg + mg * k2) + 2.0 ** -30 * (r < -88) * g["gi"] * mg, "dx")
    rec.close(dh0, e0, ee0, "dh0")
    # the formula: an open gate forgets all, a shut one nothing
    assert bool((grads[1][..., 2] == 0).all())
