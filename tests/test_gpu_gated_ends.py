"""The gated recurrence where its arguments end: batches of no sequences, decays past fp32's range."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


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
