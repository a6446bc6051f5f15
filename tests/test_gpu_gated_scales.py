"""The gated-recurrence model's operators at other decay scales c and other eps, and at sizes that take other workgroups,
against 64 bits. Bounds as in the operators' own tests, where each is derived; what differs here is derived where it
stands."""
import pytest

torch = pytest.importorskip("torch")

import test_gpu_block_norm as norms  # noqa: E402
import test_gpu_gated_recurrence as rec  # noqa: E402

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def whole_pass(x, r, i, lam, c, lengths, h0, dy, dhT, chain):
    """Forward and gradients at decay scale c against the walk in 64 bits, every output with its own bound: of dlam the sum
    over tokens of each token's own, `chain` roundings of its terms' magnitudes among them."""
    from ssmjs_amd import kernels as k
    B, L, D = x.shape
    n = lengths if lengths is not None else torch.full((B,), L, dtype=torch.int32, device="cuda")
    g = rec.gates(x, r, i, lam, c)
    hs, ms, es = rec.walk(g, n, h0)
    states, hT, dh0 = k.gated_recurrence_states(B, L, D, "cuda"), torch.empty(B, D, device="cuda"), torch.empty(B, D, device="cuda")
    y = k.gated_recurrence(x, r, i, lam, c=c, lengths=lengths, h0=h0, hT=hT, states=states)
    dx, dr, di, dlam = k.gated_recurrence_backward(dy, x, r, i, lam, states, c=c, lengths=lengths, dhT=dhT, dh0=dh0)
    torch.cuda.synchronize()
    inside = (torch.arange(L, device="cuda") < n[:, None])[..., None]
    rec.close(y, torch.where(inside, hs[:, 1:], 0.0), es[:, 1:], "y")
    rec.close(hT, hs[:, -1], es[:, -1], "hT")
    for s in range(0, L, 64):
        on = (s < n)[:, None]
        rec.close(torch.where(on, states[:, s // 64], 0.0), torch.where(on, hs[:, s], 0.0), es[:, s], f"state {s}")
    gt, mg, eg, e0, ee0 = rec.adjoint(g, dy, n, dhT)
    k2 = (g["R"] + g["I"] + 60) * U
    bi, bu = g["beta"] * g["gi"], g["b"] * g["ci"]
    rec.close(dx, gt * bi, bi * (eg + mg * k2), "dx")
    rec.close(di, gt * bu, bu.abs() * (eg + mg * k2), "di")
    p1 = g["gi"] * g["x"] * g["a"] ** 2 * g["z"] / g["beta"].clamp(min=1e-300)
    p2 = g["a"] * g["z"]
    hp, mp, ep = hs[:, :-1], ms[:, :-1], es[:, :-1]
    q = gt * (p1 - p2 * hp)
    k3 = (4 * g["R"] + g["I"] + 80 + 4 * g["z"] * (g["R"] + 24)) * U
    eq = eg * (p1.abs() + p2 * mp) + mg * (p1.abs() * k3 + p2 * (ep + k3 * mp))
    gone = 2.0 ** -126 * (1 + g["z"]) * (1 + mp) * mg
    rec.close(dr, q * g["cr"], g["cr"] * (eq + gone), "dr")
    f = torch.sigmoid(lam.double()) / torch.nn.functional.softplus(lam.double(), threshold=1e4)
    sums = (eq + gone + chain * U * mg * (p1.abs() + p2 * mp)).sum((0, 1))
    want = f * q.sum((0, 1))
    print(f"  dlam: bound / largest {float((f * sums).max() / (want.abs().max() + 1e-30)):.2e}", flush=True)
    rec.close(dlam, want, f * sums, "dlam")
    if x.dtype == torch.float32:
        # and far tighter, the sum alone: of q as this call's own dr = q (1 - sigmoid r) has it, whose second factor is within
        # 2 |r| + 9 units and whose product and quotient round twice; f is within 16
        q = dr.double() / g["cr"]
        off = f * (q.abs() * (chain + 2 * g["R"] + 27)).sum((0, 1)) * U
        print(f"  dlam of dr: bound / largest {float(off.max() / (want.abs().max() + 1e-30)):.2e}", flush=True)
        rec.close(dlam, f * q.sum((0, 1)), off, "dlam of dr")
    rec.close(dh0, e0, ee0, "dh0")


def drawn(B, L, D, dtype, seed, strided=False, ragged=False):
    x, r, i, lam, h0, gen = rec.inputs(B, L, D, dtype, seed, strided)
    dy = torch.randn(B, L, D, generator=gen, device="cuda").to(dtype)
    dhT = torch.randn(B, D, generator=gen, device="cuda")
    lengths = None
    if ragged:
        lengths = torch.randint(0, L + 1, (B,), generator=gen, device="cuda").to(torch.int32)
        lengths[0], lengths[-1] = L, 0 if B > 1 else L
    return x, r, i, lam, h0, dy, dhT, lengths


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("c", [0.0, 0.7, 20.0])
@pytest.mark.parametrize("B,L,D,strided,ragged", [(2, 13, 66, False, False), (3, 300, 33, True, True), (1, 3000, 68, False, True)])
def test_decay_scales(B, L, D, strided, ragged, c, dtype):
    print(f"[case] decay scale {c}: {B} {L} {D} {dtype}", flush=True)
    x, r, i, lam, h0, dy, dhT, lengths = drawn(B, L, D, dtype, 21, strided, ragged)
    whole_pass(x, r, i, lam, c, lengths, h0, dy, dhT, L / 8 + 48)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("c", [0.0, 0.7, 20.0])
def test_decay_scales_of_a_step(c, dtype):
    from ssmjs_amd import kernels as k
    for B, D in ((3, 5), (5, 256)):
        print(f"[case] decay scale {c}, step: {B} {D} {dtype}", flush=True)
        x, r, i, lam, h, _ = rec.inputs(B, 1, D, dtype, 22)
        hs, _, es = rec.walk(rec.gates(x, r, i, lam, c), torch.ones(B, device="cuda"), h)
        y = k.gated_recurrence_step(x[:, 0], r[:, 0], i[:, 0], lam, h, c=c)
        torch.cuda.synchronize()
        rec.close(y, hs[:, 1], es[:, 1], "y")
        rec.close(h, hs[:, 1], es[:, 1], "h")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L,D", [(40, 150, 1024), (17, 512, 2048), (520, 70, 64)])
def test_many_short_prompts(B, L, D, dtype):
    """Gradients on workgroups of four waves over more than one block of 64 steps, without lengths: a lane adds up 8 values
    a block, L / 8, the waves, rows and sequences (these in double) 16 more."""
    print(f"[case] many short prompts {B} {L} {D} {dtype}", flush=True)
    x, r, i, lam, h0, dy, dhT, _ = drawn(B, L, D, dtype, 23)
    whole_pass(x, r, i, lam, 8.0, None, h0, dy, dhT, L / 8 + 48)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L,D,strided,ragged", [(1, 5000, 516, False, False), (3, 3000, 392, True, True), (1, 6000, 302, False, False)])
def test_cut_prompts_of_many_channels(B, L, D, strided, ragged, dtype):
    """Sequences cut into segments whose first pass takes several groups of 128 channels, the last not whole (and, D = 302,
    of 64)."""
    from ssmjs_amd import _lib
    print(f"[case] cut prompts {B} {L} {D} {dtype}", flush=True)
    assert _lib.lib().ssm_gated_recurrence_workspace(B, L, D) > 0
    x, r, i, lam, h0, dy, dhT, lengths = drawn(B, L, D, dtype, 24, strided, ragged)
    whole_pass(x, r, i, lam, 8.0, lengths, h0, dy, dhT, L / 8 + 48)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("eps,size", [(0.1, 1.0), (1e-6, 1e-3), (0.0, 1.0)])
@pytest.mark.parametrize("shape", [(5, 66), (4, 768), (3, 2048), (2, 5000), (2, 9000)])
def test_eps(shape, eps, size, dtype):
    """An eps that is a visible part of the mean of squares, and none; of y as of x'."""
    from ssmjs_amd import kernels as k
    print(f"[case] norms' eps {eps} {size} {shape} {dtype}", flush=True)
    x, y, z, dx1, dn, post, scale, pre = norms.inputs(shape, dtype, 31, False)
    x, y = (x.float() * size).to(dtype), (y.float() * size).to(dtype)
    scale = scale * size
    for zz in (z, None):
        ref = norms.reference(x, y, zz, post, scale, pre, eps, dx1, dn)
        x1, n = k.block_norm(x, y, zz, post, scale, pre, eps=eps)
        got = dict(zip(("dx", "dy", "dz", "dpost", "dscale", "dpre"),
                       k.block_norm_backward(dx1, dn, x, y, zz, post, scale, pre, eps=eps)))
        torch.cuda.synchronize()
        for name, t in (got | {"x1": x1, "n": n}).items():
            if t is not None:
                norms.close(t, ref[name], f"{name} gate {zz is not None}")


def test_columns_of_many_wide_rows():
    """The weights' gradients over 24000 rows of 4100 elements, where a workgroup takes one row at a time: a lane adds T / 256
    rows, and 64 roundings cover the rest."""
    from ssmjs_amd import kernels as k
    T, D = 24000, 4100
    print(f"[case] columns of many wide rows {T} {D}", flush=True)
    x, y, _, dx1, dn, post, scale, pre = norms.inputs((T, D), torch.float32, 32, False)
    *_, dpost, dscale, dpre = k.block_norm_backward(dx1, dn, x, y, None, post, scale, pre)
    torch.cuda.synchronize()
    want = {m: [0.0, 0.0] for m in ("dpost", "dscale", "dpre")}
    chain = (T / 256 + 64) * U
    for s in range(0, T, 2000):
        rows = slice(s, s + 2000)
        ref = norms.reference(x[rows], y[rows], None, post, scale, pre, 1e-6, dx1[rows], dn[rows])
        g, eg = ref["dx"]
        n, en = ref["n"]
        yy = y[rows].double()
        w = yy * (yy.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
        v, sc, d = w * post.double(), scale.double(), dn[rows].double()
        nh, enh = n / pre.double(), en / pre.double().abs()
        for m, val, err in (("dscale", g * v, eg * v.abs() + (g * v).abs() * 46 * U),
                            ("dpost", g * sc * w, (sc * w).abs() * eg + (g * sc * w).abs() * 46 * U),
                            ("dpre", d * nh, d.abs() * enh + U * (d * nh).abs())):
            want[m][0] += val.sum(0)
            want[m][1] += (err + chain * val.abs()).sum(0)
    for m, got in (("dpost", dpost), ("dscale", dscale), ("dpre", dpre)):
        norms.close(got, want[m], m)
