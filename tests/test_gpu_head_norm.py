"""qk_norm_rope against the formula in 64 bits. A pair's outputs are held to 2^-24 of |a| + |b| (its
normed elements) times the roundings on the way: the mean of D squares 14 (its sum is a tree of at
most 8 + 6 levels; half of it after the root), 1 / sqrt 4, the products with it and w 3, cosine and
sine 4 + 4 (2 ulp, and the rounding of the reduced angle), the rotation 3: 32 in all; bfloat16
outputs to half a step, 2^-8 of the value, on top."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def reference(x, w, pos, freq, inter, eps):
    """The formula in 64 bits, and |a| + |b| of each element's pair."""
    x = x.double().cpu().numpy()
    D, R = x.shape[-1], 2 * len(freq)
    x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    if w is not None:
        x = x * w.double().cpu().numpy()
    at = np.arange(R // 2)
    a, b = (2 * at, 2 * at + 1) if inter else (at, at + R // 2)
    t = pos.cpu().numpy().astype(np.float64)[..., None, None] * freq.cpu().numpy()
    y, size = x.copy(), np.abs(x)
    y[..., a] = x[..., a] * np.cos(t) - x[..., b] * np.sin(t)
    y[..., b] = x[..., b] * np.cos(t) + x[..., a] * np.sin(t)
    size[..., a] = size[..., b] = np.abs(x[..., a]) + np.abs(x[..., b])
    assert D == y.shape[-1]
    return y, size


def check(got, ref, what):
    y, size = ref
    got_ = got.double().cpu().numpy()
    bound = 32 * 2.0 ** -24 * size + (2.0 ** -8 * np.abs(y) if got.dtype == torch.bfloat16 else 0)
    worst = float((np.abs(got_ - y) / np.maximum(bound, 1e-300)).max())
    print(f"  {what}: worst |err| / bound {worst:.3f}", flush=True)
    assert np.isfinite(got_).all() and worst <= 1


CASES = [   # rows, H, G, D, R
    ((1, 1), 1, 1, 2, 2), ((1, 1), 1, 0, 128, 128), ((1, 1), 0, 3, 64, 64), ((3, 5), 4, 2, 64, 32),
    ((2, 7), 5, 1, 128, 128), ((1, 33), 8, 8, 80, 80), ((1, 9), 2, 2, 96, 48), ((2, 3), 3, 1, 256, 64),
    ((1, 4), 2, 1, 512, 512), ((1, 4), 2, 1, 511, 510), ((1, 5), 3, 2, 7, 4), ((1, 6), 2, 2, 20, 20),
    ((2, 3), 2, 1, 128, 0), ((5, 1000), 6, 2, 64, 64), ((64,), 12, 4, 128, 64), ((4099,), 2, 1, 128, 128),
]


@pytest.mark.parametrize("rows,H,G,D,R", CASES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("inter", [False, True])
def test_matches_formula(rows, H, G, D, R, dtype, inter):
    print(f"[case] qk_norm_rope {rows} H={H} G={G} D={D} R={R} {dtype} {inter}", flush=True)
    from ssmjs_amd import kernels
    gen = torch.Generator(device="cuda").manual_seed(D + R)
    f = lambda *s: torch.randn(*s, generator=gen, device="cuda")   # noqa: E731
    q, k = f(*rows, H, D).to(dtype), f(*rows, G, D).to(dtype)
    wq, wk = 1 + 0.3 * f(D), (None if D % 3 == 0 else 1 + 0.3 * f(D))
    pos = torch.randint(0, 2_000_000, rows, generator=gen, device="cuda").to(torch.int32)
    freq = 10000.0 ** (-torch.arange(R // 2, device="cuda", dtype=torch.float64) / max(R // 2, 1))
    qo, ko = kernels.qk_norm_rope(q, k, wq, wk, pos, freq, eps=1e-5, interleaved=inter)
    torch.cuda.synchronize()
    for what, x, w, got in (("q", q, wq, qo), ("k", k, wk, ko)):
        if x.numel():
            check(got, reference(x, w, pos, freq, inter, 1e-5), what)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift", [0, 1])   # 1: rows that are not aligned
def test_views_and_in_place(dtype, shift):
    """q and k as parts of wider rows, rotated in place: the same bits as from and to tensors of
    their own, and nothing else in the rows is touched."""
    print(f"[case] qk_norm_rope in place {dtype} shift {shift}", flush=True)
    from ssmjs_amd import kernels
    B, L, H, G, D = 2, 21, 3, 2, 64
    W = (H + 2 * G) * D + 2 * shift
    gen = torch.Generator(device="cuda").manual_seed(1)
    flat = torch.randn(B * L * W + shift, generator=gen, device="cuda").to(dtype)
    rows = flat[shift:].view(B, L, W)
    before = rows.clone()
    q = rows[..., :H * D].unflatten(-1, (H, D))
    k = rows[..., H * D:(H + G) * D].unflatten(-1, (G, D))
    pos = torch.arange(B * L, device="cuda", dtype=torch.int32).view(B, L)
    freq = 100.0 ** (-torch.arange(D // 2, device="cuda", dtype=torch.float64) / (D // 2))
    w = torch.ones(D, device="cuda")
    wide = kernels.qk_norm_rope(q.contiguous(), k.contiguous(), w, w, pos, freq)
    kernels.qk_norm_rope(q, k, w, w, pos, freq, out=(q, k))
    torch.cuda.synchronize()
    if shift == 0:
        assert torch.equal(q, wide[0]) and torch.equal(k, wide[1])
    else:   # the element-wise kernel: another order of the sum of squares
        for got, x in ((q, before[..., :H * D].unflatten(-1, (H, D))),
                       (k, before[..., H * D:(H + G) * D].unflatten(-1, (G, D)))):
            check(got, reference(x, w, pos, freq, False, 1e-6), "in place")
    assert torch.equal(rows[..., (H + G) * D:], before[..., (H + G) * D:])


def test_odd_values_stay_in_their_head():
    """Zeros give zeros, and an inf or NaN reaches no other head."""
    print("[case] qk_norm_rope odd values", flush=True)
    from ssmjs_amd import kernels
    q = torch.randn(1, 6, 4, 64, device="cuda")
    q[0, 1, 2] = 0
    q[0, 2, 1, 5] = float("nan")
    q[0, 3, 0, 7] = float("inf")
    k = torch.zeros(1, 6, 1, 64, device="cuda")
    pos = torch.zeros(1, 6, dtype=torch.int32, device="cuda")
    freq = torch.ones(32, dtype=torch.float64, device="cuda")
    qo, ko = kernels.qk_norm_rope(q, k, None, None, pos, freq)
    torch.cuda.synchronize()
    bad = torch.zeros(1, 6, 4, dtype=torch.bool)
    bad[0, 2, 1] = bad[0, 3, 0] = True
    assert torch.equal(qo.isnan().any(-1).cpu(), bad)
    assert not qo[0, 1, 2].any() and not ko.any()
