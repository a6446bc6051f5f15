"""What the operators of a linear-attention layer refuse, and what their workspace queries say. The
pointers are placeholders that are never followed: every call here ends at the host's checks."""
import pytest

from ssmjs_amd import _lib

P = 1 << 20
F32, BF16 = _lib.SSM_F32, _lib.SSM_BF16
OK, INVALID, UNSUPPORTED = _lib.SSM_OK, _lib.SSM_ERR_INVALID_ARG, _lib.SSM_ERR_UNSUPPORTED


def rope(dtype=F32, q=P, ldq=256, k=P, ldk=128, pos=P, freq=P, qo=P, ldqo=256, ko=P, ldko=128, T=2,
         H=4, G=2, D=64, R=64):
    return _lib.lib().ssm_qk_norm_rope(dtype, q, ldq, k, ldk, None, None, pos, freq, 0, 1e-6, qo,
                                       ldqo, ko, ldko, T, H, G, D, R, None)


@pytest.mark.parametrize("change,status", [
    (dict(T=0), OK), (dict(H=0, G=0), OK),
    (dict(dtype=2), INVALID), (dict(T=-1), INVALID), (dict(D=0), INVALID), (dict(R=63), INVALID),
    (dict(R=66), INVALID), (dict(R=-2), INVALID), (dict(D=514, R=64), UNSUPPORTED),
    (dict(q=None), INVALID), (dict(ko=None), INVALID), (dict(pos=None), INVALID),
    (dict(freq=None), INVALID), (dict(ldq=255), INVALID), (dict(ldko=127), INVALID),
    (dict(T=1 << 30, H=16, G=16, ldq=1024, ldqo=1024, ldk=1024, ldko=1024), INVALID),
])
def test_qk_norm_rope_refuses(change, status):
    assert rope(**change) == status, _lib.lib().ssm_last_error()


def attention(dtype=BF16, q=P, ldq=512, k=P, ldk=256, v=P, ldv=256, g=P, y=P, ldy=512, B=2, L=8,
              H=4, G=2, K=128, V=128, ws=None, nws=0):
    return _lib.lib().ssm_linear_attention(dtype, q, ldq, k, ldk, v, ldv, g, 1.0, None, y, ldy, B, L,
                                           H, G, K, V, None, None, ws, nws, None)


@pytest.mark.parametrize("change,status", [
    (dict(B=0), OK), (dict(dtype=5), INVALID), (dict(B=-1), INVALID), (dict(L=-1), INVALID),
    (dict(H=4, G=3), INVALID), (dict(G=0), INVALID), (dict(K=0), INVALID), (dict(V=0), INVALID),
    (dict(K=257, ldq=2000, ldk=2000), UNSUPPORTED), (dict(q=None), INVALID), (dict(g=None), INVALID),
    (dict(y=None), INVALID), (dict(g=None, L=0), INVALID), (dict(ldq=511), INVALID),
    (dict(ldk=255), INVALID), (dict(ldv=255), INVALID), (dict(ldy=511), INVALID),
    (dict(ldv=1 << 24), INVALID), (dict(B=1 << 20, H=1 << 16, G=1, ldq=1 << 23, ldy=1 << 23), INVALID),
])
def test_linear_attention_refuses(change, status):
    assert attention(**change) == status, _lib.lib().ssm_last_error()


def test_linear_attention_workspace_agrees_with_the_launch():
    L = _lib.lib()
    assert L.ssm_linear_attention_workspace(BF16, 0, 8, 4, 128, 128) == 0
    assert L.ssm_linear_attention_workspace(BF16, 2, 0, 4, 128, 128) == 0
    assert L.ssm_linear_attention_workspace(BF16, 64, 4096, 16, 128, 128) == 0   # fills the chip
    need = L.ssm_linear_attention_workspace(BF16, 1, 8192, 4, 128, 128)
    assert need > 0 and need % (4 * 128 * 128 * 4) == 0
    big = dict(B=1, L=8192)
    assert attention(**big) == INVALID
    assert f"workspace of {need} bytes".encode() in L.ssm_last_error()
    assert attention(**big, ws=P, nws=need - 1) == INVALID
    assert attention(**big, ws=P + 8, nws=need) == INVALID
    assert b"16-byte aligned" in L.ssm_last_error()


def step(dtype=F32, q=P, ldq=512, k=P, ldk=256, v=P, ldv=256, g=P, y=P, ldy=512, h=P, B=2, H=4, G=2,
         K=128, V=128):
    return _lib.lib().ssm_linear_attention_step(dtype, q, ldq, k, ldk, v, ldv, g, 1.0, y, ldy, h, B,
                                                H, G, K, V, None)


@pytest.mark.parametrize("change,status", [
    (dict(B=0), OK), (dict(dtype=-1), INVALID), (dict(B=-1), INVALID), (dict(H=3), INVALID),
    (dict(V=0), INVALID), (dict(K=300, ldq=2000, ldk=2000), UNSUPPORTED), (dict(h=None), INVALID),
    (dict(v=None), INVALID), (dict(ldq=100), INVALID), (dict(ldv=100), INVALID),
    (dict(B=1 << 24, H=64, G=1, ldq=8192, ldy=8192), INVALID),
])
def test_linear_attention_step_refuses(change, status):
    assert step(**change) == status, _lib.lib().ssm_last_error()


def i8(x=P, ldx=256, sx=P, W=P, ldw=256, sw=P, out=F32, y=P, ldy=64, M=2, N=64, K=256, ws=None,
       nws=0):
    return _lib.lib().ssm_linear_i8(x, ldx, sx, W, ldw, sw, None, out, y, ldy, M, N, K, 0.0, ws, nws,
                                    None)


def q8(dtype=F32, x=P, ldx=256, W=P, ldw=256, sw=P, out=F32, y=P, ldy=64, M=2, N=64, K=256, ws=None,
       nws=0):
    return _lib.lib().ssm_linear_q8(dtype, x, ldx, W, ldw, sw, None, out, y, ldy, M, N, K, 0.0, ws,
                                    nws, None)


BAD_PRODUCTS = [
    (dict(M=0), OK), (dict(out=3), INVALID), (dict(M=-1), INVALID), (dict(N=0), INVALID),
    (dict(K=0), INVALID), (dict(K=131072, ldx=131072, ldw=131072), UNSUPPORTED),
    (dict(x=None), INVALID), (dict(W=None), INVALID), (dict(sw=None), INVALID),
    (dict(y=None), INVALID), (dict(ldx=255), INVALID), (dict(ldw=255), INVALID),
    (dict(ldy=63), INVALID), (dict(ldw=1 << 22), INVALID), (dict(ldx=1 << 22), INVALID),
]


@pytest.mark.parametrize("change,status", BAD_PRODUCTS + [(dict(sx=None), INVALID)])
def test_linear_i8_refuses(change, status):
    assert i8(**change) == status, _lib.lib().ssm_last_error()


@pytest.mark.parametrize("change,status", BAD_PRODUCTS + [(dict(dtype=7), INVALID)])
def test_linear_q8_refuses(change, status):
    assert q8(**change) == status, _lib.lib().ssm_last_error()


def test_product_workspaces_agree_with_the_launches():
    L = _lib.lib()
    # aligned rows of whole 256-byte blocks are read in place, x's from 65 rows on
    assert L.ssm_linear_i8_workspace(P, 256, P, 256, 65, 64, 256) == 0
    assert L.ssm_linear_i8_workspace(P, 256, P, 256, 64, 64, 256) >= 64 * 256
    assert L.ssm_linear_i8_workspace(P, 240, P, 240, 5, 64, 240) >= 5 * 256
    assert L.ssm_linear_i8_workspace(P, 256, P + 1, 256, 65, 64, 256) >= 64 * 256
    for change in (dict(K=240, ldx=240, ldw=240), dict(W=P + 8), dict(x=P + 4), dict(ldw=264)):
        c = dict(x=P, ldx=256, W=P, ldw=256, M=2, N=64, K=256) | change
        need = L.ssm_linear_i8_workspace(c["x"], c["ldx"], c["W"], c["ldw"], c["M"], c["N"], c["K"])
        assert need > 0
        for bad in (dict(), dict(ws=P, nws=need - 1), dict(ws=P + 4, nws=need)):
            assert i8(**change, **bad) == INVALID, change
            assert f"workspace of {need} bytes".encode() in L.ssm_last_error()
    need = L.ssm_linear_q8_workspace(P, 256, 2, 64, 256)
    assert need >= 2 * 256 + 8
    for bad in (dict(), dict(ws=P, nws=need - 1), dict(ws=P + 4, nws=need)):
        assert q8(**bad) == INVALID
    assert L.ssm_linear_q8_workspace(P, 250, 2, 64, 250) >= need + 64 * 256


def test_quantize_rows_refuses():
    call = _lib.lib().ssm_quantize_rows
    assert call(F32, P, 8, P, 8, P, 0, 8, None) == OK
    for a in ((9, P, 8, P, 8, P, 2, 8), (F32, None, 8, P, 8, P, 2, 8), (F32, P, 7, P, 8, P, 2, 8),
              (F32, P, 8, P, 7, P, 2, 8), (F32, P, 8, P, 8, None, 2, 8), (F32, P, 8, P, 8, P, -1, 8),
              (F32, P, 8, P, 8, P, 2, 0)):
        assert call(*a, None) == INVALID


def test_python_checks():
    torch = pytest.importorskip("torch")
    from ssmjs_amd import kernels as k
    z = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt)   # noqa: E731
    with pytest.raises(ValueError, match="HIP device"):
        k.linear_attention(z(1, 4, 2, 8), z(1, 4, 2, 8), z(1, 4, 2, 8), z(2))
    with pytest.raises(TypeError):
        k.linear_attention(z(1, 4, 2, 8, dt=torch.float16), z(1, 4, 2, 8), z(1, 4, 2, 8), z(2))
    with pytest.raises(ValueError):
        k.linear_attention(z(4, 2, 8), z(1, 4, 2, 8), z(1, 4, 2, 8), z(2))
    with pytest.raises(ValueError):
        k.linear_attention_step(z(1, 4, 2, 8), z(1, 2, 8), z(1, 2, 8), z(2), z(1, 2, 8, 8))
    with pytest.raises(ValueError):
        k.qk_norm_rope(z(1, 4, 2, 8), z(1, 3, 2, 8), None, None, z(1, 4, dt=torch.int32), None)
    with pytest.raises(TypeError):
        k.quantize_rows(z(2, 8, dt=torch.float16))
    with pytest.raises(ValueError, match="beta"):
        k.linear_q8(z(2, 8), z(4, 8, dt=torch.int8), z(4), beta=1.0)
    # rows that do not lie at one distance, heads that do not follow one another
    with pytest.raises(ValueError, match="one distance"):
        k._head_rows("q", z(4, 6, 2, 8)[:, :4])
    with pytest.raises(ValueError, match="follow one another"):
        k._head_rows("q", z(1, 4, 2, 16)[..., :8])
    assert k._head_rows("q", z(2, 4, 6, 8)[:, :, 2:5]) == 48
    assert k._head_rows("q", z(3, 1, 6, 8)[:, :, 2:5]) == 48
    assert k._head_rows("q", z(3, 6, 8)[:, :2]) == 48


def refused(status, word):
    assert status == INVALID and word in _lib.lib().ssm_last_error(), _lib.lib().ssm_last_error()


def test_overlapping_outputs_are_refused():
    """An output may be the input it is made of where that is said, and lie between the columns of
    another tensor's rows; else it shares no memory with an input. (Each call ends at these checks.)"""
    far = 1 << 30
    o = b"overlaps"
    # four rows of 4 x 64 queries (1024 bytes) and 2 x 64 keys
    a = dict(T=4, q=P, k=far, qo=2 * far, ko=3 * far)
    refused(rope(**a | dict(qo=P + 4)), o)
    refused(rope(**a | dict(qo=P, ldqo=260)), o)
    refused(rope(**a | dict(ko=P + 3 * 1024 + 1020)), o)
    refused(rope(**a | dict(qo=far - 4)), o)
    refused(rope(**a | dict(ko=2 * far + 512)), o)
    # rows of 384 elements that hold queries, keys: keys written into the queries' last column
    refused(rope(**a | dict(ldq=384, ldko=384, ko=P + 255 * 4)), o)
    b = dict(q=P, k=far, v=2 * far, y=3 * far, g=P)
    for name, at in (("q", P), ("k", far), ("v", 2 * far)):
        refused(attention(**b | dict(y=at)), o)
        refused(attention(**b | dict(y=at + 511)), o)
        refused(step(**b | dict(y=at)), o)
    refused(attention(**b | dict(ldq=1024, ldy=1024, y=P + 1000)), o)   # (the last of a row of q)
    refused(_lib.lib().ssm_quantize_rows(F32, P, 8, P + 60, 8, far, 2, 8, None), o)
    need = _lib.lib().ssm_linear_i8_workspace(P, 256, far, 256, 2, 64, 256)
    refused(i8(W=far, sw=far, sx=far, y=P + 252, ws=far, nws=need), o)


def test_more_rows_than_a_launch_counts_are_refused():
    n = 1 << 24
    far = 1 << 45
    refused(_lib.lib().ssm_quantize_rows(F32, P, 8, far, 8, P, n, 8, None), b"too many rows")
    refused(i8(M=n, y=far), b"too many rows")
    refused(q8(N=n, ldy=1 << 20), b"row stride")
    refused(attention(B=n, H=1, G=1, L=1), b"too many heads")
    refused(step(B=n, H=1, G=1, V=16, K=1), b"too many heads")
