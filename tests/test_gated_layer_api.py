"""What the operators of a gated-recurrence model refuse, and what their workspace queries say. The pointers are
placeholders that are never followed: every call here ends at the host's checks."""
import inspect

import pytest

from ssmjs_amd import _lib

F32, BF16 = _lib.SSM_F32, _lib.SSM_BF16
OK, INVALID, UNSUPPORTED = _lib.SSM_OK, _lib.SSM_ERR_INVALID_ARG, _lib.SSM_ERR_UNSUPPORTED
FAR = [(i + 1) << 40 for i in range(40)]   # places apart
NAN, INF = float("nan"), float("inf")


def caller(name, names, values):
    """A call with every operand at a place of its own, but for the changes."""
    where = dict(zip([n for n in names if n not in values], FAR))

    def call(**change):
        c = where | values | change
        assert set(c) == set(names)
        return getattr(_lib.lib(), name)(*(c[n] for n in names), None)
    return call


# bf16: rows of 100 elements, 200 bytes, two sequences of eight
forward = caller("ssm_gated_recurrence", ["dtype", "x", "ldx", "r", "ldr", "i", "ldi", "lam", "c", "lengths", "pad", "y", "ldy", "B", "L", "D",
                                          "h0", "hT", "states", "ws", "nws"],
                 dict(dtype=BF16, ldx=100, ldr=200, ldi=200, c=8.0, pad=0, ldy=100, B=2, L=8, D=100, ws=None, nws=0))
backward = caller("ssm_gated_recurrence_backward", ["dtype", "dy", "lddy", "x", "ldx", "r", "ldr", "i", "ldi", "lam", "c", "lengths", "pad",
                                                    "states", "dhT", "dx", "lddx", "dr", "lddr", "di", "lddi", "dlam", "dh0",
                                                    "B", "L", "D", "ws", "nws"],
                  dict(dtype=BF16, lddy=100, ldx=100, ldr=200, ldi=200, c=8.0, pad=0, lddx=100, lddr=100, lddi=100, B=2, L=8,
                       D=100, nws=1 << 30))
step = caller("ssm_gated_recurrence_step", ["dtype", "x", "ldx", "r", "ldr", "i", "ldi", "lam", "c", "y", "ldy", "h", "B", "D"],
              dict(dtype=BF16, ldx=100, ldr=200, ldi=200, c=8.0, ldy=100, B=2, D=100))
norm = caller("ssm_block_norm", ["dtype", "x", "ldx", "y", "ldy", "z", "ldz", "post", "scale", "pre", "eps", "x1", "ldx1", "n", "ldn", "T",
                                 "D"], dict(dtype=BF16, ldx=100, ldy=100, ldz=100, eps=1e-6, ldx1=100, ldn=100, T=4, D=100))
norm_back = caller("ssm_block_norm_backward", ["dtype", "dx1", "lddx1", "dn", "lddn", "x", "ldx", "y", "ldy", "z", "ldz", "post",
                                               "scale", "pre", "eps", "dx", "lddx", "dy", "lddy", "dz", "lddz", "dpost",
                                               "dscale", "dpre", "T", "D", "ws", "nws"],
                   dict(dtype=BF16, lddx1=100, lddn=100, ldx=100, ldy=100, ldz=100, eps=1e-6, lddx=100, lddy=100, lddz=100,
                        T=4, D=100, nws=1 << 30))
logp = caller("ssm_token_logprobs", ["dtype", "x", "ldx", "ids", "M", "N", "k", "logp", "entropy", "stats", "top", "toplp", "ws", "nws"],
              dict(dtype=BF16, ldx=100, M=4, N=100, k=3, ws=None, nws=0))
logp_back = caller("ssm_token_logprobs_backward", ["dtype", "x", "ldx", "ids", "stats", "entropy", "dlogp", "dentropy", "dx",
                                                   "lddx", "M", "N"], dict(dtype=BF16, ldx=100, lddx=100, M=4, N=100))


def said(status, want, call):
    assert status == want, (inspect.getsource(call)[:40], _lib.lib().ssm_last_error())


@pytest.mark.parametrize("change,status", [
    (dict(B=0), OK), (dict(dtype=2), INVALID), (dict(B=-1), INVALID), (dict(L=-1), INVALID), (dict(D=0), INVALID),
    (dict(c=-1.0), INVALID), (dict(c=NAN), INVALID), (dict(c=INF), INVALID), (dict(x=None), INVALID),
    (dict(r=None), INVALID), (dict(i=None), INVALID), (dict(lam=None), INVALID), (dict(y=None), INVALID),
    (dict(lam=None, L=0), INVALID), (dict(ldx=99), INVALID), (dict(ldr=99), INVALID), (dict(ldi=99), INVALID),
    (dict(ldy=99), INVALID), (dict(ldx=1 << 20), INVALID), (dict(L=(1 << 30) + 1, B=1), INVALID),
    (dict(L=(1 << 31) - 1, B=1), INVALID), (dict(B=1 << 20, D=1 << 19, ldx=1 << 19, ldr=1 << 19, ldi=1 << 19, ldy=1 << 19), INVALID),
])
def test_recurrence(change, status):
    said(forward(**change), status, forward)


@pytest.mark.parametrize("change,status", [
    (dict(dtype=7), INVALID), (dict(B=0), INVALID), (dict(L=-1), INVALID), (dict(D=0), INVALID), (dict(c=-1.0), INVALID),
    (dict(dy=None), INVALID), (dict(x=None), INVALID), (dict(states=None), INVALID), (dict(dx=None), INVALID),
    (dict(dr=None), INVALID), (dict(di=None), INVALID), (dict(dlam=None), INVALID), (dict(lam=None), INVALID),
    (dict(lddy=99), INVALID), (dict(lddx=99), INVALID), (dict(lddr=99), INVALID), (dict(lddi=99), INVALID),
    (dict(ldx=1 << 20), INVALID), (dict(L=(1 << 31) - 1, B=1), INVALID), (dict(ws=None), INVALID), (dict(nws=4), INVALID),
    (dict(ws=FAR[30] + 8), INVALID),
])
def test_recurrence_backward(change, status):
    said(backward(**change), status, backward)


@pytest.mark.parametrize("change,status", [
    (dict(B=0), OK), (dict(dtype=-1), INVALID), (dict(B=-1), INVALID), (dict(D=0), INVALID), (dict(c=NAN), INVALID),
    (dict(h=None), INVALID), (dict(x=None), INVALID), (dict(y=None), INVALID), (dict(ldx=99), INVALID), (dict(ldy=99), INVALID),
    (dict(B=1 << 20, D=1 << 20, ldx=1 << 20, ldr=1 << 20, ldi=1 << 20, ldy=1 << 20), INVALID),
])
def test_recurrence_step(change, status):
    said(step(**change), status, step)


@pytest.mark.parametrize("change,status", [
    (dict(T=0), OK), (dict(dtype=3), INVALID), (dict(T=-1), INVALID), (dict(D=0), INVALID), (dict(eps=-1.0), INVALID),
    (dict(eps=NAN), INVALID), (dict(D=16385, ldx=20000, ldy=20000, ldz=20000, ldx1=20000, ldn=20000), UNSUPPORTED),
    (dict(x=None), INVALID), (dict(y=None), INVALID), (dict(x1=None), INVALID), (dict(n=None), INVALID), (dict(ldx=99), INVALID),
    (dict(ldz=99), INVALID), (dict(ldn=99), INVALID), (dict(T=1 << 23), INVALID),
])
def test_norm(change, status):
    said(norm(**change), status, norm)


@pytest.mark.parametrize("change,status", [
    (dict(T=0), INVALID), (dict(dtype=3), INVALID), (dict(D=0), INVALID), (dict(eps=-1.0), INVALID), (dict(D=16385), UNSUPPORTED),
    (dict(dn=None), INVALID), (dict(x=None), INVALID), (dict(dx=None), INVALID), (dict(dy=None), INVALID), (dict(dz=None), INVALID),
    (dict(lddx1=99), INVALID), (dict(lddz=99), INVALID), (dict(T=1 << 23), INVALID), (dict(ws=None), INVALID), (dict(nws=4), INVALID),
    (dict(ws=FAR[30] + 4), INVALID),
])
def test_norm_backward(change, status):
    said(norm_back(**change), status, norm_back)


@pytest.mark.parametrize("change,status", [
    (dict(M=0), OK), (dict(dtype=3), INVALID), (dict(M=-1), INVALID), (dict(N=0), INVALID), (dict(k=-1), INVALID),
    (dict(k=101), INVALID), (dict(k=65), UNSUPPORTED), (dict(x=None), INVALID), (dict(ids=None), INVALID), (dict(top=None), INVALID),
    (dict(toplp=None), INVALID), (dict(ldx=99), INVALID), (dict(N=(1 << 30) + 1, ldx=1 << 31, M=1), INVALID),
    (dict(M=1 << 25), INVALID), (dict(stats=FAR[20] + 4), INVALID), (dict(M=1, N=100000, ldx=100000), INVALID),
])
def test_logprobs(change, status):
    said(logp(**change), status, logp)


@pytest.mark.parametrize("change,status", [
    (dict(M=0), OK), (dict(dtype=3), INVALID), (dict(M=-1), INVALID), (dict(N=0), INVALID), (dict(x=None), INVALID),
    (dict(stats=None), INVALID), (dict(dx=None), INVALID), (dict(ids=None), INVALID), (dict(entropy=None), INVALID),
    (dict(ldx=99), INVALID), (dict(lddx=99), INVALID), (dict(stats=FAR[20] + 4), INVALID), (dict(M=1 << 25), INVALID),
])
def test_logprobs_backward(change, status):
    said(logp_back(**change), status, logp_back)


def test_workspaces_agree_with_the_launches():
    L = _lib.lib()
    assert L.ssm_gated_recurrence_workspace(8, 4096, 2048) >= 0
    assert L.ssm_gated_recurrence_workspace(0, 8, 64) == L.ssm_gated_recurrence_workspace(2, 0, 64) == 0
    assert L.ssm_gated_recurrence_workspace(4, 100, 64) == 0   # a block a sequence
    for B, n, D in ((1, 5000, 64), (3, 70000, 515)):
        need = L.ssm_gated_recurrence_workspace(B, n, D)
        assert need > 0
        big = dict(B=B, L=n, D=D, ldx=D, ldr=D, ldi=D)
        for bad in (dict(), dict(ws=FAR[30], nws=need - 1), dict(ws=FAR[30] + 8, nws=need)):
            assert forward(**big, ldy=D, **bad) == INVALID
            assert f"{need} bytes".encode() in L.ssm_last_error() or b"16-byte aligned" in L.ssm_last_error()
        need = L.ssm_gated_recurrence_backward_workspace(B, n, D)
        assert need >= 4 * B * D
        assert backward(**big | dict(lddy=D, lddx=D, lddr=D, lddi=D), nws=need - 1) == INVALID
        assert f"{need} bytes".encode() in L.ssm_last_error()
    assert L.ssm_block_norm_backward_workspace(0, 8) == L.ssm_block_norm_backward_workspace(8, 0) == 0
    need = L.ssm_block_norm_backward_workspace(4, 100)
    assert norm_back(nws=need - 1) == INVALID and f"{need} bytes".encode() in L.ssm_last_error()
    assert L.ssm_token_logprobs_workspace(4096, 128000, 20) == 0
    need = L.ssm_token_logprobs_workspace(1, 100000, 20)
    assert need > 0
    assert logp(M=1, N=100000, ldx=100000, k=20, ws=FAR[30], nws=need - 1) == INVALID
    assert f"{need} bytes".encode() in L.ssm_last_error()


@pytest.mark.parametrize("B,L,D,cut", [
    (8, 4096, 2048, False), (4, 2048, 2048, False), (256, 1000, 1024, False), (64, 16, 1024, False), (1, 256, 64, False),
    (1, 32768, 1024, True), (1, 5000, 516, True), (2, 4000, 392, True), (3, 3000, 392, True)])
def test_room_for_segments(B, L, D, cut):
    """A forward call whose sequences are cut keeps a pair of floats for each block of 256 steps and one more, of every
    channel and sequence, to whole 16 bytes; one whose sequences are walked whole keeps nothing."""
    need = _lib.lib().ssm_gated_recurrence_workspace(B, L, D)
    assert need == ((B * (-(-L // 256) + 1) * D * 8 + 15) // 16 * 16 if cut else 0)


# What each operand covers, of the calls above: bytes from its first to past its last
ROWS, WIDE = 15 * 200 + 200, 15 * 400 + 200
SIZES = {
    forward: (dict(x=ROWS, r=WIDE, i=WIDE, lam=400, lengths=8, h0=800), dict(y=ROWS, hT=800, states=800)),
    backward: (dict(dy=ROWS, x=ROWS, r=WIDE, i=WIDE, lam=400, lengths=8, states=800, dhT=800),
               dict(dx=ROWS, dr=ROWS, di=ROWS, dlam=400, dh0=800)),
    step: (dict(x=400, r=600, i=600, lam=400), dict(y=400, h=800)),
    norm: (dict(x=800, y=800, z=800, post=400, scale=400, pre=400), dict(x1=800, n=800)),
    norm_back: (dict(dx1=800, dn=800, x=800, y=800, z=800, post=400, scale=400, pre=400),
                dict(dx=800, dy=800, dz=800, dpost=400, dscale=400, dpre=400)),
    logp: (dict(x=800, ids=16), dict(logp=16, entropy=16, stats=32, top=48, toplp=48)),
    logp_back: (dict(x=800, ids=16, stats=32, entropy=16, dlogp=16, dentropy=16), dict(dx=800)),
}
NAMES = {forward: "recurrence", backward: "gradients", step: "step", norm: "norms", norm_back: "norms' gradients",
         logp: "log probabilities", logp_back: "their gradient"}


@pytest.mark.parametrize("call,out", [(c, o) for c, (_, outs) in SIZES.items() for o in outs],
                         ids=[f"{NAMES[c]}-{o}" for c, (_, outs) in SIZES.items() for o in outs])
def test_outputs_are_apart(call, out):
    """An output that reaches into any other operand, by its first or its last bytes, is refused."""
    ins, outs = SIZES[call]
    at, size = FAR[30], outs[out]
    for other, wide in (ins | {k: v for k, v in outs.items() if k != out}).items():
        for place in (at - size + 8, at + wide // 16 * 8, at + wide - 8):
            assert call(**{other: at, out: place}) == INVALID, (other, out, place - at)
            assert b"overlap" in _lib.lib().ssm_last_error(), _lib.lib().ssm_last_error()


@pytest.mark.parametrize("call", [backward, norm_back], ids=lambda c: NAMES[c])
def test_workspaces_are_apart(call):
    ins, outs = SIZES[call]
    for other in ins | outs:
        assert call(**{other: FAR[30] + 16, "ws": FAR[30]}) == INVALID, other
        assert b"overlap" in _lib.lib().ssm_last_error(), other


def test_python_checks():
    torch = pytest.importorskip("torch")
    from ssmjs_amd import kernels as k
    z = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt)   # noqa: E731
    x, lam = z(2, 4, 8), z(8)
    for call in (lambda: k.gated_recurrence(x, x, x, lam), lambda: k.gated_recurrence_step(x[:, 0], x[:, 0], x[:, 0], lam, z(2, 8)),
                 lambda: k.block_norm(x, x), lambda: k.token_logprobs(z(2, 9), z(2, dt=torch.int32)),
                 lambda: k.gated_recurrence_backward(x, x, x, x, lam, z(2, 1, 8)), lambda: k.block_norm_backward(x, x, x, x),
                 lambda: k.token_logprobs_backward(z(2, 9), None, z(2, 2))):
        with pytest.raises(ValueError, match="HIP device"):
            call()
    with pytest.raises(TypeError):
        k.gated_recurrence(z(1, 4, 8, dt=torch.float16), x, x, lam)
    with pytest.raises(ValueError):
        k.gated_recurrence(z(4, 8), z(4, 8), z(4, 8), lam)
    with pytest.raises(TypeError):
        k.token_logprobs(z(2, 9, dt=torch.float64))
    with pytest.raises(ValueError, match="one distance"):
        k._steps("x", z(4, 6, 8)[:, :4])
    with pytest.raises(ValueError, match="contiguous"):
        k._steps("x", z(4, 6, 8).transpose(1, 2))
    assert k._steps("x", z(2, 4, 24)[..., 8:16]) == 24 and k._steps("x", z(3, 1, 24)[..., :8]) == 24
    assert k._steps("x", z(1, 1, 24)[..., :8]) == 8
    assert k._flat("x", z(5, 24)[:, :8]) == 24 and k._flat("x", z(2, 3, 4, 8)) == 8
