"""Sizes next to 2^31, whose 32-bit indices would wrap inside the kernels, are refused. The pointers are
placeholders that are never followed: every call here ends at the host's checks."""
from ssmjs_amd import _lib

F32, BF16 = _lib.SSM_F32, _lib.SSM_BF16
INVALID = _lib.SSM_ERR_INVALID_ARG
FAR = [(i + 1) << 52 for i in range(8)]
TOP = (1 << 31) - 1


def refused(status, word):
    assert status == INVALID and word in _lib.lib().ssm_last_error(), _lib.lib().ssm_last_error()


def test_rows_to_integers():
    call = _lib.lib().ssm_quantize_rows
    for K in (TOP, (1 << 30) + 1):   # (the last pieces' index and the step past them)
        refused(call(F32, FAR[0], K, FAR[1], K, FAR[2], 1, K, None), b"too long")


def test_prompts():
    L = _lib.lib()
    for n in (TOP, (1 << 30) + 1):   # (the end of the last segment and chunk)
        need = L.ssm_linear_attention_workspace(BF16, 1, n, 1, 1, 1)
        refused(L.ssm_linear_attention(BF16, FAR[0], 1, FAR[1], 1, FAR[2], 1, FAR[3], 1.0, None, FAR[4], 1, 1, n, 1, 1, 1,
                                       1, None, None, FAR[5], need, None), b"too long")


def test_heads():
    L = _lib.lib()
    for H, G in ((TOP, 1), (TOP, TOP), ((1 << 30) + 1, 0), (1 << 29, (1 << 29) + 1)):   # (their sum, and rows ahead)
        refused(L.ssm_qk_norm_rope(BF16, FAR[0], 8 * H, FAR[1], 8 * G, None, None, FAR[2], FAR[3], 0, 1e-6, FAR[4], 8 * H,
                                   FAR[5], 8 * G, 1, H, G, 8, 8, None), b"too many heads")
