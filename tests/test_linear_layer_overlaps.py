"""Outputs and states of a linear-attention layer's operators that share memory with what else a call reads
or writes are refused. The pointers are placeholders that are never followed: every call here ends at the
host's checks."""
import pytest

from ssmjs_amd import _lib

F32, BF16 = _lib.SSM_F32, _lib.SSM_BF16
INVALID = _lib.SSM_ERR_INVALID_ARG
FAR = [(i + 1) << 32 for i in range(16)]   # places apart


def refused(status):
    assert status == INVALID and b"overlap" in _lib.lib().ssm_last_error(), _lib.lib().ssm_last_error()


# B 2, L 8, H 4, G 2, K = V = 128, bf16: rows of 1024 bytes of q and y, 512 of k and v; states of 65536 bytes a
# head, 524288 in all
ROWS, KROWS, STATES = 16 * 1024, 16 * 512, 8 * 65536


def attention(**at):
    c = dict(q=FAR[0], k=FAR[1], v=FAR[2], g=FAR[3], lengths=FAR[4], y=FAR[5], h0=FAR[6], hT=FAR[7], L=8, ws=None, nws=0) | at
    return _lib.lib().ssm_linear_attention(
        BF16, c["q"], 512, c["k"], 256, c["v"], 256, c["g"], 1.0, c["lengths"], c["y"], 512, 2, c["L"], 4, 2,
        128, 128, c["h0"], c["hT"], c["ws"], c["nws"], None)


@pytest.mark.parametrize("name,size", [("q", ROWS), ("k", KROWS), ("v", KROWS), ("g", 16), ("lengths", 8), ("y", ROWS)])
def test_final_states_apart_from_the_inputs_and_outputs(name, size):
    at = FAR[9] + 16 * STATES
    for hT in (at - STATES + 4, at, at + size - 4):
        refused(attention(**{name: at, "hT": hT}))


def test_final_states_are_the_entering_ones_or_apart():
    for d in (4, -4, STATES - 4, 4 - STATES, 65536):
        refused(attention(h0=FAR[6], hT=FAR[6] + d))


@pytest.mark.parametrize("name,size", [("g", 16), ("lengths", 8), ("h0", STATES)])
def test_outputs_apart_from_the_decays_lengths_and_states(name, size):
    at = FAR[9] + STATES
    for y in (at - ROWS + 2, at, at + size - 2):
        refused(attention(**{name: at, "y": y}))


@pytest.mark.parametrize("name,size", [("q", 1), ("k", 1), ("v", 1), ("g", 1), ("lengths", 1), ("y", 1), ("h0", 1), ("hT", 1)])
def test_the_workspace_is_apart(name, size):
    L = 8192
    need = _lib.lib().ssm_linear_attention_workspace(BF16, 2, L, 4, 128, 128)
    assert need > 0
    at = FAR[9]
    refused(attention(**{name: at + need - 16}, L=L, ws=at, nws=need))


def step(**at):
    c = dict(q=FAR[0], k=FAR[1], v=FAR[2], g=FAR[3], y=FAR[5], h=FAR[6]) | at
    return _lib.lib().ssm_linear_attention_step(
        BF16, c["q"], 512, c["k"], 256, c["v"], 256, c["g"], 1.0, c["y"], 512, c["h"], 2, 4, 2, 128, 128, None)


@pytest.mark.parametrize("name,size", [("q", 2048), ("k", 1024), ("v", 1024), ("g", 16), ("y", 2048)])
def test_a_steps_state_is_apart(name, size):
    at = FAR[9] + STATES
    for h in (at - STATES + 4, at, at + size - 2):
        refused(step(**{name: at, "h": h}))


def test_a_steps_output_is_apart_from_the_decays():
    refused(step(g=FAR[5] + 2044))
    refused(step(y=FAR[3] + 14))


def products(**at):
    """Both forms: M 3, N 64, K 256, W of 16384 bytes, y of 768."""
    c = dict(x=FAR[0], sx=FAR[1], W=FAR[2], sw=FAR[3], bias=FAR[4], y=FAR[5], ws=FAR[6], nws=1 << 20) | at
    L = _lib.lib()
    yield "i8", L.ssm_linear_i8(c["x"], 256, c["sx"], c["W"], 256, c["sw"], c["bias"], F32, c["y"], 64, 3, 64, 256,
                                0.0, c["ws"], c["nws"], None)
    yield "q8", L.ssm_linear_q8(F32, c["x"], 256, c["W"], 256, c["sw"], c["bias"], F32, c["y"], 64, 3, 64, 256, 0.0,
                                c["ws"], c["nws"], None)


@pytest.mark.parametrize("name,size", [("W", 16384), ("sw", 256), ("bias", 256), ("sx", 12)])
def test_a_products_output_is_apart_from_the_weights_and_scales(name, size):
    at = FAR[9]
    for y in (at - 764, at, at + size - 4):
        for form, status in products(**{name: at, "y": y}):
            if not (form == "q8" and name == "sx"):
                refused(status)


@pytest.mark.parametrize("name", ["x", "W", "sw", "bias", "sx", "y"])
def test_a_products_workspace_is_apart(name):
    L = _lib.lib()
    for form, need in (("i8", L.ssm_linear_i8_workspace(FAR[0], 256, FAR[2], 256, 3, 64, 256)),
                       ("q8", L.ssm_linear_q8_workspace(FAR[2], 256, 3, 64, 256))):
        assert need > 0
        for f, status in products(**{name: FAR[6] + need - 16}):
            if f == form and not (f == "q8" and name == "sx"):
                refused(status)


def test_operands_that_reach_into_each_others_rows():
    """Column ranges of one buffer, and blocks in the gaps of far rows, that are a little too long."""
    L = _lib.lib()
    # W and y as column ranges of rows of 512 bytes
    refused(L.ssm_linear_i8(FAR[0], 256, FAR[1], FAR[2], 512, FAR[3], None, F32, FAR[2] + 252, 128, 3, 64, 256, 0.0, FAR[6],
                            1 << 20, None))
    # a state in the gap between two sequences' rows of q that reaches the second, or begins in the first
    for at in (FAR[0] + (1 << 21) - STATES + 4, FAR[0] + 2044):
        refused(L.ssm_linear_attention_step(F32, FAR[0], 1 << 19, FAR[1], 256, FAR[2], 256, FAR[3], 1.0, FAR[5], 512, at,
                                            2, 4, 2, 128, 128, None))


def test_quantised_scales_are_apart():
    call = _lib.lib().ssm_quantize_rows
    # x (3, 64) fp32: 768 bytes; q 192 bytes
    refused(call(F32, FAR[0], 64, FAR[1], 64, FAR[0] + 764, 3, 64, None))
    refused(call(F32, FAR[0], 64, FAR[1], 64, FAR[0] - 8, 3, 64, None))
    refused(call(F32, FAR[0], 64, FAR[1], 64, FAR[1] + 188, 3, 64, None))
    refused(call(F32, FAR[0], 64, FAR[1], 64, FAR[1] - 8, 3, 64, None))


@pytest.mark.parametrize("name,size", [("wq", 256), ("wk", 256), ("pos", 8), ("freq", 256)])
@pytest.mark.parametrize("out", ["qo", "ko"])
def test_heads_outputs_are_apart_from_the_weights_and_positions(name, size, out):
    """T 2, H 4, G 2, D 64, fp32: 2048 bytes of q, 1024 of k."""
    c = dict(q=FAR[0], k=FAR[1], wq=FAR[2], wk=FAR[3], pos=FAR[4], freq=FAR[5], qo=FAR[6], ko=FAR[7])
    c[name] = FAR[9]
    for at in (FAR[9], FAR[9] + size - 4, FAR[9] - (2048 if out == "qo" else 1024) + 4):
        c[out] = at
        refused(_lib.lib().ssm_qk_norm_rope(F32, c["q"], 256, c["k"], 128, c["wq"], c["wk"], c["pos"], c["freq"], 0, 1e-6,
                                            c["qo"], 256, c["ko"], 128, 2, 4, 2, 64, 64, None))
