"""ssm_score: log probabilities, entropies and likeliest tokens of a forward, against those that its own logits give in
64 bits (bounds of the kernel on those logits, as in its own tests)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_token_logprobs import close, reference  # noqa: E402

pytestmark = pytest.mark.gpu

CFG = {"vocabSize": 517, "dModel": 64, "numLayers": 2, "dState": 16, "dConv": 4, "expand": 2, "nHeads": 2,
       "layers": [{"type": "mamba1"}, {"type": "mamba2"}]}


@pytest.fixture(scope="module")
def model():
    from ssmjs_amd import model as M
    device = M.init_webgpu()["device"]
    m = M.HybridMambaModel(device, CFG, seed=5)
    yield m
    m.destroy()
    device.destroy()


@pytest.mark.parametrize("B,L,k", [(1, 1, 3), (2, 7, 0), (1, 30, 64), (3, 50, 5), (2, 300, 2)])
def test_score_is_what_the_logits_say(model, B, L, k):
    print(f"[case] score {B} {L} {k}", flush=True)
    ids = np.random.default_rng(L).integers(0, CFG["vocabSize"], (B, L)).astype(np.uint32)
    lg = torch.from_numpy(model.forward(ids, B, L)["logits"].reshape(B * L, -1)).cuda()
    got = model.score(ids, B, L, top=k)
    nxt = np.full((B, L), -1, np.int32)
    nxt[:, :-1] = ids[:, 1:]
    ref = reference(lg, torch.from_numpy(nxt.reshape(-1)).cuda(), max(k, 1))
    dev = lambda a: torch.from_numpy(a.reshape(B * L, -1)).cuda()   # noqa: E731
    close(dev(got["logprobs"])[:, 0], ref["logp"], "logp")
    close(dev(got["entropies"])[:, 0], ref["H"], "entropy")
    assert (got["logprobs"][:, -1] == 0).all()
    assert got["topIds"].shape == (B, L, k)
    if k:
        assert torch.equal(dev(got["topIds"].astype(np.int64)), ref["top"])
        close(dev(got["topLogprobs"]), ref["toplp"], "top logp")


def test_perplexity(model):
    """exp of the mean of what score gives is evaluate's perplexity."""
    from ssmjs_amd import model as M

    class Words:
        def encode(self, text):
            return [ord(c) % CFG["vocabSize"] for c in text]

    text = "the log probabilities of a text, token by token " * 3
    ids = np.array([Words().encode(text)], np.uint32)
    lp = model.score(ids, 1, ids.size)["logprobs"][0, :-1].astype(np.float64)
    ppl = M.MambaTrainer(model, Words()).evaluate(text)
    assert abs(np.exp(-lp.mean()) / ppl - 1) <= 1e-5


def test_refusals(model):
    from ssmjs_amd import _lib
    n = model.native
    with pytest.raises(_lib.SsmError, match="at most 64"):
        n.score(np.zeros((1, 4)), k=65)
    with pytest.raises(_lib.SsmError, match="out of range"):
        n.score(np.full((1, 4), CFG["vocabSize"]))
    a = n.score(np.zeros((1, 4)))   # (and goes on)
    assert np.isfinite(a[0]).all()
    assert n.score(np.zeros((0, 4)))[0].shape == (0, 4)
