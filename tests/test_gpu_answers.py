"""Answers drawn with cached keys and values (sheaf_b200/answers.py) against
the oracle's forward of prompt and answer as a whole, in float64: the log
probability of every drawn token, greedy tokens, and the gradient of the last
step's log probabilities in its logits."""
import numpy as np
import pytest

from oracle import dtype as odt
from oracle import models
from tests.parity import TOL_BF16, TOL_F32

pytestmark = pytest.mark.gpu

CFG = models.GPTConfig(n_layer=2, n_head=2, n_embd=128, block_size=64, vocab_size=65, batch=1, seq=64)


def _answers(kind):
    from sheaf_b200.answers import Answers
    from sheaf_b200.runtime import ELEM_BF16, ELEM_F32, Session

    s = Session(0)
    leaves, _, _ = models.gpt_inputs(CFG)
    # larger weights than at initialisation: distributions that tell tokens apart
    leaves = [a * np.float32(4) if a.ndim == 2 else a for a in leaves]
    if kind == "bf16":
        leaves = [odt.round_bf16(a) for a in leaves]
    elem = ELEM_BF16 if kind == "bf16" else ELEM_F32
    return s, leaves, Answers(s, [s.upload(a, elem) for a in leaves], n_layer=CFG.n_layer, n_head=CFG.n_head,
                              n_embd=CFG.n_embd, block_size=CFG.block_size, vocab_size=CFG.vocab_size, page_rows=8)


def _logp(leaves, ids, temperature):
    z = models.gpt_forward_logits(leaves, ids, CFG) / temperature
    z = z - z.max(-1, keepdims=True)
    return z - np.log(np.exp(z).sum(-1, keepdims=True))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("T,n,n_new,k,temperature", [(1, 3, 5, 32, 1.0), (21, 5, 12, 8, 0.8), (40, 1, 25, 1, 1.0),
                                                     (17, 70, 3, 32, 1.3)])
def test_answers(kind, T, n, n_new, k, temperature, cuda):
    s, leaves, a = _answers(kind)
    prompt = np.random.default_rng(T).integers(0, CFG.vocab_size, T)
    tokens, logp = a.draw(prompt, n, n_new, k=k, temperature=temperature, seed=3)
    ids = np.concatenate([np.repeat(prompt[None], n, 0), tokens], 1).astype(np.float32)
    want = _logp(leaves, ids[:, :-1], temperature)[:, T - 1:]
    got = np.take_along_axis(want, tokens[..., None].astype(int), -1)[..., 0]
    tol = TOL_F32 * 10 if kind == "f32" else TOL_BF16
    assert np.abs(logp - got).max() <= tol * (1 + np.abs(got).max())
    best = want.max(-1)
    if k == 1:  # greedy: the likeliest, or one that rounding cannot tell from it
        assert (best - got <= tol * (1 + np.abs(best))).all()
    # every token is among the k likeliest, to that accuracy
    kth = np.sort(want, -1)[..., -min(k, CFG.vocab_size)]
    assert (got >= kth - 2 * tol * (1 + np.abs(kth))).all()


def test_scores_and_their_gradient(cuda):
    s, leaves, a = _answers("f32")
    tokens, logp = a.draw([1, 2, 3], 4, 2, k=8)
    t = s.upload(tokens[:, 1].astype(np.float32))
    scores = s.token_logprobs(a.logits, CFG.vocab_size, targets=t)
    assert np.abs(scores["logp"].to_host() - logp[:, 1]).max() <= 1e-5
    g = np.array([1.0, -0.5, 2.0, 0.0], np.float32)
    dx = s.token_logprobs_vjp(a.logits, CFG.vocab_size, scores, targets=t, dlogp=s.upload(g)).to_host()
    z = a.logits.to_host()[:, :CFG.vocab_size].astype(np.float64)
    p = np.exp(z - z.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    want = g[:, None] * (np.eye(CFG.vocab_size)[tokens[:, 1]] - p)
    assert np.abs(dx[:, :CFG.vocab_size] - want).max() <= 1e-5


def test_answers_refuses_what_does_not_fit(cuda):
    _, _, a = _answers("f32")
    with pytest.raises(ValueError):
        a.draw(np.zeros(60), 2, 6)
    with pytest.raises(ValueError):
        a.draw([], 2, 2)


def test_session_ops_raise(cuda):
    from sheaf_b200.runtime import ELEM_F32, Session, SheafB200Error

    s = Session(0)
    x = s.upload(np.zeros((2, 8)))
    with pytest.raises(SheafB200Error):
        s.token_logprobs(x, 9)
    with pytest.raises(SheafB200Error):
        s.token_logprobs(x, 8, temperature=0.0)
    cache = s.kv_cache(2, 8, 1, 32, ELEM_F32)
    with pytest.raises(SheafB200Error):
        s.prefix_attention(cache, s.upload(np.zeros((2, 32))), s.upload(np.zeros(2), 0x10000020), scale=-1.0)
