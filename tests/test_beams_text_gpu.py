"""Many answers about one image with the text decoder (TextDecoder(kv8=True, questions=Q / beams=F)) against the CPU oracle with its
cached keys and values quantised by oracle/kv8_ref.py."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from strix_halo_maxx_b200.config import TEXT
from strix_halo_maxx_b200 import weights as wg
from strix_halo_maxx_b200.text import TextDecoder
from strix_halo_maxx_b200._lib import device_status
from oracle.tower_ref import layer_norm, linear
from helpers import rel
from test_kv8_text_gpu import layers, logits_of, quantised, NL, DEV


def model(vocab=TEXT.vocab):
    W = {k: np.asarray(v) for k, v in wg.text_weights(TEXT, seed=3, n_layers=NL, affine="random").items()}
    rng = np.random.default_rng(9)
    W["lm_w"] = (rng.standard_normal((vocab, TEXT.dim)) * 0.05).astype(np.float32)
    W["lm_b"] = (rng.standard_normal(vocab) * 0.1).astype(np.float32)
    return W, {k: torch.as_tensor(v).float() for k, v in W.items()}


def questions(k, seed):
    """k questions of different lengths: ids [k, q_len], last [k]."""
    rng = np.random.default_rng(seed)
    ids = rng.integers(1, TEXT.vocab, (k, TEXT.q_len))
    return torch.from_numpy(ids), [int(x) for x in rng.integers(0, TEXT.q_len, k)]


def held_prefix(Wt, emb, bos, dec, keep):
    with torch.no_grad():
        _, kv, _ = layers(torch.cat([Wt["wte"][bos][None], torch.from_numpy(emb)]), Wt, 0, None)
    if keep is None:
        return kv
    idx = dec.kept.cpu().long()
    return [tuple(quantised(t.gather(1, idx[i][..., None].expand(-1, -1, TEXT.head_dim))) for t in kv[i]) for i in range(NL)]


@pytest.mark.parametrize("keep", [None, 256])
def test_query_many_answers_each_question(keep):
    device_status(clear=True)
    W, Wt = model()
    emb, bos, _, _ = wg.text_inputs(TEXT, seed=5)
    dec = TextDecoder(W, TEXT, device=DEV, kv8=True, keep=keep, questions=5)
    dec.encode(torch.from_numpy(emb).to(DEV), bos)
    kv = held_prefix(Wt, emb, bos, dec, keep)
    for r, k in enumerate((5, 3, 1)):  # eagerly, then from the graph with fewer questions
        ids, last = questions(k, 20 + r)
        got = dec.query_many(ids.to(DEV), last).float().cpu()
        assert got.shape == (k, TEXT.n_yn)
        for b in range(k):
            with torch.no_grad():
                y, _, _ = layers(Wt["wte"][ids[b, :last[b] + 1]], Wt, TEXT.prefix, kv)
            assert rel(got[b], logits_of(y, last[b], Wt)) < 3e-2, (r, b)
        # and as one question alone
        one = dec.query(ids[0].to(DEV), last[0]).float().cpu()
        assert rel(got[0], one) < 3e-2
    assert device_status(clear=True) == 0


@pytest.mark.parametrize("int8", [False, True])
def test_query_many_graph_matches_eager_whatever_came_before(int8):
    W, _ = model()
    emb, bos, ids1, last1 = wg.text_inputs(TEXT, seed=5)
    dg, de = (TextDecoder(W, TEXT, device=DEV, graphs=g, int8=int8, kv8=True, questions=40) for g in (True, False))
    for d in (dg, de):
        d.encode(torch.from_numpy(emb).to(DEV), bos)
    for r in range(4):
        ids, last = questions((40, 40, 7, 40)[r], r)
        if r == 2:
            dg.query(torch.from_numpy(ids1).to(DEV), last1)  # writes into the block that the prefix ends in
        a, b = (d.query_many(ids.to(DEV), torch.tensor(last, device=DEV)).clone() for d in (dg, de))
        assert torch.equal(a, b) and torch.isfinite(a).all(), r
    assert dg.many.graph is not None


def log_prob(Wt, kv, ids, last, words):
    """The oracle's log probability of each of an answer's words after the question."""
    rows = torch.cat([ids[:last + 1], words])
    with torch.no_grad():
        y, _, _ = layers(Wt["wte"][rows], Wt, TEXT.prefix, kv)
        z = linear(layer_norm(y[last:-1], Wt["tpost_ln_w"], Wt["tpost_ln_b"], TEXT.eps), Wt["lm_w"], Wt["lm_b"])
    return torch.log_softmax(z, -1).gather(1, words[:, None])[:, 0], torch.log_softmax(z, -1)


@pytest.mark.parametrize("F,steps,keep", [(4, 6, None), (1, 5, None), (6, 4, 256)])
def test_answer_is_a_beam_search(F, steps, keep):
    device_status(clear=True)
    W, Wt = model()
    emb, bos, ids, last = wg.text_inputs(TEXT, seed=5)
    ids = torch.from_numpy(ids)
    dec = TextDecoder(W, TEXT, device=DEV, kv8=True, keep=keep, beams=F, steps=steps)
    dec.encode(torch.from_numpy(emb).to(DEV), bos)
    kv = held_prefix(Wt, emb, bos, dec, keep)
    words, scores = dec.answer(ids.to(DEV), last)
    again, scores2 = dec.answer(ids.to(DEV), last)  # from the graph
    assert torch.equal(words, again) and torch.equal(scores, scores2)
    assert words.shape == (F, steps) and len({tuple(w.tolist()) for w in words}) == F and (scores.diff() <= 0).all()
    for b in range(F):
        lp, every = log_prob(Wt, kv, ids, last, words[b])
        # bf16 GEMMs: the decoder's logits are within 3e-2 of the oracle's, of which log probabilities of this head (|logit| < 4) see a tenth
        assert abs(float(scores[b]) - float(lp.sum())) < 0.1 * steps, b
        if F == 1:
            best = every.max(-1).values
            assert (best - lp < 0.2).all()
    eager = TextDecoder(W, TEXT, device=DEV, graphs=False, kv8=True, keep=keep, beams=F, steps=steps)
    eager.encode(torch.from_numpy(emb).to(DEV), bos)
    w3, s3 = eager.answer(ids.to(DEV), last)
    assert torch.equal(words, w3) and torch.equal(scores, s3)
    assert device_status(clear=True) == 0


def test_answer_ends_with_its_word():
    """With the best beam's second word as the end, that beam stops there and keeps its score, whatever follows."""
    W, _ = model()
    emb, bos, ids, last = wg.text_inputs(TEXT, seed=5)
    ids = torch.from_numpy(ids).to(DEV)
    dec = TextDecoder(W, TEXT, device=DEV, kv8=True, beams=3, steps=5)
    dec.encode(torch.from_numpy(emb).to(DEV), bos)
    free, _ = dec.answer(ids, last)
    eos = int(free[0, 1])
    words, scores = dec.answer(ids, last, eos=eos)
    ended = [(w == eos).nonzero()[0, 0].item() for w in words if (w == eos).any()]
    assert ended and torch.isfinite(scores).all()
    for w in words:
        at = (w == eos).nonzero()
        if len(at):
            assert (w[at[0, 0]:] == eos).all()
    assert torch.equal(dec.answer(ids, last)[0], free)  # without an end again


def test_many_answers_are_refused_where_they_make_no_sense():
    W, _ = model()
    small = {k: v for k, v in W.items() if not k.startswith("lm_") or k.startswith("lm_small")}
    for kw in (dict(questions=3), dict(kv8=True, questions=-1), dict(kv8=True, beams=4), dict(kv8=True, beams=65, steps=2), dict(kv8=True, steps=3), dict(beams=2, steps=2)):
        with pytest.raises(ValueError):
            TextDecoder(W, TEXT, device=DEV, **kw)
    with pytest.raises(ValueError):
        TextDecoder(small, TEXT, device=DEV, kv8=True, beams=2, steps=2)
    dec = TextDecoder(W, TEXT, device=DEV, kv8=True, questions=2)
    ids, last = questions(3, 1)
    for call in (lambda: dec.query_many(ids.to(DEV), last), lambda: dec.query_many(ids[:2].to(DEV), last[:1]), lambda: dec.query_many(ids[:2].to(DEV), [0, TEXT.q_len]),
                 lambda: dec.query_many(ids[:2, :8].to(DEV), last[:2]), lambda: dec.answer(ids[0].to(DEV), 3)):
        with pytest.raises(ValueError):
            call()


def test_query_many_cuts_off_last_on_the_device():
    W, _ = model()
    emb, bos, _, _ = wg.text_inputs(TEXT, seed=5)
    dec = TextDecoder(W, TEXT, device=DEV, kv8=True, questions=2)
    dec.encode(torch.from_numpy(emb).to(DEV), bos)
    ids, _ = questions(2, 1)
    want = dec.query_many(ids.to(DEV), [0, TEXT.q_len - 1]).clone()
    got = dec.query_many(ids.to(DEV), torch.tensor([-5, TEXT.q_len + 1000], device=DEV))
    assert torch.equal(got, want)
