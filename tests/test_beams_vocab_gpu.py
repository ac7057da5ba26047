"""Beam search with the text decoder over lm heads of any number of words."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from strix_halo_maxx_b200.config import TEXT
from strix_halo_maxx_b200 import weights as wg
from strix_halo_maxx_b200.text import TextDecoder
from strix_halo_maxx_b200._lib import device_status
from test_beams_text_gpu import model, held_prefix, log_prob, DEV


@pytest.mark.parametrize("vocab,F,steps,keep", [(TEXT.vocab - 1, 4, 3, None), (TEXT.vocab - 7, 3, 3, 128), (77, 5, 4, None), (9, 2, 3, None)])
def test_answer_over_an_lm_head_of_odd_size(vocab, F, steps, keep):
    device_status(clear=True)
    W, Wt = model(vocab)
    emb, bos, ids, last = wg.text_inputs(TEXT, seed=5)
    ids = torch.from_numpy(ids)
    dec = TextDecoder(W, TEXT, device=DEV, kv8=True, keep=keep, beams=F, steps=steps)
    dec.encode(torch.from_numpy(emb).to(DEV), bos)
    kv = held_prefix(Wt, emb, bos, dec, keep)
    words, scores = dec.answer(ids.to(DEV), last)
    again, scores2 = dec.answer(ids.to(DEV), last)  # from the graph
    assert torch.equal(words, again) and torch.equal(scores, scores2)
    assert (words >= 0).all() and (words < vocab).all() and len({tuple(w.tolist()) for w in words}) == F and (scores.diff() <= 0).all()
    for b in range(F):  # as over a head of a multiple of 8 words
        lp, _ = log_prob(Wt, kv, ids, last, words[b])
        assert abs(float(scores[b]) - float(lp.sum())) < 0.1 * steps, b
    assert device_status(clear=True) == 0


def test_answer_with_fewer_words_than_beams():
    """The first choice has three words for eight beams; the others begin with the second."""
    W, Wt = model(3)
    emb, bos, ids, last = wg.text_inputs(TEXT, seed=5)
    ids = torch.from_numpy(ids)
    dec = TextDecoder(W, TEXT, device=DEV, kv8=True, beams=8, steps=2)
    dec.encode(torch.from_numpy(emb).to(DEV), bos)
    words, scores = dec.answer(ids.to(DEV), last)
    kv = held_prefix(Wt, emb, bos, dec, None)
    assert (words >= 0).all() and len({tuple(w.tolist()) for w in words}) == 8 and (scores.diff() <= 0).all()
    for b in range(8):
        assert abs(float(scores[b]) - float(log_prob(Wt, kv, ids, last, words[b])[0].sum())) < 0.2
    one = TextDecoder(W, TEXT, device=DEV, kv8=True, beams=8, steps=1)
    one.encode(torch.from_numpy(emb).to(DEV), bos)
    words, scores = one.answer(ids.to(DEV), last)
    assert sorted(words[:3, 0].tolist()) == [0, 1, 2] and (words[3:] == -1).all() and torch.isfinite(scores[:3]).all() and (scores[3:] == -float("inf")).all()
