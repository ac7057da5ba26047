"""Beam search with the int8 text decoder (TextDecoder(int8=True, kv8=True, beams=F)) against the oracle's int8 layers."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from strix_halo_maxx_b200.config import TEXT
from strix_halo_maxx_b200 import weights as wg
from strix_halo_maxx_b200.text import TextDecoder
from strix_halo_maxx_b200._lib import device_status
from oracle import text_ref as R
from oracle.tower_ref import layer_norm, linear
from test_beams_text_gpu import model, NL, DEV


@pytest.mark.parametrize("F", [1, 4])
def test_answer_of_the_int8_decoder(F):
    device_status(clear=True)
    W, Wt = model()
    emb, bos, ids, last = wg.text_inputs(TEXT, seed=5)
    last, steps = min(last, TEXT.q_len - 5), 5
    got = []
    for graphs in (True, False):
        dec = TextDecoder(W, TEXT, device=DEV, graphs=graphs, int8=True, kv8=True, beams=F, steps=steps)
        dec.encode(torch.from_numpy(emb).to(DEV), bos)
        got += [dec.answer(torch.from_numpy(ids).to(DEV), last) for _ in range(2)]
    words, scores = got[0]
    assert all(torch.equal(words, w) and torch.equal(scores, s) for w, s in got[1:])
    assert len({tuple(w.tolist()) for w in words}) == F and (scores.diff() <= 0).all() and device_status(clear=True) == 0
    i8 = R.quantize_weights(W, NL)
    _, (kc, vc) = R.encode(emb, bos, W, TEXT, n_layers=NL, i8=i8)
    for b in range(F):
        rows = torch.cat([torch.from_numpy(ids[:last + 1]), words[b]])[:-1]
        n = len(rows)
        with torch.no_grad():
            mask = torch.ones(n, TEXT.prefix + n, dtype=torch.bool).tril(TEXT.prefix)[None, None]
            x = R.text_layers(Wt["wte"][rows][None], W, TEXT, TEXT.prefix, *R.rope_angles(TEXT, TEXT.prefix, n), mask, [t.clone() for t in kc], [t.clone() for t in vc], NL, i8)
            z = linear(layer_norm(x[0, last:], Wt["tpost_ln_w"], Wt["tpost_ln_b"], TEXT.eps), Wt["lm_w"], Wt["lm_b"])
        want = torch.log_softmax(z, -1).gather(1, words[b][:, None]).sum()
        # the int8 decoder's logits are within 3e-2 of the oracle's norm, the 8-bit cache's within as much again; spread evenly over
        # the words, a chosen one's is off by three times that at most, and the words' sum by no more than all of them together
        assert abs(float(scores[b] - want)) < 3 * 6e-2 * float(z.square().mean().sqrt()) * steps, b
