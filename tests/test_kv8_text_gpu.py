"""The text decoder on the 8-bit KV cache (TextDecoder(kv8=True), with and without eviction of the image prefix) against the
CPU oracle with its cached keys and values quantised by oracle/kv8_ref.py."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from strix_halo_maxx_b200.config import TEXT
from strix_halo_maxx_b200 import weights as wg
from strix_halo_maxx_b200.text import TextDecoder
from strix_halo_maxx_b200._lib import device_status
from oracle import kv8_ref, text_ref as R
from oracle.tower_ref import layer_norm, linear
from helpers import assert_tokens_close, rel

DEV = "cuda"
NL = 2


def quantised(x):
    """[H, n, hd] fp32 -> the values its blocks of 64 tokens stand for, all written in one call."""
    out = torch.empty_like(x)
    for h in range(x.shape[0]):
        n = x.shape[1]
        codes, s = np.zeros(((n + 63) // 64 * 64, x.shape[2]), np.int8), np.zeros((n + 63) // 64, np.float32)
        kv8_ref.quantise(kv8_ref.bf16(x[h].numpy()), codes, s, 0)
        out[h] = torch.from_numpy(codes[:n].astype(np.float32) * s[np.arange(n) // 64][:, None])
    return out


def layers(x, W, pos, held, kept=None):
    """oracle.text_ref.text_layers over quantised keys and values: x [n, D] at positions pos ..; held: None (the prefix: no
    mask) or the layers' (k, v) [H, T, hd] before these tokens (causal).  Returns x, the layers' (k, v) and the prefix's
    attention weights [layers, H, n]."""
    H, hd, n = TEXT.heads, TEXT.head_dim, x.shape[0]
    cos, sin = R.rope_angles(TEXT, pos, n)
    kv, ws = [], []
    for i in range(NL):
        p = f"tblocks.{i}."
        h = layer_norm(x[None], W[p + "ln_w"], W[p + "ln_b"], TEXT.eps)
        q, k, v = (t.view(1, n, H, hd).transpose(1, 2) for t in linear(h, W[p + "qkv_w"], W[p + "qkv_b"]).split(H * hd, dim=-1))
        q, k = R.rope(q, cos, sin, TEXT.rot)[0], quantised(R.rope(k, cos, sin, TEXT.rot)[0])
        v = quantised(v[0])
        T0 = 0
        if held is not None:
            T0 = held[i][0].shape[1]
            k, v = torch.cat([held[i][0], k], 1), torch.cat([held[i][1], v], 1)
        s = q @ k.transpose(1, 2) / math.sqrt(hd)
        if held is not None:
            s = s.masked_fill(torch.arange(T0 + n)[None] > T0 + torch.arange(n)[:, None], -math.inf)
        a = torch.softmax(s, -1)
        ws.append(a.sum(1))
        kv.append((k, v))
        a = (a @ v).transpose(0, 1).reshape(1, n, H * hd)
        f = R.gelu_tanh(linear(h, W[p + "fc1_w"], W[p + "fc1_b"]))
        x = (linear(f, W[p + "fc2_w"], W[p + "fc2_b"]) + linear(a, W[p + "proj_w"], W[p + "proj_b"]) + x[None])[0]
    return x, kv, torch.stack(ws)


def logits_of(x, last, W):
    return linear(layer_norm(x[last][None], W["tpost_ln_w"], W["tpost_ln_b"], TEXT.eps), W["lm_small_w"], W["lm_small_b"])[0]


@pytest.mark.parametrize("keep", [None, 256])
def test_text_decoder_on_the_8_bit_cache(keep):
    device_status(clear=True)
    W = wg.text_weights(TEXT, seed=3, n_layers=NL, affine="random")
    emb, bos, ids, last = wg.text_inputs(TEXT, seed=5)
    Wt = {k: torch.as_tensor(np.asarray(v)).float() for k, v in W.items()}
    dec = TextDecoder(W, TEXT, device=DEV, kv8=True, keep=keep)
    got = dec.encode(torch.from_numpy(emb).to(DEV), bos)
    with torch.no_grad():
        x, kv, ws = layers(torch.cat([Wt["wte"][bos][None], torch.from_numpy(emb)]), Wt, 0, None)
    # a key or value is half a step of its block's scale off in both, but where bf16 inputs put it on another code: the
    # decoder's tolerance for bf16 rounding covers it
    assert_tokens_close(got.float().cpu(), x, what="prefix hidden states")
    if keep is not None:
        w = dec.attn_w[:, :, :TEXT.prefix].cpu()
        assert rel(w, ws) < 1e-2 and torch.allclose(w.sum(-1), torch.full((NL, TEXT.heads), float(TEXT.prefix)), rtol=1e-4)
        idx = dec.kept.cpu().long()
        for i in range(NL):
            for h in range(TEXT.heads):
                best = sorted(range(TEXT.prefix - 32), key=lambda j: (-float(w[i, h, j]), j))[:keep - 32]
                assert idx[i, h].tolist() == sorted(best) + list(range(TEXT.prefix - 32, TEXT.prefix))
        kv = [tuple(quantised(t.gather(1, idx[i][..., None].expand(-1, -1, TEXT.head_dim))) for t in kv[i]) for i in range(NL)]
    for r in range(2):  # the question twice: eagerly, then from its graph
        logits = dec.query(torch.from_numpy(ids).to(DEV), last).float().cpu()
        with torch.no_grad():
            y, _, _ = layers(Wt["wte"][torch.from_numpy(ids)], Wt, TEXT.prefix, kv)
        assert rel(logits, logits_of(y, last, Wt)) < 3e-2, r
    assert device_status(clear=True) == 0


@pytest.mark.parametrize("int8", [False, True])
def test_text_decoder_kv8_graphs_match_eager(int8):
    W = wg.text_weights(TEXT, seed=3, n_layers=NL, affine="random")
    emb, bos, ids, last = wg.text_inputs(TEXT, seed=5)
    dg, de = (TextDecoder(W, TEXT, device=DEV, graphs=g, int8=int8, kv8=True, keep=128) for g in (True, False))
    g = torch.Generator().manual_seed(2)
    for r in range(3):
        e = torch.from_numpy(emb).to(DEV) if r == 0 else torch.randn(TEXT.prefix - 1, TEXT.dim, generator=g).to(DEV)
        assert torch.equal(dg.encode(e, bos), de.encode(e, bos)), f"prefill {r}"
        assert torch.equal(dg.kept, de.kept)
        for k in range(2):
            q = torch.from_numpy(ids).to(DEV) if k == 0 else torch.randint(1, TEXT.vocab, (TEXT.q_len,), generator=g).to(DEV)
            assert torch.equal(dg.query(q, last), de.query(q, last)), f"question {k} after prefill {r}"
    assert dg._egraph is not None and dg._qgraph is not None


@pytest.mark.parametrize("keep", [None, 128])
def test_an_answer_does_not_depend_on_the_questions_before_it(keep):
    """The image prefix ends inside a block that the question's tokens share; a question with far larger keys before it (its
    embeddings scaled up) must leave no trace."""
    W = wg.text_weights(TEXT, seed=3, n_layers=NL, affine="random")
    W = {k: np.array(v) for k, v in W.items()}
    W["wte"][7] *= 50
    emb, bos, ids, last = wg.text_inputs(TEXT, seed=5)
    ids[ids == 7] = 8
    a, b = (TextDecoder(W, TEXT, device=DEV, kv8=True, keep=keep) for _ in range(2))
    for d in (a, b):
        d.encode(torch.from_numpy(emb).to(DEV), bos)
    for _ in range(2):
        a.query(torch.full((TEXT.q_len,), 7, device=DEV), TEXT.q_len - 1)
    assert torch.equal(a.query(torch.from_numpy(ids).to(DEV), last).clone(), b.query(torch.from_numpy(ids).to(DEV), last))


def test_keep_is_refused_where_it_makes_no_sense():
    W = wg.text_weights(TEXT, seed=3, n_layers=1)
    for kw in (dict(keep=128), dict(kv8=True, keep=100), dict(kv8=True, keep=0), dict(kv8=True, keep=768), dict(kv8=True, keep=64, keep_recent=65)):
        with pytest.raises(ValueError):
            TextDecoder(W, TEXT, device=DEV, **kw)
