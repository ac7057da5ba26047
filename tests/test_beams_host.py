"""Many answers about one context without a GPU: refusals of the entry points before any CUDA call, and the oracle's own laws."""
import numpy as np
import pytest
import torch

from strix_halo_maxx_b200 import build, ops, _lib
from oracle import beam_ref as R, kv8_ref

BF = torch.bfloat16
M = 1 << 30  # addresses that are never read


@pytest.fixture(scope="module")
def L():
    build.build()
    return _lib.lib()


def _shared(L, S=1, B=4, n=1, Hq=4, H=2, D=64, Cp=128, C=64, q=M, sq=64, out=M + (1 << 16), so=64, lens=4096, plens=4096, pk=4096, kc=4096, scale=0.125, ws=4096,
            ws_bytes=1 << 40):
    return L.vt_attn_kv8_shared(None, q, 256 * n, 256, sq, pk, 4096, 4096, 4096, Cp, plens, S, kc, 4096, 4096, 4096, C, lens, None, B, n, Hq, H, D, scale,
                                out, 256 * n, 256, so, ws, ws_bytes)


@pytest.mark.parametrize("kw,rc,word", [
    (dict(D=80), -1, b"head_dim"), (dict(C=65), -2, b"multiple of 64"), (dict(Cp=100), -2, b"multiple of 64"), (dict(Hq=5), -2, b"multiple of H"),
    (dict(n=-1), -2, b"n=-1"), (dict(S=3), -2, b"4 sequences over 3 prefixes"), (dict(S=0), -2, b"over 0 prefixes"), (dict(S=8), -2, b"over 8 prefixes"),
    (dict(q=None), -2, b"null"), (dict(out=M + (1 << 16) + 8), -2, b"16-byte"), (dict(sq=12), -2, b"16-byte"), (dict(so=100), -2, b"16-byte"), (dict(lens=None), -2, b"null"),
    (dict(plens=None), -2, b"null"), (dict(pk=None), -2, b"null"), (dict(kc=4104), -2, b"unaligned"), (dict(scale=-0.1), -2, b"scale"),
    (dict(scale=float("nan")), -2, b"scale"), (dict(scale=float("inf")), -2, b"scale"), (dict(B=2052), -2, b"at most 2048"), (dict(out=M), -2, b"out overlaps q"),
    (dict(out=M + 256), -2, b"out overlaps q"), (dict(n=0), 0, None), (dict(B=0), 0, None), (dict(B=0, S=0), 0, None)])
def test_attn_kv8_shared_refuses_on_the_host(L, kw, rc, word):
    assert _shared(L, **kw) == rc
    assert word is None or word in L.vt_last_error_string(), L.vt_last_error_string()


def _select(L, S=2, F=4, V=100, k=4, eos=5, ld=None, f32=1, logits=M, scores=M + (1 << 20), done=M + (1 << 21), out=M + (1 << 22), ws=4096, ws_bytes=1 << 40):
    return L.vt_beam_select(None, logits, V if ld is None else ld, f32, scores, done, S, F, V, k, eos, out, out + 4096 if out else None, M + (1 << 23), M + (1 << 24),
                            ws, ws_bytes)


@pytest.mark.parametrize("kw,rc,word", [
    (dict(F=0), -2, b"F=0"), (dict(F=65), -2, b"F=65"), (dict(V=0, ld=1), -2, b"V=0"), (dict(k=0), -2, b"k=0"), (dict(k=129), -2, b"k=129"), (dict(S=-1), -2, b"S=-1"),
    (dict(ld=99), -2, b"pitch of 99"), (dict(eos=100), -2, b"eos=100"), (dict(eos=-1), -2, b"eos=-1"), (dict(logits=None), -2, b"null"), (dict(logits=M + 2), -2, b"unaligned"),
    (dict(logits=M + 1, f32=0), -2, b"unaligned"), (dict(scores=None), -2, b"null"), (dict(out=None), -2, b"null"), (dict(ws=None), -2, b"workspace"), (dict(ws_bytes=8), -2, b"workspace"),
    (dict(ws=4100), -2, b"workspace"), (dict(out=M + (1 << 20)), -2, b"overlaps"), (dict(out=M + 792), -2, b"overlaps"), (dict(out=M + (1 << 21) - 28), -2, b"overlaps"),
    (dict(S=1 << 23, V=1, eos=0), -2, b"too large"), (dict(S=0), 0, None), (dict(S=0, logits=None, ws=None), 0, None)])
def test_beam_select_refuses_on_the_host(L, kw, rc, word):
    assert _select(L, **kw) == rc
    assert word is None or word in L.vt_last_error_string(), L.vt_last_error_string()


def _reorder(L, layers=1, Bs=4, C=64, dst=None, Cd=64, B=4, beams=2, H=2, D=64, base=M, parents=4096, lens=8192, new=None):
    four = lambda p: [None] * 4 if p is None else [p, p + (1 << 20), p + (1 << 21), p + (1 << 22)]
    return L.vt_kv8_reorder(None, *four(base), layers, Bs, C, *four(dst), Cd, parents, lens, B, beams, H, D, new)


@pytest.mark.parametrize("kw,rc,word", [
    (dict(D=72), -1, b"head_dim"), (dict(C=100), -2, b"multiple of 64"), (dict(dst=M + (1 << 25), Cd=96), -2, b"multiple of 64"), (dict(layers=-1), -2, b"layers=-1"),
    (dict(beams=0), -2, b"beams=0"), (dict(beams=3), -2, b"beams=3"), (dict(beams=65, B=65, Bs=65), -2, b"beams=65"), (dict(Bs=8), -2, b"divide"), (dict(parents=None), -2, b"null"),
    (dict(lens=None), -2, b"null"), (dict(base=None), -2, b"null"), (dict(dst=M), -2, b"overlaps"), (dict(dst=M + (1 << 20)), -2, b"overlaps"), (dict(new=8192), -2, b"overlaps"),
    (dict(new=4096 + 12), -2, b"overlaps"), (dict(new=M + 64), -2, b"overlaps"), (dict(dst=M + (1 << 25), new=8196), -2, b"overlaps"), (dict(layers=1 << 16, B=1 << 15, Bs=1 << 15), -2, b"too large"),
    (dict(layers=1 << 20, B=64, Bs=64), -2, b"too large"), (dict(C=1 << 25, Cd=0), -2, b"too large"), (dict(dst=M + (1 << 25), Bs=0), -2, b"no sequence"), (dict(layers=0), 0, None), (dict(B=0, Bs=0), 0, None), (dict(B=0, dst=M + (1 << 25)), 0, None)])
def test_kv8_reorder_refuses_on_the_host(L, kw, rc, word):
    assert _reorder(L, **kw) == rc
    assert word is None or word in L.vt_last_error_string(), L.vt_last_error_string()


def test_workspaces_of_empty_or_refused_problems_are_empty(L):
    for a in ((0, 0, 1, 4, 2, 64, 64, 64), (1, 0, 1, 4, 2, 64, 64, 64), (2, 3, 1, 4, 2, 64, 64, 64), (1, 1, 1, 4, 3, 64, 64, 64), (1, 1, 0, 4, 2, 64, 64, 64), (1, 1, 1, 4, 2, 72, 64, 64)):
        assert L.vt_attn_kv8_shared_ws_bytes(*a) == 0, a
    for a in ((0, 4, 10, 4), (1, 0, 10, 4), (1, 65, 10, 4), (1, 4, 0, 4), (1, 4, 10, 0), (1, 4, 10, 129)):
        assert L.vt_beam_select_ws_bytes(*a) == 0, a


@pytest.mark.parametrize("S,F,n,Hq,H,D,Cp,C", [(1, 12, 1, 32, 32, 64, 83200, 128), (1, 4, 1, 4, 4, 64, 64, 8192), (2, 2, 2, 8, 2, 128, 8192, 1024), (1, 1, 1, 1, 1, 64, 131072, 64)])
def test_attn_kv8_shared_workspace_holds_the_parts_of_runs(L, S, F, n, Hq, H, D, Cp, C):
    """Few rows over more tiles than one CTA takes: two parts of 8 rows or more for each of two CTAs an SM."""
    assert L.vt_attn_kv8_shared_ws_bytes(S, S * F, n, Hq, H, D, Cp, C) >= 2 * 2 * 148 * 8 * (D * 4 + 8)


def test_python_entry_points_refuse_wrong_types_shapes_and_layouts():
    i32 = lambda n: torch.zeros(n, dtype=torch.int32)
    p, c = ops.kv8_cache(2, 2, 64, 64, "cpu"), ops.kv8_cache(4, 2, 64, 64, "cpu")
    q, out = torch.zeros(4, 3, 4, 64, dtype=BF), torch.zeros(4, 3, 256, dtype=BF)
    x, sc = torch.zeros(8, 50), torch.zeros(8)
    c5 = ops.Kv8(*(t[None].repeat(3, *[1] * t.dim()) for t in c))
    bad = [lambda: ops.attn_kv8_shared(q.float(), p, i32(2), c, i32(4), out), lambda: ops.attn_kv8_shared(q, p, i32(1), c, i32(4), out),
           lambda: ops.attn_kv8_shared(q, p, i32(2), c, i32(2), out), lambda: ops.attn_kv8_shared(q, p, i32(2).long(), c, i32(4), out),
           lambda: ops.attn_kv8_shared(q, p, i32(2), c, i32(4), out[:, :, :128]), lambda: ops.attn_kv8_shared(q[:2], p, i32(2), c, i32(4), out[:2]),
           lambda: ops.attn_kv8_shared(q, ops.kv8_cache(2, 1, 64, 64, "cpu"), i32(2), c, i32(4), out),
           lambda: ops.attn_kv8_shared(q, p._replace(vs=p.vs.double()), i32(2), c, i32(4), out), lambda: ops.attn_kv8_shared(q, p, i32(2), c, i32(4), out, counts=sc[:4]),
           lambda: ops.attn_kv8_shared(q.transpose(2, 3), p, i32(2), c, i32(4), out),
           lambda: ops.beam_select(x.double(), sc, 4), lambda: ops.beam_select(x, sc, 3), lambda: ops.beam_select(x, sc, 0), lambda: ops.beam_select(x, sc[:4], 4),
           lambda: ops.beam_select(x.t(), sc, 4), lambda: ops.beam_select(x, sc, 4, eos=1, done=sc), lambda: ops.beam_select(x, sc.double(), 4),
           lambda: ops.beam_select(x, sc, 4, out=ops.Beams(sc, sc, sc, sc)), lambda: ops.beam_select(x[0], sc, 4),
           lambda: ops.kv8_reorder(c, i32(4), i32(4)), lambda: ops.kv8_reorder(c, i32(3), i32(4), beams=2), lambda: ops.kv8_reorder(c, i32(4), i32(3), beams=2),
           lambda: ops.kv8_reorder(c, i32(4).long(), i32(4), beams=2), lambda: ops.kv8_reorder(c, i32(4), i32(4), beams=2, dst=c), lambda: ops.kv8_reorder(c, i32(4), i32(4), dst=p),
           lambda: ops.kv8_reorder(c, i32(4), i32(4), dst=c5), lambda: ops.kv8_reorder(c5._replace(ks=c5.ks[:2]), i32(4), i32(4), beams=2),
           lambda: ops.kv8_reorder(c5._replace(k=c5.k.transpose(0, 1)), i32(4), i32(4), beams=2), lambda: ops.kv8_reorder(c, i32(4), i32(4), beams=2, new_lens=sc[:4])]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was not refused")


def test_oracle_attention_behind_a_prefix_is_attention_over_the_whole():
    """A prefix of whole blocks in front of a sequence's own: kv8_ref's attention over the two as one cache."""
    rng = np.random.default_rng(0)
    cache = lambda B, C: (*(rng.integers(-127, 128, (B, 2, C, 64), dtype=np.int8) for _ in range(2)),
                          *(rng.random((B, 2, C // 64), dtype=np.float32) * 0.02 + 0.01 for _ in range(2)))
    prefix, own, q, lens = cache(2, 128), cache(4, 64), rng.standard_normal((4, 3, 4, 64)), [0, 10, 61, 5]
    out, mag = R.attention_shared(q, prefix, [128, 128], own, lens, [3, 1, 3, 0])
    both = [np.concatenate([np.repeat(p, 2, axis=0), o], axis=2) for p, o in zip(prefix, own)]
    want, _, wmag, _ = kv8_ref.attention(q, both, [128 + x for x in lens], [3, 1, 3, 0])
    np.testing.assert_allclose(out, want, rtol=1e-12)
    np.testing.assert_allclose(mag, wmag, rtol=1e-12)


def test_oracle_totals_are_log_probabilities():
    """Of a live beam the totals less its score add up to one; a finished one has one continuation."""
    x = np.random.default_rng(1).standard_normal((4, 30))
    t = R.totals(x, [-1.0, -2.0, -3.0, -4.0], 2, 7, [False, True, False, False]).reshape(4, 30)
    np.testing.assert_allclose(np.exp(t[[0, 2, 3]] + np.array([[1.0], [3.0], [4.0]])).sum(-1), 1, rtol=1e-12)
    assert np.flatnonzero(np.isfinite(t[1])).tolist() == [7] and t[1, 7] == -2


def test_oracle_reorder_goes_round():
    """A cycle applied as often as it is long gives the cache back."""
    rng = np.random.default_rng(2)
    c = [rng.integers(-9, 9, (2, 3, 1, 64, 64), dtype=np.int8) for _ in range(2)] + [rng.random((2, 3, 1, 1), dtype=np.float32) for _ in range(2)]
    now = c
    for i in range(3):
        now, lens = R.reorder(now, [1, 2, 0], [50] * 3, 3)
        assert all(np.array_equal(a, b) for a, b in zip(now, c)) == (i == 2) and lens.tolist() == [50] * 3


@pytest.mark.parametrize("S,F,Hq,H,D,Cp,C", [(1, 4, 32, 32, 64, 768, 64), (1, 1, 32, 8, 128, 6016, 512), (4, 3, 8, 8, 64, 1024, 128), (2, 8, 32, 8, 128, 8192, 1024), (9, 1, 16, 16, 64, 2048, 64),
                                              (8, 3, 8, 1, 64, 768, 640), (16, 1, 16, 2, 128, 2048, 64), (1, 3, 128, 32, 64, 704, 448)])
def test_attn_kv8_shared_workspace_is_enough_for_fewer_tokens(L, S, F, Hq, H, D, Cp, C):
    need = [L.vt_attn_kv8_shared_ws_bytes(S, S * F, n, Hq, H, D, Cp, C) for n in range(1, 700)]
    assert need == sorted(need)


def test_an_lm_head_with_words_that_have_no_embedding_is_refused():
    from strix_halo_maxx_b200.text import TextDecoder
    with pytest.raises(ValueError, match="embeddings of 80"):
        TextDecoder({"lm_w": torch.zeros(90, 8), "wte": torch.zeros(80, 8)}, device="cpu", kv8=True, beams=2, steps=2)
