"""The 8-bit KV cache without a GPU: refusals of the entry points before any CUDA call, and the oracle's own laws (a value
is at most half a step off when its block came in one call, one step however it came)."""
import numpy as np
import pytest
import torch

from strix_halo_maxx_b200 import build, ops, _lib
from oracle import kv8_ref as R

BF = torch.bfloat16


@pytest.fixture(scope="module")
def L():
    build.build()
    return _lib.lib()


def _msg(L):
    return L.vt_last_error_string()


def _rope(L, B=1, n=1, Hq=4, H=2, D=64, tab=8, C=64, sx=512, sq=64, qkv=4096, cos=4096, lens=4096):
    return L.vt_rope_kv8(None, qkv, sx, sx, B, n, Hq, H, D, cos, 4096, tab, lens, None, None, 4096, 256, 256, sq, 4096, 4096,
                         4096, 4096, C)


@pytest.mark.parametrize("kw,rc,word", [
    (dict(D=72), -1, b"head_dim"), (dict(C=100), -2, b"multiple of 64"), (dict(C=0), -2, b"C=0"), (dict(Hq=3), -2, b"multiple of H"),
    (dict(H=0), -2, b"H=0"), (dict(n=-1), -2, b"n=-1"), (dict(tab=0), -2, b"tab=0"), (dict(sx=516), -2, b"16-byte"),
    (dict(sq=4), -2, b"16-byte"), (dict(qkv=4100), -2, b"16-byte"), (dict(cos=None), -2, b"null"), (dict(lens=None), -2, b"null"),
    (dict(B=1 << 16, H=1 << 15, Hq=1 << 15), -2, b"too large"), (dict(B=0), 0, None), (dict(n=0), 0, None)])
def test_rope_kv8_refuses_on_the_host(L, kw, rc, word):
    assert _rope(L, **kw) == rc
    assert word is None or word in _msg(L), _msg(L)


def _attn(L, B=1, n=1, Hq=4, H=2, D=64, C=64, q=4096, sq=64, out=4096, so=64, w=None, w_in=None, ws=4096, ws_bytes=1 << 40, lens=4096,
          scale=0.125):
    return L.vt_attn_kv8(None, q, 256, 256, sq, 4096, 4096, 4096, 4096, C, lens, None, B, n, Hq, H, D, 1, scale, out, 256, 256, so,
                         w, w_in, ws, ws_bytes)


@pytest.mark.parametrize("kw,rc,word", [
    (dict(D=80), -1, b"head_dim"), (dict(C=65), -2, b"multiple of 64"), (dict(Hq=5), -2, b"multiple of H"), (dict(q=None), -2, b"null"),
    (dict(out=4104), -2, b"16-byte"), (dict(sq=12), -2, b"16-byte"), (dict(so=100), -2, b"16-byte"), (dict(lens=None), -2, b"null"),
    (dict(w_in=4096), -2, b"weights_in without weights"), (dict(scale=-0.1), -2, b"scale"), (dict(scale=float("nan")), -2, b"scale"),
    (dict(scale=float("inf")), -2, b"scale"), (dict(B=2049, C=4096), -2, b"at most 2048"), (dict(w=4096, ws=None), -2, b"workspace"),
    (dict(w=4096, ws_bytes=4), -2, b"workspace"), (dict(w=4096, ws=4100), -2, b"workspace"), (dict(n=0), 0, None), (dict(B=0), 0, None)])
def test_attn_kv8_refuses_on_the_host(L, kw, rc, word):
    assert _attn(L, **kw) == rc
    assert word is None or word in _msg(L), _msg(L)


def _evict(L, B=1, H=2, D=64, C=128, keep=64, recent=8, base=1 << 20, dst=1 << 24, Cd=64, w=1 << 22, dlens=(1 << 25)):
    return L.vt_kv8_evict(None, base, base + (1 << 16), base + (1 << 17), base + (1 << 18), C, w, 1 << 23, B, H, D, keep, recent, dst,
                          dst + (1 << 16), dst + (1 << 17), dst + (1 << 18), Cd, dst + (1 << 19), dlens, dst + (1 << 20))


@pytest.mark.parametrize("kw,rc,word", [
    (dict(D=96), -1, b"head_dim"), (dict(keep=0), -2, b"keep=0"), (dict(keep=63), -2, b"keep=63"), (dict(keep=128), -2, b"keep=128"),
    (dict(recent=65), -2, b"recent=65"), (dict(recent=-1), -2, b"recent=-1"), (dict(Cd=96), -2, b"multiple of 64"),
    (dict(w=None), -2, b"null"), (dict(C=262144 + 64), -2, b"at most 262144"), (dict(dst=1 << 20), -2, b"overlaps"), (dict(dst=(1 << 20) + 64 * 64), -2, b"overlaps"),
    (dict(dlens=1 << 23), -2, b"overlaps"), (dict(B=0), 0, None)])
def test_kv8_evict_refuses_on_the_host(L, kw, rc, word):
    assert _evict(L, **kw) == rc
    assert word is None or word in _msg(L), _msg(L)


def test_workspace_of_an_empty_problem_is_empty(L):
    assert L.vt_attn_kv8_ws_bytes(0, 1, 4, 2, 64, 64, 1) == 0 and L.vt_attn_kv8_ws_bytes(1, 0, 4, 2, 64, 64, 1) == 0
    assert L.vt_attn_kv8_ws_bytes(1, 1, 4, 3, 64, 64, 1) == 0


def test_python_entry_points_refuse_wrong_types_shapes_and_layouts():
    c = ops.kv8_cache(2, 2, 100, 64, "cpu")
    assert c.k.shape == (2, 2, 128, 64) and c.ks.shape == (2, 2, 2)
    lens, cs = torch.zeros(2, dtype=torch.int32), torch.zeros(8, 16)
    qkv, q, out = torch.zeros(2, 3, 8 * 64, dtype=BF), torch.zeros(2, 3, 4, 64, dtype=BF), torch.zeros(2, 3, 256, dtype=BF)
    w = torch.zeros(2, 2, 128)
    bad = [lambda: ops.rope_kv8(qkv.float(), c, lens, cs, cs, q), lambda: ops.rope_kv8(qkv[:, :, :-8], c, lens, cs, cs, q),
           lambda: ops.rope_kv8(qkv, c, lens.long(), cs, cs, q), lambda: ops.rope_kv8(qkv, c, lens[:1], cs, cs, q),
           lambda: ops.rope_kv8(qkv, c, lens, cs[:, :8], cs, q), lambda: ops.rope_kv8(qkv, c, lens, cs, cs[:4], q),
           lambda: ops.rope_kv8(qkv, c, lens, cs, cs, q, counts=lens.float()),
           lambda: ops.rope_kv8(qkv, c._replace(ks=c.ks[:, :, :1]), lens, cs, cs, q),
           lambda: ops.rope_kv8(qkv, c._replace(k=c.k.transpose(0, 1)), lens, cs, cs, q),
           lambda: ops.attn_kv8(q.float(), c, lens, out), lambda: ops.attn_kv8(q, c, lens, out[:, :, :128]),
           lambda: ops.attn_kv8(q, c, lens, out, weights=w[:, :, :64]), lambda: ops.attn_kv8(q, c, lens, out, weights=w.double()),
           lambda: ops.attn_kv8(q, c._replace(vs=c.vs.double()), lens, out), lambda: ops.attn_kv8(q[:1], c, lens, out),
           lambda: ops.attn_kv8(q.transpose(2, 3), c, lens, out),
           lambda: ops.kv8_evict(c, w, lens, 64, 8, ops.kv8_cache(2, 1, 64, 64, "cpu"), w[:, :, :64].contiguous(), lens.clone()),
           lambda: ops.kv8_evict(c, w, lens, 64, 8, ops.kv8_cache(2, 2, 64, 64, "cpu"), w, lens.clone()),
           lambda: ops.kv8_evict(c, w[:, :1], lens, 64, 8, ops.kv8_cache(2, 2, 64, 64, "cpu"), w[:, :, :64].contiguous(), lens.clone())]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was not refused")


def test_values_are_codes_times_their_blocks_scale():
    c = ops.kv8_cache(1, 1, 128, 64, "cpu")
    c.k[0, 0, 70, 3], c.ks[0, 0, 1] = 5, 0.5
    k, v = c.values()
    assert float(k[0, 0, 70, 3]) == 2.5 and float(k.abs().sum()) == 2.5 and float(v.abs().sum()) == 0


@pytest.mark.parametrize("step", [1, 3, 64, 200])
def test_oracle_quantisation_error(step):
    """Half a step where a block is written in one call; below one step of the last scale however tokens arrive, here with
    magnitudes that grow from token to token, so that scales double again and again."""
    rng = np.random.default_rng(step)
    x = R.bf16((rng.standard_normal((200, 64)) * np.exp(0.05 * np.arange(200))[:, None]).astype(np.float32))
    codes, s = np.zeros((256, 64), np.int8), np.zeros(4, np.float32)
    for at in range(0, 200, step):
        R.quantise(x[at:at + step], codes, s, at)
    sc = s[np.arange(200) // 64].astype(np.float64)[:, None]
    err = np.abs(codes[:200].astype(np.float64) * sc - x) / sc
    # x / s is rounded once to fp32 before rint: 127 * 2^-24 of a step beside the half
    assert err.max() <= (0.5 if step >= 64 and 64 % step == 0 or step == 200 else 1.0) + 1e-5
    assert (np.abs(x).max(axis=1) <= 127.0001 * sc[:, 0]).all()
