"""The 8-bit KV cache on the GPU against oracle/kv8_ref.py: codes and scales bit for bit, attention and weights within
bounds derived from their roundings, eviction bit for bit; and the three together."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from strix_halo_maxx_b200 import ops
from strix_halo_maxx_b200.config import TEXT
from strix_halo_maxx_b200.text import rope_tables
from strix_halo_maxx_b200._lib import device_status, VtError
from oracle import kv8_ref as R

DEV, BF = "cuda", torch.bfloat16
RANGE_BIT = 1 << 9


@pytest.fixture(autouse=True)
def _status():
    device_status(clear=True)
    yield
    assert device_status(clear=True) == 0


def i32(x):
    return torch.tensor(list(x), dtype=torch.int32, device=DEV)


def np_(t):
    return t.detach().cpu().numpy().copy()


def tables(n=8192):
    cos, sin = rope_tables(TEXT.__class__(prefix=n, q_len=0), DEV)
    return cos, sin


def filled(B, H, C, D, seed, spread=0.02):
    """A cache with codes over the whole range and scales that differ from block to block."""
    g = torch.Generator(DEV).manual_seed(seed)
    k, v = ((torch.randn(B, H, C, D, device=DEV, generator=g) * 40).round().clamp(-127, 127).to(torch.int8) for _ in range(2))
    ks, vs = (torch.rand(B, H, C // 64, device=DEV, generator=g) * spread + 0.01 for _ in range(2))
    return ops.Kv8(k, v, ks, vs)


def as_np(c):
    return tuple(np_(t) for t in c)


# ------------------------------------------------------------------------------------------------ append
APPEND = [  # B, n, Hq, H, D, lens, counts
    (1, 1, 32, 32, 64, [0], None), (1, 1, 4, 4, 64, [63], None), (1, 1, 4, 2, 128, [64], None), (2, 1, 8, 1, 64, [127, 5], None),
    (1, 730, 4, 4, 64, [0], None), (1, 300, 6, 3, 128, [37], None), (3, 70, 5, 1, 64, [0, 60, 130], [70, 0, 3]),
    (4, 7, 8, 2, 128, [1, 64, 63, 250], [7, 6, 1, 0]), (1, 64, 2, 2, 64, [64], None), (1, 65, 2, 2, 64, [191], None)]


@pytest.mark.parametrize("B,n,Hq,H,D,lens,counts", APPEND)
def test_rope_kv8_writes_the_oracles_codes(B, n, Hq, H, D, lens, counts):
    C = (max(lens) + n + 127) // 64 * 64
    g = torch.Generator(DEV).manual_seed(n + D)
    # rows that grow, so that scales of blocks with tokens double
    qkv = (torch.randn(B, n, (Hq + 2 * H) * D, device=DEV, generator=g) * torch.linspace(0.2, 6, n, device=DEV)[:, None]).to(BF)
    cache = filled(B, H, C, D, 1)
    cos, sin = tables()
    ref = as_np(cache)
    before = as_np(cache)
    q = torch.full((B, n, Hq, D), 7.0, dtype=BF, device=DEV)
    ops.rope_kv8(qkv, cache, i32(lens), cos, sin, q, counts=None if counts is None else i32(counts))
    qr = R.append(np_(qkv.float()), ref, lens, np_(cos), np_(sin), Hq, counts=counts)
    for name, got, want in zip(("k", "v", "ks", "vs"), as_np(cache), ref):
        assert np.array_equal(got, want), name
    for b in range(B):
        m = n if counts is None else counts[b]
        assert (np_(q[b, m:].float()) == 7).all()
        assert np.array_equal(np_(q[b, :m].float()), R.bf16(qr[b, :m]))
        end = (lens[b] + m + 63) // 64 * 64
        for got, was in zip(as_np(cache)[:2], before[:2]):
            assert np.array_equal(got[b, :, lens[b] + m:], was[b, :, lens[b] + m:]), "slots behind the last token"
        for got, was in zip(as_np(cache)[2:], before[2:]):
            assert np.array_equal(got[b, :, end // 64:], was[b, :, end // 64:])


def test_rope_kv8_one_by_one_strided_and_repeated():
    """150 tokens one by one through strided q and qkv rows, positions apart from slots: the oracle's codes after each block; the
    last call repeated changes nothing; values within one step."""
    B, Hq, H, D, n = 2, 4, 2, 64, 150
    cos, sin = tables()
    g = torch.Generator(DEV).manual_seed(3)
    qkv = (torch.randn(n, B, (Hq + 2 * H) * D + 24, device=DEV, generator=g) * torch.linspace(0.1, 4, n, device=DEV)[:, None, None]).to(BF)
    cache, qb = ops.kv8_cache(B, H, 192, D, DEV), torch.zeros(B, 2, Hq, D + 8, dtype=BF, device=DEV)
    ref = as_np(cache)
    for t in range(n):
        row = qkv[t].view(B, 1, -1)[:, :, :(Hq + 2 * H) * D]
        lens, pos = [t, t], [t + 500, t + 11]
        ops.rope_kv8(row, cache, i32(lens), cos, sin, qb[:, 1:, :, :D], pos=i32(pos))
        qr = R.append(np_(row.float()), ref, lens, np_(cos), np_(sin), Hq, pos=pos)
        if t in (0, 62, 63, 64, n - 1):
            assert np.array_equal(np_(qb[:, 1:, :, :D].float()), R.bf16(qr))
            assert all(np.array_equal(a, b) for a, b in zip(as_np(cache), ref)), t
    once = as_np(cache)
    ops.rope_kv8(row, cache, i32(lens), cos, sin, qb[:, 1:, :, :D], pos=i32(pos))
    assert all(np.array_equal(a, b) for a, b in zip(as_np(cache), once))
    v = np_(qkv[:, :, (Hq + H) * D:(Hq + 2 * H) * D].float()).reshape(n, B, H, D).transpose(1, 2, 0, 3)
    err = np.abs(np_(cache.values()[1])[:, :, :n] - v) / once[3].repeat(64, axis=2)[:, :, :n, None]
    assert err.max() <= 1 + 1e-5
    assert (qb[:, :1] == 0).all() and (qb[..., D:] == 0).all()


def test_rope_kv8_zero_tiny_large_and_non_finite_values():
    H, D, n = 1, 64, 64
    cos, sin = tables()
    qkv = torch.zeros(6, n, 3 * D, dtype=BF, device=DEV)
    qkv[1] = 1e-39          # subnormal
    qkv[2, 3, 2 * D + 5] = float("nan")
    qkv[3, 0, 2 * D] = float("inf")
    qkv[4] = 3.0e38
    qkv[4, :, D:2 * D] = 1e38
    qkv[5, 0] = 1e-30       # the first of a block; the others 1e30 times larger, one call later
    cache = filled(6, H, 128, D, 5)
    ref = as_np(cache)
    lens = [0] * 6
    q = torch.zeros(6, n, 1, D, dtype=BF, device=DEV)
    counts = [n] * 5 + [1]
    ops.rope_kv8(qkv, cache, i32(lens), cos, sin, q, counts=i32(counts))
    R.append(np_(qkv.float()), ref, lens, np_(cos), np_(sin), 1, counts=counts)
    big = torch.ones(6, 1, 3 * D, dtype=BF, device=DEV)
    ops.rope_kv8(big, cache, i32([64, 64, 5, 64, 64, 1]), cos, sin, q[:, :1])
    R.append(np_(big.float()), ref, [64, 64, 5, 64, 64, 1], np_(cos), np_(sin), 1)
    for name, got, want in zip(("k", "v", "ks", "vs"), as_np(cache), ref):
        assert np.array_equal(got, want, equal_nan=name in ("ks", "vs")), name
    assert float(cache.vs[0, 0, 0]) == 0 and torch.isnan(cache.vs[2, 0, 0]) and torch.isnan(cache.vs[3, 0, 0])
    assert not torch.isnan(cache.ks[2, 0, 0])


def test_lengths_beyond_the_cache_are_cut_off_and_recorded():
    B, H, D, C = 4, 1, 64, 128
    cos, sin = tables()
    cache = filled(B, H, C, D, 9)
    ref = as_np(cache)
    g = torch.Generator(DEV).manual_seed(2)
    qkv = torch.randn(B, 3, 3 * D, device=DEV, generator=g).to(BF)
    q = torch.zeros(B, 3, 1, D, dtype=BF, device=DEV)
    ops.rope_kv8(qkv, cache, i32([127, 10, -5, 500]), cos, sin, q, counts=i32([3, 9, 0, 3]))
    assert device_status(clear=True) == RANGE_BIT
    R.append(np_(qkv.float()), ref, [127, 10, 0, 0], np_(cos), np_(sin), 1, counts=[1, 3, 0, 0])
    for got, want in zip(as_np(cache), ref):
        assert np.array_equal(got, want)
    for pos in (cos.shape[0], -1, 2 ** 31 - 1, -2 ** 31):
        ops.rope_kv8(qkv[:1, :1], ops.Kv8(*(t[:1] for t in cache)), i32([3]), cos, sin, q[:1, :1], pos=i32([pos]))
        assert device_status(clear=True) == RANGE_BIT, pos
    out = torch.full((B, 3, D), 5.0, dtype=BF, device=DEV)
    ops.attn_kv8(q, cache, i32([127, 10, -5, 500]), out, counts=i32([3, 9, 0, 3]))
    assert device_status(clear=True) == RANGE_BIT
    assert (out[0, 1:] == 5).all() and (out[2:] == 5).all() and (out[1] != 5).any() and (out[0, 0] != 5).any()


# ------------------------------------------------------------------------------------------------ attention
ATTN = [  # B, n, Hq, H, D, lens, counts, causal
    (1, 1, 1, 1, 64, [0], None, True), (1, 1, 4, 4, 64, [62], None, True), (1, 1, 8, 1, 64, [63], None, True),
    (2, 1, 8, 2, 128, [64, 1000], None, True), (1, 1, 32, 32, 64, [761], None, True), (1, 32, 4, 4, 64, [730], None, True),
    (3, 5, 6, 2, 64, [0, 129, 64], [5, 0, 2], True), (3, 9, 10, 2, 128, [300, 1, 77], [1, 9, 0], False),
    (1, 70, 2, 2, 64, [0], None, False), (1, 200, 4, 2, 64, [33], None, True), (1, 130, 3, 3, 128, [250], None, True),
    (2, 129, 8, 2, 64, [500, 3], [129, 100], True), (1, 300, 5, 1, 128, [0], None, True), (1, 3, 64, 1, 128, [4000], None, True),
    (5, 2, 3, 3, 64, [7, 0, 190, 64, 63], [2, 1, 0, 2, 1], False), (1, 1, 20, 1, 64, [5000], None, True)]


def check_attn(q, cache, lens, counts, causal, out, w=None, w_in=None, scale=None):
    ro, rw, mag, werr = R.attention(np_(q.float()), as_np(cache), lens, counts, causal, scale,
                                    None if w_in is None else np_(w_in))
    o, rows = np_(out.float()), ~np.isnan(ro)
    # output rounded to bf16: half a step, 2^-8 of the value; P rounded to bf16 at most 2^-8 of each term p |v|; scores
    # and sums in fp32: far below 2^-12 of the terms for the scores here (|score| < 60)
    bound = np.abs(ro) * 2.0 ** -8 + mag * (2.0 ** -8 + 2.0 ** -12)
    assert (np.abs(o - ro)[rows] <= bound[rows] * (1 + 2.0 ** -7)).all(), float((np.abs(o - ro) / bound)[rows].max())
    # the rounding errors are random: over the whole output they stay under a third of that bound
    assert np.linalg.norm((o - ro)[rows]) <= np.linalg.norm(bound[rows]) / 3
    if w is not None:
        ww, at = np_(w), ~np.isnan(rw)
        n, G = q.shape[1], q.shape[2] // cache.k.shape[1]
        # p off by the score's and the row's (fp32 sums of exponentials) relative errors; n G + 1 terms added in fp32
        tol = werr + np.abs(rw) * (2.0 ** -18 + (n * G + 1) * 2.0 ** -24) + 1e-30
        assert (np.abs(ww - rw)[at] <= tol[at]).all(), float((np.abs(ww - rw) / tol)[at].max())
    return o


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("B,n,Hq,H,D,lens,counts,causal", ATTN)
def test_attn_kv8_matches_the_oracle(B, n, Hq, H, D, lens, counts, causal, weights):
    C = (max(lens) + n + 63) // 64 * 64
    cache = filled(B, H, C, D, n + Hq)
    g = torch.Generator(DEV).manual_seed(n)
    q = (torch.randn(B, n, Hq, D, device=DEV, generator=g) * 1.5).to(BF)
    out = torch.full((B, n, Hq * D), 3.0, dtype=BF, device=DEV)
    w = torch.full((B, H, C), -1.0, device=DEV) if weights else None
    w_in = torch.rand(B, H, C, device=DEV, generator=g) if weights and n % 2 else None
    cnt = None if counts is None else i32(counts)
    ops.attn_kv8(q, cache, i32(lens), out, counts=cnt, causal=causal, weights=w, weights_in=w_in)
    check_attn(q, cache, lens, counts, causal, out, w, w_in)
    for b in range(B):
        m = n if counts is None else counts[b]
        assert (out[b, m:] == 3).all(), "rows past the count"
        assert w is None or (w[b, :, lens[b] + m:] == -1).all(), "slots behind the last token"
    again, w2 = torch.full_like(out, 3.0), None if w is None else torch.full_like(w, -1.0)
    ops.attn_kv8(q, cache, i32(lens), again, counts=cnt, causal=causal, weights=w2, weights_in=w_in)
    assert torch.equal(out, again) and (w is None or torch.equal(w, w2)), "the same call twice"


@pytest.mark.parametrize("n", [1, 6, 140])
def test_attn_kv8_strides_scale_and_weights_in_place(n):
    """q a view of a wider row, out a column range of a wider matrix, a scale of the caller's, weights accumulated in place."""
    B, Hq, H, D, L = 2, 4, 2, 64, 100
    cache = filled(B, H, 320, D, 3)
    g = torch.Generator(DEV).manual_seed(8)
    qw = (torch.randn(B, Hq, n, D + 16, device=DEV, generator=g)).to(BF)
    q = qw.transpose(1, 2)[..., 8:8 + D]
    wide = torch.zeros(B, n, Hq * D + 32, dtype=BF, device=DEV)
    out = wide[:, :, 16:16 + Hq * D]
    w = torch.rand(B, H, 320, device=DEV, generator=g)
    w0 = w.clone()
    ops.attn_kv8(q, cache, i32([L, L - 30]), out, scale=0.3, weights=w, weights_in=w)
    check_attn(q, cache, [L, L - 30], None, True, out, w, w0, scale=0.3)
    assert (wide[:, :, :16] == 0).all() and (wide[:, :, 16 + Hq * D:] == 0).all()


@pytest.mark.parametrize("n,Hq,H,D", [(1, 2, 2, 64), (3, 8, 2, 128), (200, 2, 1, 64), (150, 2, 2, 128)])
def test_attn_kv8_blocks_out_of_sight_may_hold_anything(n, Hq, H, D):
    """NaN and infinite scales and any codes behind the last token change nothing; a NaN block inside makes exactly the rows
    that see it NaN (causal rows before it stay); an all-zero block (scale 0) is a block of zeros."""
    L = 130
    C = (L + n + 63) // 64 * 64 + 128
    cache = filled(1, H, C, D, 11)
    cache.ks[:, :, 0] = 0
    cache.vs[:, :, 1] = 0
    last = (L + n - 1) // 64
    cache.ks[:, :, last + 1:] = float("nan")
    cache.vs[:, :, last + 1:] = float("inf")
    q = torch.randn(1, n, Hq, D, device=DEV, generator=torch.Generator(DEV).manual_seed(1)).to(BF)
    out, w = torch.zeros(1, n, Hq * D, dtype=BF, device=DEV), torch.zeros(1, H, C, device=DEV)
    ops.attn_kv8(q, cache, i32([L]), out, weights=w)
    check_attn(q, cache, [L], None, True, out, w)
    clean = out.clone()
    cache.vs[:, :, last] = float("nan")
    ops.attn_kv8(q, cache, i32([L]), out)
    sees = (L + torch.arange(n)) // 64 >= last
    assert torch.isnan(out[0, sees]).all()
    assert torch.equal(out[0, ~sees], clean[0, ~sees])


def test_attn_kv8_large_scores_and_peaked_rows():
    """Scores of several hundred: one key takes it all; rows whose maximum comes last, first, and grows all the way."""
    H, D, T = 3, 64, 700
    cache = filled(1, H, 704, D, 4)
    cache.k.zero_()
    cache.ks.fill_(1.0)
    cache.k[0, 0, :T, 0] = torch.linspace(-127, 127, T, device=DEV).round().to(torch.int8)
    cache.k[0, 1, :T, 0] = torch.linspace(127, -127, T, device=DEV).round().to(torch.int8)
    cache.k[0, 2, 300, 0] = 127
    for n in (1, 64, 200):
        q = torch.zeros(1, n, H, D, dtype=BF, device=DEV)
        q[..., 0] = torch.linspace(1, 40, n, device=DEV)[None, :, None]
        out = torch.zeros(1, n, H * D, dtype=BF, device=DEV)
        ops.attn_kv8(q, cache, i32([T - n]), out)
        ro, _, mag, _ = R.attention(np_(q.float()), as_np(cache), [T - n])
        # integer scores times a power of two: exact in fp32, so only the roundings of P and the output remain
        assert (np.abs(np_(out.float()) - ro) <= (np.abs(ro) + mag) * 2.0 ** -8 * 1.02 + 1e-6).all()


@pytest.mark.parametrize("n", [1, 40, 150])
def test_attn_kv8_odd_queries_and_a_zero_scale(n):
    """Rows of q that are zero, subnormal, huge, infinite or NaN change no other row; scale 0 weighs every key the same."""
    H, D, L = 2, 64, 190
    cache = filled(1, H, 384, D, 21)
    g = torch.Generator(DEV).manual_seed(n)
    q = torch.randn(1, n, 2 * H, D, device=DEV, generator=g).to(BF)
    q[0, 0, 0], q[0, 0, 1], q[0, n // 2, 2] = 0, q[0, 0, 1] * 1e-39, q[0, n // 2, 2] * 1e-30
    out = ops.attn_kv8(q, cache, i32([L]))
    check_attn(q, cache, [L], None, True, out)
    bad = q.clone()
    bad[0, 0, 3, 5], bad[0, n - 1, 1, 0], bad[0, n // 3, 2] = float("inf"), float("nan"), 3e38
    o2 = ops.attn_kv8(bad, cache, i32([L]))
    same = torch.ones(n, 2 * H, dtype=torch.bool)
    same[0, 3], same[n - 1, 1], same[n // 3, 2] = False, False, False
    a, b = out.view(n, 2 * H, D)[same.to(DEV)], o2.view(n, 2 * H, D)[same.to(DEV)]
    assert torch.equal(a, b) and torch.isnan(o2.view(n, 2 * H, D)[n - 1, 1]).all()
    flat = ops.attn_kv8(q, cache, i32([L]), scale=0.0)
    check_attn(q, cache, [L], None, True, flat, scale=0.0)


def test_attn_kv8_one_workspace_for_calls_of_every_size_and_two_streams():
    """A workspace for the largest call serves the smaller ones after it; calls on two streams with workspaces of their own
    give what they give alone."""
    H, D = 2, 64
    cache = filled(1, H, 2048, D, 2)
    ws = ops.attn_kv8_workspace(1, 300, 4, H, D, 2048, DEV, True)
    want = {}
    for n in (300, 16, 1, 90):
        g = torch.Generator(DEV).manual_seed(n)
        q, w = torch.randn(1, n, 4, D, device=DEV, generator=g).to(BF), torch.zeros(1, H, 2048, device=DEV)
        o = ops.attn_kv8(q, cache, i32([1500]), weights=w, ws=ws)
        want[n] = (q, o, w)
        check_attn(q, cache, [1500], None, True, o, w)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for r in range(10):
        for s, n in ((s1, 300), (s2, 90), (s1, 16), (s2, 1)):
            with torch.cuda.stream(s):
                w = torch.zeros(1, H, 2048, device=DEV)
                got.append((n, ops.attn_kv8(want[n][0], cache, i32([1500]), weights=w), w))
    torch.cuda.synchronize()
    for n, o, w in got:
        assert torch.equal(o, want[n][1]) and torch.equal(w, want[n][2]), n


def test_attn_kv8_of_one_row_does_not_depend_on_its_batch():
    """A sequence alone and in a batch: equal within the rounding of the split."""
    H, D = 4, 128
    cache = filled(9, H, 4096, D, 6)
    q = torch.randn(9, 1, 16, D, device=DEV, generator=torch.Generator(DEV).manual_seed(1)).to(BF)
    lens = [4000, 1, 17, 2047, 64, 63, 3000, 0, 900]
    out = ops.attn_kv8(q, cache, i32(lens))
    for b in (0, 1, 6, 7):
        one = ops.attn_kv8(q[b:b + 1], ops.Kv8(*(t[b:b + 1] for t in cache)), i32(lens[b:b + 1]))
        assert torch.allclose(one[0].float(), out[b].float(), rtol=2.0 ** -7, atol=2.0 ** -9)


# ------------------------------------------------------------------------------------------------ eviction
EVICT = [  # B, H, D, C, lens, keep, recent, dst C
    (1, 1, 64, 128, [128], 64, 0, 64), (1, 2, 64, 832, [730], 256, 32, 320), (2, 3, 128, 512, [500, 300], 448, 448, 448),
    (4, 2, 64, 1024, [1000, 64, 0, 65], 64, 7, 128), (1, 2, 128, 5056, [5001], 1024, 100, 2048), (3, 1, 64, 256, [200, 256, 193], 192, 1, 256),
    (1, 1, 128, 20480, [20001], 128, 0, 128), (1, 2, 64, 9024, [9000], 64, 0, 64), (2, 1, 64, 40000, [39999, 33000], 4096, 5, 4096),
    (1, 1, 64, 70016, [70016], 640, 1, 640), (150, 1, 64, 2112, [2100 - i for i in range(150)], 1024, 100, 1024),
    (150, 1, 64, 33024, [33000] * 2 + [500] * 148, 512, 1, 512), (1, 1, 64, 262144, [262100], 128, 64, 128)]


@pytest.mark.parametrize("ties", [False, True])
@pytest.mark.parametrize("B,H,D,C,lens,keep,recent,Cd", EVICT)
def test_kv8_evict_matches_the_oracle(B, H, D, C, lens, keep, recent, Cd, ties):
    cache = filled(B, H, C, D, keep)
    g = torch.Generator(DEV).manual_seed(C)
    w = torch.exp(3 * torch.randn(B, H, C, device=DEV, generator=g))
    w[torch.rand(B, H, C, device=DEV, generator=g) < 0.1] = 0
    if ties:  # few different weights, minus zero, NaN, infinities and negative ones among them
        w = w.log2().clamp(-1, 2).round()
        w[..., 5], w[..., 17], w[..., 40], w[..., 41] = float("nan"), float("inf"), -0.0, float("-inf")
        cache.k[:, :, 64:128] = 0
    w[..., max(lens):] = 1e30   # behind the last token: never chosen
    ref = R.evict(as_np(cache), np_(w), lens, keep, recent)
    dst = filled(B, H, Cd, D, 77)
    was = as_np(dst)
    dw, dl = torch.full((B, H, Cd), -2.0, device=DEV), i32([9] * B)
    src = as_np(cache)
    idx = ops.kv8_evict(cache, w, i32(lens), keep, recent, dst, dw, dl)
    assert np_(dl).tolist() == [min(x, keep) for x in lens]
    assert all(np.array_equal(a, b) for a, b in zip(src, as_np(cache))), "the source stays"
    got = as_np(dst)
    for b in range(B):
        L = lens[b]
        if ref[b] is None:
            nb = (L + 63) // 64
            want = (np.tile(np.arange(L), (H, 1)), src[0][b, :, :L], src[1][b, :, :L], src[2][b, :, :nb], src[3][b, :, :nb])
        else:
            want = ref[b]
        T, nb = min(L, keep), (min(L, keep) + 63) // 64
        assert np.array_equal(np_(idx)[b, :, :T], want[0]), b
        assert np.array_equal(np_(dw)[b, :, :T], np.take_along_axis(np_(w)[b], want[0], -1), equal_nan=True)
        assert (np_(dw)[b, :, T:] == -2).all()
        for x, y, z, t in ((got[0], want[1], was[0], T), (got[1], want[2], was[1], T), (got[2], want[3], was[2], nb), (got[3], want[4], was[3], nb)):
            assert np.array_equal(x[b, :, :t], y) and np.array_equal(x[b, :, t:], z[b, :, t:])


def test_kv8_evict_keeps_a_nan_block_nan_and_refuses_itself():
    cache = filled(1, 1, 256, 64, 2)
    cache.ks[0, 0, 1] = float("nan")
    w = torch.ones(1, 1, 256, device=DEV)
    w[0, 0, 64:70] = 2
    dst, dw, dl = ops.kv8_cache(1, 1, 128, 64, DEV), torch.zeros(1, 1, 128, device=DEV), i32([0])
    idx = ops.kv8_evict(cache, w, i32([256]), 128, 0, dst, dw, dl)
    assert np_(idx)[0, 0].tolist() == list(range(128))
    assert torch.isnan(dst.ks[0, 0]).tolist() == [False, True] and not torch.isnan(dst.vs).any()
    with pytest.raises(VtError, match="overlaps"):
        ops.kv8_evict(cache, w, i32([256]), 128, 0, cache, w, dl)


# ------------------------------------------------------------------------------------------------ together
def _pass(cache, small, bufs, cos, sin, L, n, H, D):
    """One use of all three: a prompt written and attended to with its weights, evicted, then one more token over the
    smaller cache."""
    q, out, w, dw, idx = bufs["q"], bufs["out"], bufs["w"], bufs["dw"], bufs["idx"]
    ops.rope_kv8(bufs["qkv"], cache, bufs["zero"], cos, sin, q)
    ops.attn_kv8(q, cache, bufs["zero"], out, weights=w, ws=bufs["ws"])
    ops.kv8_evict(cache, w, bufs["n"], 64, 16, small, dw, bufs["dl"], index=idx)
    ops.rope_kv8(bufs["one"], small, bufs["dl"], cos, sin, bufs["q1"], pos=bufs["n"])
    ops.attn_kv8(bufs["q1"], small, bufs["dl"], bufs["o1"], weights=dw, weights_in=dw, ws=bufs["ws"])


def _bufs(n, Hq, H, D, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    return {"qkv": torch.randn(1, n, (Hq + 2 * H) * D, device=DEV, generator=g).to(BF),
            "one": torch.randn(1, 1, (Hq + 2 * H) * D, device=DEV, generator=g).to(BF),
            "q": torch.zeros(1, n, Hq, D, dtype=BF, device=DEV), "q1": torch.zeros(1, 1, Hq, D, dtype=BF, device=DEV),
            "out": torch.zeros(1, n, Hq * D, dtype=BF, device=DEV), "o1": torch.zeros(1, 1, Hq * D, dtype=BF, device=DEV),
            "w": torch.zeros(1, H, 256, device=DEV), "dw": torch.zeros(1, H, 128, device=DEV), "zero": i32([0]), "n": i32([n]),
            "dl": i32([0]), "idx": torch.zeros(1, H, 64, dtype=torch.int32, device=DEV),
            "ws": ops.attn_kv8_workspace(1, n, Hq, H, D, 256, DEV, True)}


def test_write_attend_evict_and_go_on_eager_captured_and_on_another_stream():
    n, Hq, H, D = 150, 4, 2, 64
    cos, sin = tables()
    runs = []
    for mode in ("eager", "graph", "stream"):
        cache, small, bufs = ops.kv8_cache(1, H, 256, D, DEV), ops.kv8_cache(1, H, 128, D, DEV), _bufs(n, Hq, H, D, 5)
        args = (cache, small, bufs, cos, sin, 0, n, H, D)
        if mode == "eager":
            _pass(*args)
        else:
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                _pass(*args)
                if mode == "graph":
                    torch.cuda.synchronize()
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph, stream=s):
                        _pass(*args)
                    for t in (bufs["out"], bufs["o1"], bufs["w"], small.k):
                        t.zero_()
                    graph.replay()
            torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        runs.append([bufs["out"], bufs["o1"], bufs["w"], bufs["dw"], bufs["idx"], *small])
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))
    # the eager run against the oracle, step by step on its own cache
    cache, small, bufs = ops.kv8_cache(1, H, 256, D, DEV), ops.kv8_cache(1, H, 128, D, DEV), _bufs(n, Hq, H, D, 5)
    ref = as_np(cache)
    R.append(np_(bufs["qkv"].float()), ref, [0], np_(cos), np_(sin), Hq)
    _pass(cache, small, bufs, cos, sin, 0, n, H, D)
    assert all(np.array_equal(a, b) for a, b in zip(ref, as_np(cache)))
    check_attn(bufs["q"], cache, [0], None, True, bufs["out"], bufs["w"])
    (idx, k, v, ks, vs), = R.evict(ref, np_(bufs["w"]), [n], 64, 16)
    assert np.array_equal(np_(bufs["idx"])[0], idx) and np_(bufs["dl"]).tolist() == [64]
    sref = [np.zeros((1, H, 128, D), np.int8), np.zeros((1, H, 128, D), np.int8), np.zeros((1, H, 2), np.float32), np.zeros((1, H, 2), np.float32)]
    sref[0][0, :, :64], sref[1][0, :, :64], sref[2][0, :, :1], sref[3][0, :, :1] = k, v, ks, vs
    R.append(np_(bufs["one"].float()), sref, [64], np_(cos), np_(sin), Hq, pos=[n])
    assert all(np.array_equal(a, b) for a, b in zip(sref, as_np(small)))
    w_in = torch.from_numpy(np.take_along_axis(np_(bufs["w"]), idx[None], -1))
    w_in = torch.nn.functional.pad(w_in, (0, 64)).to(DEV)
    check_attn(bufs["q1"], small, [64], None, True, bufs["o1"], bufs["dw"], w_in)
