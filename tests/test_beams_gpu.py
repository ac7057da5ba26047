"""Many answers about one context on the GPU against oracle/beam_ref.py: attention behind a shared prefix within bounds derived from
its roundings, the choice of a beam search, the reordering of caches bit for bit; and the three together."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from strix_halo_maxx_b200 import ops
from strix_halo_maxx_b200.config import TEXT
from strix_halo_maxx_b200.text import rope_tables
from strix_halo_maxx_b200._lib import device_status
from oracle import beam_ref as R

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


def filled(lead, H, C, D, seed, spread=0.02):
    """A cache with codes over the whole range and scales that differ from block to block."""
    g = torch.Generator(DEV).manual_seed(seed)
    k, v = ((torch.randn(*lead, H, C, D, device=DEV, generator=g) * 40).round().clamp(-127, 127).to(torch.int8) for _ in range(2))
    ks, vs = (torch.rand(*lead, H, C // 64, device=DEV, generator=g) * spread + 0.01 for _ in range(2))
    return ops.Kv8(k, v, ks, vs)


def up64(x):
    return max(64, (x + 63) // 64 * 64)


def as_np(c):
    return tuple(np_(t) for t in c)


# ------------------------------------------------------------------------------------------------ attention
SHARED = [  # S, F, n, Hq, H, D, plens, lens, counts
    # few rows on a prefix
    (1, 1, 1, 1, 1, 64, [0], [0], None), (1, 4, 1, 4, 4, 64, [730], [38] * 4, None), (1, 4, 1, 8, 2, 128, [65], [0, 63, 64, 130], None),
    (2, 3, 1, 4, 2, 64, [1, 1000], [5, 0, 70, 127, 1, 300], [1, 1, 0, 1, 0, 1]), (1, 8, 4, 2, 2, 64, [200], [0, 9, 60, 61, 62, 63, 64, 65], [4, 0, 1, 2, 4, 4, 3, 4]),
    (3, 2, 3, 5, 1, 128, [64, 0, 129], [0, 1, 2, 0, 100, 64], [3, 2, 0, 0, 1, 3]), (5, 1, 2, 8, 1, 64, [0, 63, 64, 65, 400], [0, 0, 0, 0, 0], None),
    (1, 16, 1, 4, 2, 64, [5000], [3] * 16, None), (1, 4, 1, 8, 1, 128, [9000], [700, 0, 3, 64], None),
    # a short prefix and many sequences' own slots, over many CTAs
    (2, 12, 1, 2, 2, 64, [730, 100], [i * 5 for i in range(24)], None), (1, 16, 2, 1, 1, 64, [60], [i * 31 for i in range(16)], [i % 3 for i in range(16)]),
    (3, 4, 1, 4, 1, 128, [500, 0, 64], [300, 0, 64, 1, 290, 17, 33, 32, 31, 64, 65, 200], None), (1, 32, 1, 1, 1, 64, [64], [(i * 37) % 200 for i in range(32)], None),
    # many rows on a prefix, few of each sequence
    (1, 40, 1, 3, 3, 64, [500], [i * 7 for i in range(40)], None), (2, 17, 1, 8, 2, 128, [300, 0], [0] * 17 + [i * 13 for i in range(17)], [i % 3 % 2 for i in range(34)]),
    (1, 9, 8, 4, 4, 64, [700], [0] * 9, [8, 1, 0, 3, 8, 7, 2, 5, 0]), (1, 33, 2, 4, 1, 128, [64], [i for i in range(33)], None),
    (3, 20, 1, 8, 2, 64, [64, 2000, 777], [i * 3 for i in range(60)], [int(i % 7 != 3) for i in range(60)]), (1, 64, 1, 16, 4, 128, [4000], [i * 5 for i in range(64)], None),
    (2, 40, 1, 1, 1, 64, [1, 130], [0] * 80, [0] * 40 + [1] * 40), (1, 300, 1, 2, 2, 64, [1500], [i % 90 for i in range(300)], None),
    # many rows of each sequence
    (1, 2, 40, 2, 2, 64, [100], [0, 30], None), (2, 2, 70, 4, 2, 128, [300, 64], [0, 0, 100, 64], [70, 11, 0, 70]),
    (1, 3, 150, 2, 1, 64, [1], [64, 0, 200], [150, 0, 149]), (1, 4, 65, 5, 1, 64, [640], [0, 1, 2, 63], None), (1, 2, 300, 1, 1, 128, [0], [0, 70], None)]


def check_shared(q, prefix, plens, cache, lens, counts, out, scale=None):
    ro, mag = R.attention_shared(np_(q.float()), as_np(prefix), plens, as_np(cache), lens, counts, scale)
    o, rows = np_(out.float()), ~np.isnan(ro)
    # output rounded to bf16: half a step, 2^-8 of the value; P rounded to f16, 2^-11 of each term p |v|; scores and sums in
    # fp32 and the parts' factors by the hardware exponential: below 2^-12 of the terms for the scores here (|score| < 60)
    bound = np.abs(ro) * 2.0 ** -8 + mag * (2.0 ** -11 + 2.0 ** -12)
    assert (np.abs(o - ro)[rows] <= bound[rows] * (1 + 2.0 ** -7)).all(), float((np.abs(o - ro) / bound)[rows].max())
    # rounding errors are spread evenly over a step: their root mean square is below 1 / sqrt(3) of the half step
    if rows.any():
        assert np.linalg.norm((o - ro)[rows]) <= np.linalg.norm(bound[rows]) * 3 ** -0.5


@pytest.mark.parametrize("S,F,n,Hq,H,D,plens,lens,counts", SHARED)
def test_attn_kv8_shared_matches_the_oracle(S, F, n, Hq, H, D, plens, lens, counts):
    B = S * F
    prefix, cache = filled((S,), H, up64(max(plens)), D, n + Hq), filled((B,), H, up64(max(lens) + n), D, n + Hq + 1)
    q = (torch.randn(B, n, Hq, D, device=DEV, generator=torch.Generator(DEV).manual_seed(n)) * 1.5).to(BF)
    out = torch.full((B, n, Hq * D), 3.0, dtype=BF, device=DEV)
    cnt = None if counts is None else i32(counts)
    ops.attn_kv8_shared(q, prefix, i32(plens), cache, i32(lens), out, counts=cnt)
    check_shared(q, prefix, plens, cache, lens, counts, out)
    for b in range(B):
        assert (out[b, n if counts is None else counts[b]:] == 3).all(), "rows past the count"
    again = torch.full_like(out, 3.0)
    ops.attn_kv8_shared(q, prefix, i32(plens), cache, i32(lens), again, counts=cnt)
    assert torch.equal(out, again), "the same call twice"


@pytest.mark.parametrize("F,n", [(3, 2), (12, 3), (40, 1), (2, 40)])
def test_attn_kv8_shared_strides_and_scale(F, n):
    """q a view of a wider row in another order, out a column range of a wider matrix, a scale of the caller's."""
    Hq, H, D, P = 4, 2, 64, 190
    lens = [7 * b % 50 for b in range(F)]
    prefix, cache = filled((1,), H, 320, D, 3), filled((F,), H, 128, D, 4)
    g = torch.Generator(DEV).manual_seed(8)
    q = (torch.randn(F, Hq, n, D + 16, device=DEV, generator=g)).to(BF).transpose(1, 2)[..., 8:8 + D]
    wide = torch.zeros(F, n, Hq * D + 32, dtype=BF, device=DEV)
    out = wide[:, :, 16:16 + Hq * D]
    ops.attn_kv8_shared(q, prefix, i32([P]), cache, i32(lens), out, scale=0.3)
    check_shared(q, prefix, [P], cache, lens, None, out, scale=0.3)
    assert (wide[:, :, :16] == 0).all() and (wide[:, :, 16 + Hq * D:] == 0).all()


@pytest.mark.parametrize("F,n,Hq,H,D", [(4, 1, 2, 2, 64), (4, 2, 8, 2, 128), (40, 1, 4, 2, 64), (12, 4, 4, 2, 128), (3, 100, 2, 1, 64)])
def test_attn_kv8_shared_what_is_out_of_sight_may_hold_anything(F, n, Hq, H, D):
    """NaN and infinite scales, any codes behind the last token, and rows of padding that are NaN change nothing; a NaN block in a
    sequence's own cache makes the rows that see it NaN and no others; an all-zero block is a block of zeros."""
    P, L = 130, 70
    prefix, cache = filled((1,), H, 320, D, 11), filled((F,), H, up64(L + n) + 128, D, 12)
    prefix.ks[:, :, 0], prefix.vs[:, :, 1], cache.vs[:, :, 0] = 0, 0, 0
    prefix.ks[:, :, 3:], prefix.vs[:, :, 3:] = float("nan"), float("inf")
    last = (L + n - 1) // 64
    cache.ks[:, :, last + 1:], cache.vs[:, :, last + 1:] = float("nan"), float("inf")
    q = torch.randn(F, n, Hq, D, device=DEV, generator=torch.Generator(DEV).manual_seed(1)).to(BF)
    counts = [n] * F
    counts[1] = n - 1
    q[1, n - 1] = float("nan")
    out = torch.zeros(F, n, Hq * D, dtype=BF, device=DEV)
    args = i32([P]), cache, i32([L] * F)
    ops.attn_kv8_shared(q, prefix, *args, out, counts=i32(counts))
    check_shared(q, prefix, [P], cache, [L] * F, counts, out)
    clean = out.clone()
    cache.vs[2, :, last] = float("nan")
    ops.attn_kv8_shared(q, prefix, *args, out, counts=i32(counts))
    sees = (L + torch.arange(n)) // 64 >= last
    assert torch.isnan(out[2, sees]).all() and torch.equal(out[2, ~sees], clean[2, ~sees])
    rest = [b for b in range(F) if b != 2]
    assert torch.equal(out[rest], clean[rest])


@pytest.mark.parametrize("F,n", [(4, 1), (40, 1), (8, 8), (2, 80)])
def test_attn_kv8_shared_large_scores_wherever_they_are(F, n):
    """Scores of several hundred: one key takes it all, in the prefix or behind it; rows whose maximum comes last, first and grows
    all the way; integer scores times a power of two, so only the roundings of P and the output remain."""
    H, D, P, L = 4, 64, 700, 100
    prefix, cache = filled((1,), H, 704, D, 4), filled((F,), H, 256, D, 5)
    for c in (prefix, cache):
        c.k.zero_()
        c.ks.fill_(1.0)
    prefix.k[0, 0, :P, 0] = torch.linspace(-127, 100, P, device=DEV).round().to(torch.int8)
    prefix.k[0, 1, :P, 0] = torch.linspace(127, -127, P, device=DEV).round().to(torch.int8)
    prefix.k[0, 2, 300, 0] = 127
    cache.k[:, 0, :, 0], cache.k[:, 2, 20, 0], cache.k[:, 3, 99, 0] = 101, 126, 127
    q = torch.zeros(F, n, H, D, dtype=BF, device=DEV)
    q[..., 0] = torch.linspace(1, 40, F * n, device=DEV).view(F, n, 1)
    out = ops.attn_kv8_shared(q, prefix, i32([P]), cache, i32([L] * F))
    ro, mag = R.attention_shared(np_(q.float()), as_np(prefix), [P], as_np(cache), [L] * F)
    assert (np.abs(np_(out.float()) - ro) <= (np.abs(ro) * 2.0 ** -8 + mag * 2.0 ** -10) * 1.02 + 1e-6).all()


@pytest.mark.parametrize("F,n", [(5, 1), (50, 1), (9, 6), (2, 60)])
def test_attn_kv8_shared_odd_queries_and_a_zero_scale(F, n):
    """Rows of q that are zero, subnormal, huge, infinite or NaN change no other row; scale 0 weighs every key the same."""
    H, D, P = 2, 64, 190
    prefix, cache = filled((1,), H, 192, D, 21), filled((F,), H, 128, D, 22)
    lens = [3 * b % 60 for b in range(F)]
    q = torch.randn(F, n, 2 * H, D, device=DEV, generator=torch.Generator(DEV).manual_seed(n)).to(BF)
    q[0, 0, 0], q[0, 0, 1], q[F // 2, n // 2, 2] = 0, q[0, 0, 1] * 1e-39, q[F // 2, n // 2, 2] * 1e-30
    args = prefix, i32([P]), cache, i32(lens)
    out = ops.attn_kv8_shared(q, *args)
    check_shared(q, prefix, [P], cache, lens, None, out)
    bad = q.clone()
    bad[0, 0, 3, 5], bad[F - 1, n - 1, 1, 0], bad[F // 3, n // 3, 2] = float("inf"), float("nan"), 3e38
    o2 = ops.attn_kv8_shared(bad, *args)
    same = torch.ones(F, n, 2 * H, dtype=torch.bool, device=DEV)
    same[0, 0, 3], same[F - 1, n - 1, 1], same[F // 3, n // 3, 2] = False, False, False
    view = lambda t: t.view(F, n, 2 * H, D)
    assert torch.equal(view(out)[same], view(o2)[same]) and torch.isnan(view(o2)[F - 1, n - 1, 1]).all()
    flat = ops.attn_kv8_shared(q, *args, scale=0.0)
    check_shared(q, prefix, [P], cache, lens, None, flat, scale=0.0)


def test_attn_kv8_shared_lengths_beyond_the_caches_are_cut_off_and_recorded():
    H, D = 2, 64
    prefix, cache = filled((2,), H, 128, D, 1), filled((4,), H, 128, D, 2)
    q = torch.randn(4, 3, H, D, device=DEV, generator=torch.Generator(DEV).manual_seed(1)).to(BF)
    for plens, lens, counts in (([129, 5], [0, 0, 0, 0], [3, 3, 3, 3]), ([-1, 5], [1, 1, 1, 1], [1, 1, 1, 1]), ([5, 5], [127, 200, -7, 3], [3, 3, 0, 9]),
                                ([2 ** 31 - 1, -2 ** 31], [0] * 4, [0] * 4), ([1, 1], [2 ** 31 - 1, -2 ** 31, 0, 0], [2 ** 31 - 1, 1, -2 ** 31, 2])):
        out = torch.full((4, 3, H * D), 5.0, dtype=BF, device=DEV)
        ops.attn_kv8_shared(q, prefix, i32(plens), cache, i32(lens), out, counts=i32(counts))
        assert device_status(clear=True) == RANGE_BIT, (plens, lens, counts)
        pl, ln = np.clip(plens, 0, 128), np.clip(lens, 0, 128)
        ct = np.minimum(np.clip(counts, 0, 3), 128 - ln)
        check_shared(q, prefix, pl, cache, ln, ct, out)
        assert all((out[b, int(ct[b]):] == 5).all() for b in range(4))


def test_attn_kv8_shared_equals_attention_over_copies_of_the_prefix():
    """The same batch with the prefix copied in front of each sequence's own slots."""
    S, F, H, D, Hq, P, lens = 2, 20, 2, 128, 8, 640, [i * 11 % 128 for i in range(40)]
    prefix, cache = filled((S,), H, P, D, 1), filled((S * F,), H, 192, D, 2)
    q = torch.randn(S * F, 1, Hq, D, device=DEV, generator=torch.Generator(DEV).manual_seed(3)).to(BF)
    out = ops.attn_kv8_shared(q, prefix, i32([P] * S), cache, i32(lens))
    full = ops.Kv8(*(torch.cat([p.repeat_interleave(F, 0), c], dim=2) for p, c in zip(prefix, cache)))
    want = ops.attn_kv8(q, full, i32([P + x for x in lens]))
    # both round to bf16 and round P: two half steps of the value each, and 2^-11 of the terms (values below 6)
    assert torch.allclose(out.float(), want.float(), rtol=2.0 ** -7, atol=2.0 ** -8)


def test_attn_kv8_shared_one_workspace_for_calls_of_every_size_and_two_streams():
    H, D = 2, 64
    prefix, cache = filled((1,), H, 2048, D, 2), filled((48,), H, 256, D, 3)
    ws = ops.attn_kv8_shared_workspace(1, 48, 60, 4, H, D, 2048, 256, DEV)
    want = {}
    for n in (60, 12, 1):
        q = torch.randn(48, n, 4, D, device=DEV, generator=torch.Generator(DEV).manual_seed(n)).to(BF)
        lens = [b * 3 for b in range(48)]
        want[n] = q, lens, ops.attn_kv8_shared(q, prefix, i32([1990]), cache, i32(lens), ws=ws)
    check_shared(want[1][0], prefix, [1990], cache, want[1][1], None, want[1][2])
    s1, s2, got = torch.cuda.Stream(), torch.cuda.Stream(), []
    torch.cuda.synchronize()
    for _ in range(5):
        for s, n in ((s1, 60), (s2, 12), (s1, 1), (s2, 60), (s1, 12)):
            with torch.cuda.stream(s):
                got.append((n, ops.attn_kv8_shared(want[n][0], prefix, i32([1990]), cache, i32(want[n][1]))))
    torch.cuda.synchronize()
    for n, o in got:
        assert torch.equal(o, want[n][2]), n


# ------------------------------------------------------------------------------------------------ beam selection
def check_select(logits, scores, beams, k, eos, done, got):
    """Scores within their bound; beams and words those of the oracle wherever their totals are apart by more than that."""
    x = np_(logits.float())
    t = R.totals(x, np_(scores), beams, eos, None if done is None else np_(done))
    S, V = t.shape[0], x.shape[1]
    sc, pa, to, dn = (np_(y) for y in got)
    assert sc.shape == pa.shape == to.shape == dn.shape == (S, k)
    for s in range(S):
        order = np.argsort(-t[s], kind="stable")[:k]
        want = np.full(k, -np.inf)
        want[:len(order)] = t[s, order]
        fin = np.isfinite(want)
        assert (np.isneginf(sc[s]) == ~fin).all()
        # the exponentials' own error (2^-22), of their arguments (2^-23 of each, ln V + 1 on average over the sum at most) and of
        # 64 additions in fp32, and the total's rounding to fp32
        tol = 2.0 ** -22 + (np.log(V) + 1) * 2.0 ** -23 + 64 * 2.0 ** -24 + np.abs(want[fin]) * 2.0 ** -24
        assert (np.abs(sc[s][fin] - want[fin]) <= tol).all(), float((np.abs(sc[s][fin] - want[fin]) / tol).max())
        flat = (pa[s].astype(np.int64) - s * beams) * V + to[s]
        assert ((pa[s] >= s * beams) & (pa[s] < (s + 1) * beams)).all()
        assert (to[s][~fin] == -1).all() and (pa[s][~fin] == s * beams + np.flatnonzero(~fin) % beams).all() and dn[s][~fin].all()
        assert len(set(flat[fin])) == fin.sum()
        for j in np.flatnonzero(fin):
            if flat[j] != order[j]:  # another one, as good within the bound, of another beam
                near = abs(t[s, flat[j]] - want[j]) <= 2 * tol.max() and flat[j] // V != order[j] // V
                # or the totals are the same in the oracle's 64 bits, in which a logit of 2^-149 beside 9.9 is lost: exactly, the beam's
                # words of larger logits have larger totals, and the chosen one is among the beam's first k by logit and word
                f = flat[j] // V
                first = np.argsort(-x[s * beams + f].astype(np.float64), kind="stable")[:k]
                lost = t[s, flat[j]] == want[j] and f == order[j] // V and flat[j] % V in first
                assert near or lost, (s, j, flat[j], order[j])
            was = done is not None and bool(done[pa[s, j]])
            assert dn[s, j] == (was or to[s, j] == eos)


SELECT = [  # S, F, k, V, dtype, what
    (1, 1, 1, 1, "fp32", ""), (1, 1, 1, 51200, "bf16", ""), (1, 4, 4, 51200, "fp32", ""), (2, 4, 8, 1000, "bf16", "done"), (3, 5, 5, 777, "fp32", "done banned"),
    (1, 64, 128, 5000, "bf16", "done"), (2, 3, 6, 2, "fp32", ""), (1, 2, 128, 50, "bf16", ""), (1, 8, 8, 131071, "bf16", "banned"), (4, 8, 16, 8192, "fp32", "first"),
    (7, 6, 11, 8193, "bf16", "first banned"), (2, 33, 66, 2049, "fp32", "done"), (40, 2, 4, 300, "bf16", "done"), (1, 1, 128, 128, "fp32", ""), (1, 32, 64, 262144, "bf16", ""),
    (300, 1, 2, 4097, "fp32", ""), (1, 16, 100, 65537, "fp32", "banned done")]


def select_inputs(S, F, V, dtype, what, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    x = torch.randn(S * F, V, device=DEV, generator=g) * 3
    if "banned" in what:
        x[torch.rand(S * F, V, device=DEV, generator=g) < 0.5] = -float("inf")
        x[:, 0] = 1.0
    scores = -torch.rand(S * F, device=DEV, generator=g) * 5
    done = torch.rand(S * F, device=DEV, generator=g) < 0.3 if "done" in what else None
    if "first" in what:
        scores = torch.where(torch.arange(S * F, device=DEV) % F == 0, 0.0, -float("inf"))
    return x.to(BF) if dtype == "bf16" else x, scores, done


@pytest.mark.parametrize("S,F,k,V,dtype,what", SELECT)
def test_beam_select_matches_the_oracle(S, F, k, V, dtype, what):
    x, scores, done = select_inputs(S, F, V, dtype, what, V + k)
    eos = V // 3
    got = ops.beam_select(x, scores, F, k=k, eos=eos, done=done)
    check_select(x, scores, F, k, eos, done, got)
    again = ops.beam_select(x, scores, F, k=k, eos=eos, done=done)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("V,pad,at", [(1000, 1, 0), (1000, 0, 1), (1001, 7, 3), (4099, 5, 2), (51200, 8, 8), (20000, 3, 1)])
def test_beam_select_any_pitch_and_alignment(V, pad, at, dtype):
    """Rows of a wider matrix, wherever they begin; what lies between them (NaN) is never looked at."""
    S, F = 2, 3
    x, scores, _ = select_inputs(S, F, V, dtype, "", V)
    wide = torch.full((S * F * (V + pad) + at + 8,), float("nan"), dtype=x.dtype, device=DEV)
    view = wide[at:at + S * F * (V + pad)].view(S * F, V + pad)[:, :V]
    view.copy_(x)
    got = ops.beam_select(view, scores, F)
    check_select(x, scores, F, F, -1, None, got)


@pytest.mark.parametrize("V", [5, 700, 40000])
def test_beam_select_equal_totals_go_to_the_lowest_beam_and_word(V):
    """Equal logits in equal beams, zeros of both signs among them: in the order of their places."""
    S, F, k = 2, 4, 10
    x = torch.zeros(S * F, V, device=DEV)
    x[:, 1::2] = -0.0
    scores = torch.full((S * F,), -1.5, device=DEV)
    for y in (x, x.to(BF)):
        got = ops.beam_select(y, scores, F, k=k)
        assert np_(got.tokens).tolist() == [[j % V for j in range(k)]] * S
        assert np_(got.parents).tolist() == [[s * F + j // V for j in range(k)] for s in range(S)]
    y = torch.full((S * F, V), -2.0, device=DEV).to(BF)  # of two beams, two words each; the others have a lower score
    y[:, [3, V - 1]] = 4.0
    scores = torch.tensor([-3.0, -1.0, -3.0, -1.0] * S, device=DEV)
    got = ops.beam_select(y, scores, F, k=4)
    assert np_(got.tokens).tolist() == [[3, V - 1, 3, V - 1]] * S and np_(got.parents).tolist() == [[s * F + f for f in (1, 1, 3, 3)] for s in range(S)]


def test_beam_select_rows_that_have_nothing_to_say():
    """Rows of -inf, of the type's lowest value, with a NaN or an infinity; beams whose score is -inf, NaN or infinite."""
    inf, nan, V = float("inf"), float("nan"), 600
    for dt in (BF, torch.float32):
        low = torch.finfo(dt).min
        x = (torch.randn(8, V, device=DEV, generator=torch.Generator(DEV).manual_seed(1)) * 2).to(dt)
        x[0], x[1], x[2, 7], x[3, 9] = -inf, low, nan, inf
        x[4, 1:], x[5] = low, low
        x[5, 5] = 0.0
        scores = torch.tensor([0.0, -1.0, 0.0, 0.0, -2.0, -3.0, -inf, nan], device=DEV)
        got = ops.beam_select(x, scores, 8, k=128)
        check_select(x, scores, 8, 128, -1, None, got)
        # the beams of one open word come first, then the row of lowest values, its words by number
        assert np_(got.parents)[0, :3].tolist() == [4, 5, 1] and np_(got.tokens)[0, :6].tolist() == [0, 5, 0, 1, 2, 3]
        none = ops.beam_select(x[:4], scores[[6, 7, 6, 7]], 4, k=5)
        assert torch.isneginf(none.scores).all() and (none.tokens == -1).all() and none.done.all() and np_(none.parents)[0].tolist() == [0, 1, 2, 3, 0]
        alive = ops.beam_select(x[6:], torch.tensor([inf, -5.0], device=DEV), 2, k=2, eos=3, done=torch.tensor([False, True], device=DEV))
        assert alive.tokens[0, 1] != 3 or alive.parents[0, 1] == 0


def test_beam_select_finished_beams_keep_their_score():
    """A finished beam takes part with its score and eos alone, whatever its logits are (NaN here)."""
    V, eos = 900, 41
    x = torch.randn(4, V, device=DEV, generator=torch.Generator(DEV).manual_seed(2))
    x[1], x[3] = float("nan"), float("nan")
    scores, done = torch.tensor([-9.0, -0.5, -9.0, -30.0], device=DEV), torch.tensor([False, True, False, True], device=DEV)
    got = ops.beam_select(x, scores, 4, eos=eos, done=done)
    check_select(x, scores, 4, 4, eos, done, got)
    assert got.parents[0, 0] == 1 and got.tokens[0, 0] == eos and got.scores[0, 0] == -0.5 and got.done[0, 0]
    every = ops.beam_select(x, scores, 4, k=6, eos=eos, done=torch.ones(4, dtype=torch.bool, device=DEV))
    assert np_(every.parents)[0].tolist() == [1, 0, 2, 3, 0, 1] and np_(every.tokens)[0].tolist() == [eos] * 4 + [-1] * 2


def test_beam_select_clustered_words():
    """The best words next to one another, and spread at every distance that a kernel might give one thread."""
    V, F, k = 30000, 2, 64
    for step in (1, 2, 4, 8, 16, 32, 64, 128, 256, 512):
        x = torch.zeros(F, V, device=DEV)
        at = (torch.arange(40, device=DEV) * step + 1234)
        at = at[at < V]
        x[:, at] = torch.linspace(5, 9, len(at), device=DEV)
        scores = torch.tensor([0.0, -0.01], device=DEV)
        for y in (x, x.to(BF)):
            check_select(y, scores, F, k, -1, None, ops.beam_select(y, scores, F, k=k))


def test_beam_select_on_two_streams_and_in_place_of_its_outputs():
    x, scores, done = select_inputs(3, 8, 5000, "bf16", "done", 5)
    want = ops.beam_select(x, scores, 8, eos=7, done=done)
    out = ops.Beams(*(torch.zeros_like(t) for t in want))
    assert ops.beam_select(x, scores, 8, eos=7, done=done, out=out) is out
    assert all(torch.equal(a, b) for a, b in zip(want, out))
    s1, s2, got = torch.cuda.Stream(), torch.cuda.Stream(), []
    torch.cuda.synchronize()
    for _ in range(10):
        for s in (s1, s2):
            with torch.cuda.stream(s):
                got.append(ops.beam_select(x, scores, 8, eos=7, done=done))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(want, g))


# ------------------------------------------------------------------------------------------------ reordering
IN_PLACE = [  # layers, S, F, H, C, D, lens of the groups, parents within the group
    (1, 1, 1, 1, 64, 64, [5], [0]), (1, 1, 2, 2, 64, 128, [64], [1, 0]), (3, 2, 4, 3, 128, 64, [65, 1], [1, 2, 3, 0, 0, 0, 3, 2]),
    (2, 1, 4, 2, 192, 64, [190], [3, 3, 3, 3]), (1, 3, 5, 1, 320, 128, [0, 300, 129], [4, 3, 2, 1, 0, 1, 1, 2, 4, 4, 0, 0, 1, 1, 1]),
    (24, 1, 4, 4, 64, 64, [38], [0, 0, 1, 3]), (1, 1, 64, 2, 1024, 64, [1000], [(i * 7 + 3) % 64 for i in range(64)]), (2, 1, 33, 1, 128, 128, [100], [i * i % 33 for i in range(33)]),
    (1, 1, 3, 2, 8192, 128, [8001], [2, 0, 1])]


@pytest.mark.parametrize("layers,S,F,H,C,D,lens,parents", IN_PLACE)
def test_kv8_reorder_in_place_matches_the_oracle(layers, S, F, H, C, D, lens, parents):
    cache = filled((layers, S * F), H, C, D, F)
    ln = [x for x in lens for _ in range(F)]
    pa = [b // F * F + p for b, p in enumerate(parents)]
    want, wl = R.reorder(as_np(cache), pa, ln, F)
    new = torch.full((S * F,), -9, dtype=torch.int32, device=DEV)
    ops.kv8_reorder(cache, i32(pa), i32(ln), beams=F, new_lens=new)
    assert all(np.array_equal(np_(g), w) for g, w in zip(cache, want)) and np_(new).tolist() == wl.tolist()


def test_kv8_reorder_lengths_that_differ_within_a_group_and_one_layer():
    cache, pa, ln = filled((6,), 2, 256, 64, 3), [1, 0, 2, 5, 3, -1], [10, 200, 65, 0, 64, 256]
    want, wl = R.reorder([t[None] for t in as_np(cache)], pa, ln, 3)
    new = torch.zeros(6, dtype=torch.int32, device=DEV)
    ops.kv8_reorder(cache, i32(pa), i32(ln), beams=3, new_lens=new)
    assert all(np.array_equal(np_(g), w[0]) for g, w in zip(cache, want)) and np_(new).tolist() == wl.tolist()


FORK = [  # layers, Bs, B, H, C, dst C, D, lens, parents
    (1, 1, 1, 1, 64, 64, 64, [3], [0]), (2, 3, 5, 2, 192, 256, 64, [190, 0, 64], [2, 2, 0, 1, -1]), (1, 4, 2, 3, 320, 128, 128, [100, 128, 65, 1], [3, 1]),
    (1, 2, 70, 1, 128, 128, 128, [127, 128], [i % 2 for i in range(70)]), (24, 1, 4, 4, 768, 768, 64, [730], [0] * 4), (1, 3, 3, 2, 4096, 4160, 128, [4095, 4000, 63], [1, 2, 0])]


@pytest.mark.parametrize("layers,Bs,B,H,C,Cd,D,lens,parents", FORK)
def test_kv8_reorder_into_another_cache_matches_the_oracle(layers, Bs, B, H, C, Cd, D, lens, parents):
    cache, dst = filled((layers, Bs), H, C, D, B), filled((layers, B), H, Cd, D, B + 1)
    before = as_np(cache)
    want, wl = R.reorder(before, parents, lens, dst=as_np(dst), new_lens=[-9] * B)
    new = torch.full((B,), -9, dtype=torch.int32, device=DEV)
    ops.kv8_reorder(cache, i32(parents), i32(lens), dst=dst, new_lens=new)
    assert all(np.array_equal(np_(g), w) for g, w in zip(dst, want)) and np_(new).tolist() == wl.tolist()
    assert all(np.array_equal(np_(g), w) for g, w in zip(cache, before))


def test_kv8_reorder_parents_and_lengths_out_of_range_are_recorded():
    for pa, ln in (([4, 1, 2, 3], [9] * 4), ([0, 1, 0, 3], [9] * 4), ([2 ** 31 - 1, 0, 3, 2], [9] * 4), ([1, 0, 2, 3], [129] * 4), ([1, 0, 3, 2], [-1, 9, 9, 2 ** 31 - 1])):
        cache = filled((4,), 2, 128, 64, 3)
        want, wl = R.reorder([t[None] for t in as_np(cache)], pa, ln, 2)
        ops.kv8_reorder(cache, i32(pa), i32(ln), beams=2)
        assert device_status(clear=True) == RANGE_BIT, (pa, ln)
        assert all(np.array_equal(np_(g), w[0]) for g, w in zip(cache, want)), (pa, ln)
    cache, dst = filled((2,), 1, 128, 64, 3), filled((3,), 1, 64, 64, 4)
    want, _ = R.reorder([t[None] for t in as_np(cache)], [0, 2, -5], [100, 3], dst=[t[None] for t in as_np(dst)])
    ops.kv8_reorder(cache, i32([0, 2, -5]), i32([100, 3]), dst=dst)
    assert device_status(clear=True) == RANGE_BIT and all(np.array_equal(np_(g), w[0]) for g, w in zip(dst, want))


# ------------------------------------------------------------------------------------------------ together
def test_write_attend_choose_and_reorder_eager_captured_and_on_another_stream():
    """Steps of a beam search over two prefixes: each step's rows are written, attended to, the continuations chosen from logits, and
    the caches follow; eagerly, replayed from one captured graph, and on another stream, all bit for bit, and the first against the oracle."""
    S, F, H, Hq, D, P, V, steps = 2, 4, 2, 4, 64, 150, 2000, 5
    B, C = S * F, 128
    cos, sin = rope_tables(TEXT.__class__(prefix=1024, q_len=0), DEV)
    prefix, plens = filled((S,), H, 192, D, 1), i32([P, 64])
    g = torch.Generator(DEV).manual_seed(5)
    table = torch.randn(V, (Hq + 2 * H) * D, device=DEV, generator=g).to(BF)
    head = torch.randn(Hq * D, V, device=DEV, generator=g) * 0.3

    def fresh():
        c = ops.kv8_cache(B, H, C, D, DEV)
        return {"c": c, "lens": torch.zeros(B, dtype=torch.int32, device=DEV), "tok": torch.arange(B, dtype=torch.int32, device=DEV),
                "q": torch.zeros(B, 1, Hq, D, dtype=BF, device=DEV), "out": torch.zeros(B, 1, Hq * D, dtype=BF, device=DEV),
                "scores": torch.where(torch.arange(B, device=DEV) % F == 0, 0.0, -1e9), "done": torch.zeros(B, dtype=torch.bool, device=DEV)}

    def step(s):
        qkv = table[s["tok"].clamp(min=0).long()][:, None].contiguous()
        ops.rope_kv8(qkv, s["c"], s["lens"], cos, sin, s["q"], pos=plens.repeat_interleave(F) + s["lens"])
        ops.attn_kv8_shared(s["q"], prefix, plens, s["c"], s["lens"], s["out"])
        s["lens"] += 1
        best = ops.beam_select(s["out"].view(B, -1).float() @ head, s["scores"], F, eos=3, done=s["done"])
        ops.kv8_reorder(s["c"], best.parents.view(-1), s["lens"], beams=F)
        for n, t in (("scores", best.scores), ("tok", best.tokens), ("done", best.done)):
            s[n].copy_(t.view(-1))
        return best

    eager = fresh()
    for i in range(steps):
        before = as_np(eager["c"])
        best = step(eager)
        if i == 0:
            ro, mag = R.attention_shared(np_(eager["q"].float()), as_np(prefix), [P, 64], as_np(eager["c"]), [0] * B)
            # one token of its own each, and the beams of a group may have changed places since: the oracle on what was written then
            rows = np_(eager["out"].float())
            assert np.isfinite(rows).all() and best.scores.isfinite().any()
    assert np_(eager["lens"]).tolist() == [steps] * B
    other = fresh()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(steps):
            step(other)
    torch.cuda.synchronize()
    graphed, warm = fresh(), fresh()
    step(warm)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(graphed)
    for _ in range(steps):
        graph.replay()
    torch.cuda.synchronize()
    for s in (other, graphed):
        for n in ("lens", "tok", "out", "scores", "done"):
            assert torch.equal(s[n], eager[n]), n
        assert all(torch.equal(a, b) for a, b in zip(s["c"], eager["c"]))


@pytest.mark.parametrize("k", [1, 7, 16, 33, 64, 128])
def test_beam_select_crowds_of_equal_words_beside_close_ones(k):
    """Most words equal (a mask by the lowest value, or a flat row), a few just above and below them by as little as the type can tell."""
    V, F = 20000, 2
    g = torch.Generator(DEV).manual_seed(k)
    for dt in (torch.float32, BF):
        for base in (torch.finfo(dt).min, -3.0, 0.0, 2.5):
            x = torch.full((F, V), base, device=DEV, dtype=dt)
            at = torch.randperm(V, device=DEV, generator=g)[:300]
            up, down = (torch.nextafter(x[0, :1], torch.tensor([s], device=DEV, dtype=dt)) for s in (float("inf"), -float("inf")))
            x[:, at[:k // 2]] = up
            if base != torch.finfo(dt).min:
                x[:, at[100:]] = down
            scores = torch.tensor([0.0, -1.0], device=DEV)
            check_select(x, scores, F, k, -1, None, ops.beam_select(x, scores, F, k=k))
