"""The 8-bit KV cache where its kernels take another way than at ordinary sizes: clusters, runs of tiles over many sequences,
row groups, extreme weights, scales and queries; against oracle/kv8_ref.py or sums in 64 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from strix_halo_maxx_b200 import ops
from strix_halo_maxx_b200._lib import device_status
from oracle import kv8_ref as R
from test_kv8_gpu import BF, DEV, as_np, filled, i32, np_, tables


@pytest.fixture(autouse=True)
def _status():
    device_status(clear=True)
    yield
    assert device_status(clear=True) == 0


# ------------------------------------------------------------------------------------------------ eviction
@pytest.mark.parametrize("B,H,D,C,lens,keep,recent", [
    (1, 2, 64, 20032, [20000], 4096, 4096),            # a cluster of two; nothing is chosen by weight
    (1, 1, 128, 40000, [39999], 64, 64), (2, 1, 64, 70016, [70016, 4000], 4096, 4096), (1, 3, 64, 140032, [140000], 128, 127)])
def test_kv8_evict_over_clusters_with_few_or_no_places_left_for_weights(B, H, D, C, lens, keep, recent):
    cache = filled(B, H, C, D, recent)
    w = torch.rand(B, H, C, device=DEV, generator=torch.Generator(DEV).manual_seed(1))
    dst, dw, dl = ops.kv8_cache(B, H, keep, D, DEV), torch.zeros(B, H, keep, device=DEV), i32([0] * B)
    ref = R.evict(as_np(cache), np_(w), lens, keep, recent)
    for _ in range(3):
        idx = ops.kv8_evict(cache, w, i32(lens), keep, recent, dst, dw, dl)
        assert np_(dl).tolist() == [min(x, keep) for x in lens]
        for b in range(B):
            if ref[b] is None:
                assert np.array_equal(np_(idx)[b, :, :lens[b]], np.tile(np.arange(lens[b]), (H, 1)))
                continue
            assert np.array_equal(np_(idx)[b], ref[b][0])
            assert np.array_equal(np_(dw)[b], np.take_along_axis(np_(w)[b], ref[b][0], -1))
            for got, want in zip(as_np(dst), ref[b][1:]):
                assert np.array_equal(got[b], want)


# ------------------------------------------------------------------------------------------------ attention
def attention64(q, cache, lens, counts=None, causal=True, scale=None, w_in=None):
    """out, weights, the sums of p |v| behind each output and a bound on the error of each weight (scores in fp32, as in
    oracle.kv8_ref.attention), in 64 bits on the GPU; rows past the count and slots past the end NaN."""
    B, H, C, D = cache.k.shape
    n, Hq = q.shape[1:3]
    G, scale = Hq // H, D ** -0.5 if scale is None else scale
    nan = lambda *s: torch.full(s, float("nan"), dtype=torch.float64, device=DEV)
    out, mag, w, werr = nan(B, n, Hq, D), nan(B, n, Hq, D), nan(B, H, C), nan(B, H, C)
    for b in range(B):
        L, m = lens[b], n if counts is None else counts[b]
        T = L + m
        blk = torch.arange(T, device=DEV) // 64
        w[b, :, :T], werr[b, :, :T] = 0, 0
        if w_in is not None:
            w[b, :, :L] = w_in[b, :, :L].double()
        for h in range(H if m else 0):
            k, v = (c[b, h, :T].double() * s[b, h, blk].double()[:, None] for c, s in ((cache.k, cache.ks), (cache.v, cache.vs)))
            x = q[b, :m, h * G:h * G + G].double().reshape(m * G, D)
            z = x @ k.T * scale
            d = ((x.abs() @ k.abs().T) * (abs(scale) * D * 2.0 ** -24) + z.abs() * 2.0 ** -22)
            if causal:
                i = torch.arange(m, device=DEV).repeat_interleave(G)[:, None]
                hide = torch.arange(T, device=DEV)[None] > L + i
                z.masked_fill_(hide, -float("inf"))
                d.masked_fill_(hide, 0)
            p = torch.softmax(z, -1)
            out[b, :m, h * G:h * G + G] = (p @ v).view(m, G, D)
            mag[b, :m, h * G:h * G + G] = (p @ v.abs()).view(m, G, D)
            w[b, h, :T] += p.sum(0)
            werr[b, h, :T] += (p * 2 * d.amax(-1, keepdim=True)).sum(0)
    return out.flatten(2), w, mag.flatten(2), werr


def check64(q, cache, lens, counts, causal, out, w=None, w_in=None, scale=None, random_v=True):
    """Outputs: the rounding to bf16, half a step or 2^-8 of the value; P in 11 bits, 2^-11 of each term p |v|; scores and sums
    in fp32, below 2^-12 of the terms (|score| < 100).  Where V has both signs the roundings of P are independent and
    add in squares to an eighth of the output's own: 1.01 of it in the 2-norm, 1.1 allowed."""
    ro, rw, mag, werr = attention64(q, cache, lens, counts, causal, scale, w_in)
    at = ~torch.isnan(ro)
    err, bound = (out.double() - ro).abs()[at], (ro.abs() * 2.0 ** -8 + mag * (2.0 ** -11 + 2.0 ** -12))[at]
    assert (err <= bound * (1 + 2.0 ** -7)).all(), float((err / bound).max())
    if random_v:
        own = (ro.to(torch.bfloat16).double() - ro)[at].norm()
        assert err.norm() <= 1.1 * own, float(err.norm() / own)
    if w is not None:
        n, G, at = q.shape[1], q.shape[2] // cache.k.shape[1], ~torch.isnan(rw)
        tol = werr + rw.abs() * (2.0 ** -18 + (n * G + 1) * 2.0 ** -24) + 1e-30
        err, tol = (w.double() - rw).abs()[at], tol[at]
        assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("gap", [9.0, 15.0, 17.0, 17.6])
@pytest.mark.parametrize("n,D,T,Hq", [(1, 64, 730, 2), (1, 128, 500, 8), (32, 64, 762, 2), (32, 128, 400, 2), (5, 64, 2500, 6), (1, 128, 2500, 4)])
def test_attn_kv8_few_rows_keep_what_stands_beside_a_sink(n, D, T, Hq, gap):
    """One key takes nearly all the weight and its value is zero, so the output is made of weights e^-gap: as exact as others."""
    _sink(n, D, T, Hq, gap)


def _sink(n, D, T, Hq, gap):
    H, C = 2, (T + 63) // 64 * 64
    cache = filled(1, H, C, D, n)
    cache.k.zero_()
    cache.ks.fill_(1 / 128)
    cache.v.copy_(cache.v.abs() // 4 + 90)   # one sign: the losses would add up
    cache.k[:, :, 3, 0] = 127
    cache.v[:, :, 3] = 0
    q = torch.randn(1, n, Hq, D, device=DEV, generator=torch.Generator(DEV).manual_seed(2)).to(BF)
    q[..., 0] = 1
    out = ops.attn_kv8(q, cache, i32([T - n]), scale=gap * 128 / 127)
    check64(q, cache, [T - n], None, True, out, scale=gap * 128 / 127, random_v=False)


@pytest.mark.parametrize("n,D,T,Hq", [(1, 64, 730, 2), (2, 128, 2500, 8), (32, 64, 762, 2), (60, 64, 762, 2)])
def test_attn_kv8_queries_with_one_value_far_above_the_others(n, D, T, Hq):
    """The scores come from values 2^-22 of the row's largest, which meets keys that are zero there."""
    H, C = 2, (T + 63) // 64 * 64
    cache = filled(1, H, C, D, n)
    cache.k[..., 7] = 0
    cache.ks.fill_(1.0)
    q = (torch.randn(1, n, Hq, D, device=DEV, generator=torch.Generator(DEV).manual_seed(2)) * 2.0 ** -12).to(BF)
    q[..., 7] = 1024
    w = torch.zeros(1, H, C, device=DEV)
    out = ops.attn_kv8(q, cache, i32([T - n]), scale=16.0, weights=w)
    check64(q, cache, [T - n], None, True, out, w, scale=16.0)


@pytest.mark.parametrize("gap", [9.0, 15.0, 17.0, 17.6])
@pytest.mark.parametrize("n,D,T,Hq", [(64, 64, 730, 2), (200, 128, 1000, 4), (70, 64, 2500, 2), (300, 128, 2500, 2)])
def test_attn_kv8_many_rows_keep_what_stands_beside_a_sink(n, D, T, Hq, gap):
    _sink(n, D, T, Hq, gap)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n,Hq,H,D,L", [(730, 4, 4, 64, 0), (40, 8, 2, 128, 700), (513, 4, 2, 128, 2000), (129, 2, 2, 64, 3000), (16, 4, 2, 64, 500)])
def test_attn_kv8_rounds_its_probabilities_to_11_bits(n, Hq, H, D, L, causal):
    """The output's own rounding to bf16 is what is left of the error; V's scales differ from block to block by up to 2^12, some
    blocks are all zeros, and rows rescale (the largest scores come late)."""
    C = (L + n + 63) // 64 * 64
    cache = filled(1, H, C, D, n)
    g = torch.Generator(DEV).manual_seed(L + n)
    cache.vs.copy_(2.0 ** (torch.rand(cache.vs.shape, device=DEV, generator=g) * 12 - 6))
    cache.vs[:, :, 1::7] = 0
    cache.ks.mul_(torch.linspace(0.5, 3, C // 64, device=DEV))
    q = (torch.randn(1, n, Hq, D, device=DEV, generator=g) * 1.5).to(BF)
    w = torch.zeros(1, H, C, device=DEV)
    out = ops.attn_kv8(q, cache, i32([L]), causal=causal, weights=w)
    check64(q, cache, [L], None, causal, out, w)


def test_attn_kv8_many_rows_take_scales_over_their_whole_range():
    """V scales of 2^-100 and of 2^100, beside zeros; weights count every key."""
    H, D, n, C = 2, 64, 80, 512
    for e in (-100, -60, 60, 99):
        cache = filled(1, H, C, D, 3)
        cache.vs.mul_(2.0 ** e / 0.03)
        cache.vs.clamp_(min=2.0 ** -100)
        cache.vs[:, :, 2] = 0
        q = torch.randn(1, n, H, D, device=DEV, generator=torch.Generator(DEV).manual_seed(2)).to(BF)
        w = torch.zeros(1, H, C, device=DEV)
        out = ops.attn_kv8(q, cache, i32([C - n]), weights=w)
        check64(q, cache, [C - n], None, True, out, w)


@pytest.mark.parametrize("n,C", [(40, 2048), (40, 512), (1, 2048), (1, 512)])
@pytest.mark.parametrize("lens,counts", [([5000, 100], None), ([100, 2 ** 31 - 1], [1, 0]), ([-7, 100], [0, 1]), ([100, 64], [1, -1]), ([100, 64], [1, 2 ** 31 - 1])])
def test_attn_kv8_records_every_length_beyond_the_cache(n, C, lens, counts):
    """In every plan, and for sequences that are left without work by it; their rows stay as they were."""
    cache = filled(2, 2, C, 64, 5)
    q = torch.randn(2, n, 2, 64, device=DEV, generator=torch.Generator(DEV).manual_seed(2)).to(BF)
    out = torch.full((2, n, 128), 3.0, dtype=BF, device=DEV)
    ops.attn_kv8(q, cache, i32(lens), out, counts=None if counts is None else i32(counts))
    assert device_status(clear=True) == 1 << 9
    for b in range(2):
        L, m = min(max(lens[b], 0), C), n if counts is None else min(max(counts[b], 0), n)
        m = min(m, C - L)
        assert (out[b, m:] == 3).all() and (out[b, :m] != 3).any(-1).all()


def test_an_empty_batch_and_no_new_tokens_are_calls_that_do_nothing():
    for B, n in ((0, 3), (0, 0), (2, 0)):
        cache, q = ops.kv8_cache(B, 2, 128, 64, DEV), torch.zeros(B, n, 4, 64, dtype=BF, device=DEV)
        cos = torch.zeros(8, 16, device=DEV)
        assert ops.rope_kv8(torch.zeros(B, n, 512, dtype=BF, device=DEV), cache, i32([0] * B), cos, cos, q) is q
        assert ops.attn_kv8(q, cache, i32([0] * B)).shape == (B, n, 256)
        assert ops.attn_kv8(q, cache, i32([0] * B), weights=torch.zeros(B, 2, 128, device=DEV)).shape == (B, n, 256)
    cache = ops.kv8_cache(0, 2, 128, 64, DEV)
    w = torch.zeros(0, 2, 128, device=DEV)
    assert ops.kv8_evict(cache, w, i32([]), 64, 8, ops.kv8_cache(0, 2, 64, 64, DEV), w[:, :, :64].contiguous(), i32([])).shape == (0, 2, 64)


def test_kv8_evict_zero_codes_under_scales_far_apart():
    """Zeros stay zeros whatever their block's scale was: 1e30 beside 1e-20, whose ratio is no finite number."""
    cache = filled(1, 2, 256, 64, 2)
    cache.k[:, :, :64] = 0
    cache.v[:, :, 64:128] = 0
    cache.ks[:, :, 0], cache.vs[:, :, 1] = 1e30, 1e30
    cache.ks[:, :, 1:] = 1e-20
    cache.vs[:, :, 0], cache.vs[:, :, 2:] = 1e-20, 1e-20
    w = torch.rand(1, 2, 256, device=DEV, generator=torch.Generator(DEV).manual_seed(4))
    dst, dw, dl = ops.kv8_cache(1, 2, 128, 64, DEV), torch.zeros(1, 2, 128, device=DEV), i32([0])
    idx = ops.kv8_evict(cache, w, i32([256]), 128, 0, dst, dw, dl)
    (ri, *want), = R.evict(as_np(cache), np_(w), [256], 128, 0)
    assert np.array_equal(np_(idx)[0], ri)
    for got, x in zip(as_np(dst), want):
        assert np.array_equal(got[0], x)


def test_attn_kv8_weights_of_many_heads_over_a_very_long_cache():
    """128 query heads on one kv head over 17 million slots: (slots - length) * heads passes 31 bits."""
    C, D, G = 17_000_000, 64, 128
    g = torch.Generator(DEV).manual_seed(1)
    k, v = (torch.randint(-127, 128, (1, 1, C, D), dtype=torch.int8, device=DEV, generator=g) for _ in range(2))
    ks, vs = (torch.rand(1, 1, C // 64, device=DEV, generator=g) * 0.01 + 0.01 for _ in range(2))
    cache = ops.Kv8(k, v, ks, vs)
    q = torch.randn(1, 1, G, D, device=DEV, generator=g).to(BF)
    w = torch.zeros(1, 1, C, device=DEV)
    out = ops.attn_kv8(q, cache, i32([C - 1]), weights=w)
    x, step = q[0, 0].double() * D ** -0.5, 64 * 15625
    vals = lambda c, s, at: c[0, 0, at:at + step].double() * s[0, 0, at // 64:(at + step) // 64].double().repeat_interleave(64)[:, None]
    lse = torch.stack([torch.logsumexp(x @ vals(k, ks, at).T, -1) for at in range(0, C, step)]).logsumexp(0)
    o = torch.zeros(G, D, dtype=torch.float64, device=DEV)
    for at in range(0, C, step):
        p = torch.exp(x @ vals(k, ks, at).T - lse[:, None])
        o += p @ vals(v, vs, at)
        # scores of up to 30 in fp32, 128 rows: far below 2^-12 of a weight
        assert torch.allclose(w[0, 0, at:at + step].double(), p.sum(0), rtol=2.0 ** -12, atol=0), at
    # means of 17 million values of both signs: small beside the values, whose rounded weights and fp32 sums leave 2^-12 of their size
    assert (out[0, 0].view(G, D).double() - o).abs().max() <= o.abs().max() * 2.0 ** -8 + 2.0 ** -12


FEW = [  # B, n, Hq, H, D, C, lens, counts: D = 128 with two row groups (17 to 32 rows), whole items and runs; two of eight rows in runs
    (3, 8, 8, 2, 128, 512, [400, 0, 33], [8, 3, 5]), (2, 5, 4, 1, 128, 512, [500, 31], [5, 1]), (4, 8, 8, 2, 128, 2048, [2000, 1, 64, 1500], [8, 4, 0, 2]),
    (2, 6, 20, 4, 128, 4096, [4000, 900], None), (3, 7, 8, 2, 128, 1024, [512, 1000, 0], [7, 0, 4]), (2, 4, 8, 2, 128, 2048, [1111, 2000], None),
    (3, 4, 12, 3, 64, 2048, [1999, 5, 1025], [4, 1, 3]), (5, 8, 12, 3, 64, 4096, [3000, 0, 4088, 64, 2000], [8, 5, 2, 0, 8]), (40, 1, 32, 8, 128, 2048, [50 * i for i in range(40)], None)]


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("B,n,Hq,H,D,C,lens,counts", FEW)
def test_attn_kv8_few_rows_in_every_plan(B, n, Hq, H, D, C, lens, counts, causal, weights):
    _attend(B, n, Hq, H, D, C, lens, counts, causal, weights)


MANY = [  # runs of tiles that end inside an item, hold whole ones and begin another; sequences of every length, idle ones among them
    (6, 300, 32, 16, 64, 1856, [1500, 300, 0, 700, 64, 1000], [300, 211, 300, 0, 1, 130]), (5, 90, 16, 8, 128, 2176, [2000, 1500, 0, 1900, 37], [90, 0, 60, 17, 90]),
    (4, 140, 8, 8, 128, 1664, [1500, 640, 1, 1024], None), (1, 600, 12, 4, 64, 2560, [1900], None), (7, 64, 32, 8, 128, 1600, [1536, 1000, 500, 250, 100, 50, 0], [64, 0, 64, 33, 64, 0, 64]),
    (3, 65, 5, 1, 64, 4160, [4000, 0, 2048], [65, 65, 30]), (12, 40, 20, 10, 64, 1600, [130 * i for i in range(12)], [40 - 3 * i for i in range(12)]),
    (3, 200, 4, 2, 64, 1536, [1300, 0, 512], [200, 200, 0])]


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("B,n,Hq,H,D,C,lens,counts", MANY)
def test_attn_kv8_many_rows_in_every_plan(B, n, Hq, H, D, C, lens, counts, causal, weights):
    _attend(B, n, Hq, H, D, C, lens, counts, causal, weights)


def _attend(B, n, Hq, H, D, C, lens, counts, causal, weights):
    cache = filled(B, H, C, D, n + Hq)
    g = torch.Generator(DEV).manual_seed(n)
    # keys that grow along the cache, so that rows rescale late in a run
    cache.ks.mul_(torch.linspace(0.4, 2.5, C // 64, device=DEV))
    q = (torch.randn(B, n, Hq, D, device=DEV, generator=g) * 1.5).to(BF)
    out = torch.full((B, n, Hq * D), 3.0, dtype=BF, device=DEV)
    w = torch.full((B, H, C), -1.0, device=DEV) if weights else None
    w_in = torch.rand(B, H, C, device=DEV, generator=g) if weights else None
    ops.attn_kv8(q, cache, i32(lens), out, counts=None if counts is None else i32(counts), causal=causal, weights=w, weights_in=w_in)
    check64(q, cache, lens, counts, causal, out, w, w_in)
    for b in range(B):
        m = n if counts is None else counts[b]
        assert (out[b, m:] == 3).all() and (w is None or (w[b, :, lens[b] + m:] == -1).all())


@pytest.mark.parametrize("n", [1, 5, 70])
def test_rows_side_by_side_in_one_buffer(n):
    """q beside qkv, and out beside q, as columns of one matrix: the same numbers as in buffers of their own."""
    B, Hq, H, D = 2, 4, 2, 64
    g = torch.Generator(DEV).manual_seed(n)
    wide = torch.randn(B, n, 1024, device=DEV, generator=g).to(BF)
    qkv, q, out = wide[..., :512], wide[..., 512:768].view(B, n, Hq, D), wide[..., 768:]
    cos, sin = tables()
    a, b = (filled(B, H, 256, D, 4) for _ in range(2))
    q2 = ops.rope_kv8(qkv.clone(), b, i32([3, 90]), cos, sin, torch.zeros(B, n, Hq, D, dtype=BF, device=DEV))
    ops.rope_kv8(qkv, a, i32([3, 90]), cos, sin, q)
    ops.attn_kv8(q, a, i32([3, 90]), out)
    assert torch.equal(q, q2) and torch.equal(out, ops.attn_kv8(q2, b, i32([3, 90])))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("gap,at,e", [(12.0, 0, 0), (25.0, 0, 0), (40.0, 0, 0), (25.0, 200, 0), (40.0, 200, 0), (40.0, 129, 0), (12.0, 0, -85), (40.0, 0, 90), (40.0, 200, 90)])
@pytest.mark.parametrize("n,D,T,Hq", [(64, 64, 730, 2), (200, 128, 1000, 4), (70, 64, 2500, 2), (300, 128, 2500, 2)])
def test_attn_kv8_many_rows_beside_a_block_of_zero_values(n, D, T, Hq, gap, at, e):
    """The key that takes the weight lies in a block whose values are all zero (scale 0): it counts in the sum alone, and what
    the others add up to is as exact as without it, e^-40 of its weight or not, and with scales around 2^e."""
    H, C = 2, (T + 63) // 64 * 64
    cache = filled(1, H, C, D, n)
    cache.k.zero_()
    cache.ks.fill_(1 / 128)
    cache.v.copy_(cache.v.abs() // 4 + 90)
    cache.k[:, :, at, 0] = 127
    cache.vs.mul_(2.0 ** e)
    cache.vs[:, :, at // 64] = 0
    cache.vs[:, :, 7] = 2.0 ** -90   # and one whose values are next to nothing
    q = torch.randn(1, n, Hq, D, device=DEV, generator=torch.Generator(DEV).manual_seed(2)).to(BF)
    q[..., 0] = 1
    w = torch.zeros(1, H, C, device=DEV)
    out = ops.attn_kv8(q, cache, i32([T - n]), causal=False, scale=gap * 128 / 127, weights=w)
    check64(q, cache, [T - n], None, False, out, w, scale=gap * 128 / 127, random_v=False)
