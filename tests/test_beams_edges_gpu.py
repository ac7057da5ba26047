"""Many answers about one context where they are likeliest to go wrong: blocks of zero values beside sinks, groups of very many query heads,
offsets beyond 32 bits, workspaces of several calls in one graph."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from strix_halo_maxx_b200 import ops
from strix_halo_maxx_b200._lib import device_status
from oracle import beam_ref as R
from test_beams_gpu import DEV, BF, as_np, check_select, check_shared, filled, i32, np_, up64


@pytest.fixture(autouse=True)
def _status():
    device_status(clear=True)
    yield
    assert device_status(clear=True) == 0


@pytest.mark.parametrize("gap", [2.0, 12.0, 25.0, 40.0])
@pytest.mark.parametrize("F,n,D", [(4, 1, 64), (40, 1, 64), (20, 2, 128), (2, 70, 64), (2, 150, 128), (64, 1, 128)])
def test_attn_kv8_shared_beside_blocks_of_zero_values(F, n, D, gap):
    """Blocks whose values are all zero (scale 0) hold keys `gap` nats above or below all others, in the prefix and in the sequences' own
    slots: they count in the sum alone, and the other terms keep their bits."""
    H, P, L = 2, 330, 130
    prefix, cache = filled((1,), H, 384, D, 5, spread=0.0), filled((F,), H, up64(L + n), D, 6, spread=0.0)
    g = torch.Generator(DEV).manual_seed(F)
    q = torch.randn(F, n, H, D, device=DEV, generator=g).to(BF) * 0.3
    q[..., 0] = 1.0
    for c in (prefix, cache):
        c.ks.fill_(0.01)
        c.k[..., 0] = 0
    step = int(gap * D ** 0.5 / 0.01)  # a score of gap: q[0] k[0] 0.01 D^-1/2, k's codes end at 127: the scales of these blocks are larger
    for c, block, sign in ((prefix, 0, 1), (prefix, 3, -1), (cache, 1, 1)):
        c.vs[:, :, block] = 0
        c.ks[:, :, block] = max(step / 100, 1) * 0.01
        c.k[:, :, block * 64:block * 64 + 64, 1:] = 0
        c.k[:, :, block * 64 + 7, 0] = sign * min(step, 100)
    out = ops.attn_kv8_shared(q, prefix, i32([P]), cache, i32([L] * F))
    ro, mag = R.attention_shared(np_(q.float()), as_np(prefix), [P], as_np(cache), [L] * F)
    # the sinks leave exp(-gap) of the output: its own size is what errors are held to.  With many rows P's f16 has 11 bits down to 2^-21 of
    # the row's largest product with a V scale (no zero block has one), 2^-38 of it below that.  The kernel for few rows of a sequence, which
    # may take either cache, knows weights only: below 2^-29 of the largest (1 at most) a term is off by 2^-40 of it
    bound = np.abs(ro) * 2.0 ** -8 + mag * (2.0 ** -10 + 2.0 ** -11) + 1e-30
    if n <= 32:
        bound += 2.0 ** -40 * (P + L + n) * 127 * float(max(prefix.vs.max(), cache.vs.max()))
    err = np.abs(np_(out.float()) - ro)
    assert (err <= bound).all(), float((err / bound).max())


BIG = [  # S, F, n, Hq, H, D, P, L: many query heads a kv head, one token's heads over several items
    (1, 2, 1, 150, 1, 64, 200, 30), (1, 1, 1, 33, 1, 128, 70, 64), (2, 3, 2, 130, 2, 128, 64, 1), (1, 1, 3, 300, 1, 64, 0, 0), (1, 5, 1, 257, 1, 64, 1, 63)]


@pytest.mark.parametrize("S,F,n,Hq,H,D,P,L", BIG)
def test_attn_kv8_shared_of_many_query_heads(S, F, n, Hq, H, D, P, L):
    B = S * F
    prefix, cache = filled((S,), H, up64(P), D, 1), filled((B,), H, up64(L + n), D, 2)
    q = torch.randn(B, n, Hq, D, device=DEV, generator=torch.Generator(DEV).manual_seed(Hq)).to(BF)
    counts = [n - b % 2 for b in range(B)]
    out = torch.zeros(B, n, Hq * D, dtype=BF, device=DEV)
    ops.attn_kv8_shared(q, prefix, i32([P] * S), cache, i32([L] * B), out, counts=i32(counts))
    check_shared(q, prefix, [P] * S, cache, [L] * B, counts, out)


@pytest.mark.parametrize("F", [2, 40])
def test_attn_kv8_shared_offsets_beyond_32_bits(F):
    """The last of nine heads of a prefix of 2^21 slots: its codes lie beyond 2^31 bytes."""
    H, D, P = 9, 128, (1 << 21) - 5
    prefix, cache = ops.kv8_cache(1, H, 1 << 21, D, DEV), filled((F,), H, 64, D, 3)
    g = torch.Generator(DEV).manual_seed(1)
    for t in prefix[:2]:
        t[0, H - 1] = torch.randint(-127, 128, (1 << 21, D), dtype=torch.int8, device=DEV, generator=g)
    for t in prefix[2:]:
        t.fill_(0.01)
    q = torch.randn(F, 1, H, D, device=DEV, generator=g).to(BF)
    out = ops.attn_kv8_shared(q, prefix, i32([P]), cache, i32([5] * F)).view(F, H, D)[:, H - 1]
    for f in (0, F - 1):
        kf, vf = (torch.cat([p[0, H - 1, :P].double() * float(torch.tensor(0.01)), c[f, H - 1, :6].double() * s[f, H - 1, 0].double()])
                  for p, c, s in zip(prefix[:2], cache[:2], cache[2:]))
        p = torch.softmax(kf @ q[f, 0, H - 1].double() * D ** -0.5, 0)
        want, mag = p @ vf, p @ vf.abs()
        # outputs average two million values to nearly nothing: held to the rounding of P (2^-11, random over the terms) and of sums in fp32
        assert ((out[f].double() - want).abs() <= want.abs() * 2.0 ** -8 + mag * 2.0 ** -11).all()


def test_kv8_reorder_offsets_beyond_32_bits():
    layers, B, H, C, D = 2, 4, 8, 1 << 19, 128
    c = ops.kv8_cache(layers * B, H, C, D, DEV)
    c = ops.Kv8(*(t.view(layers, B, *t.shape[1:]) for t in c))
    assert c.k.numel() > 1 << 31
    g = torch.Generator(DEV).manual_seed(2)
    lens, parents = [100, C, 70, 64], [1, 0, 3, 2]
    for t in c[:2]:
        t[:, :, :, :128] = torch.randint(-127, 128, (layers, B, H, 128, D), dtype=torch.int8, device=DEV, generator=g)
        t[:, 1, :, C - 64:] = torch.randint(-127, 128, (layers, H, 64, D), dtype=torch.int8, device=DEV, generator=g)
    for t in c[2:]:
        t.copy_(torch.rand(t.shape, device=DEV, generator=g))
    probe = lambda c: [torch.cat([t[:, :, :, :(128 if i < 2 else 2)], t[:, :, :, -(64 if i < 2 else 1):]], 3).clone() for i, t in enumerate(c)]
    before = probe(c)
    ops.kv8_reorder(c, i32(parents), i32(lens), beams=4)
    after = probe(c)
    for i, (b, a) in enumerate(zip(before, after)):
        for seq, p in enumerate(parents):
            T = lens[p]
            n = T if i < 2 else (T + 63) // 64
            head = b.shape[3] - (64 if i < 2 else 1)
            want = b[:, seq].clone()
            want[:, :, :min(n, head)] = b[:, p, :, :min(n, head)]
            if T == C:
                want[:, :, head:] = b[:, p, :, head:]
            assert torch.equal(a[:, seq], want), (i, seq)


def test_beam_select_offsets_beyond_32_bits():
    S, V = 40, 1 << 26
    g = torch.Generator(DEV).manual_seed(3)
    x = torch.empty(S, V, dtype=BF, device=DEV)
    for s in range(S):
        x[s] = torch.randn(V, device=DEV, generator=g, dtype=torch.float32).to(BF)
    x[39, [5, V - 3]] = 30.0
    x[38, V - 1] = 25.0
    got = ops.beam_select(x, torch.zeros(S, device=DEV), 1, k=4)
    for s in (0, 38, 39):
        row = x[s].double()
        lp = torch.log_softmax(row, 0)
        best = torch.sort(row, descending=True, stable=True).indices[:4]
        assert got.tokens[s].tolist() == best.tolist() and (got.parents[s] == s).all()
        # 2^26 words of one size, 64 at a time in fp32: 2^-18 of the sum at most, and the total's rounding
        assert ((got.scores[s].double() - lp[best]).abs() < 2.0 ** -18 + 2.0 ** -20).all()


def test_two_steps_in_one_graph_share_a_workspace():
    """Calls of different sizes one after another in one captured graph, with the same workspaces."""
    H, D, F = 2, 64, 6
    prefix, cache = filled((1,), H, 2048, D, 2), filled((F,), H, 256, D, 3)
    ws = ops.attn_kv8_shared_workspace(1, F, 40, 4, H, D, 2048, 256, DEV)
    qs = [torch.randn(F, n, 4, D, device=DEV, generator=torch.Generator(DEV).manual_seed(n)).to(BF) for n in (40, 1, 7)]
    outs = [torch.zeros(F, q.shape[1], 4 * D, dtype=BF, device=DEV) for q in qs]
    lens, plens = i32([9 * f for f in range(F)]), i32([2000])
    x, scores = torch.randn(F, 700, device=DEV), torch.zeros(F, device=DEV)
    sel = torch.empty(1 << 20, dtype=torch.uint8, device=DEV)

    def run():
        for q, o in zip(qs, outs):
            ops.attn_kv8_shared(q, prefix, plens, cache, lens, o, ws=ws)
        return ops.beam_select(x, scores, F, ws=sel), ops.beam_select(x[:2], scores[:2], 2, k=9, ws=sel)

    want = [t.clone() for b in run() for t in b] + [o.clone() for o in outs]
    for q, o in zip(qs, outs):
        check_shared(q, prefix, [2000], cache, np_(lens), None, o)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for o in outs:
        o.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, [t for b in got for t in b] + outs))


@pytest.mark.parametrize("dt", [torch.float32, BF])
@pytest.mark.parametrize("F,k", [(1, 1), (2, 4), (3, 16), (1, 33), (2, 128)])
@pytest.mark.parametrize("allowed", [1, 40, 150, 3000])
def test_beam_select_few_words_allowed_that_stand_together(dt, F, k, allowed):
    """All words but a few runs of neighbours at one value: more words than k above it, in fewer parts of a chunk than k."""
    V = 20000
    g = torch.Generator(DEV).manual_seed(allowed + k)
    for base in (torch.finfo(dt).min, -1e4, 0.0):
        x = torch.full((F, V), base, device=DEV, dtype=dt)
        for f in range(F):
            for v0 in (f * 5, 8192 + 4093, 16384):
                x[f, v0:v0 + allowed] = (torch.rand(allowed, device=DEV, generator=g) * 9 + 1).to(dt)
        scores = torch.linspace(0, -1, F, device=DEV)
        check_select(x, scores, F, k, -1, None, ops.beam_select(x, scores, F, k=k))


@pytest.mark.parametrize("S,F,n,Hq,H,D,plens", [(3, 4, 5, 24, 3, 64, [1500, 0, 1]), (5, 4, 5, 24, 3, 64, [1500, 0, 64, 65, 1]), (3, 20, 4, 8, 2, 128, [1100, 0, 2])])
def test_attn_kv8_shared_shares_of_one_tile_that_follow_one_another(S, F, n, Hq, H, D, plens):
    """Items of few tiles behind the last tile of the item before: one half of a CTA has nothing in a share, and all of the next."""
    B = S * F
    q = (torch.randn(B, n, Hq, D, device=DEV, generator=torch.Generator(DEV).manual_seed(B)) * 1.5).to(BF)
    for r in range(20):
        lens = [(b * 7 + r) % 3 % 2 for b in range(B)]
        prefix, cache = filled((S,), H, 1536, D, r), filled((B,), H, 64, D, r + 100)
        out = ops.attn_kv8_shared(q, prefix, i32(plens), cache, i32(lens))
        ro, mag = R.attention_shared(np_(q.float()), as_np(prefix), plens, as_np(cache), lens)
        # as for all shapes, and 2^-32 of a row's largest product with a V scale (0.03 at most) for each term of 127 below 2^-21 of it
        bound = np.abs(ro) * 2.0 ** -8 + mag * (2.0 ** -11 + 2.0 ** -12) + 2.0 ** -32 * 0.03 * 127 * (max(plens) + n + 1)
        assert (np.abs(np_(out.float()) - ro) <= bound * (1 + 2.0 ** -7)).all(), r
