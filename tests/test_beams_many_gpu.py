"""Attention behind shared prefixes with as many sequences as a call takes, and with many prefixes, against the formula in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from strix_halo_maxx_b200 import ops
from test_beams_gpu import DEV, BF, _status, filled, i32


def values(codes, scales, T):
    """The first T slots in 64 bits [.., T, D]."""
    return codes[..., :T, :].double() * scales.double().repeat_interleave(64, -1)[..., :T, None]


def formula(q, prefix, plens, cache, lens, scale):
    """-> out and the sums of p |v| behind it, [B, n, Hq, D] in 64 bits."""
    B, n, Hq, D = q.shape
    F, H, P, T = B // len(plens), cache.k.shape[1], max(plens), max(lens) + n
    out, mag = (torch.empty(B, n, Hq, D, dtype=torch.float64, device=DEV) for _ in range(2))
    step = max(1, (1 << 26) // ((P + T) * Hq * n))
    own, pre = torch.tensor(lens, device=DEV), torch.tensor(plens, device=DEV).repeat_interleave(F)
    j, i = torch.arange(P + T, device=DEV), torch.arange(n, device=DEV)
    for b in range(0, B, step):
        at = torch.arange(b, min(b + step, B), device=DEV)
        k, v = (torch.cat([values(p[at // F], ps[at // F], P), values(c[at], cs[at], T)], -2).repeat_interleave(Hq // H, 1)
                for p, ps, c, cs in ((prefix.k, prefix.ks, cache.k, cache.ks), (prefix.v, prefix.vs, cache.v, cache.vs)))
        sees = torch.where(j < P, j < pre[at, None, None], j - P <= own[at, None, None] + i[:, None])
        z = (q[at].double().transpose(1, 2) @ k.transpose(-1, -2) * scale).masked_fill(~sees[:, None], -float("inf"))
        p = torch.softmax(z, -1)
        out[at], mag[at] = (p @ v).transpose(1, 2), (p @ v.abs()).transpose(1, 2)
    return out, mag


MANY = [  # S, F, n, Hq, H, D, capacity of the prefixes, of the others, longest prefix, most own tokens
    # few rows on a prefix, in runs: 32 rows of as many sequences as there may be; a sequence a prefix; 128 wide
    (64, 32, 1, 1, 1, 64, 16448, 64, 300, 60), (2048, 1, 1, 32, 1, 64, 128, 64, 128, 63), (1024, 2, 1, 8, 1, 128, 128, 64, 128, 63), (3, 8, 1, 6, 2, 64, 17000 // 64 * 64, 320, 9000, 300),
    # more: one tile of codes in flight beside the longest lists, of 128 and 256 rows, in whole items and in runs
    (2048, 1, 1, 32, 1, 128, 128, 64, 128, 63), (2048, 1, 16, 16, 1, 128, 64, 64, 64, 48), (1950, 1, 16, 16, 1, 128, 1920, 64, 200, 48),
    # two thousand sequences on one prefix, their own slots in the same kernel and in another one
    (1, 2000, 1, 2, 1, 64, 16576, 64, 3000, 63), (1, 2000, 1, 2, 1, 64, 4096, 256, 3000, 255), (2, 1000, 1, 4, 2, 128, 2048, 192, 1000, 150),
    # many prefixes, some of them empty, in runs
    (40, 5, 2, 16, 2, 64, 8192, 128, 1500, 100), (300, 3, 3, 5, 1, 128, 4096, 64, 200, 61), (1000, 2, 70, 2, 1, 64, 3200, 128, 150, 58)]


@pytest.mark.parametrize("S,F,n,Hq,H,D,Cp,C,P,L", MANY)
def test_attn_kv8_shared_of_many_sequences_and_prefixes(S, F, n, Hq, H, D, Cp, C, P, L):
    B = S * F
    plens, lens = [(s * 53 + 7) % (P + 1) if s % 11 != 3 else 0 for s in range(S)], [(b * 37) % (L + 1) for b in range(B)]
    plens[0] = P
    counts = [(b * 5) % (n + 1) if b % 3 == 1 else n for b in range(B)]
    prefix, cache = filled((S,), H, Cp, D, 1), filled((B,), H, C, D, 2)
    q = (torch.randn(B, n, Hq, D, device=DEV, generator=torch.Generator(DEV).manual_seed(3)) * 1.5).to(BF)
    outs = [torch.full((B, n, Hq * D), 3.0, dtype=BF, device=DEV) for _ in range(2)]
    for out in outs:
        ops.attn_kv8_shared(q, prefix, i32(plens), cache, i32(lens), out, counts=i32(counts))
    assert torch.equal(*outs), "the same call twice"
    ro, mag = formula(q, prefix, plens, cache, lens, D ** -0.5)
    out = outs[0].view(B, n, Hq, D).double()
    rows = torch.arange(n, device=DEV) < i32(counts)[:, None]
    assert (out[~rows] == 3).all(), "rows past the count"
    # the bounds of tests/test_beams_gpu.py: the output's rounding to bf16, P's to f16, scores of a few units in fp32
    err, bound = (out - ro).abs()[rows], (ro.abs() * 2.0 ** -8 + mag * (2.0 ** -11 + 2.0 ** -12))[rows]
    assert (err <= bound * (1 + 2.0 ** -7)).all(), float((err / bound).max())
    assert err.norm() <= bound.norm() * 3 ** -0.5
