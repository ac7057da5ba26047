"""The 8-bit KV cache's operators in plain numpy, one sequence and head at a time: the cache write in the fp32 steps
that define its codes, attention and eviction from their definitions in 64 bits.  No counterpart in the reference
(its cache is bf16, moondream/gpu/md2fast.py:186-191)."""
import numpy as np

BLK = 64
F = np.float32


def bf16(x):
    """fp32 rounded to bf16 (nearest even), as fp32; finite values and infinities."""
    u = np.ascontiguousarray(x, dtype=F).view(np.uint32).astype(np.uint64)
    u = (u + 0x7fff + ((u >> 16) & 1)) & 0xffff0000
    return u.astype(np.uint32).view(F).reshape(np.shape(x))


def rope(x, cos, sin):
    """x [n, heads, D] fp32 (bf16 values), cos / sin [n, 16] -> rotated, fp32, each operation rounded."""
    a, b, c, s = x[..., :16], x[..., 16:32], cos[:, None].astype(F), sin[:, None].astype(F)
    y = x.copy()
    y[..., 0:32:2] = a * c - b * s
    y[..., 1:32:2] = a * s + b * c
    return y


def quantise(x, codes, scales, length):
    """x [n, D] fp32 into codes [C, D] int8 / scales [C / 64] fp32 (in place) from slot `length` on."""
    n = len(x)
    for blk in range(length // BLK, (length + n - 1) // BLK + 1 if n else 0):
        lo, hi = max(blk * BLK, length), min((blk + 1) * BLK, length + n)
        new, held = x[lo - length:hi - length], lo - blk * BLK
        need = F(np.abs(new).max()) / F(127) if np.isfinite(new).all() else F(np.nan)
        old = scales[blk] if held else F(0)
        if old == 0:
            s = need
        elif np.isnan(old) or np.isnan(need):
            s = F(np.nan)
        else:
            s, j = old, 0
            while s < need:
                s, j = F(s * F(2)), j + 1
            if j:
                codes[blk * BLK:lo] = np.rint(codes[blk * BLK:lo].astype(np.float64) * 0.5 ** j)
        codes[lo:hi] = np.clip(np.rint(new / s), -127, 127) if s > 0 else 0
        scales[blk] = s


def append(qkv, cache, lens, cos, sin, Hq, pos=None, counts=None):
    """qkv [B, n, (Hq + 2 H) D] fp32, cache (k, v, ks, vs) arrays updated in place -> q [B, n, Hq, D] fp32, rotated and
    not rounded (rows past the count zero)."""
    k, v, ks, vs = cache
    B, H, C, D = k.shape
    n = qkv.shape[1]
    q = np.zeros((B, n, Hq, D), F)
    for b in range(B):
        m = n if counts is None else int(counts[b])
        p = (int(lens[b]) if pos is None else int(pos[b])) + np.arange(m)
        x = qkv[b, :m].reshape(m, Hq + 2 * H, D)
        q[b, :m] = rope(x[:, :Hq], cos[p], sin[p])
        kr = rope(x[:, Hq:Hq + H], cos[p], sin[p])
        kr = np.where(np.isfinite(kr), bf16(kr), kr)
        for h in range(H):
            quantise(kr[:, h], k[b, h], ks[b, h], int(lens[b]))
            quantise(x[:, Hq + H + h], v[b, h], vs[b, h], int(lens[b]))
    return q


def attention(q, cache, lens, counts=None, causal=True, scale=None, weights_in=None):
    """q [B, n, Hq, D] -> out [B, n, Hq D] (64 bits, NaN rows past the count), weights [B, H, C] (NaN past the end), the sums
    of p |v| behind each output and a bound on the rounding of a score in fp32 behind each weight (same shapes)."""
    k8, v8, ks, vs = cache
    B, H, C, D = k8.shape
    n, Hq = q.shape[1:3]
    scale = D ** -0.5 if scale is None else scale
    out, mag = np.full((B, n, Hq * D), np.nan), np.zeros((B, n, Hq * D))
    w, werr = np.full((B, H, C), np.nan), np.zeros((B, H, C))
    for b in range(B):
        L, m = int(lens[b]), n if counts is None else int(counts[b])
        T = L + m
        blk = np.arange(T) // BLK
        see = np.arange(T)[None] <= (L + np.arange(m)[:, None] if causal else np.full((m, 1), T))
        w[b, :, :T] = 0
        if weights_in is not None:
            w[b, :, :L] = weights_in[b, :, :L]
        for hq in range(Hq):
            h = hq // (Hq // H)
            k = k8[b, h, :T].astype(np.float64) * ks[b, h, blk].astype(np.float64)[:, None]
            v = v8[b, h, :T].astype(np.float64) * vs[b, h, blk].astype(np.float64)[:, None]
            for i in range(m):
                t = np.flatnonzero(see[i])
                qi = q[b, i, hq].astype(np.float64)
                with np.errstate(invalid="ignore"):
                    z = k[t] @ qi * scale
                    p = np.exp(z - z.max())
                    p /= p.sum()
                    out[b, i, hq * D:(hq + 1) * D] = p @ v[t]
                    mag[b, i, hq * D:(hq + 1) * D] = p @ np.abs(v[t])
                    w[b, h, t] += p
                    d = np.abs(k[t]) @ np.abs(qi) * abs(scale) * D * 2.0 ** -24 + np.abs(z) * 2.0 ** -22
                    werr[b, h, t] += p * 2 * d.max()
    return out, w, mag, werr


def evict(cache, weights, lens, keep, recent):
    """-> for each sequence None (copied) or (index [H, keep], k, v, ks, vs) with the new codes and scales."""
    k8, v8, ks, vs = cache
    B, H, C, D = k8.shape
    res = []
    for b in range(B):
        L = int(lens[b])
        if L <= keep:
            res.append(None)
            continue
        idx = np.zeros((H, keep), np.int64)
        new = [np.zeros((H, keep, D), np.int8), np.zeros((H, keep, D), np.int8), np.zeros((H, keep // BLK), F),
               np.zeros((H, keep // BLK), F)]
        for h in range(H):
            old = weights[b, h, :L - recent].astype(np.float64)
            rank = np.where(np.isnan(old), np.inf, old)
            top = sorted(range(L - recent), key=lambda j: (not np.isnan(old[j]), -rank[j], j))[:keep - recent]
            idx[h] = np.array(sorted(top) + list(range(L - recent, L)))
            for codes, sc, nc, ns in ((k8, ks, new[0], new[2]), (v8, vs, new[1], new[3])):
                x = codes[b, h, idx[h]].astype(F) * sc[b, h, idx[h] // BLK][:, None]
                for blk in range(keep // BLK):
                    y = x[blk * BLK:(blk + 1) * BLK]
                    s = F(np.abs(y).max()) / F(127)
                    ns[h, blk] = s
                    nc[h, blk * BLK:(blk + 1) * BLK] = np.clip(np.rint(y / s), -127, 127) if s > 0 else 0
        res.append((idx, *new))
    return res
