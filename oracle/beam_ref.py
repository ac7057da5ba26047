"""Many answers about one context, restated in numpy with 64 bits: attention behind a shared prefix, the choice of a beam search and
the reordering of caches.  The reference has no counterpart (it asks one question at a time, md2fast.py:208-212); the cache is
the one of kv8_ref."""
import numpy as np

from .kv8_ref import BLK


def _values(cache, w, b, h, T):
    codes, scale = cache[w], cache[w + 2]
    return codes[b, h, :T].astype(np.float64) * scale[b, h, np.arange(T) // BLK].astype(np.float64)[:, None]


def attention_shared(q, prefix, plens, cache, lens, counts=None, scale=None):
    """q [B, n, Hq, D]; prefix, cache (k, v, ks, vs) of S prefixes and B sequences -> out [B, n, Hq D] (NaN rows past the count) and
    the sums of p |v| behind each output."""
    S, H, _, D = prefix[0].shape
    B, n, Hq = q.shape[:3]
    scale = D ** -0.5 if scale is None else scale
    out, mag = np.full((B, n, Hq * D), np.nan), np.zeros((B, n, Hq * D))
    for b in range(B):
        s, L, m = b // (B // S), int(lens[b]), n if counts is None else int(counts[b])
        P = int(plens[s])
        for hq in range(Hq):
            h = hq // (Hq // H)
            k, v = (np.concatenate([_values(prefix, w, s, h, P), _values(cache, w, b, h, L + m)]) for w in (0, 1))
            for i in range(m):
                T = P + L + i + 1
                with np.errstate(invalid="ignore"):
                    z = k[:T] @ q[b, i, hq].astype(np.float64) * scale
                    p = np.exp(z - z.max())
                    p /= p.sum()
                    out[b, i, hq * D:(hq + 1) * D] = p @ v[:T]
                    mag[b, i, hq * D:(hq + 1) * D] = p @ np.abs(v[:T])
    return out, mag


def totals(logits, scores, beams, eos=-1, done=None):
    """[S, beams V] 64-bit totals of every continuation, -inf where there is none."""
    x = np.asarray(logits, np.float64)
    B, V = x.shape
    res = np.full((B, V), -np.inf)
    for b in range(B):
        if done is not None and done[b]:
            res[b, eos] = scores[b] if np.isfinite(scores[b]) else -np.inf
            continue
        with np.errstate(all="ignore"):
            top = x[b].max()
            t = float(scores[b]) + ((x[b] - top) - np.log(np.exp(x[b] - top).sum()))
        res[b] = np.where(np.isfinite(t), t, -np.inf)
    return res.reshape(B // beams, beams * V)


def reorder(cache, parents, lens, beams=None, dst=None, new_lens=None):
    """cache (k, v, ks, vs) [layers, Bs, ...], dst likewise (None: in place) -> the tensors and lengths afterwards."""
    out = [t.copy() for t in (dst if dst is not None else cache)]
    B = out[0].shape[1]
    res = np.zeros(B, np.int64) if new_lens is None else np.array(new_lens)
    for b in range(B):
        p = int(parents[b])
        lo, hi = (b // beams * beams, b // beams * beams + beams) if dst is None else (0, cache[0].shape[1])
        if not lo <= p < hi:
            if dst is None:
                res[b] = lens[b]
            continue
        T = min(max(int(lens[p]), 0), cache[0].shape[3], out[0].shape[3])
        nb = (T + BLK - 1) // BLK
        for i, t in enumerate(cache):
            m = T if i < 2 else nb
            out[i][:, b, :, :m] = t[:, p, :, :m]
        res[b] = T
    return out, res
