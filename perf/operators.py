"""Workloads of the 8-bit key / value cache: writing new tokens into it, attention over it, and eviction from it.

The cache of one layer holds, for B sequences x H heads x C slots (C a multiple of 64) x D dims, int8 codes k, v
[B, H, C, D] and one fp32 scale per 64 slots and head ks, vs [B, H, C / 64]; a value is code * scale.  lens[b] is the
number of tokens that sequence b holds before a call, counts[b] <= n the number of new ones (rows past it are padding).

  append   rotary embedding of new q / k rows, and k / v quantised into the cache
  attn     attention of the new rows over the cache (their own tokens in it already), and, where asked for, the
           attention weight that each slot received, summed over rows and over the query heads of its group
  evict    each head keeps the most recent tokens and those with the largest weight, in order, in another cache

run() computes them with elementary torch operations, or, where `own` is true, by the framework's entry points.
"""
import math

import torch

own = False

BLOCK = 64        # slots that share a scale
ROT = 32          # rotary dims of a head
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


# ---------------------------------------------------------------------------------------------------- cases
def _append(name, B, n, Hq, H, D, L, ragged=False):
    return {"name": name, "op": "append", "B": B, "n": n, "Hq": Hq, "H": H, "D": D, "L": L, "ragged": ragged}


def _attn(name, B, n, Hq, H, D, L, causal=True, weights=False, ragged=False):
    return {"name": name, "op": "attn", "B": B, "n": n, "Hq": Hq, "H": H, "D": D, "L": L, "causal": causal,
            "weights": weights, "ragged": ragged}


def _evict(name, B, H, D, L, keep, recent, ragged=False):
    return {"name": name, "op": "evict", "B": B, "H": H, "D": D, "L": L, "keep": keep, "recent": recent, "ragged": ragged}


def listed():
    return [
        # the text decoder's layer (32 heads x 64): one more token after the 730-token image prefix and a question
        _append("append 1 token", 1, 1, 32, 32, 64, 762),
        # the image prefix itself, into an empty cache
        _append("append prefix", 1, 730, 32, 32, 64, 0),
        # a served batch with grouped heads: up to 7 new tokens a sequence, at lengths that differ
        _append("append batch", 48, 7, 32, 8, 128, 4099, ragged=True),
        # the image prefix attends to itself without a mask, and leaves the weights that eviction goes by
        _attn("attn prefix", 1, 730, 32, 32, 64, 0, causal=False, weights=True),
        # a 32-token question over the prefix
        _attn("attn question", 1, 32, 32, 32, 64, 730),
        # one token of an answer
        _attn("attn 1 token", 1, 1, 32, 32, 64, 761, weights=True),
        # a served batch, one token for each sequence, at lengths that differ
        _attn("attn batch", 64, 1, 32, 8, 128, 8191, ragged=True),
        # one token over a long context, with the weights
        _attn("attn long", 1, 1, 32, 8, 128, 131007, weights=True),
        # a chunk of a long prompt over what is already there
        _attn("attn chunk", 1, 2048, 32, 8, 128, 6001),
        # the image prefix of all 24 layers at once down to 256 tokens a head
        _evict("evict prefix", 24, 32, 64, 730, 256, 32),
        # a served batch down to 2048 tokens a head
        _evict("evict batch", 32, 8, 128, 16385, 2048, 256, ragged=True),
        # one long context
        _evict("evict long", 1, 8, 128, 131071, 8192, 1024),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: heads 64 or 128 wide, groups of 1 to 8, one sequence to 64, lengths over their whole range."""
    op = rng.choice(("append", "attn", "attn", "evict"))
    D = rng.choice((64, 128))
    H = rng.choice((1, 2, 4, 8, 16, 32)) if D == 64 else rng.choice((1, 2, 3, 4, 8))
    G = rng.choice((1, 1, 2, 4, 5, 8)) if H <= 8 else 1
    B = _log(rng, 1, 64)
    ragged = B > 1 and rng.random() < 0.7
    if op == "append":
        n = rng.choice((1, 1, _log(rng, 2, 1500)))
        L = rng.choice((0, _log(rng, 1, 6000)))
        while B * H * (L + n) * D > 48 * 8 * 4200 * 128:
            B, n, L = (B + 1) // 2, max(1, n // 2), L // 2
        return _append("", B, n, G * H, H, D, L, ragged and B > 1)
    if op == "attn":
        n = rng.choice((1, 1, _log(rng, 2, 64), _log(rng, 65, 2048)))
        L = _log(rng, 1, 131000)
        while B * H * (L + n) * D > 64 * 8 * 6200 * 128 or B * G * H * n * (L + n) * D > 2048 * 7025 * 32 * 128:
            if n > 64 and rng.random() < 0.5:
                n = n // 2 + 1
            elif B > 1 and rng.random() < 0.5:
                B = (B + 1) // 2
            else:
                L = L // 2 + 1
        return _attn("", B, n, G * H, H, D, L, rng.random() < 0.75, rng.random() < 0.5, ragged and B > 1)
    L = _log(rng, 65, 131000)
    while B * H * L * D > 32 * 8 * 12000 * 128:
        B, L = (B + 1) // 2, max(65, L // 2)
    keep = BLOCK * max(1, _log(rng, max(1, L // 16), L) // BLOCK)
    return _evict("", B, H, D, L, keep, min(keep, _log(rng, 1, keep)), ragged and B > 1)


def _lens(c):
    """Tokens that each sequence holds, a function of the case alone: L, or from about L / 2 to L."""
    L = c["L"]
    return [L - (b * 7919) % (L // 2 + 1) if c["ragged"] else L for b in range(c["B"])]


def _counts(c):
    """New tokens of each sequence: n, or in a ragged batch 0 (an idle sequence) to n."""
    n = c["n"]
    return [n - (b * 5) % (n + 1) if c["ragged"] and n > 1 else n for b in range(c["B"])]


def _capacity(c):
    return (c["L"] + c.get("n", 0) + BLOCK - 1) // BLOCK * BLOCK + BLOCK


# ---------------------------------------------------------------------------------------------------- inputs
def _cache(B, H, C, D, g, dev):
    """Codes and scales as quantised keys and values have them: near-normal values, some channels larger, scales that
    differ from block to block."""
    gain = torch.rand(2, 1, H, 1, D, device=dev, generator=g) * 0.8 + 0.6
    codes = [torch.empty(B, H, C, D, dtype=torch.int8, device=dev) for _ in range(2)]
    for w in range(2):
        for b in range(B):
            x = torch.randn(H, C, D, device=dev, generator=g) * 32.0 * gain[w, 0]
            codes[w][b] = x.round().clamp(-127, 127).to(torch.int8)
    ks, vs = (torch.rand(B, H, C // BLOCK, device=dev, generator=g) * 0.02 + 0.015 for _ in range(2))
    return codes[0], codes[1], ks, vs


def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    B, H, D = c["B"], c["H"], c["D"]
    C = _capacity(c)
    s = {"case": dict(c), "cache": _cache(B, H, C, D, g, dev),
         "lens": torch.tensor(_lens(c), dtype=torch.int32, device=dev)}
    if c["op"] != "evict":
        n, Hq = c["n"], c["Hq"]
        s["counts"] = torch.tensor(_counts(c), dtype=torch.int32, device=dev) if c["ragged"] else None
        s["q"] = torch.zeros(B, n, Hq, D, dtype=BF16, device=dev)
    if c["op"] == "append":
        s["qkv"] = torch.randn(B, n, (Hq + 2 * H) * D, device=dev, generator=g).to(BF16)
        inv = 10000.0 ** (-torch.arange(0, ROT, 2, dtype=F64, device=dev) / ROT)
        ang = torch.arange(C, dtype=F64, device=dev)[:, None] * inv[None]
        s["cos"], s["sin"] = torch.cos(ang).float(), torch.sin(ang).float()
    elif c["op"] == "attn":
        s["q"] = (torch.randn(B, n, Hq, D, device=dev, generator=g) * 1.7).to(BF16)
        s["out"] = torch.zeros(B, n, Hq * D, dtype=BF16, device=dev)
        s["w_in"] = torch.rand(B, H, C, device=dev, generator=g) if c["weights"] else None
        s["w"] = torch.zeros(B, H, C, device=dev) if c["weights"] else None
    else:
        # weights as attention leaves them: a few slots with most of it, many with little, some with none at all
        w = torch.exp(2.5 * torch.randn(B, H, C, device=dev, generator=g))
        s["w"] = w * (torch.rand(B, H, C, device=dev, generator=g) > 0.05)
        Cd = c["keep"] + BLOCK
        s["dst"] = tuple(torch.zeros(B, H, Cd, D, dtype=torch.int8, device=dev) for _ in range(2)) + \
            tuple(torch.zeros(B, H, Cd // BLOCK, device=dev) for _ in range(2))
        s["dst_w"] = torch.zeros(B, H, Cd, device=dev)
        s["dst_lens"] = torch.zeros(B, dtype=torch.int32, device=dev)
        s["index"] = torch.zeros(B, H, c["keep"], dtype=torch.int32, device=dev)
    return s


# ---------------------------------------------------------------------------------------------------- the passes
def run(state):
    s = state
    c = s["case"]
    if own:
        from strix_halo_maxx_b200 import ops
        cache = ops.Kv8(*s["cache"])
        if c["op"] == "append":
            ops.rope_kv8(s["qkv"], cache, s["lens"], s["cos"], s["sin"], s["q"], counts=s["counts"])
        elif c["op"] == "attn":
            ops.attn_kv8(s["q"], cache, s["lens"], s["out"], counts=s["counts"], causal=c["causal"], weights=s["w"],
                         weights_in=s["w_in"])
        else:
            ops.kv8_evict(cache, s["w"], s["lens"], c["keep"], c["recent"], ops.Kv8(*s["dst"]), s["dst_w"], s["dst_lens"],
                          index=s["index"])
    elif c["op"] == "append":
        _plain_append(s)
    elif c["op"] == "attn":
        _plain_attn(s)
    else:
        _plain_evict(s)
    # codes are whole numbers, to be equal one by one
    if c["op"] == "append":
        return {"q": s["q"], **dict(zip(("k", "v", "ks", "vs"), s["cache"]))}
    if c["op"] == "attn":
        return {"out": s["out"], "w": s["w"]} if c["weights"] else {"out": s["out"]}
    return {**dict(zip(("k", "v", "ks", "vs"), s["dst"])), "w": s["dst_w"], "lens": s["dst_lens"], "index": s["index"]}


def _rope(x, cos, sin):
    """x [B, n, heads, D] fp32, cos / sin [B, n, 1, 16]: dims i and 16 + i rotate into dims 2i and 2i + 1."""
    a, b = x[..., :ROT // 2], x[..., ROT // 2:ROT]
    r = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    return torch.cat([r, x[..., ROT:]], dim=-1)


def _plain_append(s):
    c, lens = s["case"], s["lens"].long()
    B, n, Hq, H, D = (c[k] for k in ("B", "n", "Hq", "H", "D"))
    dev = lens.device
    cnt = s["counts"].long() if s["counts"] is not None else torch.full((B,), n, device=dev)
    C = s["cache"][0].shape[2]
    i = torch.arange(n, device=dev)
    at = (lens[:, None] + i).clamp(max=s["cos"].shape[0] - 1)
    cos, sin = s["cos"][at][:, :, None], s["sin"][at][:, :, None]
    x = s["qkv"].float().view(B, n, Hq + 2 * H, D)
    s["q"].copy_(torch.where((i < cnt[:, None])[..., None, None], _rope(x[:, :, :Hq], cos, sin).to(BF16), s["q"]))
    # k is rounded to bf16 as the bf16 cache holds it, then quantised
    k = _rope(x[:, :, Hq:Hq + H], cos, sin).to(BF16).float()
    _quantise(k, s["cache"][0], s["cache"][2], lens, cnt)
    _quantise(x[:, :, Hq + H:], s["cache"][1], s["cache"][3], lens, cnt)


def _quantise(x, codes, scales, lens, cnt):
    """x [B, n, H, D] fp32 into slots lens .. lens + cnt - 1.  A block that gets its first tokens, or holds only zeros,
    takes the scale max|x| / 127; one that holds tokens keeps its scale, doubled as often as the new ones need."""
    B, n, H, D = x.shape
    dev = x.device
    nb = (n - 1) // BLOCK + 2
    bi = torch.arange(B, device=dev)
    blk = lens[:, None] // BLOCK + torch.arange(nb, device=dev)                             # [B, nb]
    blk_in = blk.clamp(max=scales.shape[2] - 1)
    slot = blk[..., None] * BLOCK + torch.arange(BLOCK, device=dev)                         # [B, nb, 64]
    i = slot - lens[:, None, None]
    new = (i >= 0) & (i < cnt[:, None, None])
    held = i < 0
    xs = x[bi[:, None, None], i.clamp(0, n - 1)]                                            # [B, nb, 64, H, D]
    xs = torch.where(new[..., None, None], xs, torch.zeros((), device=dev))
    need = xs.abs().amax(dim=(2, 4))                                                        # [B, nb, H]
    need = need / torch.full_like(need, 127.0)
    old_s = scales[bi[:, None], :, blk_in]                                                  # [B, nb, H]
    fresh = ~held.any(-1)[..., None] | (old_s == 0)
    (mn, en), (ms, es) = torch.frexp(need), torch.frexp(old_s)
    k = torch.where(need > old_s, en - es + (ms < mn).int(), torch.zeros_like(en))
    k = torch.where(fresh, torch.zeros_like(k), k)
    s = torch.where(fresh, need, torch.ldexp(old_s, k))
    old = codes.view(B, H, -1, BLOCK, D)[bi[:, None], :, blk_in].permute(0, 1, 3, 2, 4)     # [B, nb, 64, H, D]
    shifted = torch.ldexp(old.float(), -k[:, :, None, :, None]).round().to(torch.int8)
    q = (xs / torch.where(s > 0, s, torch.ones_like(s))[:, :, None, :, None]).round().clamp(-127, 127).to(torch.int8)
    res = torch.where(new[..., None, None], q, torch.where(held[..., None, None], shifted, old))
    any_new = new.any(-1)[..., None]
    # _capacity() leaves a spare block, so that no two of these blocks are clamped to the same one
    codes.view(B, H, -1, BLOCK, D)[bi[:, None], :, blk_in] = torch.where(any_new[..., None, None], res.permute(0, 1, 3, 2, 4),
                                                                     old.permute(0, 1, 3, 2, 4))
    scales[bi[:, None], :, blk_in] = torch.where(any_new, s, old_s)


def _plain_attn(s):
    c, lens = s["case"], s["lens"].long()
    B, n, Hq, H, D = (c[k] for k in ("B", "n", "Hq", "H", "D"))
    G, dev = Hq // H, lens.device
    cnt = s["counts"].long() if s["counts"] is not None else torch.full((B,), n, device=dev)
    k8, v8, ks, vs = s["cache"]
    C = min(k8.shape[2], (c["L"] + n + BLOCK - 1) // BLOCK * BLOCK)
    k, v = ((t[:, :, :C].float().view(B, H, -1, BLOCK, D) * sc[:, :, :C // BLOCK, None, None]).view(B, H, C, D)
            for t, sc in ((k8, ks), (v8, vs)))
    i, j = torch.arange(n, device=dev), torch.arange(C, device=dev)
    limit = lens[:, None] + (i + 1 if c["causal"] else cnt[:, None].expand(B, n))           # keys that row i sees
    row = i < cnt[:, None]                                                                  # [B, n] rows that count
    q = s["q"].float().view(B, n, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * n, D)
    sc = (q @ k.transpose(-1, -2)).view(B, H, G, n, C) * D ** -0.5
    sc.masked_fill_((j >= limit[..., None])[:, None, None], -math.inf)
    sc -= sc.amax(-1, keepdim=True)
    sc.exp_()
    sc /= sc.sum(-1, keepdim=True)
    o = (sc.view(B, H, G * n, C) @ v).view(B, H, G, n, D).permute(0, 3, 1, 2, 4).reshape(B, n, Hq * D)
    s["out"].copy_(torch.where(row[..., None], o.to(BF16), s["out"]))
    if c["weights"]:
        sc *= row[:, None, None, :, None]
        w = sc.sum((2, 3))
        w = torch.where((j < lens[:, None])[:, None], w + s["w_in"][:, :, :C], w)           # new slots begin at 0
        s["w"][:, :, :C] = torch.where((j < (lens + cnt)[:, None])[:, None], w, s["w"][:, :, :C])


def _plain_evict(s):
    c, lens = s["case"], s["lens"].long()
    B, H, D, keep, recent = (c[k] for k in ("B", "H", "D", "keep", "recent"))
    dev = lens.device
    k8, v8, ks, vs = s["cache"]
    C, Cd = k8.shape[2], s["dst"][0].shape[2]
    j = torch.arange(C, device=dev)
    over = lens > keep                                                                      # [B] sequences that lose tokens
    # the recent ones first, then by weight, the lowest slot where weights are equal; slots past the end last
    rank = torch.where((j < lens[:, None])[:, None], s["w"], torch.full((), -1.0, device=dev))
    rank = torch.where(((j >= lens[:, None] - recent) & (j < lens[:, None]))[:, None], torch.full((), math.inf, device=dev), rank)
    by = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    by = torch.nn.functional.pad(by, (0, max(0, keep - by.shape[-1])))
    idx = torch.sort(by, dim=-1).values
    slots = torch.arange(keep, device=dev)
    idx = torch.where(over[:, None, None], idx, slots.clamp(max=C - 1))                      # [B, H, keep]
    new_len = lens.clamp(max=keep)
    valid = slots < new_len[:, None]                                                        # [B, keep]
    s["index"].copy_(torch.where(valid[:, None], idx, s["index"]))
    s["dst_w"][..., :keep] = torch.where(valid[:, None], s["w"].gather(-1, idx), s["dst_w"][..., :keep])
    s["dst_lens"].copy_(new_len)
    blocks = valid.view(B, 1, keep // BLOCK, BLOCK).any(-1)
    bi, hi = torch.arange(B, device=dev)[:, None, None], torch.arange(H, device=dev)[None, :, None]
    _requantise(k8[bi, hi, idx], ks.gather(-1, idx // BLOCK), ks, s["dst"][0], s["dst"][2], over, valid, blocks)
    _requantise(v8[bi, hi, idx], vs.gather(-1, idx // BLOCK), vs, s["dst"][1], s["dst"][3], over, valid, blocks)


def _requantise(codes, scale, old, dst, dst_s, over, valid, blocks):
    """codes [B, H, keep, D] with a scale each: sequences that lost tokens get new scales max|value| / 127 and codes;
    the others are copied."""
    B, H, keep, D = codes.shape
    x = (codes.float() * scale[..., None]).view(B, H, keep // BLOCK, BLOCK, D)
    s = x.abs().amax((3, 4))
    s = s / torch.full_like(s, 127.0)
    q = (x / torch.where(s > 0, s, torch.ones_like(s))[..., None, None]).round().clamp(-127, 127).to(torch.int8)
    q = torch.where(over[:, None, None, None], q.view(B, H, keep, D), codes)
    dst[:, :, :keep] = torch.where(valid[:, None, :, None], q, dst[:, :, :keep])
    nb = keep // BLOCK
    same = torch.nn.functional.pad(old[..., :nb], (0, max(0, nb - old.shape[-1])))
    s = torch.where(over[:, None, None], s, same)
    dst_s[..., :nb] = torch.where(blocks, s, dst_s[..., :nb])


# ---------------------------------------------------------------------------------------------------- work
def work(case):
    """Bytes: codes, scales, rows and weights read or written once each.  Operations: two products of D for each pair
    of a row and a key that it sees (attention), or a handful for each value that is quantised."""
    c = case
    lens, H, D = _lens(c), c["H"], c["D"]
    if c["op"] == "append":
        tok = sum(_counts(c))
        return {"bytes": tok * (c["Hq"] * D * 4 + 2 * H * D * 3) + c["B"] * H * 16, "flops": tok * (c["Hq"] + 2 * H) * D * 4}
    if c["op"] == "attn":
        cnt, G = _counts(c), c["Hq"] // H
        keys = sum(a + b if b else 0 for a, b in zip(lens, cnt))
        pairs = sum(b * a + b * (b + 1) // 2 if c["causal"] else b * (a + b) for a, b in zip(lens, cnt))
        bytes_ = keys * H * (2 * D + 8 / BLOCK + (8 if c["weights"] else 0)) + sum(cnt) * c["Hq"] * D * 4
        return {"bytes": bytes_, "flops": 4.0 * pairs * G * H * D}
    kept = sum(min(a, c["keep"]) for a in lens)
    return {"bytes": H * (4 * sum(lens) + kept * (4 * D + 4 + 4 + 16 / BLOCK)), "flops": kept * H * D * 2 * 4}


# ---------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attn": _exact_attn, "evict": _exact_evict}[case["op"]](s)


def _exact_append(s):
    """The rotated q, and v's scales.  k's scales have no one right value: they are 1/127 of a value rounded to bf16,
    and one at a border of that rounding may go either way.  Codes are whole numbers."""
    c = s["case"]
    B, n, Hq, H, D = (c[k] for k in ("B", "n", "Hq", "H", "D"))
    lens, cnt = _lens(c), _counts(c)
    q, vs = s["q"].double(), s["cache"][3].double().clone()
    for b in range(B):
        m = cnt[b]
        if m == 0:
            continue
        x = s["qkv"][b, :m].double().view(m, Hq + 2 * H, D)
        cs, sn = s["cos"][lens[b]:lens[b] + m].double()[:, None], s["sin"][lens[b]:lens[b] + m].double()[:, None]
        y = x[:, :Hq].clone()
        y[..., 0:ROT:2] = x[:, :Hq, :16] * cs - x[:, :Hq, 16:32] * sn
        y[..., 1:ROT:2] = x[:, :Hq, :16] * sn + x[:, :Hq, 16:32] * cs
        q[b, :m] = y
        for blk in range(lens[b] // BLOCK, (lens[b] + m - 1) // BLOCK + 1):
            lo, hi = max(blk * BLOCK, lens[b]), min((blk + 1) * BLOCK, lens[b] + m)
            need = x[lo - lens[b]:hi - lens[b], Hq + H:].abs().amax((0, 2)) / 127.0
            have = vs[b, :, blk].clone()
            grown = have * torch.exp2(torch.ceil(torch.log2((need / have).clamp(min=1.0))))
            vs[b, :, blk] = grown if lo > blk * BLOCK else need
    return {"q": q, "k": None, "v": None, "ks": None, "vs": vs}


def _exact_attn(s):
    c = s["case"]
    B, n, Hq, H, D = (c[k] for k in ("B", "n", "Hq", "H", "D"))
    G, (k8, v8, ks, vs) = Hq // H, s["cache"]
    lens, cnt = _lens(c), _counts(c)
    out = s["out"].double()
    w = s["w"].double() if c["weights"] else None
    for b in range(B):
        m, T = cnt[b], lens[b] + cnt[b]
        if m == 0:
            if w is not None:
                w[b, :, :T] = s["w_in"][b, :, :T].double()
            continue
        at = torch.arange(T, device=k8.device) // BLOCK
        see = torch.arange(T, device=k8.device)[None] <= lens[b] + torch.arange(m, device=k8.device)[:, None]
        for h in range(H):
            k = k8[b, h, :T].double() * ks[b, h, at].double()[:, None]
            v = v8[b, h, :T].double() * vs[b, h, at].double()[:, None]
            tot = torch.zeros(T, dtype=F64, device=k8.device)
            for u in range(h * G, h * G + G):
                z = s["q"][b, :m, u].double() @ k.T / math.sqrt(D)
                if c["causal"]:
                    z = z.masked_fill(~see, -math.inf)
                p = torch.softmax(z, dim=-1)
                out[b, :m, u * D:(u + 1) * D] = p @ v
                tot += p.sum(0)
            if w is not None:
                tot[:lens[b]] += s["w_in"][b, h, :lens[b]].double()
                w[b, h, :T] = tot
    return {"out": out, "w": w} if c["weights"] else {"out": out}


def _exact_evict(s):
    """Scales and weights of the kept tokens; codes, lengths and slots are whole numbers."""
    c = s["case"]
    B, H, D, keep, recent = (c[k] for k in ("B", "H", "D", "keep", "recent"))
    k8, v8, ks, vs = s["cache"]
    lens = _lens(c)
    dks, dvs, dw = (t.double() for t in (s["dst"][2], s["dst"][3], s["dst_w"]))
    for b in range(B):
        T = lens[b]
        if T <= keep:
            nb = (T + BLOCK - 1) // BLOCK
            dks[b, :, :nb], dvs[b, :, :nb], dw[b, :, :T] = ks[b, :, :nb].double(), vs[b, :, :nb].double(), s["w"][b, :, :T].double()
            continue
        order = torch.argsort(-s["w"][b, :, :T - recent].double(), dim=-1, stable=True)[:, :keep - recent]
        tail = torch.arange(T - recent, T, device=k8.device).expand(H, recent)
        idx = torch.cat([order.sort(-1).values, tail], dim=-1)
        dw[b, :, :keep] = s["w"][b].double().gather(-1, idx)
        for codes, scale, to in ((k8, ks, dks), (v8, vs, dvs)):
            top = codes[b].abs().amax(-1).gather(-1, idx).double() * scale[b].double().gather(-1, idx // BLOCK)
            to[b, :, :keep // BLOCK] = top.view(H, -1, BLOCK).amax(-1) / 127.0
    return {"k": None, "v": None, "ks": dks, "vs": dvs, "w": dw, "lens": None, "index": None}
