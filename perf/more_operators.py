"""Workloads of many answers about one context: attention of sequences that share a prefix, the choice of a beam search, and the
reordering of caches that follows it.

A cache holds, for B sequences x H heads x C slots (C a multiple of 64) x D dims, int8 codes k, v [B, H, C, D] and one fp32
scale per 64 slots and head ks, vs [B, H, C / 64]; a value is code * scale.  Of layers, it has their number in front.

  shared   S prefixes, F sequences on each: sequence b holds lens[b] tokens of its own behind the plens[b // F] of prefix
           b // F, and counts[b] <= n new ones, which its own cache has already.  Row i sees the whole prefix and
           its own slots 0 .. lens[b] + i
  select   the k best of a group's F x V continuations by score + log softmax(logits), in order, the lowest beam * V + token
           first where totals are equal; a finished beam goes on as it is, with its one token
  reorder  sequence b becomes sequence parents[b]: in place for the beams of a group, or into another cache

run() computes them with elementary torch operations, or, where `own` is true, by the framework's entry points.
"""
import math

import torch

own = False

BLOCK = 64        # slots that share a scale
VOCAB = 51200     # the text decoder's vocabulary
BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32


# ---------------------------------------------------------------------------------------------------- cases
def _shared(name, S, F, n, Hq, H, D, P, L, ragged=False):
    return {"name": name, "op": "shared", "S": S, "F": F, "n": n, "Hq": Hq, "H": H, "D": D, "P": P, "L": L, "ragged": ragged}


def _select(name, S, F, k, V, dtype="bf16", done=False, first=False, banned=False):
    return {"name": name, "op": "select", "S": S, "F": F, "k": k, "V": V, "dtype": dtype, "done": done, "first": first,
            "banned": banned}


def _reorder(name, layers, S, F, H, D, L, ragged=False, sources=0):
    """sources: 0 in place among the F beams of each of S groups, else into another cache from that many sequences."""
    return {"name": name, "op": "reorder", "layers": layers, "S": S, "F": F, "H": H, "D": D, "L": L, "ragged": ragged,
            "sources": sources}


def listed():
    return [
        # one layer of the text decoder (32 heads x 64): four beams of one answer, a token each, behind the image prefix
        _shared("shared beams", 1, 4, 1, 32, 32, 64, 730, 38),
        # 32 questions of up to 32 tokens about one image, at once
        _shared("shared questions", 1, 32, 32, 32, 32, 64, 730, 0, ragged=True),
        # a served batch: eight images, twelve sequences on each, a token each
        _shared("shared images", 8, 12, 1, 32, 32, 64, 730, 60, ragged=True),
        # 64 conversations behind one long instruction, a token each
        _shared("shared prompt", 1, 64, 1, 32, 8, 128, 8191, 1001, ragged=True),
        # sixteen short answers about one long document, a token each
        _shared("shared document", 1, 16, 1, 32, 8, 128, 131007, 65),
        # eight continuations of one context, a chunk of 256 tokens each
        _shared("shared chunk", 1, 8, 256, 32, 8, 128, 6001, 511, ragged=True),
        # one answer's four beams
        _select("select beams", 1, 4, 4, VOCAB, "fp32"),
        # 32 answers' eight beams, some of them finished, twice as many candidates as beams
        _select("select batch", 32, 8, 16, VOCAB, done=True),
        # many wide beams over a vocabulary of odd size, some words banned
        _select("select wide", 16, 32, 32, 100003, "fp32", banned=True),
        # all 24 layers of the text decoder: four beams of one answer
        _reorder("reorder beams", 24, 1, 4, 32, 64, 38),
        # the same for a served batch of answers that differ in length
        _reorder("reorder batch", 24, 8, 8, 32, 64, 250, ragged=True),
        # one layer's batch with grouped heads, forked out of 16 contexts into another cache
        _reorder("reorder fork", 1, 1, 64, 8, 128, 4099, ragged=True, sources=16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: heads 64 or 128 wide, groups of 1 to 8 query heads, prefixes and own lengths over their whole range."""
    op = rng.choice(("shared", "shared", "select", "reorder"))
    D = rng.choice((64, 128))
    H = rng.choice((1, 2, 4, 8, 16, 32)) if D == 64 else rng.choice((1, 2, 3, 4, 8))
    if op == "shared":
        G = rng.choice((1, 1, 2, 4, 5, 8)) if H <= 8 else 1
        S, F = rng.choice((1, 1, _log(rng, 2, 16))), _log(rng, 1, 64)
        n = rng.choice((1, 1, 1, _log(rng, 2, 64), _log(rng, 65, 300)))
        P, L = _log(rng, 1, 131000), rng.choice((0, _log(rng, 1, 2000)))
        while S * H * D * (P + F * (L + n)) > 8 * 128 * 130000 or \
                S * F * H * G * n * D * (P + (L + n) * S) > 8 * 256 * 32 * 128 * 6500:
            c = rng.random()
            if n > 8 and c < 0.4:
                n = n // 2 + 1
            elif S > 1 and c < 0.6:
                S = (S + 1) // 2
            elif F > 1 and c < 0.7:
                F = (F + 1) // 2
            else:
                P, L = P // 2 + 1, L // 2
        return _shared("", S, F, n, G * H, H, D, P, L, rng.random() < 0.6)
    if op == "select":
        F, V = _log(rng, 1, 32), rng.choice((VOCAB, _log(rng, 500, 130000)))
        S = _log(rng, 1, 32)
        while S * F * V > 16 * 32 * 100003:
            S = S // 2
        return _select("", S, F, rng.choice((F, F, min(2 * F, 64))), V, rng.choice(("bf16", "fp32")), rng.random() < 0.4,
                       rng.random() < 0.2, rng.random() < 0.3)
    layers, F, S = rng.choice((1, 2, 24)), _log(rng, 2, 32), _log(rng, 1, 16)
    L = _log(rng, 1, 4000)
    while layers * S * F * H * L * D > 24 * 64 * 32 * 180 * 64:
        S, L = (S + 1) // 2, L // 2 + 1
    return _reorder("", layers, S, F, H, D, L, rng.random() < 0.6, rng.choice((0, 0, max(1, S * F // 4))))


def _plens(c):
    """Tokens of each prefix, a function of the case alone."""
    P = c["P"]
    return [P - (s * 977) % (P // 4 + 1) if c["ragged"] else P for s in range(c["S"])]


def _lens(c):
    """Tokens that each sequence holds: L, or from about L / 2 to L (of beams: the same in a group)."""
    L, F = c["L"], c["F"]
    if c["op"] == "reorder":
        if c["sources"]:
            return [L - (b * 7919) % (L // 2 + 1) if c["ragged"] else L for b in range(c["sources"])]
        return [L - (b // F * 7919) % (L // 2 + 1) if c["ragged"] else L for b in range(c["S"] * F)]
    return [L - (b * 7919) % (L // 2 + 1) if c["ragged"] else L for b in range(c["S"] * F)]


def _counts(c):
    """New tokens of each sequence: n, or in a ragged batch from about n / 4 to n, and now and then none (an idle sequence)."""
    n, B = c["n"], c["S"] * c["F"]
    if not c["ragged"]:
        return [n] * B
    return [0 if b % 9 == 8 else n - (b * 5) % (n * 3 // 4 + 1) for b in range(B)]


def _parents(c):
    """The sequence that each becomes: beams mostly follow the better ones of their group, a few stay; forks go round."""
    F = c["F"]
    if c["sources"]:
        return [(b * 5 + b // 7) % c["sources"] for b in range(c["S"] * F)]
    return [b // F * F + ((b % F) * (b % F) * 5 // (3 * F + 1) + b // F * (b % 3)) % F for b in range(c["S"] * F)]


def _capacity(tokens):
    return (tokens + BLOCK - 1) // BLOCK * BLOCK + BLOCK


# ---------------------------------------------------------------------------------------------------- inputs
def _cache(lead, H, C, D, g, dev):
    """Codes and scales as quantised keys and values have them: near-normal values, some channels larger, scales that
    differ from block to block."""
    gain = torch.rand(2, H, 1, D, device=dev, generator=g) * 0.8 + 0.6
    B = math.prod(lead)
    codes = [torch.empty(B, H, C, D, dtype=torch.int8, device=dev) for _ in range(2)]
    step = max(1, (1 << 26) // (H * C * D))
    for w in range(2):
        for b in range(0, B, step):
            x = torch.randn(min(step, B - b), H, C, D, device=dev, generator=g).mul_(32.0).mul_(gain[w])
            codes[w][b:b + step] = x.round_().clamp_(-127, 127).to(torch.int8)
    ks, vs = (torch.rand(*lead, H, C // BLOCK, device=dev, generator=g) * 0.02 + 0.015 for _ in range(2))
    return codes[0].view(*lead, H, C, D), codes[1].view(*lead, H, C, D), ks, vs


def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    i32 = lambda x: torch.tensor(x, dtype=I32, device=dev)
    s = {"case": dict(c)}
    B = c["S"] * c["F"]
    if c["op"] == "shared":
        n, Hq, H, D = (c[k] for k in ("n", "Hq", "H", "D"))
        s["prefix"], s["plens"] = _cache((c["S"],), H, _capacity(c["P"]), D, g, dev), i32(_plens(c))
        s["cache"], s["lens"] = _cache((B,), H, _capacity(c["L"] + n), D, g, dev), i32(_lens(c))
        s["counts"] = i32(_counts(c)) if c["ragged"] else None
        s["q"] = (torch.randn(B, n, Hq, D, device=dev, generator=g) * 1.7).to(BF16)
        s["out"] = torch.zeros(B, n, Hq * D, dtype=BF16, device=dev)
    elif c["op"] == "select":
        S, F, V = c["S"], c["F"], c["V"]
        x = torch.randn(B, V, device=dev, generator=g) * 2.5
        # a few words stand out in each row, as they do in text
        top = torch.randint(0, V, (B, 5), device=dev, generator=g)
        x.scatter_add_(1, top, torch.rand(B, 5, device=dev, generator=g) * 8.0)
        if c["banned"]:
            x.masked_fill_(torch.rand(V, device=dev, generator=g) < 0.2, -math.inf)
        s["eos"] = V // 3
        if c["banned"]:
            x[:, s["eos"]] = -1.0
        s["logits"] = x.to(BF16) if c["dtype"] == "bf16" else x
        s["scores"] = -torch.rand(B, device=dev, generator=g) * 6.0 - 10.0
        s["done"] = torch.rand(B, device=dev, generator=g) < (0.25 if c["done"] else -1.0)
        if c["first"]:  # the first step of an answer: its beams are one
            s["scores"] = torch.where(torch.arange(B, device=dev) % F == 0, torch.zeros_like(s["scores"]), -math.inf)
            s["done"].zero_()
    else:
        H, D, layers, src = c["H"], c["D"], c["layers"], c["sources"]
        C = _capacity(c["L"])
        s["cache"], s["lens"], s["parents"] = _cache((layers, src or B), H, C, D, g, dev), i32(_lens(c)), i32(_parents(c))
        s["dst"] = tuple(torch.zeros(layers, B, *t.shape[2:], dtype=t.dtype, device=dev) for t in s["cache"]) if src else None
        s["new_lens"] = torch.zeros(B, dtype=I32, device=dev)
    return s


# ---------------------------------------------------------------------------------------------------- the passes
def run(state):
    s = state
    c = s["case"]
    if c["op"] == "shared":
        if own:
            from strix_halo_maxx_b200 import ops
            ops.attn_kv8_shared(s["q"], ops.Kv8(*s["prefix"]), s["plens"], ops.Kv8(*s["cache"]), s["lens"], s["out"],
                                counts=s["counts"])
        else:
            _plain_shared(s)
        return {"out": s["out"]}
    if c["op"] == "select":
        if own:
            from strix_halo_maxx_b200 import ops
            return ops.beam_select(s["logits"], s["scores"], c["F"], k=c["k"], eos=s["eos"], done=s["done"])._asdict()
        return _plain_select(s)
    if own:
        from strix_halo_maxx_b200 import ops
        ops.kv8_reorder(ops.Kv8(*s["cache"]), s["parents"], s["lens"], beams=None if c["sources"] else c["F"],
                        dst=ops.Kv8(*s["dst"]) if c["sources"] else None, new_lens=s["new_lens"])
    else:
        _plain_reorder(s)
    return {**dict(zip(("k", "v", "ks", "vs"), s["dst"] or s["cache"])), "lens": s["new_lens"]}


def _values(cache, T):
    """fp32 values [B, H, T', D] of the blocks that hold the first T slots."""
    k8, v8, ks, vs = cache
    B, H, C, D = k8.shape
    T = min(C, (T + BLOCK - 1) // BLOCK * BLOCK)
    return ((t[:, :, :T].float().view(B, H, -1, BLOCK, D) * sc[:, :, :T // BLOCK, None, None]).view(B, H, T, D)
            for t, sc in ((k8, ks), (v8, vs)))


def _plain_shared(s):
    c, lens, plens = s["case"], s["lens"].long(), s["plens"].long()
    S, F, n, Hq, H, D = (c[k] for k in ("S", "F", "n", "Hq", "H", "D"))
    B, G, dev = S * F, Hq // H, lens.device
    cnt = s["counts"].long() if s["counts"] is not None else torch.full((B,), n, device=dev)
    q = s["q"].float().view(B, n, H, G, D).permute(0, 2, 3, 1, 4)                            # [B, H, G, n, D]
    kp, vp = _values(s["prefix"], c["P"])
    k, v = _values(s["cache"], c["L"] + n)
    i, jp, j = torch.arange(n, device=dev), torch.arange(kp.shape[2], device=dev), torch.arange(k.shape[2], device=dev)
    # scores over the prefix, once for the rows of all of its sequences
    qp = q.reshape(S, F, H, G * n, D).transpose(1, 2).reshape(S, H, F * G * n, D)
    zp = (qp @ kp.transpose(-1, -2)) * D ** -0.5
    zp.masked_fill_((jp >= plens[:, None])[:, None, None], -math.inf)
    z = (q.reshape(B, H, G * n, D) @ k.transpose(-1, -2)).view(B, H, G, n, -1) * D ** -0.5
    z.masked_fill_((j > lens[:, None, None] + i[:, None])[:, None, None], -math.inf)
    z = z.view(B, H, G * n, -1)
    split = lambda t: t.view(S, H, F, G * n, -1).transpose(1, 2).reshape(B, H, G * n, -1)    # of a prefix's rows, by sequence
    join = lambda t: t.view(S, F, H, G * n, -1).transpose(1, 2).reshape(S, H, F * G * n, -1)
    top = torch.maximum(split(zp.amax(-1, keepdim=True)), z.amax(-1, keepdim=True))
    zp.sub_(join(top)).exp_()
    z.sub_(top).exp_()
    total = split(zp.sum(-1, keepdim=True)) + z.sum(-1, keepdim=True)
    o = (split(zp @ vp) + z @ v) / total
    o = o.view(B, H, G, n, D).permute(0, 3, 1, 2, 4).reshape(B, n, Hq * D)
    s["out"].copy_(torch.where((i < cnt[:, None])[..., None], o.to(BF16), s["out"]))


def _plain_select(s):
    c, x = s["case"], s["logits"].double()
    S, F, k, V = (c[k] for k in ("S", "F", "k", "V"))
    # in 64 bits: candidates of different beams lie as close together as their scores do by chance
    top = x.amax(-1, keepdim=True)
    total = s["scores"].double()[:, None] + (x - (top + (x - top).exp().sum(-1, keepdim=True).log()))
    words = torch.arange(V, device=x.device)
    held = torch.where(words == s["eos"], s["scores"].double()[:, None], -math.inf)          # a finished beam's one candidate
    total = torch.where(s["done"][:, None], held, total)
    total = torch.where(total.isnan(), -math.inf, total).view(S, F * V)
    value, at = torch.sort(total, dim=-1, descending=True, stable=True)
    value, at = value[:, :k], at[:, :k]
    none = value == -math.inf
    rows = torch.arange(S, device=x.device)[:, None] * F
    parents = rows + torch.where(none, torch.arange(k, device=x.device) % F, at // V)
    tokens = torch.where(none, -1, at % V)
    done = none | (tokens == s["eos"]) | s["done"][parents]
    return {"scores": value.float(), "parents": parents.int(), "tokens": tokens.int(), "done": done}


def _plain_reorder(s):
    src, dst = s["cache"], s["dst"] or s["cache"]
    at = s["parents"].long()
    lens = s["lens"].long()[at]                                                              # of what each becomes
    slot = torch.arange(src[0].shape[3], device=at.device) < lens[:, None]
    block = torch.arange(src[2].shape[3], device=at.device) * BLOCK < lens[:, None]
    for a, b in zip(src[:2], dst[:2]):
        b.copy_(torch.where(slot[None, :, None, :, None], a[:, at], b))
    for a, b in zip(src[2:], dst[2:]):
        b.copy_(torch.where(block[None, :, None], a[:, at], b))
    s["new_lens"].copy_(lens)


# ---------------------------------------------------------------------------------------------------- work
def work(case):
    """Bytes: codes, scales, rows and logits read or written once each, a prefix once for all of its sequences, what several
    sequences become once, and none that stay as they are.  Operations: two products of D for each pair of a row and a key
    that it sees, or a handful for each logit."""
    c = case
    if c["op"] == "shared":
        D, H, G, F = c["D"], c["H"], c["Hq"] // c["H"], c["F"]
        lens, cnt, plens = _lens(c), _counts(c), _plens(c)
        keys = sum(plens) + sum(a + b for a, b in zip(lens, cnt) if b)
        pairs = sum(b * (plens[i // F] + a) + b * (b + 1) // 2 for i, (a, b) in enumerate(zip(lens, cnt)))
        return {"bytes": keys * H * (2 * D + 8 / BLOCK) + sum(cnt) * c["Hq"] * D * 4, "flops": 4.0 * pairs * G * H * D}
    if c["op"] == "select":
        B = c["S"] * c["F"]
        return {"bytes": B * (c["V"] * (2 if c["dtype"] == "bf16" else 4) + 5) + c["S"] * c["k"] * 13, "flops": 4.0 * B * c["V"]}
    lens, parents = _lens(c), _parents(c)
    moved = [(b, p) for b, p in enumerate(parents) if c["sources"] or p != b]
    tokens = sum(lens[p] for p in {p for _, p in moved}) + sum(lens[p] for _, p in moved)
    return {"bytes": c["layers"] * c["H"] * tokens * (2 * c["D"] + 8 / BLOCK) + 12 * len(parents), "flops": 0.0}


# ---------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"shared": _exact_shared, "select": _exact_select, "reorder": _exact_reorder}[case["op"]](s)


def _exact_shared(s):
    c = s["case"]
    n, Hq, H, D, F = (c[k] for k in ("n", "Hq", "H", "D", "F"))
    G, lens, cnt, plens = Hq // H, _lens(c), _counts(c), _plens(c)
    out = s["out"].double()

    def value(codes, scale, b, h, T):
        at = torch.arange(T, device=codes.device) // BLOCK
        return codes[b, h, :T].double() * scale[b, h, at].double()[:, None]

    for p in range(c["S"]):
        for h in range(H):
            kp, vp = (value(s["prefix"][w], s["prefix"][w + 2], p, h, plens[p]) for w in range(2))
            for b in range(p * F, p * F + F):
                m, T = cnt[b], lens[b] + cnt[b]
                if m == 0:
                    continue
                k, v = (torch.cat([t, value(s["cache"][w], s["cache"][w + 2], b, h, T)]) for w, t in enumerate((kp, vp)))
                see = torch.arange(len(k), device=k.device)[None] <= plens[p] + lens[b] + torch.arange(m, device=k.device)[:, None]
                q = s["q"][b, :m, h * G:(h + 1) * G].double().transpose(0, 1)               # [G, m, D]
                z = (q @ k.T / math.sqrt(D)).masked_fill(~see, -math.inf)
                out[b, :m, h * G * D:(h + 1) * G * D] = (torch.softmax(z, dim=-1) @ v).transpose(0, 1).reshape(m, G * D)
    return {"out": out}


def _exact_select(s):
    """The scores of the choice; beams, words and flags are whole numbers."""
    c = s["case"]
    S, F, k, V = (c[k] for k in ("S", "F", "k", "V"))
    best = []
    for b in range(S * F):
        if bool(s["done"][b]):
            row = s["scores"][b:b + 1].double()
        else:
            x = s["logits"][b].double()
            row = torch.topk(torch.log_softmax(x, dim=-1), min(k, V)).values + s["scores"][b].double()
        best.append(torch.nn.functional.pad(row, (0, k - len(row)), value=-math.inf))
    scores = torch.topk(torch.stack(best).view(S, F * k), k, dim=-1).values
    return {"scores": scores, "parents": None, "tokens": None, "done": None}


def _exact_reorder(s):
    """The scales of the blocks that each sequence gets; codes and lengths are whole numbers."""
    c = s["case"]
    lens, res = _lens(c), {"k": None, "v": None, "lens": None}
    for name, old, to in (("ks", s["cache"][2], (s["dst"] or s["cache"])[2]), ("vs", s["cache"][3], (s["dst"] or s["cache"])[3])):
        res[name] = to.double()
        for b, p in enumerate(_parents(c)):
            blocks = (lens[p] + BLOCK - 1) // BLOCK
            res[name][:, b, :, :blocks] = old[:, p, :, :blocks].double()
    return res
