"""The moondream2 text decoder that consumes the tower's features, on B200: FastMD2's image prefill and question
prefill (moondream/gpu/md2fast.py:169-212) with the tower's kernels plus the rotary / KV-cache and causal
attention kernels of csrc/text.cu.

Per layer (md2fast.py:169-199, the parallel block):
    h = LN(x)                                   vt_layernorm, bf16
    qkv = h Wqkv^T + b                          vt_gemm (N = 3 x 2048)
    rope(q, k), cache k / v                     vt_rope_qkv
    a = attention                               prefix: tcgen05 attention over its 730 keys (no mask, as
                                                md2fast.py:182-183); question: vt_attn_causal over the cache
    x += a Wproj^T + b                          vt_gemm, fp32 residual epilogue
    x += gelu_tanh(h W1^T + b1) W2^T + b2       vt_gemm (GELU epilogue), vt_gemm + residual
The yes / no logits are LN(x[last]) Wyn^T + byn (md2fast.py:210-212).  The four linears run either as the
tower's bf16 tcgen05 GEMMs (int8=False, the reference's FastMD2 with tlin_cls=HLin) or as W8A8 int8 tcgen05
GEMMs (int8=True, tlin_cls=HI8Lin, md2fast.py:88, 112-113): per layer the LN output is quantised once, in the
LayerNorm kernel (vt_layernorm_quant), and shared by qkv and fc1 (md2fast.py:174); the attention output and the
fc1 output (GELU fused into its epilogue) are quantised before proj and fc2 (vt_quant_rows + vt_gemm_i8,
ops.I8Lin).  The KV caches ([layers][H][762][64]
bf16) live on the device, owned by this object: encode() fills positions 0 .. 729, query() 730 .. 761.

kv8=True holds the caches in 8 bits with a scale per 64 tokens and head (ops.Kv8: half the bytes): vt_rope_kv8 writes
them and vt_attn_kv8 reads them, for the prefix (no mask) and for the question (causal).  keep=N then evicts: each
head of each layer keeps the N image-prefix tokens that the prefix's own attention weighed most (the last keep_recent
among them in any case), and questions attend to those; their positions go on at 730.

Many answers about one image (kv8=True) share its prefix, which vt_attn_kv8_shared reads once for all:
    questions=Q      query_many() answers up to Q questions at once; the reference asks one after another (md2fast.py:208-212)
    beams=F, steps=N answer() is a beam search of F beams and N words over the whole lm head (weights lm_w [vocab, dim], lm_b):
                     each step writes the beams' words into their caches, attends, chooses (vt_beam_select) and lets the caches of all
                     layers follow the choice (vt_kv8_reorder), replayed from one CUDA graph.
"""
from types import SimpleNamespace

import torch

from .config import TEXT, TextConfig
from . import ops
from .ops import BF16
from .tower import _dev_mat, _dev_vec

F32 = torch.float32


def rope_tables(cfg: TextConfig, device, more=0):
    """cos, sin fp32 [ctx + more, rot / 2]: angle pos * theta^(-2i / rot), evaluated in float64."""
    inv = cfg.theta ** (-torch.arange(0, cfg.rot, 2, dtype=torch.float64) / cfg.rot)
    ang = torch.arange(cfg.ctx + more, dtype=torch.float64)[:, None] * inv[None]
    return torch.cos(ang).float().contiguous().to(device), torch.sin(ang).float().contiguous().to(device)


class TextDecoder:
    def __init__(self, weights, cfg: TextConfig = TEXT, device="cuda", graphs=True, int8=False, kv8=False, keep=None,
                 keep_recent=32, questions=0, beams=0, steps=0):
        if keep is not None and (not kv8 or keep <= 0 or keep % ops.KV8_BLOCK or keep >= cfg.prefix or
                                 not 0 <= keep_recent <= keep):
            raise ValueError(f"keep={keep}: needs kv8, a multiple of {ops.KV8_BLOCK} below the prefix of {cfg.prefix} tokens, "
                             f"and 0 <= keep_recent={keep_recent} <= keep")
        if (questions or beams) and not kv8 or questions < 0 or not 0 <= beams <= 64 or (steps <= 0) != (beams == 0):
            raise ValueError(f"questions={questions}, beams={beams} (at most 64), steps={steps}: need kv8, and steps with beams")
        if beams and "lm_w" not in weights:
            raise ValueError("beams need the whole lm head: weights lm_w [vocab, dim] and lm_b")
        if beams and weights["lm_w"].shape[0] > weights["wte"].shape[0]:  # a chosen word is the next step's input
            raise ValueError(f"an lm head of {weights['lm_w'].shape[0]} words, embeddings of {weights['wte'].shape[0]}")
        self.cfg = cfg
        self.use_graphs = graphs
        self.int8 = int8
        self.kv8, self.keep, self.keep_recent = kv8, keep, keep_recent
        self._qgraph = self._egraph = None
        dev = self.dev = torch.device(device)
        if dev.type == "cuda" and dev.index is None:
            dev = self.dev = torch.device("cuda", torch.cuda.current_device())
        W = weights
        self.n_layers = sum(1 for k in W if k.endswith(".qkv_w"))
        self.wte = _dev_vec(W["wte"], dev)
        self.layers = []
        for i in range(self.n_layers):
            p = f"tblocks.{i}."
            b = {"ln_w": _dev_vec(W[p + "ln_w"], dev), "ln_b": _dev_vec(W[p + "ln_b"], dev)}
            for n in ("qkv", "proj", "fc1", "fc2"):
                if int8:
                    b[n] = ops.I8Lin(W[p + n + "_w"], W[p + n + "_b"], dev)
                    continue
                b[n + "_w"], b[n + "_ld"] = _dev_mat(W[p + n + "_w"], dev)
                b[n + "_b"] = _dev_vec(W[p + n + "_b"], dev)
            self.layers.append(b)
        self.post_w, self.post_b = _dev_vec(W["tpost_ln_w"], dev), _dev_vec(W["tpost_ln_b"], dev)
        self.yn_w, self.yn_ld = _dev_mat(W["lm_small_w"], dev)
        self.yn_b = _dev_vec(W["lm_small_b"], dev)
        self.cos, self.sin = rope_tables(cfg, dev, steps)
        D, H, hd, P = cfg.dim, cfg.heads, cfg.head_dim, cfg.prefix
        R = max(P, questions * cfg.q_len, beams)  # rows of the largest pass
        self.x = torch.empty(R, D, dtype=F32, device=dev)
        self.h = torch.empty(R, D, dtype=BF16, device=dev)
        self.qkv = torch.empty(R, 3 * D, dtype=BF16, device=dev)
        self.qflat = torch.empty(H * R * hd, dtype=BF16, device=dev)
        self.a = torch.zeros(R, D, dtype=BF16, device=dev)
        self.f = torch.empty(R, cfg.ff, dtype=BF16, device=dev)
        if kv8:
            self._init_kv8(dev)
            self.many = self._many(questions, cfg.q_len, cfg.q_len, dev) if questions else None
            self.beam = self._many(beams, 1, cfg.q_len + steps, dev) if beams else None
            if beams:
                self._init_beams(W, steps, dev)
        else:
            self.kc = torch.zeros(self.n_layers, H, cfg.ctx, hd, dtype=BF16, device=dev)
            self.vc = torch.zeros(self.n_layers, H, cfg.ctx, hd, dtype=BF16, device=dev)
        self.hl = torch.empty(1, D, dtype=BF16, device=dev)
        self.xl = torch.empty(1, D, dtype=F32, device=dev)
        self._ids = torch.zeros(cfg.q_len, dtype=torch.int64, device=dev)
        self._last = torch.zeros(1, dtype=torch.int64, device=dev)
        self._bos = torch.zeros(1, dtype=torch.int64, device=dev)
        self._emb = torch.zeros(P - 1, D, dtype=F32, device=dev)
        self.logits = torch.empty(1, 8, dtype=F32, device=dev)
        self.attn = ops.VtAttn(H, P, hd, dev)
        if int8:  # quantised activations (padded 16-byte row pitches) and their per-token scales
            pad = lambda k: (k + ops.I8_PAD + 15) // 16 * 16
            self.hq = torch.empty(R, pad(D), dtype=torch.int8, device=dev)[:, :D]
            self.aq = torch.empty(R, pad(D), dtype=torch.int8, device=dev)[:, :D]
            self.fq = torch.empty(R, pad(cfg.ff), dtype=torch.int8, device=dev)[:, :cfg.ff]
            self.hs, self.as_, self.fs = (torch.empty(R, dtype=F32, device=dev) for _ in range(3))
        # split-K workspace of the question's GEMMs (32 rows; the widest output is fc1's)
        self.ws = ops.gemm_workspace(cfg.q_len, max(3 * D, cfg.ff), dev)

    def _init_kv8(self, dev):
        """The layers' 8-bit caches: the layers are the batch of one eviction call, each alone a batch of one sequence."""
        cfg, L = self.cfg, self.n_layers
        H, hd, P = cfg.heads, cfg.head_dim, cfg.prefix
        i32 = lambda x, n: torch.full((n,), x, dtype=torch.int32, device=dev)
        self.kv = self.kv_q = ops.kv8_cache(L, H, cfg.ctx, hd, dev)  # the prefix's, the question's
        self.len_0, self.len_p = i32(0, 1), i32(P, L)
        self.len_q = self.len_p                                      # tokens before the question
        if self.keep is not None:
            self.kv_q = ops.kv8_cache(L, H, self.keep + cfg.q_len, hd, dev)
            self.len_q = i32(0, L)
            self.attn_w = torch.zeros(L, H, self.kv.k.shape[2], device=dev)
            self.attn_w_q = torch.zeros(L, H, self.kv_q.k.shape[2], device=dev)
            self.kept = torch.zeros(L, H, self.keep, dtype=torch.int32, device=dev)
        # The prefix ends inside a block, whose scale a question's tokens may double for good: its codes and scales are put back
        # before each question, so that no answer depends on the questions before it
        b = P // ops.KV8_BLOCK
        self.tail = [t[:, :, b * ops.KV8_BLOCK:P] for t in (self.kv.k, self.kv.v)] + [t[:, :, b] for t in (self.kv.ks, self.kv.vs)] \
            if self.keep is None and P % ops.KV8_BLOCK else []
        self.tail_saved = [t.clone(memory_format=torch.contiguous_format) for t in self.tail]
        self.ws8 = ops.attn_kv8_workspace(1, P, H, H, hd, self.kv.k.shape[2], dev, self.keep is not None)

    def _many(self, B, n, slots, dev):
        """B sequences behind the image prefix, n new tokens each, with caches of their own for `slots` tokens in every layer."""
        cfg, L = self.cfg, self.n_layers
        kv = ops.Kv8(*(t.view(L, B, *t.shape[1:]) for t in ops.kv8_cache(L * B, cfg.heads, slots, cfg.head_dim, dev)))
        m = SimpleNamespace(B=B, kv=kv, ids=torch.zeros(B * n, dtype=torch.int64, device=dev), rows=torch.zeros(B, dtype=torch.int64, device=dev),
                            x=torch.empty(B, cfg.dim, dtype=F32, device=dev), h=torch.empty(B, cfg.dim, dtype=BF16, device=dev), graph=None)
        m.lens, m.counts = (torch.zeros(B, dtype=torch.int32, device=dev) for _ in range(2))
        m.pos = torch.full((B,), cfg.prefix, dtype=torch.int32, device=dev)
        m.ws8 = ops.attn_kv8_shared_workspace(1, B, n, cfg.heads, cfg.heads, cfg.head_dim, self.kv_q.k.shape[2], kv.k.shape[3], dev)
        m.ws = ops.gemm_workspace(B * n, max(3 * cfg.dim, cfg.ff), dev) if B * n <= 128 else None
        return m

    def _init_beams(self, W, steps, dev):
        cfg, m = self.cfg, self.beam
        F, V = m.B, W["lm_w"].shape[0]
        self.lm_w, self.lm_ld = _dev_mat(W["lm_w"], dev)
        self.lm_b = _dev_vec(W["lm_b"], dev)
        m.logits = torch.zeros(F, ops._pad8(V), dtype=F32, device=dev)[:, :V]  # the GEMM's rows begin on 32 bytes
        m.best = ops.Beams(*(torch.zeros(1, F, dtype=d, device=dev) for d in (F32, torch.int32, torch.int32, torch.bool)))
        m.ws_select = torch.empty(ops.lib().vt_beam_select_ws_bytes(1, F, V, F), dtype=torch.uint8, device=dev)
        m.first = torch.full((F,), -float("inf"), dtype=F32, device=dev)  # a search begins with one beam
        m.first[0] = 0.0
        m.scores, m.done, m.new_lens = m.first.clone(), torch.zeros(F, dtype=torch.bool, device=dev), torch.zeros_like(m.lens)
        m.tokens, m.parents = (torch.zeros(steps, F, dtype=torch.int32, device=dev) for _ in range(2))
        m.n_first = torch.zeros(1, dtype=torch.int32, device=dev)
        m.first_ws8 = ops.attn_kv8_shared_workspace(1, 1, cfg.q_len, cfg.heads, cfg.heads, cfg.head_dim, self.kv_q.k.shape[2], m.kv.k.shape[3], dev)

    def _attend_many(self, i, qkv, m, B, n, counts, ws8, a):
        """Rotary, cache write and attention of the n new rows of the first B sequences of m behind the prefix, into a [B n, D]."""
        cfg = self.cfg
        cache, prefix = ops.Kv8(*(t[i, :B] for t in m.kv)), ops.Kv8(*(t[i:i + 1] for t in self.kv_q))
        q = self.qflat[:B * n * cfg.dim].view(B, n, cfg.heads, cfg.head_dim)
        ops.rope_kv8(qkv.view(B, n, 3 * cfg.dim), cache, m.lens[:B], self.cos, self.sin, q, pos=m.pos[:B], counts=counts)
        ops.attn_kv8_shared(q, prefix, self.len_q[i:i + 1], cache, m.lens[:B], a.view(B, n, cfg.dim), counts=counts, ws=ws8)

    def _attend_kv8(self, i, qkv, n, full, a):
        """Rotary, cache write and attention of layer i's n new tokens on the 8-bit cache, into a [n, D]."""
        cfg = self.cfg
        cache = ops.Kv8(*(t[i:i + 1] for t in (self.kv if full else self.kv_q)))
        lens = self.len_0 if full else self.len_q[i:i + 1]
        q = self.qflat[:n * cfg.dim].view(1, n, cfg.heads, cfg.head_dim)
        ops.rope_kv8(qkv[None], cache, lens, self.cos, self.sin, q, pos=self.len_0 if full else self.len_p[i:i + 1])
        w = self.attn_w[i:i + 1] if full and self.keep is not None else None
        ops.attn_kv8(q, cache, lens, a[None], causal=not full, weights=w, ws=self.ws8)

    def _layers(self, n, pos0, full):
        H, hd = self.cfg.heads, self.cfg.head_dim
        q = self.qflat[:H * n * hd].view(H, n, hd)
        # the question's GEMMs are too small to fill the GPU: split K
        self._run(n, None if full else self.ws, lambda i, qkv, a: self._attend(i, qkv, q, n, pos0, full, a))

    def _run(self, n, ws, attend):
        """All layers on the n rows of x; attend(i, qkv, a): layer i's attention."""
        cfg = self.cfg
        D, Fh = cfg.dim, cfg.ff
        x, h, qkv, a, f = self.x[:n], self.h[:n], self.qkv[:n], self.a[:n], self.f[:n]
        if self.int8:
            return self._run_i8(n, ws, attend)
        for i, b in enumerate(self.layers):
            ops.layer_norm(x, b["ln_w"], b["ln_b"], cfg.eps, out=h)
            ops.gemm(h, b["qkv_w"], b["qkv_ld"], D, 3 * D, b["qkv_b"], out=qkv, ws=ws)
            attend(i, qkv, a)
            ops.gemm(a, b["proj_w"], b["proj_ld"], D, D, b["proj_b"], res=x, out=x, ws=ws)
            ops.gemm(h, b["fc1_w"], b["fc1_ld"], D, Fh, b["fc1_b"], gelu=True, out=f, ws=ws)
            ops.gemm(f, b["fc2_w"], b["fc2_ld"], Fh, D, b["fc2_b"], res=x, out=x, ws=ws)

    def _attend(self, i, qkv, q, n, pos0, full, a):
        """Rotary, cache write and attention of layer i's n new tokens at pos0 .., into a [n, D]."""
        if self.kv8:
            return self._attend_kv8(i, qkv, n, full, a)
        ops.rope_qkv(qkv, pos0, self.cos, self.sin, q, self.kc[i], self.vc[i])
        if full:  # the prefix: no mask, its own n keys (md2fast.py:182-183)
            self.attn(q[None], self.kc[i][None, :, pos0:pos0 + n], self.vc[i][None, :, pos0:pos0 + n], out=a[None])
        else:     # the question: causal over the cache (md2fast.py:184-185 with the query mask)
            ops.attn_causal(q, self.kc[i], self.vc[i], pos0, a)

    def _run_i8(self, n, ws, attend):
        """The same layers with the W8A8 linears (HI8Lin, md2fast.py:169-199 with SHARE_QUANT)."""
        cfg = self.cfg
        x, h, qkv, a, f = self.x[:n], self.h[:n], self.qkv[:n], self.a[:n], self.f[:n]
        hq, aq, fq = self.hq[:n], self.aq[:n], self.fq[:n]
        hs, as_, fs = self.hs[:n], self.as_[:n], self.fs[:n]
        for i, b in enumerate(self.layers):
            # LN + per-token quantisation in one kernel; the int8 rows are shared by qkv and fc1 (md2fast.py:174)
            pre = ops.layer_norm_quant(x, b["ln_w"], b["ln_b"], cfg.eps, hq, hs)
            b["qkv"](h, pre=pre, out=qkv, ws=ws)
            attend(i, qkv, a)
            b["proj"](a, pre=b["proj"].quant(a, aq, as_), res=x, out=x, ws=ws)
            b["fc1"](h, gelu=True, pre=pre, out=f, ws=ws)
            b["fc2"](f, pre=b["fc2"].quant(f, fq, fs), res=x, out=x, ws=ws)

    def encode(self, emb, bos):
        """Image prefill (md2fast.py:201-206): emb [729, D] fp32 / bf16 on the device, bos id.  The image
        features and the bos id go into static device buffers, so with graphs=True every prefill after the
        first replays one CUDA graph of its ~190 launches (same kernels and buffers as the eager path)."""
        self._emb.copy_(emb)
        self._bos.fill_(int(bos))
        if not self.use_graphs:
            self._encode()
        elif self._egraph is None:
            self._encode()  # first prefill eagerly (one-time library and buffer set-up), then capture
            self._egraph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self._egraph):
                self._encode()
        else:
            self._egraph.replay()
        return self.x

    def _encode(self):
        torch.index_select(self.wte, 0, self._bos, out=self.x[:1])
        self.x[1:self.cfg.prefix].copy_(self._emb)
        self._layers(self.cfg.prefix, 0, True)
        if self.keep is not None:
            ops.kv8_evict(self.kv, self.attn_w, self.len_p, self.keep, self.keep_recent, self.kv_q, self.attn_w_q,
                          self.len_q, index=self.kept)
        if self.kv8:
            for t, saved in zip(self.tail, self.tail_saved):
                saved.copy_(t)

    def query(self, ids, last):
        """Question prefill (md2fast.py:208-212): ids [q_len] int64 on the device, `last` the index of the
        question's last real token -> yes / no logits [n_yn] fp32.  The ids and `last` go into static
        device buffers, so with graphs=True (default) every question after the first replays one CUDA graph
        of the ~170 launches (same kernels and buffers as the eager path, bit-identical logits)."""
        cfg = self.cfg
        self._ids.copy_(ids)
        self._last.fill_(int(last))
        if not self.use_graphs:
            self._query()
        elif self._qgraph is None:
            self._query()  # first question eagerly (one-time library set-up), then capture
            self._qgraph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self._qgraph):
                self._query()
        else:
            self._qgraph.replay()
        return self.logits[0, :cfg.n_yn]

    def _query(self):
        cfg = self.cfg
        torch.index_select(self.wte, 0, self._ids, out=self.x[:cfg.q_len])
        if self.kv8:
            for t, saved in zip(self.tail, self.tail_saved):
                t.copy_(saved)
        self._layers(cfg.q_len, cfg.prefix, False)
        torch.index_select(self.x, 0, self._last, out=self.xl)
        ops.layer_norm(self.xl, self.post_w, self.post_b, cfg.eps, out=self.hl)
        ops.gemm(self.hl, self.yn_w, self.yn_ld, cfg.dim, cfg.n_yn, self.yn_b, out=self.logits[:, :cfg.n_yn], ws=self.ws)


    def _replay(self, m, fn):
        """fn eagerly the first time (one-time library set-up), then captured, and replayed from there on."""
        if not self.use_graphs:
            fn()
        elif m.graph is None:
            fn()
            m.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(m.graph):
                fn()
        else:
            m.graph.replay()

    def _restore_tail(self):
        for t, saved in zip(self.tail, self.tail_saved):
            t.copy_(saved)

    def query_many(self, ids, last):
        """Up to `questions` questions about the image at once: ids [k, q_len] int64 and last [k] (ints or int64) as query() takes
        them -> yes / no logits [k, n_yn] fp32, equal to query()'s up to the rounding of the keys' blocks (a question's keys share no
        block with the image's here).  A `last` outside the question is refused where it is on the host, and cut off where it is on the
        device.  The static buffers and the graph are those of all `questions`; fewer leave the rest idle."""
        cfg, m = self.cfg, self.many
        if m is None or ids.dim() != 2 or ids.shape[1] != cfg.q_len or not 0 < ids.shape[0] <= m.B or len(last) != ids.shape[0]:
            raise ValueError(f"query_many: ids {tuple(ids.shape)} for {0 if m is None else m.B} questions of {cfg.q_len} tokens")
        k = ids.shape[0]
        last = torch.as_tensor(last)
        if last.device.type == "cpu" and not bool(((last >= 0) & (last < cfg.q_len)).all()):
            raise ValueError("query_many: last lies outside the question")
        last = last.to(device=self.dev, dtype=torch.int64).clamp(0, cfg.q_len - 1)
        m.ids.view(m.B, -1)[:k].copy_(ids)
        m.counts.zero_()
        m.counts[:k].copy_(last + 1)
        m.rows[:k].copy_(torch.arange(k, device=self.dev) * cfg.q_len + last)
        self._replay(m, self._query_many)
        return m.logits[:k, :cfg.n_yn]

    def _query_many(self):
        cfg, m = self.cfg, self.many
        if not hasattr(m, "logits"):
            m.logits = torch.zeros(m.B, 8, dtype=F32, device=self.dev)
        n = m.B * cfg.q_len
        torch.index_select(self.wte, 0, m.ids, out=self.x[:n])
        self._restore_tail()
        self._run(n, m.ws, lambda i, qkv, a: self._attend_many(i, qkv, m, m.B, cfg.q_len, m.counts, m.ws8, a))
        torch.index_select(self.x, 0, m.rows, out=m.x)
        ops.layer_norm(m.x, self.post_w, self.post_b, cfg.eps, out=m.h)
        ops.gemm(m.h, self.yn_w, self.yn_ld, cfg.dim, cfg.n_yn, self.yn_b, out=m.logits[:, :cfg.n_yn], ws=m.ws)

    def answer(self, ids, last, eos=-1):
        """Beam search for the answer to one question (ids [q_len] int64, `last` as query() takes them): `beams` beams of `steps` words
        each.  A beam that chooses the word eos is finished (eos < 0: none is) and repeats it at no cost.  Returns (words int64
        [beams, steps], scores fp32 [beams]) on the CPU, the best beam first; scores are sums of log probabilities."""
        cfg, m = self.cfg, self.beam
        if m is None or ids.shape != (cfg.q_len,) or not 0 <= int(last) < cfg.q_len:
            raise ValueError(f"answer: ids {tuple(ids.shape)}, last {last} for {0 if m is None else m.B} beams and a question of {cfg.q_len} tokens")
        if m.graph is not None and m.eos != int(eos):
            m.graph = None
        m.eos = int(eos)
        steps = m.tokens.shape[0]
        self._ids.copy_(ids)
        self._last.fill_(int(last))
        m.n_first.fill_(int(last) + 1)
        m.lens.zero_()
        m.done.zero_()
        m.scores.copy_(m.first)
        m.pos.fill_(cfg.prefix)
        self._first_word()
        m.tokens[0], m.parents[0] = m.best.tokens[0], m.best.parents[0]
        for s in range(1, steps):
            self._replay(m, self._next_word)
            m.tokens[s], m.parents[s] = m.best.tokens[0], m.best.parents[0]
        tokens, parents = m.tokens.cpu().long(), m.parents.cpu().long()
        words, at = torch.empty(m.B, steps, dtype=torch.int64), torch.arange(m.B)
        for s in reversed(range(steps)):
            words[:, s], at = tokens[s][at], parents[s][at]
        return words, m.scores.cpu()

    def _first_word(self):
        """The question, as the first beam's."""
        cfg, m = self.cfg, self.beam
        torch.index_select(self.wte, 0, self._ids, out=self.x[:cfg.q_len])
        self._restore_tail()
        self._run(cfg.q_len, self.ws, lambda i, qkv, a: self._attend_many(i, qkv, m, 1, cfg.q_len, m.n_first, m.first_ws8, a))
        m.lens[:1] += m.n_first
        torch.index_select(self.x, 0, self._last, out=m.x[:1])
        self._choose(1)

    def _next_word(self):
        m = self.beam
        torch.index_select(self.wte, 0, m.ids, out=self.x[:m.B])
        self._run(m.B, m.ws, lambda i, qkv, a: self._attend_many(i, qkv, m, m.B, 1, None, m.ws8, a))
        m.lens += 1
        m.x.copy_(self.x[:m.B])
        self._choose(m.B)

    def _choose(self, n):
        """From the hidden rows of the first n beams: the best continuations, and the beams' caches after them."""
        cfg, m = self.cfg, self.beam
        V = m.logits.shape[1]
        ops.layer_norm(m.x[:n], self.post_w, self.post_b, cfg.eps, out=m.h[:n])
        ops.gemm(m.h[:n], self.lm_w, self.lm_ld, cfg.dim, V, self.lm_b, out=m.logits[:n])
        ops.beam_select(m.logits, m.scores, m.B, eos=m.eos, done=m.done if m.eos >= 0 else None, out=m.best, ws=m.ws_select)
        ops.kv8_reorder(m.kv, m.best.parents[0], m.lens, beams=m.B, new_lens=m.new_lens)
        m.lens.copy_(m.new_lens)
        torch.add(m.lens, cfg.prefix, out=m.pos)
        m.scores.copy_(m.best.scores[0])
        m.done.copy_(m.best.done[0])
        m.ids.copy_(m.best.tokens[0].clamp(min=0))


def op_times(dev, n=20, reps=5):
    """Warm time (us) of each kernel of a decoder layer at the prefill (730) and question (32) row counts:
    every op captured n times in one CUDA graph, replayed `reps` times; inputs L2-resident."""
    F32_ = torch.float32

    def graph_us(fn):
        fn()
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            fn()
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                for _ in range(n):
                    fn()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        e0.record()
        for _ in range(reps):
            g.replay()
        e1.record()
        torch.cuda.synchronize()
        return round(e0.elapsed_time(e1) / (n * reps) * 1000, 2)

    D, Fh = TEXT.dim, TEXT.ff
    out = {}
    for M in (TEXT.prefix, TEXT.q_len):
        ws = ops.gemm_workspace(M, Fh, dev) if M == TEXT.q_len else None
        x = torch.randn(M, D, device=dev)
        w_ln, b_ln = torch.ones(D, device=dev), torch.zeros(D, device=dev)
        h = torch.empty(M, D, device=dev, dtype=BF16)
        hq, hs = torch.empty(M, D, device=dev, dtype=torch.int8), torch.empty(M, device=dev)
        f = torch.randn(M, Fh, device=dev).to(BF16)
        fq, fs = torch.empty(M, Fh, device=dev, dtype=torch.int8), torch.empty(M, device=dev)
        r = {"ln": graph_us(lambda: ops.layer_norm(x, w_ln, b_ln, 1e-5, out=h)),
             "ln_quant": graph_us(lambda: ops.layer_norm_quant(x, w_ln, b_ln, 1e-5, hq, hs)),
             "quant_2048": graph_us(lambda: ops.quant_rows(h, hq, hs)),
             "quant_8192": graph_us(lambda: ops.quant_rows(f, fq, fs))}
        for name, N, K, res, gelu in (("qkv", 3 * D, D, False, False), ("proj", D, D, True, False),
                                      ("fc1", Fh, D, False, True), ("fc2", D, Fh, True, False)):
            a = torch.randn(M, K, device=dev).to(BF16)
            wt = torch.randn(N, K, device=dev) * 0.02
            bias = torch.zeros(N, device=dev)
            lin, wb = ops.I8Lin(wt, bias, dev), wt.to(BF16)
            aq, asc = ops.quant_rows(a)
            o = torch.zeros(M, N, device=dev, dtype=F32_ if res else BF16)
            rr = o if res else None
            r[name + "_bf16"] = graph_us(lambda: ops.gemm(a, wb, K, K, N, bias, gelu=gelu, res=rr, out=o, ws=ws))
            r[name + "_i8"] = graph_us(lambda: ops.gemm_i8(aq, asc, lin.wq, lin.ldw, K, N, lin.sw, bias, gelu=gelu,
                                                           res=rr, out=o, ws=ws))
        out[M] = r
    return out


def main(argv=None):
    """python -m strix_halo_maxx_b200.text [--int8] [--bf16] [--kv8 [--keep N] [--questions Q] [--beams F]] [--reps N] [--eager] [--layers L] [--ops]: the decoder on
    device-random weights (weights.text_weights_device); prints the mean prefill / question ms of each
    selected variant (both by default).  With --reps 0 it runs one eager prefill and one question per variant
    and prints nothing else: the command to put under a profiler's launch list."""
    import argparse
    from .weights import text_weights_device
    ap = argparse.ArgumentParser()
    ap.add_argument("--int8", action="store_true")
    ap.add_argument("--bf16", action="store_true")
    ap.add_argument("--kv8", action="store_true", help="the KV cache in 8 bits")
    ap.add_argument("--keep", type=int, default=None, help="with --kv8: image-prefix tokens a head keeps for the questions")
    ap.add_argument("--questions", type=int, default=0, help="with --kv8: also so many questions at once")
    ap.add_argument("--beams", type=int, default=0, help="with --kv8: also a beam search of 16 words with so many beams")
    ap.add_argument("--reps", type=int, default=20)
    ap.add_argument("--eager", action="store_true", help="no CUDA-graph replay")
    ap.add_argument("--layers", type=int, default=None, help="fewer layers than the model's 24 (small profiles)")
    ap.add_argument("--ops", action="store_true", help="warm per-kernel times of one layer (op_times) instead")
    a = ap.parse_args(argv)
    if a.ops:
        for M, r in op_times(torch.device("cuda", torch.cuda.current_device())).items():
            print(M, r, flush=True)
        return
    variants = [v for v, on in (("bf16", a.bf16), ("int8", a.int8)) if on] or ["bf16", "int8"]
    dev = torch.device("cuda", torch.cuda.current_device())
    W = text_weights_device(TEXT, dev, seed=0, n_layers=a.layers)
    g = torch.Generator(device=dev).manual_seed(1)
    if a.beams:
        W["lm_w"], W["lm_b"] = torch.randn(51200, TEXT.dim, device=dev, generator=g) * 0.02, torch.zeros(51200, device=dev)
        W["wte"] = torch.randn(51200, TEXT.dim, device=dev, generator=g)
    emb = torch.randn(TEXT.prefix - 1, TEXT.dim, device=dev, generator=g)
    ids = torch.randint(1, TEXT.vocab, (TEXT.q_len,), device=dev, generator=g)
    for v in variants:
        dec = TextDecoder(W, TEXT, device=dev, graphs=not a.eager and a.reps > 0, int8=(v == "int8"), kv8=a.kv8,
                          keep=a.keep, questions=a.questions, beams=a.beams, steps=16 if a.beams else 0)
        res = {}
        runs = [("prefill_ms", lambda: dec.encode(emb, 0)), ("question_ms", lambda: dec.query(ids, TEXT.q_len - 1))]
        if a.questions:
            qs, ql = ids[None].repeat(a.questions, 1), torch.full((a.questions,), TEXT.q_len - 1, device=dev)
            runs.append((f"questions_{a.questions}_ms", lambda: dec.query_many(qs, ql)))
        if a.beams:
            runs.append((f"answer_{a.beams}x16_ms", lambda: dec.answer(ids, TEXT.q_len - 1)))
        for name, fn in runs:
            if a.reps <= 0:
                fn()
                continue
            for _ in range(3):
                fn()
            torch.cuda.synchronize()
            e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            e0.record()
            for _ in range(a.reps):
                fn()
            e1.record()
            torch.cuda.synchronize()
            res[name] = round(e0.elapsed_time(e1) / a.reps, 4)
        torch.cuda.synchronize()
        if res:
            print(v + ("_kv8" if a.kv8 else ""), res, flush=True)
        del dec


if __name__ == "__main__":
    main()
