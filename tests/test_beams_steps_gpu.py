"""Steps of a beam search, each call's outputs against the oracle on what the steps before have left."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from strix_halo_maxx_b200 import ops
from strix_halo_maxx_b200.config import TEXT
from strix_halo_maxx_b200.text import rope_tables
from oracle import beam_ref as R, kv8_ref
from test_beams_gpu import DEV, BF, _status, as_np, check_select, check_shared, filled, i32, np_


@pytest.mark.parametrize("S,F,Hq,H,D,plens,eos", [(2, 4, 4, 2, 64, [150, 64], 3), (1, 40, 8, 2, 128, [190], 7), (3, 5, 2, 2, 64, [0, 1, 130], -1), (2, 33, 2, 2, 64, [77, 128], 5)])
def test_write_attend_choose_and_reorder_step_by_step(S, F, Hq, H, D, plens, eos):
    V, steps, B, start = 2000, 4, S * F, 62  # own tokens pass a block's end
    cos, sin = rope_tables(TEXT.__class__(prefix=1024, q_len=0), DEV)
    prefix, c = filled((S,), H, 192, D, 1), ops.kv8_cache(B, H, 128, D, DEV)
    g = torch.Generator(DEV).manual_seed(5)
    table = torch.randn(V, (Hq + 2 * H) * D, device=DEV, generator=g).to(BF)
    head = torch.randn(Hq * D, V, device=DEV, generator=g) * 0.3
    q, out = torch.zeros(B, 1, Hq, D, dtype=BF, device=DEV), torch.zeros(B, 1, Hq * D, dtype=BF, device=DEV)
    tok, lens = torch.arange(B, device=DEV) % 11, torch.zeros(B, dtype=torch.int32, device=DEV)
    scores, done = torch.where(torch.arange(B, device=DEV) % F == 0, 0.0, -1e9), torch.zeros(B, dtype=torch.bool, device=DEV)
    held = [t.copy() for t in as_np(c)]  # the oracle's cache
    # what every sequence holds before the first step, of all beams their own
    first = torch.randn(B, start, (Hq + 2 * H) * D, device=DEV, generator=g).to(BF)
    qs = torch.zeros(B, start, Hq, D, dtype=BF, device=DEV)
    pos = np.repeat(plens, F)
    ops.rope_kv8(first, c, lens, cos, sin, qs, pos=i32(pos))
    kv8_ref.append(np_(first.float()), held, [0] * B, np_(cos), np_(sin), Hq, pos=pos)
    lens += start
    for i in range(steps):
        T = start + i
        qkv = table[tok][:, None].contiguous()
        ops.rope_kv8(qkv, c, lens, cos, sin, q, pos=i32(plens).repeat_interleave(F) + lens)
        want_q = kv8_ref.append(np_(qkv.float()), held, [T] * B, np_(cos), np_(sin), Hq, pos=pos + T)
        assert np.array_equal(np_(q.float()), kv8_ref.bf16(want_q)), i
        assert all(np.array_equal(a, b) for a, b in zip(as_np(c), held)), i
        ops.attn_kv8_shared(q, prefix, i32(plens), c, lens, out)
        check_shared(q, prefix, plens, ops.Kv8(*(torch.from_numpy(t) for t in held)), [T] * B, None, out)
        lens += 1
        logits = out.view(B, -1).float() @ head
        best = ops.beam_select(logits, scores, F, eos=eos, done=done if eos >= 0 else None)
        check_select(logits, scores, F, F, eos, done if eos >= 0 else None, best)
        new = torch.zeros_like(lens)
        ops.kv8_reorder(c, best.parents.view(-1), lens, beams=F, new_lens=new)
        after, to = R.reorder([t[None] for t in held], np_(best.parents).reshape(-1), [T + 1] * B, F)
        held = [t[0].copy() for t in after]
        assert all(np.array_equal(a, b) for a, b in zip(as_np(c), held)) and np_(new).tolist() == to.tolist() == [T + 1] * B, i
        tok, scores, done = best.tokens.view(-1).long().clamp(min=0), best.scores.view(-1).clone(), best.done.view(-1).clone()
    assert (best.parents.view(S, F) != torch.arange(B, device=DEV).view(S, F)).any()
