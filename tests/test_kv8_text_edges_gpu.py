"""The text decoder on the 8-bit cache before its first image."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from strix_halo_maxx_b200.config import TEXT
from strix_halo_maxx_b200 import weights as wg
from strix_halo_maxx_b200.text import TextDecoder


@pytest.mark.parametrize("graphs", [False, True])
def test_a_question_before_any_image_sees_an_empty_cache(monkeypatch, graphs):
    """As on the bf16 cache, whose slots start as zeros: no answer from what memory happened to hold."""
    W = wg.text_weights(TEXT, seed=3, n_layers=1, affine="random")
    _, _, ids, last = wg.text_inputs(TEXT, seed=5)
    ids = torch.from_numpy(ids).cuda()
    a = TextDecoder(W, TEXT, graphs=graphs, kv8=True)
    like = torch.empty_like
    monkeypatch.setattr(torch, "empty_like", lambda t, **kw: like(t, **kw).fill_(77))
    b = TextDecoder(W, TEXT, graphs=graphs, kv8=True)
    for t in a.tail_saved:
        t.zero_()
    for _ in range(2):
        assert torch.equal(a.query(ids, last), b.query(ids, last))
