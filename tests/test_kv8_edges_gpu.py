"""The 8-bit KV cache where its kernels take another way than at ordinary sizes: clusters, runs of tiles over many sequences,
row groups, extreme weights, scales and queries; against oracle/kv8_ref.py or sums in 64 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from strix_halo_maxx_b200 import ops
from strix_halo_maxx_b200._lib import device_status
from oracle import kv8_ref as R
from test_kv8_gpu import DEV, as_np, filled, i32, np_


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
