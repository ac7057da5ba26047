"""Refusals of overlapping rows and empty batches by the 8-bit cache's entry points, before any CUDA call (no GPU)."""
import pytest

from strix_halo_maxx_b200 import build, _lib

Q = 1 << 20  # addresses that are never read


@pytest.fixture(scope="module")
def L():
    build.build()
    return _lib.lib()


# q [B][n][4][64] within or beside the rows of qkv, 8 x 64 = 512 elements (1024 bytes) of each token
OVER = [  # B, n, qkv strides, q's first byte after qkv's, q strides (b, t, h)
    (1, 1, (512, 512), 0, (256, 256, 64)), (2, 3, (1536, 512), 0, (1536, 512, 64)), (2, 3, (1536, 512), 1008, (1536, 512, 64)),
    (2, 3, (1536, 512), 512, (768, 256, 64)), (1, 4, (0, 512), -256 * 2 + 16, (0, 512, 64)), (3, 1, (512, 0), 1024, (512, 0, 64)), (1, 2, (0, 768), 1024 + 16, (0, 768, 64))]


@pytest.mark.parametrize("B,n,sx,at,sq", OVER)
def test_rope_kv8_refuses_q_over_qkv(L, B, n, sx, at, sq):
    rc = L.vt_rope_kv8(None, Q, *sx, B, n, 4, 2, 64, 4096, 4096, 64, 4096, None, None, Q + at, *sq, 4096, 4096, 4096, 4096, 64)
    assert rc == -2 and b"q overlaps qkv" in L.vt_last_error_string()


@pytest.mark.parametrize("n", [1, 5, 40])
def test_attn_kv8_refuses_out_over_q(L, n):
    for at, so in ((0, (512 * n, 512, 64)), (16, (256 * n, 256, 64)), (512 * n - 16, (256 * n, 256, 64))):
        rc = L.vt_attn_kv8(None, Q, 256 * n, 256, 64, 4096, 4096, 4096, 4096, 64, 4096, None, 2, n, 4, 2, 64, 1, 0.125, Q + at, *so,
                           None, None, 4096, 1 << 40)
        assert rc == -2 and b"out overlaps q" in L.vt_last_error_string(), (n, at)


def test_an_empty_batch_needs_no_pointers(L):
    no = [None] * 4
    assert L.vt_rope_kv8(None, None, 512, 512, 0, 1, 4, 2, 64, None, None, 8, None, None, None, None, 256, 256, 64, *no, 64) == 0
    assert L.vt_attn_kv8(None, None, 256, 256, 64, *no, 64, None, None, 0, 1, 4, 2, 64, 1, 0.125, None, 256, 256, 64, None, None, None, 0) == 0
    assert L.vt_kv8_evict(None, *no, 128, None, None, 0, 2, 64, 64, 8, *no, 64, None, None, None) == 0
