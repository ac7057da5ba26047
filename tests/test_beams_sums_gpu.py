"""The sums of beam_select: what many unlikely words add to a likely one."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from strix_halo_maxx_b200 import ops

DEV, BF = "cuda", torch.bfloat16


def row(V, at, dt):
    """One word at 0 and V - 1 at x, 1,024 of which add up to a little less than 2^-24, half a step of fp32 behind 1 -> logits, exp(x)."""
    x = torch.tensor(np.log(0.98 * 2.0 ** -34)).to(dt)
    while 1024 * np.exp(float(x)) >= 2.0 ** -24:
        x = torch.nextafter(x, torch.tensor(-100.0, dtype=dt))
    z = torch.full((V,), float(x), dtype=dt, device=DEV)
    z[at] = 0
    return z, float(np.exp(float(x)))


def bound(V, c):
    """c = exp(x): fp32 may lose the other 63 words of the likely one's 64; exponentials (d = 24) and sums of 64 are within 25 2^-22 + 63 2^-24
    < 2^-16 of theirs; the total is rounded to fp32."""
    return 63 * c + (V - 1) * c * (2.0 ** -16 + 2.0 ** -24)


@pytest.mark.parametrize("dt", [torch.float32, BF])
@pytest.mark.parametrize("V,at", [(8192, 0), (8192, 4099), (8192, 8191), (3 * 8192 + 5, 8192 + 77), (100003, 60001), (1023, 500)])
def test_beam_select_unlikely_words_count(dt, V, at):
    z, c = row(V, at, dt)
    pitched = torch.zeros(2, V + 1, dtype=dt, device=DEV)[:, :V]  # rows that are read a word at a time
    pitched.copy_(z.expand(2, V))
    for x in (z[None], pitched):
        got = ops.beam_select(x, torch.zeros(len(x), device=DEV), 1)
        for s in range(len(x)):
            assert got.tokens[s].item() == at
            assert abs(got.scores[s].item() + np.log1p((V - 1) * c)) <= bound(V, c), (s, got.scores[s].item(), np.log1p((V - 1) * c))


@pytest.mark.parametrize("dt", [torch.float32, BF])
def test_beam_select_order_of_beams_that_differ_by_them(dt):
    """One beam's likely word shares its row with unlikely ones, the other's is alone, with a score that lies between."""
    V = 8192
    z, c = row(V, 5, dt)
    alone = torch.full((V,), -float("inf"), dtype=dt, device=DEV)
    alone[9] = 0
    score = -0.5 * np.log1p((V - 1) * c)
    got = ops.beam_select(torch.stack([z, alone]), torch.tensor([0.0, score], dtype=torch.float32, device=DEV), 2)
    assert got.parents[0].tolist() == [1, 0] and got.tokens[0].tolist() == [9, 5]
