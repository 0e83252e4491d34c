"""beam_select: beams whose scores differ by little, where terms of the sum of exponentials are small against it.

A term goes through 8 sums in a lane, 3 that put a lane's together and 6 over the lanes, and is off by 3 * 2^-24 itself: a log sum is off by less than 20 * 2^-24
= 1.2e-6 where, as here, nearly all of it comes from terms at the maximum (others are off by 2.3 * 2^-24 times their distance from it besides)."""

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V,W", [(8192, 64), (131072, 4), (128003, 26)])
@pytest.mark.parametrize("first", [0, 1])
def test_small_terms_count(gpu, V, W, first):
    """A row of ones and of 63 terms of 0.95 * 2^-24 beside each, none of which changes a sum that begins with the one, but which are 3.6e-6 of all together: with
    scores 1.8e-6 apart, that decides between it and a row of equal logits."""
    import torch
    from tensorpack_amd.sampling import beam_select
    small = np.float32(math.log(0.95 * 2.0 ** -24))
    row = np.full(V, small, np.float32)
    at = np.arange(V)
    row[(at % 4096 < 512) & (at % 8 == 0)] = 0.0
    sum64 = np.exp(row.astype(np.float64)).sum()
    assert abs(math.log(sum64) - math.log((row == 0).sum()) - 63 * 0.95 * 2.0 ** -24) < 2e-7
    logits = np.zeros((1, W, V), np.float32)
    logits[0, first] = row
    logits[0, 2:] = row[::-1]
    far = np.float32(math.log(sum64) - math.log(V) - 1.8e-6)         # the row lies 1.8e-6 below the equal ones
    assert abs(float(far) - (math.log(sum64) - math.log(V) - 1.8e-6)) < 3e-7
    scores = np.full((1, W), -np.inf, np.float32)
    scores[0, first], scores[0, 1 - first] = far, 0.0
    got = beam_select(torch.from_numpy(logits).to(gpu), torch.from_numpy(scores).to(gpu), n=1)
    assert got[2].item() == 1 - first and got[1].item() == 0
    assert abs(got[0].item() + math.log(V)) < 20 * 2.0 ** -24 + 2.0 ** -24 * math.log(V)
    scores[0, first] = far + np.float32(3.6e-6)                      # and now as much above
    got = beam_select(torch.from_numpy(logits).to(gpu), torch.from_numpy(scores).to(gpu), n=1)
    assert got[2].item() == first and got[1].item() == 0
