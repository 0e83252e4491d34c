"""Factors that fp32 cannot hold are refused as other bad arguments are, without a GPU."""

import math

import pytest
import torch

from tensorpack_amd import attention, rotary


@pytest.mark.parametrize("bad", [1e39, math.inf, math.nan, 2.0 ** 128])
def test_too_large(monkeypatch, bad):
    monkeypatch.setattr(rotary, "require_gpu", lambda device=None: torch.device("cpu"))
    with pytest.raises(ValueError):
        attention._scale(bad, 64)
    for amplitude in (bad, -bad):
        with pytest.raises(ValueError):
            rotary.Rotary(8, amplitude=amplitude)
    top = (2 - 2 ** -23) * 2.0 ** 127
    assert attention._scale(top, 64) == top and rotary.Rotary(8, amplitude=-top).amplitude == -top
    assert attention._scale(None, 64) == 0.125
