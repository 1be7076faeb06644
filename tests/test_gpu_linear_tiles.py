"""linear_act in float32 where its products take 128 x 128 tiles, with the epilogue behind them. Bounds are
those of the operator's own tests."""

from __future__ import annotations

import pytest
import torch

import test_gpu_linear as linear

pytestmark = pytest.mark.gpu


# 64 x 32 tiles of 128 with partly filled ones at both edges: eight whole rounds of the device, where they pay from
# K = 745 on; loads of 16 bytes (K a multiple of 4) and of single words
@pytest.mark.parametrize("K", [900, 901])
@pytest.mark.parametrize("act", ["gelu", "none"])
def test_large_tiles(dev, K, act):
    args = linear._inputs(dev, 8190, 4090, K, torch.float32, seed=17)
    linear._check(*args, act, linear._call(*args, act))
