"""Dropout's generator against the values published with it: Philox 4x32-10 at counter 0 under
key 0 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011,
the known answers of its authors' library)."""

import pytest
import torch

import mamba_hip

pytestmark = pytest.mark.gpu
WORDS = [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_known_answer(dev, dtype):
    """An element is kept up to the threshold that is its word, and dropped above."""
    x, rng = torch.ones(2, 4, dtype=dtype, device=dev), torch.tensor([0, -3], device=dev)
    for e, w in enumerate(WORDS):
        for rows in (x, torch.ones(2, 5, dtype=dtype, device=dev)[:, :4]):  # one row of 8, and rows apart
            assert mamba_hip.dropout(rows, w / 2 ** 32, rng, 3)[0, e] != 0
            assert mamba_hip.dropout(rows, (w + 1) / 2 ** 32, rng, 3)[0, e] == 0
