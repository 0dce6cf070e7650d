"""What F8 refuses of its sources before the library sees them, without a GPU."""
import numpy as np
import pytest
import torch

import ming_dit_amd as m


@pytest.mark.parametrize("codes,scales", [
    (np.zeros((32, 288), np.uint8)[:, ::2], np.zeros((1, 2), np.float32)),      # every other column
    (np.zeros((32, 160), np.uint8)[:, :144], np.zeros((1, 2), np.float32)),     # wider rows
    (np.zeros((144, 32), np.uint8).T, np.zeros((1, 2), np.float32)),
    (torch.zeros(32, 160, dtype=torch.uint8)[:, :144], torch.zeros(1, 2)),
    (torch.zeros(32, 144, dtype=torch.uint8), torch.zeros(1, 1).expand(1, 2)),
    (torch.zeros(2, 32, 144, dtype=torch.uint8), torch.zeros(2, 1).expand(2, 2)),
])
def test_sources_that_are_not_consecutive(codes, scales):
    with pytest.raises(ValueError, match="consecutive"):
        m.F8(None, codes, scales, 32)


@pytest.mark.parametrize("codes,scales", [
    (np.zeros((32, 144), np.uint8), np.zeros((1, 2), np.int32)),
    (torch.zeros(32, 144, dtype=torch.uint8), torch.zeros(1, 2, dtype=torch.int32)),
    (np.zeros((32, 144), np.uint8), np.zeros((1, 2), np.float64)),
    (np.zeros((32, 144), np.uint8), np.zeros((2, 2), np.float32)),
    (np.zeros((32, 144), np.uint16), np.zeros((1, 2), np.float32)),
    (np.zeros((2, 2, 32, 144), np.uint8), np.zeros((4, 2), np.float32)),
    (np.zeros((24, 144), np.uint8), np.zeros((1, 2), np.float32)),
])
def test_sources_of_another_kind(codes, scales):
    with pytest.raises(ValueError):
        m.F8(None, codes, scales, 32)
