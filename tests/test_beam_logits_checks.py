"""Logits of other dimensions than the selection of beams takes are refused alike, with and without num."""

import pytest
import torch

from ojasx_amd import beam_select


@pytest.mark.parametrize("num", [None, 2])
@pytest.mark.parametrize("shape", [(), (10,), (3, 10), (2, 3, 4, 10)])
def test_refused(shape, num):
    with pytest.raises(RuntimeError):
        beam_select(torch.zeros(shape), torch.zeros(2, 3), num)
