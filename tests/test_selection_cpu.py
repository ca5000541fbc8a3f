"""What a recorded selection notes for later ones, without a GPU."""
import pytest
import torch

from cvmm_codex_amd import api


@pytest.mark.parametrize("n", [32768, 1 << 20, 0, -1])
def test_refused_counts_are_not_noted(n):
    """The next selection of the size would bring the count to a kernel that refuses it."""
    routing = api._Routing(torch.zeros(12345, dtype=torch.int32), 5)
    routing.counts(8)
    assert api._expert_guess[(12345, 5)] == 8
    routing.counts(n)
    assert api._expert_guess[(12345, 5)] == 8
    routing.counts(32767)
    assert api._expert_guess[(12345, 5)] == 32767
