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


@pytest.mark.parametrize("copied", [False, True])
def test_ids_that_are_handed_out_are_counted_again(copied):
    """Whoever reads raw_sel may write it; the histogram made with the ids' copy would then
    not be theirs, and the sort would place routes by it."""
    ids = torch.zeros(4, 3, dtype=torch.int32)
    routing = api._Routing(ids.view(-1), 3, (8, torch.zeros(1)))
    sel = api.CVMMSel._deferred(ids, routing, False, None)
    if copied:
        sel = sel.clone()
    assert sel._raw_shape_tensor().shape == (4, 3) and routing.counted is not None
    assert sel.raw_sel.data_ptr() == ids.data_ptr()
    assert routing.counts(8) is None
