"""A recorded selection whose ids are written before its first use."""
import pytest
import torch

import cvmm_codex_amd as C

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,k,E", [(50, 2, 8), (700, 4, 32), (9000, 8, 64)])
def test_raw_ids_written_before_the_first_use(T, k, E):
    g = torch.Generator().manual_seed(0)
    ids = torch.randint(0, E, (T, k), generator=g).cuda()
    x = torch.randn(T, 64, generator=g).cuda().bfloat16()
    keys = torch.randn(E, 64, 32, generator=g).cuda().bfloat16()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        C.cvmm(x, C.cvmm_prepare_sel2(ids), keys)   # (the size and its expert count are known from here on)
        sel = C.cvmm_prepare_sel2(ids)
        sel.raw_sel.fill_(E - 1)
        sel.raw_sel[::2] = 3
        y = C.cvmm(x, sel, keys)
        other = ids.clone().fill_(E - 1)
        other[::2] = 3
        exp = C.cvmm(x, C.cvmm_prepare_sel2(other), keys)
    assert torch.equal(y, exp)
