"""Workspaces of the adapters' products, without a GPU."""
import pytest

from cvmm_codex_amd import _native as N


@pytest.fixture(scope="module")
def lib():
    if not N.available():
        from cvmm_codex_amd import build
        build.build(verbose=False)
    return N.lib()


@pytest.mark.parametrize("rows", [40, 4000])
def test_room_for_the_copies_that_are_made(lib, rows):
    """Each operand's room by itself: a rank of 4 copies adapters, not the projection."""
    n, d_in, d_out, r = 2, 8192, 152064, 4
    size = lambda copied, weight=1: lib.cvmm_lora_workspace_bytes(rows, n, d_in, d_out, r, N.BF16, weight, copied)
    none = size(0)
    room = {N.LORA_COPY_X: rows * d_in * 2, N.LORA_COPY_WEIGHT: d_in * d_out * 2,
            N.LORA_COPY_A: n * d_in * 8 * 2, N.LORA_COPY_B: n * d_out * 8 * 2}
    for bit, values in room.items():
        assert values <= size(bit) - none <= values + 512
    pair = size(N.LORA_COPY_A | N.LORA_COPY_B)
    assert pair - none <= room[N.LORA_COPY_A] + room[N.LORA_COPY_B] + 1024
    assert size(N.LORA_COPY_ALL) >= none + sum(room.values())
    # without a projection there is nothing of it to copy
    assert size(N.LORA_COPY_WEIGHT, 0) == size(0, 0)
