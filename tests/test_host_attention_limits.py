"""What attention plans ask for at the limits of a launch, without a device."""
from __future__ import annotations

from hyle_amd import compute as hc

DT, D = hc.DataType, hc.TensorDesc.dense
CTX = hc.Context.planning_only()
BF16, I32 = DT.kBFloat16, DT.kInt32


def test_a_split_whose_blocks_no_grid_holds_is_not_planned():
    """256 threads to a block: 2^24 blocks are one too many."""
    def plan(sequences):
        return hc.prepare(CTX, hc.PagedAttention(), D(BF16, [sequences, 4, 8]), D(BF16, [64, 2, 4, 16, 8]), D(I32, [sequences, 64]), D(I32, [sequences]))
    fits, past = plan(2 ** 22 - 2 ** 14), plan(2 ** 22)
    assert fits.dispatch_count() == 2 and fits.workspace_requirement().size > 0
    assert past.dispatch_count() == 1 and past.workspace_requirement().size == 0
