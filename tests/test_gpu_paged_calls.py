"""Calls of the paged-cache operators on the GPU that a server makes beside the plain ones: operands that share memory, batches
with rows of no request, prompts beside drafted requests."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_layout_refuses_a_table_over_its_inputs(fp8lin, gpu):
    """An output table that overlaps the input table elsewhere than at its beginning, or another input, raises; side by side rows
    of one buffer are taken."""
    ints = dict(dtype=torch.int32, device=gpu)
    lengths, counts, free = torch.tensor([3, 40], **ints), torch.tensor([1, 2], **ints), torch.arange(20, **ints)
    buf = torch.full((5, 8), -1, **ints)
    wide = torch.full((2, 16), -1, **ints)
    for table, out in ((buf[1:3], buf[2:4]), (buf[1:3], buf[:2]), (buf[1:3], free[:16].view(2, 8)), (wide[:, :8], wide[:, 4:12])):
        with pytest.raises(fp8lin.Fp8linError):
            fp8lin.paged_layout(lengths, counts, table, free, 3, 16, out=out)
    got = fp8lin.paged_layout(lengths, counts, wide[:, :8], free, 3, 16, out=wide[:, 8:])
    # one page for position 3, then entry 2 for positions 40 and 41
    assert got.block_table.tolist() == [[0] + [-1] * 7, [-1, -1, 1] + [-1] * 5] and got.slots.tolist() == [3, 24, 25]
    assert (wide[:, :8] == -1).all()
