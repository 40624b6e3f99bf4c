"""Attention of an odd number of query heads on a KV head, of more columns than CTAs: columns that begin inside a share and go on in the next."""
import pytest
import torch

from test_gpu_paged import attend, ops  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu

TILE, MIN_TILES, WIDE_CTAS = 64, 2, {64: 3, 96: 2, 128: 2}


def cut_inside(lengths, D):
    """How many columns (of one KV head) begin inside a CTA's share and end behind it."""
    tiles = [-(-n // TILE) for n in lengths]
    grid = WIDE_CTAS[D] * torch.cuda.get_device_properties(0).multi_processor_count
    assert sum(n > 0 for n in tiles) > grid                   # (equal shares, not whole parts of columns)
    size, at, cut = max(MIN_TILES, -(-sum(tiles) // grid)), 0, 0
    for n in tiles:
        cut += n > 0 and at % size > 0 and at // size != (at + n - 1) // size
        at += n
    return cut


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("group", [9, 11, 13, 15])
def test_columns_cut_inside_shares(ops, group, D, dtype):  # noqa: F811
    requests = 480 if D == 64 else 330
    lengths = [(37 * b) % 331 for b in range(requests)]
    assert cut_inside(lengths, D) > 50
    attend(ops, lengths, group, 1, D, dtype, page=16, seed=group)


@pytest.mark.parametrize("group", [9, 15])
def test_a_workspace_of_even_groups(ops, group):  # noqa: F811
    """A workspace of one shape serves odd groups, even ones and long columns, one after the other."""
    lengths = [(37 * b) % 331 for b in range(330)]
    ws = ops.paged_attn_workspace(330, 16, 1, 128, "cuda")
    for heads in (group, 16, group - 1, group):
        attend(ops, lengths, heads, 1, 128, torch.float16, workspace=ws)
    attend(ops, [9000, 3], group, 1, 128, torch.bfloat16, workspace=ws)
