"""GPU tests of a head's losses and gradients where their rows' shares become many: 64 rows each, added up by one block from 2,048 on."""

import pytest
import torch

from test_hip_trunk_ends import check_gradients, check_loss, dtype, loss_case  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [64 * 2047, 64 * 2047 + 1, 64 * 2048, 64 * 2049 + 1, 64 * 4096 + 63, 64 * 4099])
@pytest.mark.parametrize("masked", [0.0, 0.5, 1.0])
def test_rows_are_packed_in_their_order(rows, masked, dtype):  # noqa: F811
    x, weight, targets, m = loss_case(dtype, rows, 11, 9, masked=masked, places=torch.int32 if rows % 2 else torch.int64)
    lse = check_loss(x, weight, targets)
    check_gradients(x, weight, targets, lse, m(rows, dtype=torch.float32), None)


def test_shares_of_which_most_have_no_target(dtype):  # noqa: F811
    """Targets in a few shares far from each other, the last row's among them."""
    rows = 64 * 5000 + 17
    x, weight, targets, m = loss_case(dtype, rows, 11, 9, masked=0.0)
    keep = torch.zeros(rows, dtype=torch.bool)
    keep[[0, 63, 64, 64 * 2048, 64 * 4095 + 5, rows - 1]] = True
    keep[100000:100300] = True
    targets[~keep.cuda()] = 11
    lse = check_loss(x, weight, targets)
    check_gradients(x, weight, targets, lse, m(rows, dtype=torch.float32), None)
