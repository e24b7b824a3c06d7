"""group_norm over very many small groups, few of them a sample."""
import pytest
import torch
from test_group_norm_gpu import check, make
from test_group_norm_wide_gpu import plain, timed

import h100_gdn_cuda_b200 as gdn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape,G", [((3000, 159, 8), 2), ((2100, 40, 32), 1), ((700, 33, 4 * 20), 4), ((700, 31, 4 * 20), 4), ((2500, 600, 3), 1)], ids=str)
def test_shapes(shape, G):
    for dtype in (torch.bfloat16, torch.float32):
        x, z, w, b = make(shape, dtype)
        check(gdn.group_norm(x, G, w, b, z), x, G, w, b, z)
        check(gdn.group_norm(x, G, w, b), x, G, w, b)


@pytest.mark.parametrize("shape", [(16384, 256, 8), (5378, 851, 1)], ids=str)
def test_not_slower_than_elementary_operations(shape):
    x, _, w, b = make(shape, torch.bfloat16)
    assert timed(lambda: gdn.group_norm(x, 1, w, b)) < timed(lambda: plain(x, w, b))
