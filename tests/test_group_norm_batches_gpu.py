"""group_norm of a sample alone and in a batch: the number of groups decides between the kernels, so the bits may differ; both are within the bound of
test_group_norm_gpu.py, and the same call repeats itself."""
import pytest
import torch
from test_group_norm_gpu import check, make

import h100_gdn_cuda_b200 as gdn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape,G", [((5, 1300, 64), 4), ((300, 40, 48), 4), ((1100, 33, 32), 4), ((7, 4096), 32), ((3, 2500, 640), 32), ((600, 9000), 2)], ids=str)
def test_alone_and_in_a_batch(shape, G, dtype):
    x, z, w, b = make(shape, dtype)
    y = gdn.group_norm(x, G, w, b, z)
    assert torch.equal(y, gdn.group_norm(x, G, w, b, z))
    for i in (0, shape[0] // 2, shape[0] - 1):
        one = slice(i, i + 1)
        check(gdn.group_norm(x[one], G, w, b, z[one]), x[one], G, w, b, z[one])
        check(y[one], x[one], G, w, b, z[one])
