"""group_norm over groups of more channels than a CTA sweeps at once, in pieces and not."""
import pytest
import torch
from test_group_norm_gpu import check, make

import h100_gdn_cuda_b200 as gdn

pytestmark = pytest.mark.gpu

# one group of many rows; several; widths whose pieces are alike and whose last one is shorter, a prime among them; more parts than are joined at
# once; few sweeps; as many groups as CTAs fit the SMs
SHAPES = [((1, 700, 4096), 1), ((2, 300, 2 * 2080), 2), ((3, 90, 6144), 1), ((1, 200, 1001), 1), ((1, 120, 4099), 1), ((2, 60, 2 * 5534), 2), ((1, 6000, 2050), 1),
          ((4, 2, 9000), 1), ((1, 1, 70000), 1), ((1300, 5, 2056), 1), ((1, 33, 20, 4104), 1)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape,G", SHAPES, ids=str)
def test_shapes(shape, G, dtype):
    x, z, w, b = make(shape, dtype, 3.0)
    check(gdn.group_norm(x, G, w, b, z), x, G, w, b, z)
    check(gdn.group_norm(x, G, w.bfloat16(), None), x, G, w.bfloat16())
    check(gdn.group_norm(x, G, None, b, None, 1e-3, False), x, G, None, b, None, 1e-3, False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_views(dtype):
    """Rows that start anywhere (single values are what is left of wide accesses) and rows of a wider tensor."""
    x, z, w, b = make((2, 100, 2 * 4224), dtype)
    for xv, zv in ((x[..., 1:4225], z[..., 2:4226]), (x[..., 8:4232], z[..., 4224:]), (x[:, ::3, :4224], z[:, :34, :4224])):
        check(gdn.group_norm(xv, 2, w[:4224], b[:4224], zv), xv, 2, w[:4224], b[:4224], zv)


def test_large_mean_and_nan():
    x, z, w, b = make((2, 200, 2 * 4096), torch.float32, 1000.0)
    check(gdn.group_norm(x, 2, w, b, z), x, 2, w, b, z)
    x[1, 7, 4096 + 3000] = float("nan")  # stays in its group
    y = gdn.group_norm(x, 2, w, b)
    assert bool(torch.isnan(y[1, :, 4096:]).all()) and bool(torch.isfinite(y[1, :, :4096]).all()) and bool(torch.isfinite(y[0]).all())


def plain(x, w, b):
    u = x.float()
    u = u - u.mean((1, 2), keepdim=True)
    u = u * torch.rsqrt((u * u).mean((1, 2), keepdim=True) + 1e-5) * w + b
    return (u / (1 + torch.exp(-u))).to(x.dtype)


def timed(f):
    f()
    times = []
    for _ in range(3):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        f()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b))
    return min(times)


@pytest.mark.parametrize("shape", [(1, 8192, 4096), (2, 3204, 2771)], ids=str)
def test_not_slower_than_elementary_operations(shape):
    """A group is spread over the GPU (a tenth of their time; on one CTA it was forty times as long)."""
    x, _, w, b = make(shape, torch.bfloat16)
    assert timed(lambda: gdn.group_norm(x, 1, w, b)) < timed(lambda: plain(x, w, b))
