"""group_norm against the formula in 64 bits.

Bound: with n values in a group, mean and variance are fp32 sums in trees or runs of at most a few thousand terms joined pairwise; a
group of very many values is off by less than (64 + sqrt(n)) u, u = 2^-24, of the mean of the values' sizes.  u = (x - m) r w + b then is off by at most
  E = (64 + sqrt(n)) u (|x| + mean|x|) r |w| + 16 u (|u| + |b|) ,  r = 1 / sqrt(var + eps)
SiLU has a slope of at most 1.1 and costs a few more roundings; a gate multiplies by |act(z)|; the result is rounded once (half a step)."""
import math

import pytest
import torch

import h100_gdn_cuda_b200 as gdn
from oracle import gdn_oracle as O

pytestmark = pytest.mark.gpu


def check(y, x, G, w=None, b=None, z=None, eps=1e-5, activation=True):
    assert y.shape == x.shape and y.dtype == x.dtype
    ref = O.group_norm_ref(x, G, w, b, z, eps, activation)
    lin = O.group_norm_ref(x, G, w, b, None, eps, False)
    N, C = x.shape[0], x.shape[-1]
    xs = x.double().reshape(N, -1, G, C // G)
    n = xs.shape[1] * xs.shape[3]
    size = (xs.abs() + xs.abs().mean((1, 3), keepdim=True)) / torch.sqrt(xs.var((1, 3), unbiased=False, keepdim=True) + eps)
    size = size.reshape(x.shape) * (1 if w is None else w.double().abs())
    u = 2.0 ** -24
    E = (64 + math.sqrt(n)) * u * size + 16 * u * (lin.abs() + (0 if b is None else b.double().abs()))
    if z is not None:
        gate = z.double() * torch.sigmoid(z.double()) if activation else z.double()
        E = E * gate.abs() + 16 * u * ref.abs()
    elif activation:
        E = 1.1 * E + 16 * u * lin.abs()
    tol = E + torch.finfo(x.dtype).eps / 2 * (ref.abs() + E) + 1e-30
    err = (y.double() - ref).abs()
    assert bool((err <= tol).all()), (err / tol).max().item()


def make(shape, dtype, offset=0.0, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    C = shape[-1]
    x = (torch.randn(*shape, generator=gen, device="cuda") + offset).to(dtype)
    z = torch.randn(*shape, generator=gen, device="cuda").to(dtype)
    return x, z, torch.randn(C, generator=gen, device="cuda"), torch.randn(C, generator=gen, device="cuda")


SHAPES = [((1, 8), 1), ((3, 4096), 32), ((5, 128), 128), ((7, 96), 3), ((2, 1040), 1), ((33, 2 * 1500), 2), ((300, 3 * 80), 3), ((2, 5, 12), 4),
          ((2, 7, 9), 3), ((1, 1000, 64), 8), ((4, 4095, 40), 2), ((2, 33, 17, 30), 3), ((1, 300, 4100), 1), ((3, 50, 5000), 1000), ((2, 2000, 6), 6), ((1, 1, 4, 1, 16), 2),
          ((1, 60000, 48), 2), ((2, 9001, 40), 1), ((1, 40000, 320), 5), ((2, 300, 700), 7), ((70, 40, 64), 2), ((1, 50001, 3), 1)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape,G", SHAPES, ids=str)
def test_shapes(shape, G, dtype):
    x, z, w, b = make(shape, dtype)
    check(gdn.group_norm(x, G, w, b, z), x, G, w, b, z)
    check(gdn.group_norm(x, G, w.bfloat16(), None), x, G, w.bfloat16())
    check(gdn.group_norm(x, G, None, b, activation=False), x, G, None, b, activation=False)
    check(gdn.group_norm(x, G, None, None, z, 1e-3, False), x, G, None, None, z, 1e-3, False)


@pytest.mark.parametrize("shape,G", [((64, 256), 2), ((2, 3000, 64), 4)], ids=str)
def test_large_mean(shape, G):
    """A mean 1000 times the spread costs no more digits than the values themselves have."""
    x, z, w, b = make(shape, torch.float32, 1000.0)
    check(gdn.group_norm(x, G, w, b, z), x, G, w, b, z)


@pytest.mark.parametrize("shape,G", [((6, 256), 2), ((2, 700, 64), 4)], ids=str)
def test_constant_groups_and_nan(shape, G):
    x, z, w, b = make(shape, torch.float32)
    x[0] = 3.0
    check(gdn.group_norm(x, G, w, b), x, G, w, b)
    x[1, ..., 0] = math.nan  # stays in its group
    y = gdn.group_norm(x, G, w, b)
    W = shape[-1] // G
    assert bool(torch.isnan(y[1, ..., :W]).all()) and bool(torch.isfinite(y[1, ..., W:]).all()) and bool(torch.isfinite(y[0]).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_views(dtype):
    x, z, w, b = make((4, 600, 48), dtype)
    wide = torch.cat([x, z], -1)
    for xv, zv in ((wide[..., :48], wide[..., 48:]), (x.transpose(0, 1).contiguous().transpose(0, 1), z), (x.transpose(1, 2).contiguous().transpose(1, 2), z),
                   (torch.cat([x.flatten()[:1], x.flatten()])[1:].view_as(x), z), (x, z[:, :1].expand_as(z)), (x[:1].expand_as(x), z)):
        check(gdn.group_norm(xv, 6, w, b, zv), xv, 6, w, b, zv)
    rows = torch.cat([x[0], z[0]], -1)[:, :48]
    check(gdn.group_norm(rows, 6, w, b), rows, 6, w, b)
    four = x.view(4, 20, 30, 48).transpose(1, 2)
    check(gdn.group_norm(four, 6, w, b), four, 6, w, b)


def test_same_bits_alone_and_in_a_batch():
    x, z, w, b = make((5, 1300, 64), torch.bfloat16)
    y = gdn.group_norm(x, 4, w, b, z)
    assert torch.equal(y, gdn.group_norm(x, 4, w, b, z))


def test_nothing_to_do():
    for shape in ((0, 16), (2, 0, 16), (0, 5, 16)):
        assert gdn.group_norm(torch.zeros(shape, device="cuda"), 4).shape == shape


def test_large():
    """More than 2^31 elements."""
    x = torch.empty(2 ** 19 + 3, 4096, dtype=torch.bfloat16, device="cuda")
    x.normal_(generator=torch.Generator(device="cuda").manual_seed(0))
    y = gdn.group_norm(x, 32)
    check(y[-50:], x[-50:], 32)
    check(y[:50], x[:50], 32)


def test_refusals():
    x, z, w, b = make((2, 5, 12), torch.float32)
    for bad in (lambda: gdn.group_norm(x, 5), lambda: gdn.group_norm(x, 0), lambda: gdn.group_norm(x, -3), lambda: gdn.group_norm(x.half(), 3),
                lambda: gdn.group_norm(x.cpu(), 3), lambda: gdn.group_norm(x[0, 0], 3), lambda: gdn.group_norm(x, 3, w[:6]),
                lambda: gdn.group_norm(x, 3, w, b.bfloat16()), lambda: gdn.group_norm(x, 3, w.double()), lambda: gdn.group_norm(x, 3, z=z[:1]),
                lambda: gdn.group_norm(x, 3, z=z.bfloat16()), lambda: gdn.group_norm(x, 3, w.cpu())):
        with pytest.raises(RuntimeError):
            bad()


# around the limits of the kernel that keeps a group in shared memory: 16 KB, 72 KB, 176 and 224 KB of a group, rows of whole sectors and not, more
# groups than SMs, very many small groups, a width that only pairs or single values divide
WHOLE = [((2, 1023, 64), 4), ((1, 2304, 32), 2), ((1, 2305, 32), 2), ((1, 7167, 32), 2), ((1, 7169, 32), 2), ((1, 4481, 60), 3), ((1, 3001, 60), 3),
         ((40, 500, 80), 4), ((40, 700, 80), 4), ((1100, 40, 32), 2), ((3, 900, 22), 2), ((3, 2000, 21), 3), ((1, 9, 9000), 1), ((2, 3, 4100), 2), ((1, 13, 8200), 1)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape,G", WHOLE, ids=str)
def test_groups_in_shared_memory(shape, G, dtype):
    x, z, w, b = make(shape, dtype, 3.0)
    check(gdn.group_norm(x, G, w, b, z), x, G, w, b, z)
    check(gdn.group_norm(x, G, w, b), x, G, w, b)
    check(gdn.group_norm(x, G, None, None, None, 1e-5, False), x, G, None, None, None, 1e-5, False)


@pytest.mark.parametrize("shape,G", [((70000, 200, 3), 1), ((70000, 40, 32), 2)], ids=str)
def test_more_samples_than_a_grid_has_rows(shape, G):
    x, z, w, b = make(shape, torch.bfloat16)
    y, gated = gdn.group_norm(x, G, w, b), gdn.group_norm(x, G, w, b, z)
    for at in (slice(0, 40), slice(65500, 65570), slice(69960, 70000)):
        check(y[at], x[at], G, w, b)
        check(gated[at], x[at], G, w, b, z[at])


@pytest.mark.parametrize("shape,G", [((3, 4, 64), 2), ((2, 300, 64), 4), ((2, 9000, 40), 2), ((1, 30, 4100), 1)], ids=str)
def test_in_place_through_the_library(shape, G):
    """y may be x or z itself."""
    import ctypes as C
    from h100_gdn_cuda_b200 import _cabi as cabi
    x, z, w, b = make(shape, torch.bfloat16)
    N, L, ch = shape
    lib = cabi.load()
    ws = torch.empty(lib.gdn_group_norm_workspace_bytes(N, L, ch, G) + 16, dtype=torch.uint8, device="cuda")
    for onto_z in (False, True):
        want = gdn.group_norm(x, G, w, b, z if onto_z else None)
        xc, zc = x.clone(), z.clone()
        a = cabi.GroupNormArgs()
        y = zc if onto_z else xc
        a.x, a.z, a.y, a.weight, a.bias = xc.data_ptr(), zc.data_ptr() if onto_z else None, y.data_ptr(), w.data_ptr(), b.data_ptr()
        a.samples, a.rows, a.channels, a.groups = N, L, ch, G
        for n in ("x", "z", "y"):
            setattr(a, n + "_stride_sample", L * ch)
            setattr(a, n + "_stride_row", ch)
        a.dtype, a.param_dtype, a.eps, a.silu = cabi.GDN_BF16, cabi.GDN_F32, 1e-5, 1
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        cabi.check(lib.gdn_group_norm(C.byref(a), torch.cuda.current_stream().cuda_stream), "group_norm")
        assert torch.equal(y, want)


def test_two_captured_graphs_and_another_stream():
    """Graphs that were captured from the same call, replayed on two streams at once and on new inputs."""
    shapes = [((2, 9000, 40), 2), ((4, 600, 64), 4)]
    data = [make(shape, torch.bfloat16) + (G,) for shape, G in shapes]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for x, z, w, b, G in data:
            gdn.group_norm(x, G, w, b, z)
    side.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append([gdn.group_norm(x, G, w, b, z) for x, z, w, b, G in data])
        graphs.append(g)
    for x, *_ in data:
        x.mul_(-1.5).add_(0.25)
    want = [gdn.group_norm(x, G, w, b, z) for x, z, w, b, G in data]
    torch.cuda.synchronize()
    for _ in range(3):
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))
