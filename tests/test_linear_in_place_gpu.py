"""gdn_linear_chunked with final_state = initial_state: chains that stay whole, cut ones (whose last segment would write the state before the
first has read it) and wide heads, at the bits of a call with two states."""
import ctypes as C

import pytest
import torch

from h100_gdn_cuda_b200 import _cabi as cabi
from h100_gdn_cuda_b200 import api

pytestmark = pytest.mark.gpu


def run(p, cu, s_in, s_out):
    shape, q, k, v, g, state, _, _ = api._linear_inputs(p["q"], p["k"], p["v"], p["g"], s_in, cu, False, True)
    assert state.data_ptr() == s_in.data_ptr()
    lib, packed = cabi.load(), cu is not None
    out = torch.zeros_like(v)
    need = lib.gdn_linear_chunked_workspace_bytes(C.byref(shape))
    ws = torch.full((need + 256,), 255, dtype=torch.uint8, device="cuda")  # NaN wherever nothing was written
    a = cabi.LinearChunkedArgs(shape, *(api._linear_tokens(t, packed) for t in (q, k, v, out)), g, api._linear_state(s_in), api._linear_state(s_out), 0.1,
                               cabi.GDN_F32 if s_in.dtype == torch.float32 else cabi.GDN_BF16, ws.data_ptr(), need)
    cabi.check(lib.gdn_linear_chunked(C.byref(a), torch.cuda.current_stream().cuda_stream), "chunked")
    torch.cuda.synchronize()
    assert bool((ws[need:] == 255).all())
    return out, need


# B, T (packed: lengths), kh, vh, dk, dv, cut
SHAPES = [(1, 3000, 2, 4, 128, 128, True), (2, 4000, 1, 3, 64, 128, True), (5, 3330, 4, 32, 64, 64, True), (1, 2500, 1, 2, 128, 200, True),
          (3, 200, 2, 4, 128, 128, False), (1, 70, 1, 2, 200, 64, False), (4, [3000, 1, 0, 2000], 2, 4, 128, 64, True),
          (35, [2000] * 33 + [0, 1], 1, 1, 64, 64, True), (3, [130, 0, 5], 8, 32, 128, 128, False)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(str(sum(x)) if isinstance(x, list) else str(x) for x in s))
def test_in_place(shape, dtype):
    B, T, kh, vh, dk, dv, cut = shape
    gen = torch.Generator(device="cuda").manual_seed(0)
    packed = isinstance(T, list)
    lead = (sum(T),) if packed else (B, T)

    def normal(*s):
        return torch.randn(*s, generator=gen, device="cuda")
    p = dict(q=normal(*lead, kh, dk).bfloat16(), k=normal(*lead, kh, dk).bfloat16(), v=normal(*lead, vh, dv).bfloat16(),
             g=-0.05 * torch.rand(*lead, vh, generator=gen, device="cuda"))
    cu = torch.tensor([0] + torch.tensor(T).cumsum(0).tolist(), dtype=torch.int32, device="cuda") if packed else None
    s0 = normal(B, vh, dv, dk).to(dtype)
    apart, mine = torch.empty_like(s0), s0.clone()
    want, need = run(p, cu, s0, apart)
    assert (need > 0) == cut
    for _ in range(3):
        mine.copy_(s0)
        got, _ = run(p, cu, mine, mine)
        assert torch.equal(got, want) and torch.equal(mine, apart)

