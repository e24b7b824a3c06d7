"""Offsets of packed sequences that are out of order or out of range: what lies around the outputs, the states and the workspace stays as it was, and
the state of the first sequence, whose offsets are in order, is right.  (test_linear_offsets_cpu.py walks the same offsets without a GPU.)"""
import ctypes as C

import pytest
import torch

from h100_gdn_cuda_b200 import _cabi as cabi
from h100_gdn_cuda_b200 import api
from oracle import gdn_oracle as O

pytestmark = pytest.mark.gpu
GUARD = 4096


def guarded(n, dtype, fill):
    """A tensor of n entries with GUARD of them on both sides, and what checks those."""
    whole = torch.full((n + 2 * GUARD,), fill, dtype=dtype, device="cuda")
    return whole[GUARD:GUARD + n], lambda: bool((whole[:GUARD] == fill).all()) and bool((whole[GUARD + n:] == fill).all())


# offsets, tokens, whether chains are cut into segments
CASES = [([0, 90, 40, 1 << 30], 150, False), ([0, 70, 2000, 149], 150, False), ([0, 6000, 0, 6000, 0, 6000], 6000, False), ([0, 5000, -7, 2 ** 31 - 1], 6000, True),
         ([-2 ** 31, 100, 50, 6001], 6000, True), ([0, 20000, 0, 20000, 0, 20000], 20000, True)]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("cu,total,cut", CASES, ids=str)
def test_surroundings(cu, total, cut, in_place):
    kh, vh, d, seqs = 1, 2, 64, len(cu) - 1
    gen = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (torch.randn(total, h, d, generator=gen, device="cuda").bfloat16() for h in (kh, kh, vh))
    g = -0.1 * torch.rand(total, vh, generator=gen, device="cuda")
    s0 = torch.randn(seqs, vh, d, d, generator=gen, device="cuda")
    offsets = torch.tensor(cu, dtype=torch.int32, device="cuda")
    shape, *_ = api._linear_inputs(q, k, v, g, s0, offsets, False, False)
    lib, stream = cabi.load(), torch.cuda.current_stream().cuda_stream
    need = lib.gdn_linear_chunked_workspace_bytes(C.byref(shape))
    assert (need > 0) == cut
    out, out_ok = guarded(v.numel(), torch.bfloat16, 7.0)
    state, state_ok = guarded(s0.numel(), torch.float32, 7.0)
    first, first_ok = guarded(s0.numel(), torch.float32, 7.0)
    ws, ws_ok = guarded(need, torch.uint8, 7)
    out, state, first = out.view_as(v), state.view_as(s0), first.view_as(s0)
    first.copy_(s0)
    final = first if in_place else state
    gate = cabi.TokenScalar(g.data_ptr(), cabi.GDN_F32, 0, *g.stride())
    tensors = [api._linear_tokens(t, True) for t in (q, k, v, out)]
    n = min(max(cu[1], 0), total)
    ref, sref = O.linear_attention_ref(q[None, :n], k[None, :n], v[None, :n], g[None, :n], 1.0, s0[:1])
    chunked = cabi.LinearChunkedArgs(shape, *tensors, gate, api._linear_state(first), api._linear_state(final), 1.0, cabi.GDN_F32, ws.data_ptr() if need else None, need)
    cabi.check(lib.gdn_linear_chunked(C.byref(chunked), stream), "chunked")
    torch.cuda.synchronize()
    assert out_ok() and state_ok() and first_ok() and ws_ok()
    assert (final[0].double() - sref[0]).norm() <= 2.0 ** -15 * sref.norm()  # (the first sequence's slots are there whatever follows)
    first.copy_(s0)
    recurrent = cabi.LinearRecurrentArgs(shape, *tensors, gate, api._linear_state(first), api._linear_state(final), None, None, 0, 1.0, 0, cabi.GDN_F32)
    cabi.check(lib.gdn_linear_recurrent(C.byref(recurrent), stream), "recurrent")
    torch.cuda.synchronize()
    assert out_ok() and state_ok() and first_ok()
    assert (final[0].double() - sref[0]).norm() <= 2.0 ** -15 * sref.norm()
