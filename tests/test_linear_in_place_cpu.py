"""States of linear attention updated in place: what is refused of it, and where the states of cut chains lie (no GPU needed)."""
import ctypes as C

import pytest

from h100_gdn_cuda_b200 import _cabi as cabi

P = 1 << 20  # stands for a device address; nothing is launched


def _tokens(shape, heads):
    return cabi.TokenTensor(P, shape.seq_len * heads * 64, heads * 64, 64)


@pytest.mark.parametrize("entry", ["gdn_linear_chunked", "gdn_linear_recurrent"])
@pytest.mark.parametrize("strides", [(4096, 2 * 4096), (4 * 4096, 8 * 4096)], ids=str)
def test_other_strides_are_refused(entry, strides):
    from h100_gdn_cuda_b200 import build
    build.build()
    lib = cabi.load()
    shape = cabi.Shape(batch=2, seq_len=10, total_tokens=20, num_k_heads=2, num_v_heads=4, head_dim_k=64, head_dim_v=64)
    states = cabi.State(P, 4 * 4096, 4096), cabi.State(P, *strides)
    names = ("initial_state", "final_state") if entry == "gdn_linear_chunked" else ("state_in", "state_out")
    make = cabi.LinearChunkedArgs if entry == "gdn_linear_chunked" else cabi.LinearRecurrentArgs
    a = make(shape=shape, q=_tokens(shape, 2), k=_tokens(shape, 2), v=_tokens(shape, 4), out=_tokens(shape, 4), scale=1.0, **dict(zip(names, states)))
    assert getattr(lib, entry)(C.byref(a), None) == -1 and b"same strides" in lib.gdn_last_error()


@pytest.mark.parametrize("lens,seg_chunks,per", [([3000, 1, 0, 2000], 4, 4), ([2000] * 33 + [0, 1], 8, 1), ([1], 3, 2), ([64 * 12, 64 * 12 + 1, 0, 0, 63], 3, 6)], ids=str)
def test_places_of_packed_segments(lens, seg_chunks, per):
    """As the kernels count them: every segment of a sequence has a place of its own below the count that the workspace is made for; the last one's,
    in which the first segment finds the initial state, among them."""
    items = (len(lens) + sum(lens) // (64 * seg_chunks)) * per
    seen, slot = set(), 0
    for n in lens:
        segments = max(1, -(-(-(-n // 64)) // seg_chunks))
        assert slot + segments <= items // per
        for s in range(segments):
            for rest in range(per):
                place = (slot + s) * per + rest
                assert place < items and place not in seen
                seen.add(place)
        slot += segments
