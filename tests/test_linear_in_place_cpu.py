"""final_state = initial_state of gdn_linear_chunked: what is refused of it, and where the states of cut chains lie (no GPU needed)."""
import ctypes as C

import pytest

from h100_gdn_cuda_b200 import _cabi as cabi

P = 1 << 20  # stands for a device address; nothing is launched


def test_other_strides_are_refused():
    from h100_gdn_cuda_b200 import build
    build.build()
    lib = cabi.load()
    shape = cabi.Shape(batch=2, seq_len=10, total_tokens=20, num_k_heads=2, num_v_heads=4, head_dim_k=64, head_dim_v=64)

    def tokens(heads):
        return cabi.TokenTensor(P, 10 * heads * 64, heads * 64, 64)
    a = cabi.LinearChunkedArgs(shape=shape, q=tokens(2), k=tokens(2), v=tokens(4), out=tokens(4), scale=1.0,
                               initial_state=cabi.State(P, 4 * 64 * 64, 64 * 64), final_state=cabi.State(P, 64 * 64, 2 * 64 * 64))
    assert lib.gdn_linear_chunked(C.byref(a), None) == -1 and b"same strides" in lib.gdn_last_error()


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
