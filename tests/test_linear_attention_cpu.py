"""What the library refuses of linear attention and group norm, before any CUDA call (no GPU needed)."""
import ctypes as C

import pytest

from h100_gdn_cuda_b200 import _cabi as cabi

P = 1 << 20  # stands for a device address; nothing is launched


@pytest.fixture(scope="module")
def lib():
    from h100_gdn_cuda_b200 import build
    build.build()
    return cabi.load()


def _shape(**kw):
    d = dict(batch=2, seq_len=10, total_tokens=20, num_k_heads=2, num_v_heads=4, head_dim_k=64, head_dim_v=64)
    d.update(kw)
    return cabi.Shape(**d)


def _tokens(shape, heads, dim, ptr=P):
    return cabi.TokenTensor(ptr, shape.seq_len * heads * dim, heads * dim, dim)


def _recurrent(shape=None, **kw):
    s = shape or _shape()
    d = dict(shape=s, q=_tokens(s, s.num_k_heads, s.head_dim_k), k=_tokens(s, s.num_k_heads, s.head_dim_k),
             v=_tokens(s, s.num_v_heads, s.head_dim_v), out=_tokens(s, s.num_v_heads, s.head_dim_v),
             gate=cabi.TokenScalar(P, cabi.GDN_F32, 0, 0, 1), state_in=cabi.State(P, 4 * 64 * 64, 64 * 64), state_out=cabi.State(2 * P, 4 * 64 * 64, 64 * 64), scale=1.0)
    d.update(kw)
    return cabi.LinearRecurrentArgs(**d)


def _chunked(shape=None, **kw):
    s = shape or _shape()
    d = dict(shape=s, q=_tokens(s, s.num_k_heads, s.head_dim_k), k=_tokens(s, s.num_k_heads, s.head_dim_k),
             v=_tokens(s, s.num_v_heads, s.head_dim_v), out=_tokens(s, s.num_v_heads, s.head_dim_v),
             gate=cabi.TokenScalar(P, cabi.GDN_F32, 0, 0, 1), scale=1.0)
    d.update(kw)
    return cabi.LinearChunkedArgs(**d)


BAD_SHAPES = [dict(batch=0), dict(seq_len=0), dict(num_v_heads=3), dict(num_k_heads=0), dict(head_dim_k=60), dict(head_dim_k=264), dict(head_dim_v=0),
              dict(head_dim_v=20), dict(head_dim_k=-8)]


@pytest.mark.parametrize("bad", BAD_SHAPES, ids=str)
def test_shapes(lib, bad):
    s = _shape(**bad)
    assert lib.gdn_linear_recurrent(C.byref(_recurrent(s)), None) == -1 and lib.gdn_last_error()
    assert lib.gdn_linear_chunked(C.byref(_chunked(s)), None) == -1


@pytest.mark.parametrize("name", ["q", "k", "v", "out"])
@pytest.mark.parametrize("what", ["null", "misaligned", "token", "head", "broadcast_batch", "broadcast_token", "broadcast_head"])
def test_token_tensors(lib, name, what):
    heads = 2 if name in "qk" else 4
    t = cabi.TokenTensor(P, 10 * heads * 64, heads * 64, 64)
    if what == "null":
        t.ptr = None
    elif what == "misaligned":
        t.ptr = P + 8
    elif what == "token":
        t.stride_token += 4
    elif what == "head":
        t.stride_head = 32
    else:
        setattr(t, "stride_" + what.split("_")[1], 0)
    assert lib.gdn_linear_recurrent(C.byref(_recurrent(**{name: t})), None) == -1
    assert lib.gdn_linear_chunked(C.byref(_chunked(**{name: t})), None) == -1


def test_states_and_options(lib):
    st = cabi.State
    for bad in (dict(state_in=st(P + 4, 16384, 4096)), dict(state_out=st(P, 16384, 4100)), dict(state_dtype=2), dict(gate=cabi.TokenScalar(P, 7, 0, 0, 1)),
                dict(store_step_state=1, state_out=st(None, 0, 0)), dict(store_step_state=1, state_in=st(P, 16384, 4096), state_out=st(P, 16384, 4096)),
                dict(state_indices=P, num_slots=4, store_step_state=1), dict(state_indices=P, num_slots=0), dict(state_indices=P, num_slots=4, state_in=st(None, 0, 0))):
        assert lib.gdn_linear_recurrent(C.byref(_recurrent(**bad)), None) == -1, bad
    assert lib.gdn_linear_recurrent(None, None) == -1 and lib.gdn_linear_chunked(None, None) == -1
    assert lib.gdn_linear_chunked(C.byref(_chunked(state_dtype=5)), None) == -1
    assert lib.gdn_linear_chunked(C.byref(_chunked(final_state=st(P + 2, 16384, 4096))), None) == -1


def test_group_norm(lib):
    def args(**kw):
        d = dict(x=P, y=P, samples=2, rows=5, channels=12, groups=3, x_stride_sample=60, x_stride_row=12, y_stride_sample=60, y_stride_row=12, eps=1e-5)
        d.update(kw)
        return cabi.GroupNormArgs(**d)
    for bad in (dict(groups=5), dict(groups=0), dict(channels=0), dict(samples=-1), dict(rows=-1), dict(dtype=2), dict(param_dtype=-1)):
        assert lib.gdn_group_norm(C.byref(args(**bad)), None) == -1, bad
    assert lib.gdn_group_norm(None, None) == -1
    # short groups need no workspace, long ones one entry per part and group
    assert lib.gdn_group_norm_workspace_bytes(16, 1, 4096, 32) == 0
    assert lib.gdn_group_norm_workspace_bytes(16, 4096, 4096, 32) > 0
    assert lib.gdn_group_norm_workspace_bytes(16, 4096, 4096, 33) == 0


@pytest.mark.parametrize("struct,name", [(cabi.GroupNormArgs, "GdnGroupNormArgs"), (cabi.LinearRecurrentArgs, "GdnLinearRecurrentArgs"),
                                         (cabi.LinearChunkedArgs, "GdnLinearChunkedArgs")])
def test_struct_sizes(struct, name, tmp_path):
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    (tmp_path / "s.c").write_text('#include <stdio.h>\n#include "gdn_b200.h"\nint main(void) { printf("%%zu", sizeof(%s)); return 0; }\n' % name)
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")], check=True)
    assert int(subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout) == C.sizeof(struct)
