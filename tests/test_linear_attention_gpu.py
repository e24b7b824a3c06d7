"""Linear attention with decay against the recurrence in 64 bits.

Bounds.  A half step of a type t is u(t) = eps / 2 relative (bf16 2^-8, fp32 2^-24).  With A = scale sum |S| |q|, the recurrence taken on
absolute values, and R the same for the state:
  token by token: sums of fp32 products; a value passes at most T decays (each off by a few u(fp32), exp included) and a sum of dk terms:
      |o - ref| <= u(bf16) |ref| + F A ,   |S - ref| <= u(state) |ref| + F R ,   F = (dk + 16 T + 32) u(fp32)
  in chunks the operands of the products are bf16: values with their decay and scores (intra part), the state and, where a chunk forgets
  much, the queries with their decay (inter part); of the state's increment the values:
      |o - ref| <= u(bf16) |ref| + (2 u(bf16) + u(bf16)^2 + F) A ,   |S - ref| <= u(state) |ref| + (u(bf16) + F) R
Every rounding there is independent of the others and v has random signs: the error's norm stays below 2 u(bf16) of the result's."""
import math

import pytest
import torch

import h100_gdn_cuda_b200 as gdn
from oracle import gdn_oracle as O

pytestmark = pytest.mark.gpu
U16, U32 = 2.0 ** -8, 2.0 ** -24


def make(B, T, kh, vh, dk, dv, gate="head", state=torch.float32, seed=0, packed=False):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")
    lead = (T,) if packed else (B, T)
    p = dict(q=normal(*lead, kh, dk).bfloat16(), k=normal(*lead, kh, dk).bfloat16(), v=normal(*lead, vh, dv).bfloat16())
    p["g"] = {"head": -torch.rand(vh, generator=gen, device="cuda") * 0.3, "none": None,
              "token": -torch.nn.functional.softplus(normal(*lead, vh)),
              "token16": -torch.nn.functional.softplus(normal(*lead, vh)).bfloat16()}[gate]
    p["s"] = None if state is None else normal(B, vh, dv, dk).to(state)
    return p


def check(o, s, p, chunked, steps=False, scale=None, tokens=None):
    """Padded results against the recurrence (`tokens`: of every sequence, the rest is not looked at)."""
    dk, T = p["q"].shape[-1], p["v"].shape[1]
    scale = dk ** -0.5 if scale is None else scale
    ref, sref = O.linear_attention_ref(p["q"], p["k"], p["v"], p["g"], scale, p["s"], steps)
    mag, smag = O.linear_attention_ref(p["q"].abs(), p["k"].abs(), p["v"].abs(), p["g"], abs(scale), None if p["s"] is None else p["s"].abs(), steps)
    F = (dk + 16 * T + 32) * U32
    us = U32 if s.dtype == torch.float32 else U16
    assert o.dtype == torch.bfloat16 and o.shape == ref.shape and s.shape == sref.shape
    tol = U16 * ref.abs() + ((2 * U16 + U16 ** 2 if chunked else 0) + F) * mag
    stol = us * sref.abs() + ((U16 if chunked else 0) + F) * smag
    err, serr = (o.double() - ref).abs(), (s.double() - sref).abs()
    assert bool((err <= tol).all()), (err / tol.clamp_min(1e-300)).max().item()
    assert bool((serr <= stol).all()), (serr / stol.clamp_min(1e-300)).max().item()
    if ref.numel() > 4096 and ref.norm() > 0:
        assert err.norm() <= 2 * U16 * ref.norm() and serr.norm() <= 2 * U16 * sref.norm()


SHAPES = [(1, 1, 1, 1, 128, 128), (3, 1, 2, 6, 64, 64), (2, 5, 1, 3, 128, 128), (1, 63, 2, 2, 64, 128), (2, 64, 1, 2, 128, 64),
          (1, 65, 2, 4, 8, 16), (1, 130, 1, 2, 100, 36), (2, 257, 2, 2, 96, 200), (1, 70, 1, 1, 200, 64), (1, 40, 1, 2, 256, 256),
          (1, 1000, 1, 2, 128, 128)]


@pytest.mark.parametrize("gate,state", [("head", torch.float32), ("token", torch.bfloat16), ("token16", None), ("none", torch.float32)])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_chunked(shape, gate, state):
    p = make(*shape, gate=gate, state=state)
    if gate == "none":  # without a decay the values of a chain only add up: keep them near one another
        p["g"] = None
    o, s = gdn.linear_attention_chunked(p["q"], p["k"], p["v"], p["g"], None, p["s"])
    assert s.dtype == (state or torch.bfloat16)
    check(o, s, p, True)


@pytest.mark.parametrize("gate,state", [("head", torch.float32), ("token", torch.bfloat16), ("token16", None), ("none", torch.float32)])
@pytest.mark.parametrize("shape", [s for s in SHAPES if s[1] <= 70], ids=str)
def test_recurrent(shape, gate, state):
    p = make(*shape, gate=gate, state=state)
    o, s = gdn.linear_attention_recurrent(p["q"], p["k"], p["v"], p["s"], p["g"], inference_mode=gdn.Decode)
    check(o, s, p, False)
    o2, s2 = gdn.linear_attention_recurrent(p["q"], p["k"], p["v"], p["s"], p["g"], inference_mode=gdn.SpecVerify)
    assert torch.equal(o, o2)
    check(o2, s2, p, False, steps=True)


@pytest.mark.parametrize("scale", [0.0, -0.7, 3.0])
def test_scale(scale):
    p = make(2, 100, 2, 4, 64, 64)
    check(*gdn.linear_attention_chunked(p["q"], p["k"], p["v"], p["g"], scale, p["s"]), p, True, scale=scale)
    check(*gdn.linear_attention_recurrent(p["q"], p["k"], p["v"], p["s"], p["g"], scale=scale), p, False, scale=scale)


@pytest.mark.parametrize("chunked", [True, False])
def test_resets_and_extreme_gates(chunked):
    """-inf, the type's lowest value and very fast decays forget exactly, wherever in a chunk they stand."""
    p = make(2, 200, 1, 3, 64, 64, gate="token")
    p["g"][:, ::7] = -math.inf
    p["g"][:, 3::11] = torch.finfo(torch.float32).min
    p["g"][:, 5::13] = -90.0
    p["g"][0, :, 1] = 0.0
    p["g"][1, :, 2] = -math.inf
    call = ((lambda: gdn.linear_attention_chunked(p["q"], p["k"], p["v"], p["g"], None, p["s"])) if chunked else
            (lambda: gdn.linear_attention_recurrent(p["q"], p["k"], p["v"], p["s"], p["g"])))
    o, s = call()
    assert bool(torch.isfinite(o).all()) and bool(torch.isfinite(s).all())
    check(o, s, p, chunked)


LENS = [[1], [64, 1, 0, 65], [0, 0, 3], [130, 5, 64, 63, 0, 200], [700] + [1] * 40]


@pytest.mark.parametrize("chunked", [True, False])
@pytest.mark.parametrize("lens", LENS, ids=str)
def test_packed(lens, chunked):
    """Sequences of a packed batch are on their own: neighbours hold NaN and infinities.  Rows behind the last one are left alone."""
    behind, total = 9, sum(lens)
    p = make(len(lens), total + behind, 2, 4, 128, 64, gate="token", packed=True)
    cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    for poisoned in range(2):
        q, k, v = p["q"].clone(), p["k"].clone(), p["v"].clone()
        for i, n in enumerate(lens):
            if i % 2 == poisoned:
                a = int(cu[i])
                q[a:a + n], k[a:a + n], v[a:a + n] = math.nan, math.inf, math.nan
        for t in (q, k, v):
            t[total:] = math.nan
        if chunked:
            o, s = gdn.linear_attention_chunked(q, k, v, p["g"], None, p["s"], cu)
        else:
            o, s = gdn.linear_attention_recurrent(q, k, v, p["s"], p["g"], cu)
        for i, n in enumerate(lens):
            if i % 2 == poisoned:
                continue
            a = int(cu[i])
            if n == 0:
                assert torch.equal(s[i], p["s"][i])
                continue
            one = {x: p[x][None, a:a + n] for x in "qkvg"}
            check(o[None, a:a + n], s[i:i + 1], dict(one, s=p["s"][i:i + 1]), chunked)


def test_rows_behind_the_last_sequence_and_bad_offsets():
    """Through the library itself, so that what is not written can be seen."""
    import ctypes as C
    from h100_gdn_cuda_b200 import _cabi as cabi, api
    p = make(3, 150, 1, 2, 64, 64, packed=True)
    for cu, good in (([0, 64, 64, 130], True), ([0, 90, 40, 1 << 30], False), ([-5, -1, 2000, 149], False)):
        cu = torch.tensor(cu, dtype=torch.int32, device="cuda")
        shape, q, k, v, g, s_in, _, _ = api._linear_inputs(p["q"], p["k"], p["v"], p["g"], p["s"], cu, False, False)
        out, final = torch.full_like(v, 7.0), torch.empty_like(s_in)
        lib = cabi.load()
        ws = torch.empty(lib.gdn_linear_chunked_workspace_bytes(C.byref(shape)) + 256, dtype=torch.uint8, device="cuda")
        a = cabi.LinearChunkedArgs(shape, *(api._linear_tokens(t, True) for t in (q, k, v, out)), g, api._linear_state(s_in),
                                   api._linear_state(final), 1.0, cabi.GDN_F32, ws.data_ptr(), ws.numel())
        cabi.check(lib.gdn_linear_chunked(C.byref(a), torch.cuda.current_stream().cuda_stream), "chunked")
        r = cabi.LinearRecurrentArgs(shape, *(api._linear_tokens(t, True) for t in (q, k, v, out)), g, api._linear_state(s_in),
                                     api._linear_state(final), None, None, 0, 1.0, 0, cabi.GDN_F32)
        torch.cuda.synchronize()
        if good:
            assert bool((out[130:] == 7.0).all())
        cabi.check(lib.gdn_linear_recurrent(C.byref(r), torch.cuda.current_stream().cuda_stream), "recurrent")
        torch.cuda.synchronize()
        if good:
            assert bool((out[130:] == 7.0).all())


@pytest.mark.parametrize("chunked", [True, False])
def test_views(chunked):
    """Slices of a fused projection, time-contiguous gates, broadcast heads and batches, unaligned and transposed states."""
    B, T, kh, vh, d = 2, 90, 2, 4, 64
    p = make(B, T, kh, vh, d, d, gate="token")
    fused = torch.cat([p["q"].flatten(2), p["k"].flatten(2), p["v"].flatten(2)], -1)
    q, k, v = (t.unflatten(-1, (-1, d)) for t in fused.split([kh * d, kh * d, vh * d], -1))
    g = p["g"].transpose(1, 2).contiguous().transpose(1, 2)

    def call(q, k, v, g, s):
        return gdn.linear_attention_chunked(q, k, v, g, None, s) if chunked else gdn.linear_attention_recurrent(q, k, v, s, g)
    base = call(p["q"], p["k"], p["v"], p["g"], p["s"])
    unaligned = torch.empty(p["s"].numel() + 1, device="cuda")[1:].view_as(p["s"]).copy_(p["s"])
    odd = torch.empty(v.numel() + 3, dtype=v.dtype, device="cuda")[3:].view(v.shape).copy_(v)
    for got in (call(q, k, v, g, p["s"]), call(q, k, v, g, p["s"].transpose(-1, -2).contiguous().transpose(-1, -2)), call(q, k, odd, g, unaligned)):
        assert all(torch.equal(a, b) for a, b in zip(base, got))
    wide = dict(p, q=p["q"][:1, :, :1].expand(B, T, kh, d), k=p["k"][:1, :, :1].expand(B, T, kh, d), v=p["v"][:, :1].expand(B, T, vh, d),
                g=p["g"][:1, :, :1].expand(B, T, vh), s=p["s"][:1, :1].expand(B, vh, d, d))
    check(*call(wide["q"], wide["k"], wide["v"], wide["g"], wide["s"]), wide, chunked)


@pytest.mark.parametrize("state", [torch.float32, torch.bfloat16])
def test_pool_and_in_place(state):
    B, T, kh, vh, d = 5, 3, 1, 2, 128
    p = make(B, T, kh, vh, d, d, state=state)
    ref = gdn.linear_attention_recurrent(p["q"], p["k"], p["v"], p["s"], p["g"])
    mine = p["s"].clone()
    o, s = gdn.linear_attention_recurrent(p["q"], p["k"], p["v"], mine, p["g"], inplace_state=True)
    assert s is mine and torch.equal(o, ref[0]) and torch.equal(mine, ref[1])
    pool = torch.randn(9, vh, d, d, device="cuda").to(state)
    slots = torch.tensor([4, -1, 0, 9, 8], dtype=torch.int32, device="cuda")  # -1 and 9 are not slots: left out
    keep = pool.clone()
    for i in (0, 2, 4):
        pool[slots[i].long()] = keep[slots[i].long()] = p["s"][i]
    o, s = gdn.linear_attention_recurrent(p["q"], p["k"], p["v"], pool, p["g"], state_indices=slots)
    assert s is pool
    for i in (0, 2, 4):
        assert torch.equal(o[i], ref[0][i]) and torch.equal(pool[slots[i].long()], ref[1][i])
        keep[slots[i].long()] = ref[1][i]
    assert torch.equal(pool, keep)


def test_accepted_tokens():
    p = make(5, 4, 2, 2, 64, 64)
    cap = torch.tensor([0, 1, 3, 4, 9], dtype=torch.int32, device="cuda")
    o, s = gdn.linear_attention_recurrent(p["q"], p["k"], p["v"], p["s"], p["g"], num_accepted_tokens=cap)
    for i, n in enumerate([0, 1, 3, 4, 4]):
        if n == 0:
            assert torch.equal(s[i], p["s"][i])
        else:
            one = {x: p[x][i:i + 1, :n] for x in "qkv"}
            check(o[i:i + 1, :n], s[i:i + 1], dict(one, g=p["g"], s=p["s"][i:i + 1]), False)


def test_offsets_beyond_32_bits():
    """Slots of a pool and tokens that lie more than 2^32 bytes (2^31 elements) from the start."""
    vh, d = 32, 128
    slots = 2 ** 31 // (vh * d * d) + 2
    pool = torch.empty(slots, vh, d, d, dtype=torch.bfloat16, device="cuda")
    p = make(2, 1, 16, vh, d, d, state=torch.bfloat16)
    idx = torch.tensor([slots - 1, 0], dtype=torch.int32, device="cuda")
    pool[slots - 1], pool[0] = p["s"][0], p["s"][1]
    o, s = gdn.linear_attention_recurrent(p["q"], p["k"], p["v"], pool, p["g"], state_indices=idx)
    check(o, torch.stack([pool[slots - 1], pool[0]]), p, False)
    del pool, s
    T, st = 70, 2 ** 25
    p = make(1, T, 1, 1, 64, 64)
    v = torch.empty(T * st, dtype=torch.bfloat16, device="cuda").as_strided((1, T, 1, 64), (T * st, st, 64, 1))
    v.copy_(p["v"])
    check(*gdn.linear_attention_chunked(p["q"], p["k"], v, p["g"], None, p["s"]), p, True)
    check(*gdn.linear_attention_recurrent(p["q"], p["k"], v, p["s"], p["g"]), p, False)


def test_nothing_to_do():
    p = make(2, 3, 1, 2, 64, 64)
    for B, T in ((0, 3), (2, 0)):
        q, k, v, s0 = p["q"][:B, :T], p["k"][:B, :T], p["v"][:B, :T], p["s"][:B]
        for o, s in (gdn.linear_attention_chunked(q, k, v, p["g"], None, s0), gdn.linear_attention_recurrent(q, k, v, s0, p["g"])):
            assert o.shape == v.shape and torch.equal(s, s0)
        o, s = gdn.linear_attention_chunked(q, k, v, p["g"])
        assert s.shape == s0.shape and not s.any()
    cu = torch.zeros(3, dtype=torch.int32, device="cuda")
    empty = [p[x][0, :0] for x in "qkv"]
    for o, s in (gdn.linear_attention_chunked(*empty, p["g"], None, p["s"], cu), gdn.linear_attention_recurrent(*empty, p["s"], p["g"], cu)):
        assert o.shape == (0, 2, 64) and torch.equal(s, p["s"])


def test_streams_and_graphs():
    """On a side stream; captured twice, the two graphs replayed one after the other and again on new inputs, at the bits of eager calls."""
    p = make(2, 700, 2, 4, 128, 128, gate="token")
    other = make(2, 700, 2, 4, 128, 128, gate="token", seed=1)
    names = "qkvg"

    def call(x):
        a = gdn.linear_attention_chunked(x["q"], x["k"], x["v"], x["g"], None, x["s"])
        b = gdn.linear_attention_recurrent(x["q"][:, :2], x["k"][:, :2], x["v"][:, :2], a[1], x["g"][:, :2])
        n = gdn.group_norm(a[0].view(2, 700, -1), 4)
        return [*a, *b, n]
    want, want_other = call(p), call(other)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(p)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    bufs = {x: p[x].clone() for x in (*names, "s")}
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(bufs))
        graphs.append(g)
    for src, ref in ((p, want), (other, want_other)):
        for x in bufs:
            bufs[x].copy_(src[x])
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(ref, o))


@pytest.mark.parametrize("front", ["ext", "ctypes", "module"])
def test_front_ends(front, monkeypatch):
    from h100_gdn_cuda_b200 import api, gdn_cuda
    f = gdn
    if front == "ctypes":
        monkeypatch.setattr(api, "_ext", False)
    if front == "module":
        f = gdn_cuda
    p = make(2, 70, 1, 2, 100, 36)
    check(*f.linear_attention_chunked(p["q"], p["k"], p["v"], p["g"], initial_state=p["s"]), p, True)
    check(*f.linear_attention_recurrent(p["q"], p["k"], p["v"], p["s"], p["g"]), p, False)
    r = make(3, 2, 1, 2, 64, 64)
    check(*f.linear_attention_recurrent(r["q"], r["k"], r["v"], r["s"].clone(), r["g"], inplace_state=True), r, False)
    idx = torch.arange(3, dtype=torch.int32, device="cuda")
    check(*f.linear_attention_recurrent(r["q"], r["k"], r["v"], r["s"].clone(), r["g"], state_indices=idx), r, False)
    check(*f.linear_attention_recurrent(r["q"], r["k"], r["v"], r["s"], r["g"], inference_mode=2), r, False, steps=True)
    x = torch.randn(4, 9, 24, device="cuda")
    assert (f.group_norm(x, 3).double() - O.group_norm_ref(x, 3)).abs().max() < 1e-5


def test_block_run():
    """A prompt in two slices, then single tokens, each with its gated norm: the whole run against the recurrence."""
    B, T, kh, vh, d = 2, 150, 2, 4, 128
    p = make(B, T, kh, vh, d, d, gate="token")
    z = torch.randn(B, T, vh * d, device="cuda").bfloat16()
    w, b = torch.rand(vh * d, device="cuda") + 0.5, torch.randn(vh * d, device="cuda")
    state, outs = p["s"], []
    for a, e in ((0, 100), (100, 147), (147, 148), (148, 149), (149, 150)):
        part = [p[x][:, a:e] for x in "qkv"]
        if e - a > 1:
            o, state = gdn.linear_attention_chunked(*part, p["g"][:, a:e], None, state)
        else:
            o, state = gdn.linear_attention_recurrent(*part, state, p["g"][:, a:e], inplace_state=True)
        rows = B * (e - a)
        outs.append(gdn.group_norm(o.reshape(rows, vh * d), vh, w, b, z[:, a:e].reshape(rows, vh * d)).view(B, e - a, -1))
    ref, sref = O.linear_attention_ref(p["q"], p["k"], p["v"], p["g"], d ** -0.5, p["s"])
    ref = O.group_norm_ref(ref.reshape(B * T, vh * d), vh, w, b, z.reshape(B * T, vh * d)).view(B, T, -1)
    # (the norm takes outputs that are off by up to 2 u(bf16) in norm and rounded to bf16, and rounds once more)
    err = torch.cat(outs, 1).double() - ref
    assert err.norm() <= 4 * U16 * ref.norm() and (state.double() - sref).norm() <= 2 * U16 * sref.norm()


def test_refusals():
    p = make(2, 4, 2, 4, 64, 64)
    q, k, v, g, s = p["q"], p["k"], p["v"], p["g"], p["s"]
    idx = torch.zeros(2, dtype=torch.int32, device="cuda")
    R, Cc = gdn.linear_attention_recurrent, gdn.linear_attention_chunked
    for bad in (lambda: R(q.float(), k, v, s, g), lambda: R(q.cpu(), k, v, s, g), lambda: R(q, k[:, :3], v, s, g), lambda: R(q, k, v[:1], s, g),
                lambda: R(q, k, v, s, g[:3]), lambda: R(q, k, v, s, g.double()), lambda: R(q, k, v, s, g.cpu()), lambda: R(q, k, v, s[:1], g),
                lambda: R(q, k, v, s.half(), g), lambda: R(q, k, v, s[..., :32], g), lambda: R(q, k, v[:, :, :3], s, g),
                lambda: R(q, k, v, None, g, inplace_state=True), lambda: R(q, k, v, None, g, state_indices=idx),
                lambda: R(q, k, v, s, g, state_indices=idx[:1]), lambda: R(q, k, v, s, g, state_indices=idx.long()),
                lambda: R(q, k, v, s, g, inference_mode=2, inplace_state=True), lambda: R(q, k, v, s, g, num_accepted_tokens=idx[:1]),
                lambda: R(q, k, v, s.transpose(-1, -2), g, inplace_state=True), lambda: R(q[0], k[0], v[0], s, g),
                lambda: R(q, k, v, s, g, cu_seqlens=idx), lambda: Cc(q, k, v, g, None, s[:1]), lambda: Cc(q, k, v, g, None, s, idx),
                lambda: Cc(q[0], k[0], v[0], g, None, s, idx.cpu()), lambda: Cc(q[0], k[0], v[0], g, None, s, idx.long()),
                lambda: Cc(*(torch.zeros(1, 2, 1, 264, dtype=torch.bfloat16, device="cuda"),) * 3)):
        with pytest.raises(RuntimeError):
            bad()


# cut into segments or not: one long chain, chains of a last round that is not full (160 on 148 SMs), chains of very different decay side by side,
# each tile shape
CUT = [((1, 4000, 1, 2, 128, 128), torch.bfloat16), ((5, 3330, 4, 32, 64, 64), torch.float32), ((1, 2500, 2, 4, 64, 128), None), ((2, 2049, 1, 3, 128, 40), torch.float32),
       ((1, 3000, 1, 1, 72, 256), torch.bfloat16)]


@pytest.mark.parametrize("shape,state", CUT, ids=str)
def test_cut_chains(shape, state):
    p = make(*shape, gate="token", state=state)
    p["g"] *= torch.exp2(4 - 12 * torch.rand(shape[3], generator=torch.Generator(device="cuda").manual_seed(1), device="cuda"))  # forgets in a token, or in hundreds
    check(*gdn.linear_attention_chunked(p["q"], p["k"], p["v"], p["g"], None, p["s"]), p, True)


@pytest.mark.parametrize("lens", [[3000, 1, 0, 2000], [0, 1200, 64, 1], [300] * 33 + [0, 1], [1] * 100], ids=lambda x: "%d of %d" % (len(x), sum(x)))
def test_packed_cut_chains(lens):
    total = sum(lens)
    p = make(len(lens), total, 1, 2, 64, 64, gate="token", state=torch.bfloat16, packed=True)
    p["g"] *= 0.02
    cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    o, s = gdn.linear_attention_chunked(p["q"], p["k"], p["v"], p["g"], None, p["s"], cu)
    for i, n in enumerate(lens):
        a = int(cu[i])
        if n == 0:
            assert torch.equal(s[i], p["s"][i])
        elif i in (0, 1, 2, 3, 34, len(lens) - 1):
            check(o[None, a:a + n], s[i:i + 1], dict({x: p[x][None, a:a + n] for x in "qkvg"}, s=p["s"][i:i + 1]), True)


def test_two_calls_at_once():
    """Two cut prompts on two streams at the same time, at the bits of one after the other."""
    ps = [make(1, 3000, 2, 4, 128, 128, gate="token", seed=i) for i in range(2)]
    want = [gdn.linear_attention_chunked(p["q"], p["k"], p["v"], p["g"], None, p["s"]) for p in ps]
    streams = [torch.cuda.Stream() for _ in ps]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for p, st in zip(ps, streams):
            with torch.cuda.stream(st):
                got.append(gdn.linear_attention_chunked(p["q"], p["k"], p["v"], p["g"], None, p["s"]))
        torch.cuda.synchronize()
        for (o, s), (o2, s2) in zip(got, want):
            assert torch.equal(o, o2) and torch.equal(s, s2)


@pytest.mark.parametrize("gate", ["head", "token", "none"])
@pytest.mark.parametrize("shape", [(2, 64, 1, 2, 128, 128), (2, 257, 2, 4, 64, 64), (1, 2000, 2, 4, 128, 128), (1, 900, 2, 2, 96, 200), (160, 200, 1, 1, 128, 64)], ids=str)
def test_fp32_states_of_prompts(shape, gate):
    """An fp32 state is more exact than bf16 values are: these go into it in two parts, 2^-16 off at most.  A decay is 2 to the difference of two sums
    of log2-decays below 64 each, of six roundings of half a step, 2^-19, with ln 2 in front: 2^-16 as well.  Products and sums are fp32; the
    errors of a sum's terms are independent, so the sum of both bounds, 2^-15, holds for the norm."""
    p = make(*shape, gate=gate)
    o, s = gdn.linear_attention_chunked(p["q"], p["k"], p["v"], p["g"], None, p["s"])
    ref, sref = O.linear_attention_ref(p["q"], p["k"], p["v"], p["g"], shape[4] ** -0.5, p["s"], False)
    assert s.dtype == torch.float32 and (s.double() - sref).norm() <= 2.0 ** -15 * sref.norm()
    check(o, s, p, True)


@pytest.mark.parametrize("gate", ["head", "token"])
def test_bf16_states_of_prompts(gate):
    """They are the fp32 ones (test_fp32_states_of_prompts), rounded once: half a step at most for every value, and 2^-15 of the norm beside that."""
    p = make(1, 2000, 2, 4, 128, 128, gate=gate, state=torch.bfloat16)
    o, s = gdn.linear_attention_chunked(p["q"], p["k"], p["v"], p["g"], None, p["s"])
    _, sref = O.linear_attention_ref(p["q"], p["k"], p["v"], p["g"], 128 ** -0.5, p["s"], False)
    excess = ((s.double() - sref).abs() - U16 * sref.abs()).clamp_min(0)
    assert s.dtype == torch.bfloat16 and excess.norm() <= 2.0 ** -15 * sref.norm()


@pytest.mark.parametrize("tokens", [70, 3000])
def test_no_states_through_the_library(tokens):
    """initial, final and new states may be NULL; a workspace that is too small or unaligned is refused."""
    import ctypes as C
    from h100_gdn_cuda_b200 import _cabi as cabi, api
    p = make(1, tokens, 1, 2, 64, 64, gate="token", state=None)
    shape, q, k, v, g, _, _, _ = api._linear_inputs(p["q"], p["k"], p["v"], p["g"], None, None, False, False)
    lib, st, none = cabi.load(), torch.cuda.current_stream().cuda_stream, cabi.State(None, 0, 0)
    need = lib.gdn_linear_chunked_workspace_bytes(C.byref(shape))
    ws = torch.empty(need + 256, dtype=torch.uint8, device="cuda")
    want = gdn.linear_attention_chunked(p["q"], p["k"], p["v"], p["g"])[0]
    for dtype in (cabi.GDN_F32, cabi.GDN_BF16):
        out = torch.full_like(v, 7.0)
        a = cabi.LinearChunkedArgs(shape, *(api._linear_tokens(t, False) for t in (q, k, v, out)), g, none, none, 64 ** -0.5, dtype, ws.data_ptr(), need)
        cabi.check(lib.gdn_linear_chunked(C.byref(a), st), "chunked")
        assert torch.equal(out, want)
        if need:
            for ptr, size in ((ws.data_ptr(), need - 1), (ws.data_ptr() + 16, need), (None, 0)):
                a.workspace, a.workspace_bytes = ptr, size
                assert lib.gdn_linear_chunked(C.byref(a), st) == -4
        if tokens < 100:
            r = cabi.LinearRecurrentArgs(shape, *(api._linear_tokens(t, False) for t in (q, k, v, out)), g, none, none, None, None, 0, 64 ** -0.5, 0, dtype)
            cabi.check(lib.gdn_linear_recurrent(C.byref(r), st), "recurrent")
            # (lanes hold other columns where states are fp32: sums in another order, so within the module's bound and not at the same bits)
            ref, _ = O.linear_attention_ref(p["q"], p["k"], p["v"], p["g"], 64 ** -0.5, None, False)
            mag, _ = O.linear_attention_ref(p["q"].abs(), p["k"].abs(), p["v"].abs(), p["g"], 64 ** -0.5, None, False)
            assert bool(((out.double() - ref).abs() <= U16 * ref.abs() + (64 + 16 * tokens + 32) * U32 * mag).all())
            if dtype == cabi.GDN_BF16:
                assert torch.equal(out, gdn.linear_attention_recurrent(p["q"], p["k"], p["v"], None, p["g"])[0])
    assert need > 0 or tokens < 100
