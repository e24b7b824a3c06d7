"""Linear attention's prompts with values, keys and gates that are not finite: nothing of a token reaches the tokens in front of it, another sequence,
another head, or (of a value) another column."""
import math

import pytest
import torch

import h100_gdn_cuda_b200 as gdn

pytestmark = pytest.mark.gpu


def inputs(B, T, kh, vh, dk, dv, strong, packed=False):
    gen = torch.Generator(device="cuda").manual_seed(0)

    def normal(*s):
        return torch.randn(*s, generator=gen, device="cuda")
    lead = (B * T,) if packed else (B, T)
    p = dict(q=normal(*lead, kh, dk).bfloat16(), k=normal(*lead, kh, dk).bfloat16(), v=normal(*lead, vh, dv).bfloat16(),
             gate=-torch.nn.functional.softplus(normal(*lead, vh)) * (8.0 if strong else 0.05), initial_state=normal(B, vh, dv, dk))
    if packed:
        p["cu_seqlens"] = torch.arange(B + 1, dtype=torch.int32, device="cuda") * T
    return p


def call(p):
    return gdn.linear_attention_chunked(p["q"], p["k"], p["v"], p["gate"], None, p["initial_state"], p.get("cu_seqlens"))


# whole and ragged chunks, both widths of a tile and columns past one, cut chains
SHAPES = [(2, 150, 1, 2, 128, 128), (2, 150, 2, 2, 64, 64), (1, 200, 1, 1, 64, 200), (2, 128, 1, 2, 128, 40), (1, 3000, 1, 2, 128, 128)]


@pytest.mark.parametrize("packed", [False, True], ids=["padded", "packed"])
@pytest.mark.parametrize("strong", [False, True], ids=["weak", "strong"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_values(shape, strong, packed):
    B, T, kh, vh, dk, dv = shape
    p = inputs(*shape, strong, packed)
    o, s = (t.view(B, -1, *t.shape[-2:]) for t in call(p))
    # (sequence, token, head, column): the first of a chunk and the last, the sequence's last, neighbours, one column twice
    spots = [(0, 0, 0, 0, math.nan), (0, 63, vh - 1, dv - 1, math.inf), (B - 1, T - 1, 0, 7, -math.inf), (B - 1, 70, vh - 1, 17, math.inf),
             (B - 1, 75, vh - 1, 17, math.nan), (B - 1, 71, vh - 1, 18, -math.inf), (0, 64, 0, dv // 2, math.nan), (0, 127, 0, 33, math.inf)]
    bad = dict(p, v=p["v"].clone())
    first, v = torch.full((B, vh, dv), T, device="cuda"), bad["v"].view(B, T, vh, dv)
    for b, t, h, c, x in spots:
        v[b, t, h, c] = x
        first[b, h, c] = min(int(first[b, h, c]), t)
    o2, s2 = (t.view(B, -1, *t.shape[-2:]) for t in call(bad))
    reached = torch.arange(T, device="cuda")[None, :, None, None] >= first[:, None]
    assert torch.equal(torch.where(reached, 0, o2), torch.where(reached, 0, o))
    assert not bool(torch.isfinite(o2[reached]).any())
    rows = (first < T)[..., None].expand_as(s)
    assert torch.equal(torch.where(rows, 0, s2), torch.where(rows, 0, s)) and not bool(torch.isfinite(s2[rows]).any())


def test_rows_of_padding():
    """A batch of prompts of unequal length, padded with NaN: what belongs to the prompts is as without it."""
    p = inputs(3, 200, 2, 4, 128, 128, False)
    o, _ = call(p)
    bad = {x: p[x].clone() for x in ("q", "k", "v", "gate")}
    for b, n in enumerate((1, 70, 191)):
        for t in bad.values():
            t[b, n:] = math.nan
    o2, _ = call(dict(p, **bad))
    for b, n in enumerate((1, 70, 191)):
        assert (o2[b, :n].double() - o[b, :n].double()).norm() <= 2.0 ** -7 * o[b, :n].double().norm()
        assert bool(torch.isnan(o2[b, n:]).all())


@pytest.mark.parametrize("strong", [False, True], ids=["weak", "strong"])
@pytest.mark.parametrize("name", ["q", "k", "gate"])
def test_other_inputs(name, strong):
    """A query reaches its own token, a key and a gate theirs and what follows."""
    B, T, t = 2, 150, 90
    p = inputs(B, T, 1, 2, 128, 64, strong)
    o, s = call(p)
    bad = dict(p, **{name: p[name].clone()})
    bad[name][0, t, 0] = math.nan
    o2, s2 = call(bad)
    assert torch.equal(o2[1], o[1]) and torch.equal(s2[1], s[1])
    if name == "q":
        assert torch.equal(s2, s) and not bool(torch.isfinite(o2[0, t]).any())
        o2[0, t] = o[0, t]
        assert torch.equal(o2, o)
    elif name == "k":
        assert torch.equal(o2[0, :t], o[0, :t]) and not bool(torch.isfinite(o2[0, t:]).any())
    else:  # (the chunk takes the other form of the decays: the same up to roundings of scores and queries, two half steps)
        assert (o2[0, :t, 0].double() - o[0, :t, 0].double()).norm() <= 2.0 ** -7 * o[0, :t, 0].double().norm()
        assert not bool(torch.isfinite(o2[0, t:, 0]).any()) and torch.equal(o2[0, :, 1], o[0, :, 1])
