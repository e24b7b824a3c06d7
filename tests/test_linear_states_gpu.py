"""fp32 states of linear attention's prompts against 64 bits, heads that forget slowly, and chunks that forget all."""
import math

import pytest
import torch

import h100_gdn_cuda_b200 as gdn
from oracle import gdn_oracle as O

pytestmark = pytest.mark.gpu


def normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


@pytest.mark.parametrize("heads,bound", [(80, 2.0 ** -16), (4, 2.0 ** -15)], ids=["whole", "cut"])
def test_a_state_alone(heads, bound):
    """Values of zero: a state only decays, by e^{g T}, over 1024 chunks.  Chains that stay whole (more than half as many as SMs) and cut ones.

    The exponent, E = 28.4 in log2 at most, is off by the gate's conversion (two half steps, 2^-24 of it each) and by a chunk's sum (seven), 9 2^-24 E, and by half a
    step of 2^-18 each where the state takes an exponent of up to 60 and gives it back: 1.9e-5, of which ln 2 is 1.3e-5.  Two powers of two, 2^-22 each: below 2^-16.  Cut chains take
    a power of two, rounded, in each of up to 37 segments: 37 (2^-22 + 2^-24) = 1.1e-5 more, below 2^-15."""
    T, d = 65536, 64
    gen = torch.Generator(device="cuda").manual_seed(0)
    q, k = normal(gen, 1, T, 1, d).bfloat16(), normal(gen, 1, T, 1, d).bfloat16()
    v = torch.zeros(1, T, heads, d, dtype=torch.bfloat16, device="cuda")
    s0 = normal(gen, 1, heads, d, d)
    g = -torch.linspace(1e-4, 3e-4, heads, device="cuda")
    _, s = gdn.linear_attention_chunked(q, k, v, g, None, s0)
    ref = torch.exp(g.double() * T)[None, :, None, None] * s0.double()
    assert bool(((s.double() - ref).abs() <= bound * ref.abs()).all()), ((s.double() - ref).abs() / ref.abs()).amax((0, 2, 3))


@pytest.mark.parametrize("heads", [80, 4], ids=["whole", "cut"])
def test_slow_decays(heads):
    """The same with values, as a part of the state's norm.  Values enter in two parts, within 2^-16; decays as above, within 2^-16.  Sums on the tensor cores are
    cut off rather than rounded: a step of 2^-23 at most for each of the eight sums of 16 products that 64 tokens are, over the min(T, 1 / -g) tokens that a
    head remembers."""
    T, d = 16384, 64
    gen = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = normal(gen, 1, T, 1, d).bfloat16(), normal(gen, 1, T, 1, d).bfloat16(), normal(gen, 1, T, heads, d).bfloat16()
    s0 = normal(gen, 1, heads, d, d)
    g = -torch.logspace(-6, -1, heads, base=10.0, device="cuda")
    _, s = gdn.linear_attention_chunked(q, k, v, g, None, s0)
    ages = torch.arange(T - 1, -1, -1, dtype=torch.float64, device="cuda")
    for h in range(0, heads, max(1, heads // 10)):
        ref = (v[0, :, h].double() * torch.exp(g[h].double() * ages)[:, None]).T @ k[0, :, 0].double() + torch.exp(g[h].double() * T) * s0[0, h].double()
        memory = min(T, -1 / g[h].item())
        assert (s[0, h].double() - ref).norm() <= (2.0 ** -15 + memory / 8 * 2.0 ** -23) * ref.norm()


@pytest.mark.parametrize("gates", ["strong", "resets", "lowest"])
@pytest.mark.parametrize("shape", [(2, 327, 1, 3, 128, 128), (2, 1000, 2, 4, 64, 64), (1, 2000, 2, 4, 128, 64)], ids=str)
def test_decays_that_forget_all(shape, gates):
    """Chunks that forget by more than 2^-120, with decays as fused_gdn_gating makes them, with a token in three that resets, and with the type's lowest
    value in every other: what is left of a decay where it matters is a sum of few and small numbers, so that only the values' two parts count,
    2^-16, and 9 half steps of R 2^-R <= 0.53, R being the decay's log2: 2^-21.  As above a part of the norm, of each head."""
    B, T, kh, vh, dk, dv = shape
    gen = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = normal(gen, B, T, kh, dk).bfloat16(), normal(gen, B, T, kh, dk).bfloat16(), normal(gen, B, T, vh, dv).bfloat16()
    s0 = normal(gen, B, vh, dv, dk)
    if gates == "strong":
        g = -(1 + 15 * torch.rand(vh, generator=gen, device="cuda")) * torch.nn.functional.softplus(normal(gen, B, T, vh))
        g[..., 0] *= 0.3
    else:
        g = -0.02 * torch.rand(B, T, vh, generator=gen, device="cuda")
        if gates == "resets":
            g[:, 1:-40:3] = -math.inf
        else:
            g[:, 1:-20:2] = torch.finfo(torch.float32).min
    _, s = gdn.linear_attention_chunked(q, k, v, g, None, s0)
    _, ref = O.linear_attention_ref(q, k, v, g, dk ** -0.5, s0)
    err = (s.double() - ref).flatten(2).norm(dim=-1) / ref.flatten(2).norm(dim=-1)
    assert bool((err <= 2.0 ** -16 + 2.0 ** -21).all()), err


@pytest.mark.parametrize("gate", ["head", "token", "none"])
@pytest.mark.parametrize("shape", [(2, 1, 1, 1, 128, 128), (1, 65, 2, 4, 8, 16), (2, 257, 2, 2, 96, 200), (1, 130, 1, 2, 104, 40), (1, 1000, 1, 2, 128, 128), (1, 3000, 1, 1, 64, 64)], ids=str)
def test_every_value(shape, gate):
    """Value by value, against the same sum of absolute values R: two parts of the values and decays as above, each 2^-16 at most, the tensor cores' sums as above, fp32
    states at the end."""
    B, T, kh, vh, dk, dv = shape
    gen = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = normal(gen, B, T, kh, dk).bfloat16(), normal(gen, B, T, kh, dk).bfloat16(), normal(gen, B, T, vh, dv).bfloat16()
    s0 = normal(gen, B, vh, dv, dk)
    g = {"head": -0.3 * torch.rand(vh, generator=gen, device="cuda"), "token": -torch.nn.functional.softplus(normal(gen, B, T, vh)), "none": None}[gate]
    _, s = gdn.linear_attention_chunked(q, k, v, g, None, s0)
    _, ref = O.linear_attention_ref(q, k, v, g, 1.0, s0)
    _, size = O.linear_attention_ref(q.abs(), k.abs(), v.abs(), g, 1.0, s0.abs())
    err = (s.double() - ref).abs()
    tol = (2.0 ** -15 + T / 8 * 2.0 ** -23) * size + 2.0 ** -24 * ref.abs()
    assert bool((err <= tol).all()), (err / tol).max().item()
