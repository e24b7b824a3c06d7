"""Linear attention and group norm as users of this package have them done, as measurable cases.

  decode   linear_attention_recurrent, one token per sequence, on states in place or in a pool
  verify   linear_attention_recurrent over a few draft tokens per sequence, a state kept per token
  prefill  linear_attention_chunked on padded batches
  packed   linear_attention_chunked on packed sequences of unequal length
  norm     group_norm, one sample per token (a group per head, gated) or one per sequence or image
  block    a prompt through linear_attention_chunked and the gated group_norm that follows it

Head counts and dims are those of the package's benchmark and tests (16 key heads, 32 value heads, head dim 128, their shards,
head dim 64) or odd neighbours of them.  Inputs: q, k = silu(N(0, 1)), v ~ N(0, 1), states ~ N(0, 0.02).  Decays are one per head,
a geometric series of rates from 1/2 down to 1/256, or one per token and head, -exp(A_log) softplus(a + dt_bias).
"""
import math

import torch

own = False


def listed():
    return [
        # one user's next token: a single short launch is all there is
        dict(name="decode_b1", op="decode", B=1, kh=16, vh=32, dk=128, dv=128, state="f32", where="inplace", gate="head"),
        # a serving engine's running batch, one slot of the state pool per sequence, a decay per token
        dict(name="decode_pool_b24", op="decode", B=24, kh=16, vh=32, dk=128, dv=128, state="bf16", where="pool", gate="token"),
        # a full batch: 537 MB of fp32 states updated where they lie
        dict(name="decode_b256", op="decode", B=256, kh=32, vh=32, dk=128, dv=128, state="f32", where="inplace", gate="head"),
        # draft tokens scored with a state kept per token, so that the caller can roll back; an odd batch
        dict(name="verify_b13_t5", op="verify", B=13, T=5, kh=16, vh=32, dk=128, dv=128, state="bf16", gate="head"),
        # the smallest configuration: a short prompt, head dim 64, no state yet
        dict(name="prefill_b1_t256_d64", op="prefill", B=1, T=256, kh=4, vh=4, dk=64, dv=64, state=None, gate="head"),
        # the benchmark's padded prefill
        dict(name="prefill_b4_t4096", op="prefill", B=4, T=4096, kh=16, vh=32, dk=128, dv=128, state="f32", gate="head"),
        # a GPU's share of a long-context layer whose value heads are spread over eight: few, very long chains
        dict(name="prefill_b2_t131072_h4", op="prefill", B=2, T=131072, kh=2, vh=4, dk=128, dv=128, state="bf16", gate="head"),
        # the benchmark's packed batch: 16 prompts of log-normal lengths, a decay per token
        dict(name="packed_16x32768", op="packed", n=16, tokens=32768, kh=16, vh=32, dk=128, dv=128, state="f32", gate="token"),
        # the heads' outputs of a decode step: a handful of rows, latency is all there is
        dict(name="norm_tokens_24", op="norm", N=24, L=1, C=4096, G=32, dtype="bf16", gated=True),
        # the same of a prefill batch: 16384 tokens of 32 heads
        dict(name="norm_tokens_16384", op="norm", N=16384, L=1, C=4096, G=32, dtype="bf16", gated=True),
        # statistics over whole sequences, 20 channels a group, an odd length
        dict(name="norm_rows_n4_l4095", op="norm", N=4, L=4095, C=640, G=32, dtype="bf16", gated=False),
        # one slice of a long prompt: attention continuing from the state of the slice before, then the gated norm
        dict(name="block_b1_t7919", op="block", B=1, T=7919, kh=16, vh=32, dk=128, dv=128, state="f32", gate="token"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["decode", "decode", "verify", "prefill", "prefill", "long", "packed", "norm", "norm", "rows", "block"])
    kh, vh = rng.choice([(16, 32), (32, 32), (8, 16), (4, 8), (2, 4)])
    dk, dv = rng.choice([(128, 128), (128, 128), (64, 64), (64, 128), (96, 80)])
    heads = dict(kh=kh, vh=vh, dk=dk, dv=dv, gate=rng.choice(["head", "token"]))
    state = rng.choice(["f32", "bf16"])
    if op == "decode":
        return dict(op="decode", B=_log(rng, 1, 256), state=state, where=rng.choice(["inplace", "pool", "new"]), **heads)
    if op == "verify":
        return dict(op="verify", B=_log(rng, 1, 32), T=rng.randint(2, 8), state=state, **heads)
    if op in ("prefill", "block"):
        B = _log(rng, 1, 8)
        return dict(op=op, B=B, T=_log(rng, 33, 16384 // B), state=rng.choice(["f32", "bf16", None]), **heads)
    if op == "long":
        return dict(op="prefill", B=rng.choice([1, 2]), T=_log(rng, 8192, 100000), state=state, **dict(heads, kh=2, vh=4))
    if op == "packed":
        n = _log(rng, 2, 48)
        return dict(op="packed", n=n, tokens=_log(rng, 64 * n, 32768), state=state, **heads)
    dtype, gated = rng.choice(["bf16", "bf16", "f32"]), rng.random() < 0.6
    if op == "norm":
        width = rng.choice([64, 128, 128, 80, 256])
        G = rng.choice([4, 8, 16, 32])
        return dict(op="norm", N=_log(rng, 1, 16384), L=1, C=G * width, G=G, dtype=dtype, gated=gated)
    G = rng.choice([8, 16, 32])
    return dict(op="norm", N=_log(rng, 1, 16), L=_log(rng, 16, 8192), C=G * rng.choice([4, 8, 10, 16, 20, 40]), G=G, dtype=dtype, gated=gated)


def _lengths(n, total, seed):
    """`n` lengths of at least one token that sum to `total`, log-normally distributed."""
    gen = torch.Generator().manual_seed(seed)
    w = torch.exp(torch.randn(n, generator=gen, dtype=torch.float64))
    lens = [1 + int(x) for x in (w / w.sum() * (total - n)).floor()]
    lens[max(range(n), key=lambda i: lens[i])] += total - sum(lens)
    return lens


_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    s = dict(case)
    if case["op"] == "norm":
        t = _TYPES[case["dtype"]]
        shape = (case["N"], case["C"]) if case["L"] == 1 else (case["N"], case["L"], case["C"])
        # channels have their own offsets and spreads, as activations do
        s["x"] = (normal(*shape) * (0.5 + torch.rand(case["C"], generator=gen, device="cuda")) + 0.5 * normal(case["C"])).to(t)
        s["z"] = normal(*shape).to(t) if case["gated"] else None
        s["weight"], s["bias"] = 1 + 0.1 * normal(case["C"]), 0.1 * normal(case["C"])
        return s
    kh, vh, dk, dv = case["kh"], case["vh"], case["dk"], case["dv"]
    if case["op"] == "packed":
        lens = _lengths(case["n"], case["tokens"], seed)
        lead, seqs = (case["tokens"],), case["n"]
        s["cu_host"] = [sum(lens[:i]) for i in range(len(lens) + 1)]
        s["cu_seqlens"] = torch.tensor(s["cu_host"], dtype=torch.int32, device="cuda")
    else:
        lead, seqs = (case["B"], case.get("T", 1)), case["B"]
        s["cu_seqlens"] = None
    s["q"] = torch.nn.functional.silu(normal(*lead, kh, dk)).bfloat16()
    s["k"] = torch.nn.functional.silu(normal(*lead, kh, dk)).bfloat16()
    s["v"] = normal(*lead, vh, dv).bfloat16()
    if case["gate"] == "head":
        s["g"] = -torch.exp2(-1 - 7 * torch.arange(vh, device="cuda") / max(vh - 1, 1)).float()
    else:
        a_log = torch.log(torch.rand(vh, generator=gen, device="cuda") * 15 + 1) - 4
        s["g"] = -torch.exp(a_log) * torch.nn.functional.softplus(normal(*lead, vh) + 0.1 * normal(vh))
    s["state0"] = s["index"] = None
    if case["state"] is not None:
        slots = seqs + 8 if case.get("where") == "pool" else seqs
        s["state0"] = (normal(slots, vh, dv, dk) * 0.02).to(_TYPES[case["state"]])
        if case.get("where") == "pool":
            s["index"] = torch.randperm(slots, generator=gen, device="cuda")[:seqs].int()
    if case["op"] == "block":
        s["z"] = normal(*lead, vh, dv).bfloat16()
        s["weight"], s["bias"] = 1 + 0.1 * normal(vh * dv), 0.1 * normal(vh * dv)
    return s


# ------------------------------------------------------------------ the plain forms: fp32, rounded at the end
def _per_v_head(x, vh):
    return x.repeat_interleave(vh // x.shape[-2], dim=-2)


def _plain_chunks(q, k, v, g, state, scale, chunk=128):
    """q, k (B, T, kh, dk), v (B, T, vh, dv), g (vh) or (B, T, vh), state (B, vh, dv, dk) or None -> fp32 out, state."""
    B, T, vh, dv = v.shape
    S = torch.zeros(B, vh, dv, q.shape[-1], device=v.device) if state is None else state.float()
    out = torch.empty(B, T, vh, dv, device=v.device)
    for t in range(0, T, chunk):
        n = min(chunk, T - t)
        qc, kc = (_per_v_head(x[:, t:t + n].float(), vh).transpose(1, 2) for x in (q, k))
        vc = v[:, t:t + n].float().transpose(1, 2)
        gc = g.double().expand(B, n, vh) if g.dim() == 1 else g[:, t:t + n].double()
        G = gc.transpose(1, 2).cumsum(-1)
        later = torch.ones(n, n, dtype=torch.bool, device=v.device).triu(1)
        decay = torch.exp((G[..., :, None] - G[..., None, :]).masked_fill(later, -math.inf)).float()
        o = ((qc @ kc.transpose(-1, -2)) * decay) @ vc + torch.exp(G).float()[..., None] * (qc @ S.transpose(-1, -2))
        out[:, t:t + n] = (scale * o).transpose(1, 2)
        left = torch.exp(G[..., -1:] - G).float()[..., None]
        S = torch.exp(G[..., -1]).float()[..., None, None] * S + (vc * left).transpose(-1, -2) @ kc
    return out, S


def _plain_chunked(s):
    scale = s["dk"] ** -0.5
    t = _TYPES[s["state"]] if s["state"] else torch.bfloat16
    if s["cu_seqlens"] is None:
        out, S = _plain_chunks(s["q"], s["k"], s["v"], s["g"], s["state0"], scale)
        return out.bfloat16(), S.to(t)
    outs, states = [], []
    for i, (a, b) in enumerate(zip(s["cu_host"], s["cu_host"][1:])):
        g = s["g"] if s["g"].dim() == 1 else s["g"][None, a:b]
        o, S = _plain_chunks(s["q"][None, a:b], s["k"][None, a:b], s["v"][None, a:b], g, s["state0"][i:i + 1], scale)
        outs.append(o[0])
        states.append(S[0])
    return torch.cat(outs).bfloat16(), torch.stack(states).to(t)


def _plain_recurrent(s):
    q, k, v, g = s["q"].float(), s["k"].float(), s["v"].float(), s["g"].float()
    B, T, vh, _ = v.shape
    q, k = _per_v_head(q, vh), _per_v_head(k, vh)
    pool, index = s["state0"], s["index"]
    S = (pool if index is None else pool[index.long()]).float()
    outs, steps = [], []
    for t in range(T):
        gt = g if g.dim() == 1 else g[:, t]
        S = torch.exp(gt)[..., None, None] * S + v[:, t, :, :, None] * k[:, t, :, None, :]
        outs.append(s["dk"] ** -0.5 * (S * q[:, t, :, None, :]).sum(-1))
        steps.append(S)
    out = torch.stack(outs, 1).bfloat16()
    if s["op"] == "verify":
        return out, torch.stack(steps, 1).to(pool.dtype)
    if s["where"] == "new":
        return out, S.to(pool.dtype)
    if index is None:
        pool.copy_(S)
    else:
        pool[index.long()] = S.to(pool.dtype)
    return out, pool


def _plain_norm(x, G, weight, bias, z):
    N, C = x.shape[0], x.shape[-1]
    y = x.float().view(N, -1, G, C // G)
    centred = y - y.mean((1, 3), keepdim=True)
    y = centred * torch.rsqrt((centred * centred).mean((1, 3), keepdim=True) + 1e-5)
    y = y.reshape(x.shape) * weight + bias
    u = y if z is None else z.float()
    act = u / (1 + torch.exp(-u))
    return (act if z is None else y * act).to(x.dtype)


# ------------------------------------------------------------------ one pass
def run(state):
    s = state
    if own:
        import h100_gdn_cuda_b200 as gdn
        if s["op"] == "norm":
            return gdn.group_norm(s["x"], s["G"], s["weight"], s["bias"], s["z"])
        if s["op"] == "decode":
            return gdn.linear_attention_recurrent(s["q"], s["k"], s["v"], s["state0"], s["g"], inference_mode=gdn.Decode,
                                                  inplace_state=s["where"] == "inplace", state_indices=s["index"])
        if s["op"] == "verify":
            return gdn.linear_attention_recurrent(s["q"], s["k"], s["v"], s["state0"], s["g"], inference_mode=gdn.SpecVerify)
        out, final = gdn.linear_attention_chunked(s["q"], s["k"], s["v"], s["g"], None, s["state0"], s["cu_seqlens"])
        if s["op"] == "block":
            rows, C = s["B"] * s["T"], s["vh"] * s["dv"]
            return gdn.group_norm(out.view(rows, C), s["vh"], s["weight"], s["bias"], s["z"].view(rows, C)), final
        return out, final
    if s["op"] == "norm":
        return _plain_norm(s["x"], s["G"], s["weight"], s["bias"], s["z"])
    if s["op"] in ("decode", "verify"):
        return _plain_recurrent(s)
    if s["op"] == "block":
        t = _TYPES[s["state"]] if s["state"] else torch.bfloat16
        out, S = _plain_chunks(s["q"], s["k"], s["v"], s["g"], s["state0"], s["dk"] ** -0.5)
        rows, C = s["B"] * s["T"], s["vh"] * s["dv"]
        return _plain_norm(out.view(rows, C).bfloat16(), s["vh"], s["weight"], s["bias"], s["z"].view(rows, C)), S.to(t)
    return _plain_chunked(s)


# ------------------------------------------------------------------ the definition in 64 bits, token by token
def _exact_tokens(q, k, v, g, S, scale, steps=False):
    """One group of equally long sequences: the state is the sum of decayed products, walked in place."""
    vh = v.shape[-2]
    rep = vh // q.shape[-2]
    S = S.double().clone()
    out = torch.empty(v.shape, dtype=torch.float64, device=v.device)
    kept = torch.empty(*v.shape[:2], *S.shape[1:], dtype=torch.float64, device=v.device) if steps else None
    lam = torch.exp(g.double())
    for t in range(v.shape[1]):
        kt = k[:, t].double().repeat_interleave(rep, dim=1)
        qt = q[:, t].double().repeat_interleave(rep, dim=1)
        S.mul_((lam if lam.dim() == 1 else lam[:, t])[..., None, None])
        S.addcmul_(v[:, t].double()[..., None], kt[..., None, :])
        out[:, t] = torch.einsum("bhvk,bhk->bhv", S, qt) * scale
        if steps:
            kept[:, t] = S
    return out, S, kept


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(s["x"].double(), s)
    q, k, v, g, S0 = s["q"], s["k"], s["v"], s["g"], s["state0"]
    scale = 1 / math.sqrt(case["dk"])
    seqs = case["n"] if case["op"] == "packed" else case["B"]
    zero = torch.zeros(seqs, case["vh"], case["dv"], case["dk"], dtype=torch.float64, device=v.device)
    if case["op"] == "packed":
        out, final = torch.empty(v.shape, dtype=torch.float64, device=v.device), zero
        for i in range(seqs):
            a, b = s["cu_host"][i], s["cu_host"][i + 1]
            o, S, _ = _exact_tokens(q[None, a:b], k[None, a:b], v[None, a:b], g if g.dim() == 1 else g[None, a:b], S0[i:i + 1], scale)
            out[a:b], final[i] = o[0], S[0]
        return out, final
    if case["op"] == "verify":
        out, _, kept = _exact_tokens(q, k, v, g, S0, scale, steps=True)
        return out, kept
    if case["op"] == "decode":
        index = s["index"]
        out, S, _ = _exact_tokens(q, k, v, g, S0 if index is None else S0[index.long()], scale)
        if index is None:
            return out, S
        pool = S0.double()
        pool[index.long()] = S
        return out, pool
    out, final, _ = _exact_tokens(q, k, v, g, zero if S0 is None else S0, scale)
    if case["op"] == "block":
        rows, C = case["B"] * case["T"], case["vh"] * case["dv"]
        s["G"] = case["vh"]
        s["z"] = s["z"].view(rows, C)
        return _exact_norm(out.view(rows, C), s), final
    return out, final


def _exact_norm(x, s):
    G, C = s["G"], x.shape[-1]
    groups = x.reshape(x.shape[0], -1, G, C // G).transpose(1, 2).reshape(x.shape[0], G, -1)
    var, mean = torch.var_mean(groups, dim=-1, correction=0)
    per_channel = [t.repeat_interleave(C // G, dim=-1).reshape(x.shape[0], *[1] * (x.dim() - 2), C) for t in (mean, var)]
    y = (x - per_channel[0]) / torch.sqrt(per_channel[1] + 1e-5) * s["weight"].double() + s["bias"].double()
    if s["z"] is None:
        return y * torch.sigmoid(y)
    z = s["z"].double()
    return y * z * torch.sigmoid(z)


def work(case):
    if case["op"] == "norm":
        n, size = case["N"] * case["L"] * case["C"], 2 if case["dtype"] == "bf16" else 4
        return {"bytes": n * size * (3 if case["gated"] else 2) + 8 * case["C"], "flops": n * (14 if case["gated"] else 12)}
    kh, vh, dk, dv = case["kh"], case["vh"], case["dk"], case["dv"]
    seqs = case["n"] if case["op"] == "packed" else case["B"]
    tokens = case["tokens"] if case["op"] == "packed" else case["B"] * case.get("T", 1)
    size = 4 if case["state"] == "f32" else 2
    one = vh * dv * dk * size
    moved = tokens * (4 * kh * dk + 4 * vh * dv) + (4 * vh * tokens if case["gate"] == "token" else 4 * vh)
    moved += (seqs * one if case["state"] else 0) + (tokens if case["op"] == "verify" else seqs) * one
    flops = tokens * vh * 4 * dk * dv
    if case["op"] == "block":  # the norm reads the gate beside the heads' outputs, which need not leave the chip, and writes y
        moved += tokens * vh * dv * 2 + 8 * vh * dv
        flops += tokens * vh * dv * 14
    return {"bytes": moved, "flops": flops}
