"""CPU oracle for the Gated DeltaNet hot path.  TEST INFRASTRUCTURE ONLY.

This file restates, in plain fp32/fp64 torch on the CPU, the arithmetic that the
reference library (kingsleykimm/h100_gdn_cuda) computes on the GPU.  It is the
checker for the CUDA kernels and the timed CPU baseline of the benchmark; it
is never imported by the product package, which fails loudly when its CUDA
library is missing.

Parity pin: the reference stores no golden vectors (all of its tests draw
fresh random inputs and compare against an in-process formula or against the
third-party `flash-linear-attention` package, pinned at 0.4.1 in the
reference's uv.lock).  The oracle is therefore pinned against fixtures
generated by that package's pure-PyTorch naive recurrence (version 0.5.1 was
importable when the fixtures were made; see tests/golden/make_golden.py) and
against hand-derived known answers in tests/test_oracle.py.

Which reference lines each function follows:

* `recurrent_ref`         – canonical token recurrence as written in the
                            reference's own test oracle,
                            test/test_cpp/test_gdn_recurrent.cpp:165-217
                            (gate applied before S·k), qk-norm epsilon from
                            gdn_cuda/include/gdn_cuda/kernels/sm90_bf16_gdn_recurrent.cuh:299,350,
                            default scale from csrc/apis/gdn_forward.cpp:195,
                            accepted-token cut-off from sm90_bf16_gdn_recurrent.cuh:126-128.
* `gating_ref`            – gdn_cuda/include/gdn_cuda/kernels/gdn_helpers.cuh:76-90.
* `chunk_local_cumsum_ref`– gdn_helpers.cuh:142-256.
* `prepare_chunk_indices`, `prepare_cu_chunks`
                          – csrc/jit/utils/common.hpp:245-278 and
                            test/test_cpp/test_utils.h:81-105.
* `transpose_mn_major_ref`– csrc/apis/layout.hpp:13-57.
* `compute_u_w_ref`, `seq_state_update_ref`, `compute_o_ref`
                          – per-stage quantities of the chunked algorithm
                            (test/test_cpp/test_gdn_compute_u_w.cpp:138-167,
                            test_gdn_seq_state_passing.cpp:155-171,
                            test_gdn_fwd.cpp:258-281) with the canonical W
                            `(I+A)^-1 diag(beta*exp(g)) K`.

Layouts (same as the reference): q,k (B,T,kh,dk) or (N,kh,dk); v,o (B,T,vh,dv)
or (N,vh,dv); beta,g (B,T,vh) or (N,vh); state (B|S, vh, dv, dk).
"""
from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple

import torch

CHUNK = 64


# --------------------------------------------------------------------------
# varlen metadata
# --------------------------------------------------------------------------
def prepare_cu_chunks(cu_seqlens: Sequence[int], chunk: int = CHUNK) -> list:
    """Exclusive prefix sum of ceil(len/chunk) per sequence (S+1 entries)."""
    out = [0]
    for s in range(len(cu_seqlens) - 1):
        n = int(cu_seqlens[s + 1]) - int(cu_seqlens[s])
        out.append(out[-1] + (n + chunk - 1) // chunk)
    return out


def prepare_chunk_indices(cu_seqlens: Sequence[int], chunk: int = CHUNK) -> list:
    """Flat [seq_idx, chunk_idx_in_seq, ...] pairs, one per chunk."""
    out = []
    for s in range(len(cu_seqlens) - 1):
        n = int(cu_seqlens[s + 1]) - int(cu_seqlens[s])
        for c in range((n + chunk - 1) // chunk):
            out += [s, c]
    return out


# --------------------------------------------------------------------------
# helpers
# --------------------------------------------------------------------------
def gating_ref(A_log: torch.Tensor, dt_bias: torch.Tensor, a: torch.Tensor,
               b: torch.Tensor, threshold: float = 20.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """beta = sigmoid(b); g = -exp(A_log) * softplus(a + dt_bias), fp32 result."""
    A = A_log.float().reshape(-1)[: a.shape[-1]]
    x = a.float() + dt_bias.float()
    sp = torch.where(x <= threshold, torch.log1p(torch.exp(torch.clamp(x, max=threshold))), x)
    g = -torch.exp(A) * sp
    beta = torch.sigmoid(b.float())
    return beta, g


def _seq_bounds(B: int, T: int, cu_seqlens):
    if cu_seqlens is None:
        return [(b * T, (b + 1) * T) for b in range(B)]
    cu = [int(x) for x in cu_seqlens]
    return [(cu[i], cu[i + 1]) for i in range(len(cu) - 1)]


def chunk_local_cumsum_ref(g: torch.Tensor, cu_seqlens=None, chunk: int = CHUNK) -> torch.Tensor:
    """Inclusive prefix sum of g restarted every `chunk` tokens of each sequence.

    g is token-major: (B,T,H) or (N,H).  fp32 result of the same shape."""
    if cu_seqlens is None:
        B, T, H = g.shape
        flat = g.float().reshape(B * T, H)
    else:
        B, T = 0, 0
        flat = g.float()
    out = torch.zeros_like(flat)
    for (bos, eos) in _seq_bounds(B, T, cu_seqlens):
        for c0 in range(bos, eos, chunk):
            c1 = min(c0 + chunk, eos)
            out[c0:c1] = torch.cumsum(flat[c0:c1], dim=0)
    return out.reshape(g.shape)


def transpose_mn_major_ref(x: torch.Tensor, alignment: int = 16) -> torch.Tensor:
    """(..., mn, k) -> tensor of logical shape (..., mn_aligned, k) whose
    stride(-2) is 1 (storage (..., k, mn_aligned)); pad rows are zero."""
    mn, k = x.shape[-2], x.shape[-1]
    per = alignment // x.element_size()
    mn_al = (mn + per - 1) // per * per
    store = torch.zeros(*x.shape[:-2], k, mn_al, dtype=x.dtype)
    store[..., :mn] = x.transpose(-1, -2)
    return store.transpose(-1, -2)


def l2norm_ref(x: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    return x * torch.rsqrt((x * x).sum(-1, keepdim=True) + eps)


# --------------------------------------------------------------------------
# the recurrence (the layer semantics; parity target of every kernel)
# --------------------------------------------------------------------------
def recurrent_ref(q, k, v, beta, g, initial_state=None, scale: Optional[float] = None,
                  is_qk_norm: bool = False, cu_seqlens=None, num_accepted_tokens=None,
                  store_step_state: bool = False, dtype=torch.float32):
    """Token-by-token Gated DeltaNet.

        S <- exp(g_t) S ;  S <- S + beta_t (v_t - S k_t) k_t^T ;  o_t = scale * S q_t

    Inputs are taken as given (round them to bf16 first to model the API) and
    promoted to `dtype`.  Returns (o, state) where state is the final state
    (S, vh, dv, dk), or every per-token state (B,T,vh,dv,dk)/(N,vh,dv,dk) when
    `store_step_state`.  Tokens past `num_accepted_tokens[s]` are not
    processed: their outputs (and step states) stay zero.
    """
    varlen = cu_seqlens is not None
    if varlen:
        N, kh, dk = q.shape
        vh, dv = v.shape[-2:]
        B, T = len(cu_seqlens) - 1, 0
        qf, kf, vf = q.to(dtype), k.to(dtype), v.to(dtype)
        bf, gf = beta.to(dtype), g.to(dtype)
    else:
        B, T, kh, dk = q.shape
        vh, dv = v.shape[-2:]
        N = B * T
        qf, kf, vf = (x.to(dtype).reshape(N, *x.shape[2:]) for x in (q, k, v))
        bf, gf = beta.to(dtype).reshape(N, vh), g.to(dtype).reshape(N, vh)
    if scale is None:
        scale = 1.0 / math.sqrt(dk)
    if is_qk_norm:
        qf, kf = l2norm_ref(qf), l2norm_ref(kf)
    rep = vh // kh
    qf = qf.repeat_interleave(rep, dim=1)          # (N, vh, dk)
    kf = kf.repeat_interleave(rep, dim=1)
    bounds = _seq_bounds(B, T, cu_seqlens)
    nseq = len(bounds)
    S = torch.zeros(nseq, vh, dv, dk, dtype=dtype)
    if initial_state is not None:
        S = initial_state.to(dtype).clone()
    o = torch.zeros(N, vh, dv, dtype=dtype)
    steps = torch.zeros(N, vh, dv, dk, dtype=dtype) if store_step_state else None
    lens = [e - b for b, e in bounds]
    if num_accepted_tokens is not None:
        lens = [min(l, int(a)) for l, a in zip(lens, num_accepted_tokens)]
    starts = torch.tensor([b for b, _ in bounds])
    lens_t = torch.tensor(lens)
    for t in range(max(lens) if lens else 0):
        act = torch.nonzero(lens_t > t).flatten()
        idx = starts[act] + t
        Sa = S[act] * torch.exp(gf[idx])[..., None, None]
        kt, qt, vt = kf[idx], qf[idx], vf[idx]
        r = vt - torch.einsum("shvk,shk->shv", Sa, kt)
        Sa = Sa + (bf[idx][..., None] * r)[..., None] * kt[..., None, :]
        o[idx] = scale * torch.einsum("shvk,shk->shv", Sa, qt)
        S[act] = Sa
        if store_step_state:
            steps[idx] = Sa
    if not varlen:
        o = o.reshape(B, T, vh, dv)
        if store_step_state:
            steps = steps.reshape(B, T, vh, dv, dk)
    return o, (steps if store_step_state else S)


# --------------------------------------------------------------------------
# per-stage quantities of the chunked algorithm (for the low-level wrappers)
# --------------------------------------------------------------------------
def _chunks(B, T, cu_seqlens):
    """Yield (seq, chunk_idx_in_seq, tok0, tok1) for every 64-token chunk."""
    for s, (bos, eos) in enumerate(_seq_bounds(B, T, cu_seqlens)):
        for c, c0 in enumerate(range(bos, eos, CHUNK)):
            yield s, c, c0, min(c0 + CHUNK, eos)


def _flat(x, varlen):
    return x if varlen else x.reshape(-1, *x.shape[2:])


def compute_u_w_ref(k, v, beta, g_cum, cu_seqlens=None, dtype=torch.float32):
    """U = T V, W = T (K * exp(g_cum)), T = (I + tril(diag(beta) K K^T * Gamma, -1))^-1 diag(beta),
    Gamma_ij = exp(g_cum_i - g_cum_j).  g_cum is the chunk-local cumsum, token-major."""
    varlen = cu_seqlens is not None
    B, T = (0, 0) if varlen else k.shape[:2]
    kf, vf, bf, gf = (_flat(x.to(dtype), varlen) for x in (k, v, beta, g_cum))
    kh, vh = kf.shape[1], vf.shape[1]
    rep = vh // kh
    u = torch.zeros_like(vf)
    w = torch.zeros(vf.shape[0], vh, kf.shape[-1], dtype=dtype)
    for _, _, c0, c1 in _chunks(B, T, cu_seqlens):
        n = c1 - c0
        for h in range(vh):
            K = kf[c0:c1, h // rep]
            gc = gf[c0:c1, h]
            bt = bf[c0:c1, h]
            diff = gc[:, None] - gc[None, :]
            lower = torch.tril(torch.ones(n, n, dtype=torch.bool), -1)
            Gam = torch.where(lower, torch.exp(torch.where(lower, diff, torch.zeros_like(diff))),
                              torch.zeros_like(diff))
            A = (K @ K.T) * Gam * bt[:, None]
            Tm = torch.linalg.solve_triangular(torch.eye(n, dtype=dtype) + A,
                                               torch.diag(bt), upper=False)
            u[c0:c1, h] = Tm @ vf[c0:c1, h]
            w[c0:c1, h] = Tm @ (K * torch.exp(gc)[:, None])
    if not varlen:
        u = u.reshape(B, T, *u.shape[1:])
        w = w.reshape(B, T, *w.shape[1:])
    return u, w


def seq_state_update_ref(k, u, w, g_cum, initial_state=None, cu_seqlens=None,
                         dtype=torch.float32):
    """Chunk-to-chunk state pass.  Returns (h, u_new, final_state): h[c] is the
    state entering chunk c, laid out (B,nc,vh,dv,dk) or (total_chunks,vh,dv,dk)."""
    varlen = cu_seqlens is not None
    B, T = (0, 0) if varlen else k.shape[:2]
    kf, uf, wf, gf = (_flat(x.to(dtype), varlen) for x in (k, u, w, g_cum))
    kh, vh = kf.shape[1], uf.shape[1]
    dv, dk = uf.shape[-1], kf.shape[-1]
    rep = vh // kh
    bounds = _seq_bounds(B, T, cu_seqlens)
    S = torch.zeros(len(bounds), vh, dv, dk, dtype=dtype)
    if initial_state is not None:
        S = initial_state.to(dtype).clone()
    hs = []
    un = torch.zeros_like(uf)
    for s, _, c0, c1 in _chunks(B, T, cu_seqlens):
        hs.append(S[s].clone())
        for h in range(vh):
            K = kf[c0:c1, h // rep]
            gc = gf[c0:c1, h]
            Un = uf[c0:c1, h] - wf[c0:c1, h] @ S[s, h].T
            un[c0:c1, h] = Un
            gl = gc[-1]
            S[s, h] = S[s, h] * torch.exp(gl) + Un.T @ (K * torch.exp(gl - gc)[:, None])
    hcat = torch.stack(hs) if hs else torch.zeros(0, vh, dv, dk, dtype=dtype)
    if not varlen:
        nc = (T + CHUNK - 1) // CHUNK
        hcat = hcat.reshape(B, nc, vh, dv, dk)
        un = un.reshape(B, T, vh, dv)
    return hcat, un, S


def compute_o_ref(q, k, u_new, h, g_cum, scale=None, cu_seqlens=None, dtype=torch.float32):
    """O = scale * (exp(g_cum) * Q h^T + tril(Q K^T * Gamma) U_new) per chunk."""
    varlen = cu_seqlens is not None
    B, T = (0, 0) if varlen else q.shape[:2]
    qf, kf, uf, gf = (_flat(x.to(dtype), varlen) for x in (q, k, u_new, g_cum))
    hf = h.to(dtype)
    if not varlen:
        hf = hf.reshape(-1, *hf.shape[2:])
    kh, vh = kf.shape[1], uf.shape[1]
    rep = vh // kh
    if scale is None:
        scale = 1.0 / math.sqrt(qf.shape[-1])
    o = torch.zeros_like(uf)
    for ci, (_, _, c0, c1) in enumerate(_chunks(B, T, cu_seqlens)):
        n = c1 - c0
        for hd in range(vh):
            Q, K = qf[c0:c1, hd // rep], kf[c0:c1, hd // rep]
            gc = gf[c0:c1, hd]
            diff = gc[:, None] - gc[None, :]
            low = torch.tril(torch.ones(n, n, dtype=torch.bool))
            Gam = torch.where(low, torch.exp(torch.where(low, diff, torch.zeros_like(diff))),
                              torch.zeros_like(diff))
            P = (Q @ K.T) * Gam
            o[c0:c1, hd] = scale * (torch.exp(gc)[:, None] * (Q @ hf[ci, hd].T) + P @ uf[c0:c1, hd])
    if not varlen:
        o = o.reshape(B, T, *o.shape[1:])
    return o


def chunked_ref(q, k, v, beta, g, initial_state=None, scale=None, cu_seqlens=None,
                dtype=torch.float32):
    """Composition of the three chunked stages in full precision (no bf16
    intermediates).  Must agree with `recurrent_ref` to rounding; used to
    check the stage formulas themselves."""
    gc = chunk_local_cumsum_ref(g, cu_seqlens).to(dtype)
    u, w = compute_u_w_ref(k, v, beta, gc, cu_seqlens, dtype)
    h, un, S = seq_state_update_ref(k, u, w, gc, initial_state, cu_seqlens, dtype)
    o = compute_o_ref(q, k, un, h, gc, scale, cu_seqlens, dtype)
    return o, S


# --------------------------------------------------------------------------
# error metrics used by the parity tests
# --------------------------------------------------------------------------
# --------------------------------------------------------------------------
# layer-adjacent steps (the reference leaves them to its callers; published definitions restated)
# --------------------------------------------------------------------------
def causal_conv1d_ref(x, weight, bias=None, initial_state=None, cu_seqlens=None, activation: bool = True):
    """Depthwise causal conv along tokens + SiLU.  x (B,T,C) or packed (N,C); weight (C,W); initial_state
    (sequences, W-1, C) = the W-1 inputs before each sequence.  Returns (y, final_state) in fp32."""
    W = weight.shape[1]
    varlen = cu_seqlens is not None
    xs = x.float()
    if not varlen:
        B, T, C_ = xs.shape
        bounds = [(b * T, (b + 1) * T) for b in range(B)]
        xs = xs.reshape(B * T, C_)
    else:
        C_ = xs.shape[1]
        bounds = [(int(cu_seqlens[i]), int(cu_seqlens[i + 1])) for i in range(len(cu_seqlens) - 1)]
    y = torch.zeros_like(xs)
    fin = torch.zeros(len(bounds), W - 1, C_)
    wf = weight.float()
    for s_, (b0, b1) in enumerate(bounds):
        hist = torch.zeros(W - 1, C_) if initial_state is None else initial_state[s_].float()
        ext = torch.cat([hist, xs[b0:b1]], dim=0)          # (W-1+L, C)
        for t in range(b1 - b0):
            acc = (ext[t:t + W] * wf.t()).sum(0)
            if bias is not None:
                acc = acc + bias.float()
            y[b0 + t] = torch.nn.functional.silu(acc) if activation else acc
        fin[s_] = ext[ext.shape[0] - (W - 1):]
    return (y if varlen else y.reshape(x.shape)), fin


def gated_rmsnorm_ref(x, z, weight, eps: float = 1e-6):
    xf, zf = x.float(), z.float()
    return xf * torch.rsqrt((xf * xf).mean(-1, keepdim=True) + eps) * weight.float() * torch.nn.functional.silu(zf)


def rel_fro(x: torch.Tensor, ref: torch.Tensor) -> float:
    x, ref = x.double(), ref.double()
    d = ref.norm().item()
    return (x - ref).norm().item() / (d if d > 0 else 1.0)


def max_abs_over_max(x: torch.Tensor, ref: torch.Tensor) -> float:
    x, ref = x.double(), ref.double()
    d = ref.abs().max().item() if ref.numel() else 0.0
    return (x - ref).abs().max().item() / (d if d > 0 else 1.0) if ref.numel() else 0.0


# --------------------------------------------------------------------------
# linear attention with decay, group norm (no counterpart in the reference)
# --------------------------------------------------------------------------
def linear_attention_ref(q, k, v, g, scale, state=None, steps=False):
    """S <- e^g S + v k^T, o = scale S q, token by token in fp64.  Padded layouts; g (vh), (B,T,vh) or None.
    Returns (out, final state or the state after every token)."""
    B, T, vh, dv = v.shape
    rep = vh // q.shape[2]
    q, k, v = (x.double() for x in (q, k, v))
    q, k = q.repeat_interleave(rep, 2), k.repeat_interleave(rep, 2)
    g = torch.zeros(vh, device=v.device) if g is None else g
    lam = torch.exp(g.double()).expand(B, T, vh) if g.dim() == 1 else torch.exp(g.double())
    S = torch.zeros(B, vh, dv, q.shape[-1], dtype=torch.float64, device=v.device) if state is None else state.double()
    out, kept = torch.empty_like(v), []
    for t in range(T):
        S = lam[:, t, :, None, None] * S + v[:, t, :, :, None] * k[:, t, :, None, :]
        out[:, t] = scale * (S * q[:, t, :, None, :]).sum(-1)
        if steps:
            kept.append(S)
    return out, (torch.stack(kept, 1) if steps else S)


def group_norm_ref(x, groups, weight=None, bias=None, z=None, eps=1e-5, activation=True):
    """Channels-last group norm in fp64; silu(u), or u * silu(z)."""
    N, C = x.shape[0], x.shape[-1]
    y = x.double().reshape(N, -1, groups, C // groups)
    y = (y - y.mean((1, 3), keepdim=True)) / torch.sqrt(y.var((1, 3), unbiased=False, keepdim=True) + eps)
    y = y.reshape(x.shape)
    y = y if weight is None else y * weight.double()
    y = y if bias is None else y + bias.double()
    a = y if z is None else z.double()
    a = a * torch.sigmoid(a) if activation else a
    return a if z is None else y * a
