// Linear attention with decay, token by token (decode, draft runs, wide heads).  Per token t of a sequence and v-head:
//     S <- e^g S + v k^T ,   o = scale S q          (S: dv x dk, rows independent of one another)
// One CTA per 32 rows of a state; the rows stay in registers over all tokens of the call, in fp32.
#pragma once
#include <cuda_bf16.h>

#include "pairs.cuh"
#include "prefill_common.cuh"

namespace gdn {

constexpr int kLinRows = 32;      // state rows of a CTA
constexpr int kLinThreads = 128;  // 4 warps of 8 rows

struct LinRecurrentParams {
    TokenView q, k, v, out;
    ScalarView gate;  // log-decay; ptr == NULL: none
    const void* state_in;
    void* state_out;
    long long si_ss, si_sh, so_ss, so_sh;  // strides of a slot (a token with step states) and a head, in elements
    const int* cu_seqlens;
    const int* num_accepted;
    const int* state_idx;
    long long total_tokens;
    int batch, seq_len, kh, vh, dk, dv, num_slots, store_step;
    float scale;
};

// One token per sequence.  HBM-bound (the state in and out): nothing is kept beyond a row's own arithmetic, so that many CTAs, all of their loads
// out at once, fit an SM.  Columns as below.
template <int LPR, bool kF32>
__global__ void __launch_bounds__(kLinThreads, LPR == 32 ? 5 : kF32 ? 8 : 10) gdn_linear_decode_kernel(const LinRecurrentParams p) {
    using namespace ptx;
    using namespace pairs;
    constexpr int kRowsAtOnce = 32 / LPR;
    constexpr int kIter = 8 / kRowsAtOnce;
    grid_dep_wait();
    grid_dep_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int l = lane % LPR, sub = lane / LPR;
    const int row_tiles = (p.dv + kLinRows - 1) / kLinRows;
    const int unit = blockIdx.x / row_tiles, tile = blockIdx.x - unit * row_tiles;
    const int seq = unit / p.vh, head = unit - seq * p.vh, khead = head / (p.vh / p.kh);
    const int slot = p.state_idx ? p.state_idx[seq] : seq;
    const int c0 = kF32 ? 4 * l : 8 * l, c1 = kF32 ? 4 * (LPR + l) : 8 * l + 4;
    const bool in0 = c0 < p.dk, in1 = c1 < p.dk;
    const int row0 = tile * kLinRows + warp * 8 + sub;  // + kRowsAtOnce * i
    // the token's inputs do not depend on the slot
    const uint2 zero = make_uint2(0u, 0u);
    const __nv_bfloat16* const qt = p.q.ptr + seq * p.q.sb + khead * p.q.sh;
    const __nv_bfloat16* const kt = p.k.ptr + seq * p.k.sb + khead * p.k.sh;
    const unsigned short* const vt = reinterpret_cast<const unsigned short*>(p.v.ptr + seq * p.v.sb + head * p.v.sh);
    const uint2 q0 = in0 ? __ldg(reinterpret_cast<const uint2*>(qt + c0)) : zero, q1 = in1 ? __ldg(reinterpret_cast<const uint2*>(qt + c1)) : zero;
    const uint2 k0 = in0 ? __ldg(reinterpret_cast<const uint2*>(kt + c0)) : zero, k1 = in1 ? __ldg(reinterpret_cast<const uint2*>(kt + c1)) : zero;
    const uint32_t gate = p.gate.ptr ? p.gate.load_bits(seq, 0, head) : 0u;
    unsigned short v[kIter];
#pragma unroll
    for (int i = 0; i < kIter; ++i) {
        const int row = row0 + kRowsAtOnce * i;
        v[i] = row < p.dv ? __ldg(vt + row) : static_cast<unsigned short>(0);
    }
    if (p.state_idx && (slot < 0 || slot >= p.num_slots)) return;  // padding sequence
    uint4 a[kIter], b[kF32 ? kIter : 1];  // the state as it lies
    const long long base = slot * p.si_ss + head * p.si_sh + static_cast<long long>(row0) * p.dk;
#pragma unroll
    for (int i = 0; i < kIter; ++i) {
        const bool in = p.state_in && row0 + kRowsAtOnce * i < p.dv;
        const long long at = base + kRowsAtOnce * i * p.dk;
        a[i] = make_uint4(0u, 0u, 0u, 0u);
        if (kF32) {
            const float* src = static_cast<const float*>(p.state_in) + at;
            b[i] = make_uint4(0u, 0u, 0u, 0u);
            if (in && in0) a[i] = *reinterpret_cast<const uint4*>(src + c0);
            if (in && in1) b[i] = *reinterpret_cast<const uint4*>(src + c1);
        } else if (in && in0) {
            a[i] = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.state_in) + at + c0);
        }
    }
    const float decay = __expf(p.gate.value(gate));
    const f2 d2 = pk(decay, decay);
    f2 k[4] = {pk(bf16_lo(k0.x), bf16_hi(k0.x)), pk(bf16_lo(k0.y), bf16_hi(k0.y)), pk(bf16_lo(k1.x), bf16_hi(k1.x)), pk(bf16_lo(k1.y), bf16_hi(k1.y))};
    f2 q[4] = {pk(bf16_lo(q0.x), bf16_hi(q0.x)), pk(bf16_lo(q0.y), bf16_hi(q0.y)), pk(bf16_lo(q1.x), bf16_hi(q1.x)), pk(bf16_lo(q1.y), bf16_hi(q1.y))};
    const long long to = slot * p.so_ss + head * p.so_sh + static_cast<long long>(row0) * p.dk;
    float o[kIter];
#pragma unroll
    for (int i = 0; i < kIter; ++i) {
        const float vf = __uint_as_float(static_cast<uint32_t>(v[i]) << 16);
        const f2 v2 = pk(vf, vf);
        f2 s[4];
        if (kF32) {
            s[0] = pk(a[i].x, a[i].y); s[1] = pk(a[i].z, a[i].w);
            s[2] = pk(b[i].x, b[i].y); s[3] = pk(b[i].z, b[i].w);
        } else {
            s[0] = pk(bf16_lo(a[i].x), bf16_hi(a[i].x)); s[1] = pk(bf16_lo(a[i].y), bf16_hi(a[i].y));
            s[2] = pk(bf16_lo(a[i].z), bf16_hi(a[i].z)); s[3] = pk(bf16_lo(a[i].w), bf16_hi(a[i].w));
        }
        f2 sum = 0ull;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            s[e] = fma2(s[e], d2, mul2(v2, k[e]));
            sum = fma2(s[e], q[e], sum);
        }
        float lo, hi;
        unpk(sum, lo, hi);
        o[i] = lo + hi;
        if (p.state_out && row0 + kRowsAtOnce * i < p.dv) {
            const long long at = to + kRowsAtOnce * i * p.dk;
            if (kF32) {
                float* dst = static_cast<float*>(p.state_out) + at;
                float4 x, y;
                unpk(s[0], x.x, x.y); unpk(s[1], x.z, x.w);
                unpk(s[2], y.x, y.y); unpk(s[3], y.z, y.w);
                if (in0) *reinterpret_cast<float4*>(dst + c0) = x;
                if (in1) *reinterpret_cast<float4*>(dst + c1) = y;
            } else if (in0) {
                *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.state_out) + at + c0) = make_uint4(pack2(s[0]), pack2(s[1]), pack2(s[2]), pack2(s[3]));
            }
        }
    }
#pragma unroll
    for (int m = LPR / 2; m > 0; m >>= 1)
#pragma unroll
        for (int i = 0; i < kIter; ++i) o[i] += __shfl_xor_sync(0xffffffffu, o[i], m);
    __nv_bfloat16* const op = p.out.ptr + seq * p.out.sb + head * p.out.sh;
#pragma unroll
    for (int i = 0; i < kIter; ++i) {
        const int row = row0 + kRowsAtOnce * i;
        if (l == 0 && row < p.dv) op[row] = __float2bfloat16(p.scale * o[i]);
    }
}

// LPR lanes share a row, 8 columns each: dk <= 8 LPR.  bf16 states: lane l holds columns 8 l .. 8 l + 7.  fp32 states: columns
// 4 l .. and 4 (LPR + l) .., so that a warp's 16-byte accesses are contiguous.
template <int LPR, bool kF32>
__global__ void __launch_bounds__(kLinThreads, LPR == 32 ? 4 : 7) gdn_linear_recurrent_kernel(const LinRecurrentParams p) {
    using namespace ptx;
    using namespace pairs;
    constexpr int kRowsAtOnce = 32 / LPR;
    constexpr int kIter = 8 / kRowsAtOnce;  // rows per thread
    grid_dep_wait();
    grid_dep_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int l = lane % LPR, sub = lane / LPR;
    const int row_tiles = (p.dv + kLinRows - 1) / kLinRows;
    const int tile = blockIdx.x % row_tiles;
    const long long unit = blockIdx.x / row_tiles;
    const int head = static_cast<int>(unit % p.vh);
    const int seq = static_cast<int>(unit / p.vh);
    const int khead = head / (p.vh / p.kh);
    int slot = seq;
    if (p.state_idx) {
        slot = p.state_idx[seq];
        if (slot < 0 || slot >= p.num_slots) return;  // padding sequence
    }
    long long batch = seq, tok0 = 0, tokens = p.seq_len, step0 = static_cast<long long>(seq) * p.seq_len;
    if (p.cu_seqlens) {
        const long long bos = min(max(static_cast<long long>(p.cu_seqlens[seq]), 0ll), p.total_tokens);
        const long long eos = min(max(static_cast<long long>(p.cu_seqlens[seq + 1]), bos), p.total_tokens);
        batch = 0;
        tok0 = step0 = bos;
        tokens = eos - bos;
    }
    if (p.num_accepted) tokens = min(tokens, max(static_cast<long long>(p.num_accepted[seq]), 0ll));

    // columns of this thread's two halves
    const int c0 = kF32 ? 4 * l : 8 * l, c1 = kF32 ? 4 * (LPR + l) : 8 * l + 4;
    const bool in0 = c0 < p.dk, in1 = c1 < p.dk;
    const int row0 = tile * kLinRows + warp * 8 + sub;  // + kRowsAtOnce * i
    auto state_offset = [&](int i) { return static_cast<long long>(row0 + kRowsAtOnce * i) * p.dk; };
    f2 S[kIter][4];
    if (p.state_in) {
        const long long base = static_cast<long long>(slot) * p.si_ss + static_cast<long long>(head) * p.si_sh;
#pragma unroll
        for (int i = 0; i < kIter; ++i) {
            const bool row_in = row0 + kRowsAtOnce * i < p.dv;
            if (kF32) {
                const float* src = static_cast<const float*>(p.state_in) + base + state_offset(i);
                const float4 a = row_in && in0 ? *reinterpret_cast<const float4*>(src + c0) : make_float4(0.f, 0.f, 0.f, 0.f);
                const float4 b = row_in && in1 ? *reinterpret_cast<const float4*>(src + c1) : make_float4(0.f, 0.f, 0.f, 0.f);
                S[i][0] = pk(a.x, a.y); S[i][1] = pk(a.z, a.w);
                S[i][2] = pk(b.x, b.y); S[i][3] = pk(b.z, b.w);
            } else {
                const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(p.state_in) + base + state_offset(i);
                const uint4 a = row_in && in0 ? *reinterpret_cast<const uint4*>(src + c0) : make_uint4(0u, 0u, 0u, 0u);
                S[i][0] = pk(bf16_lo(a.x), bf16_hi(a.x)); S[i][1] = pk(bf16_lo(a.y), bf16_hi(a.y));
                S[i][2] = pk(bf16_lo(a.z), bf16_hi(a.z)); S[i][3] = pk(bf16_lo(a.w), bf16_hi(a.w));
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < kIter; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) S[i][e] = 0ull;
    }
    auto store_state = [&](long long where) {
        const long long base = where * p.so_ss + static_cast<long long>(head) * p.so_sh;
#pragma unroll
        for (int i = 0; i < kIter; ++i) {
            if (row0 + kRowsAtOnce * i >= p.dv) continue;
            if (kF32) {
                float* dst = static_cast<float*>(p.state_out) + base + state_offset(i);
                float4 a, b;
                unpk(S[i][0], a.x, a.y); unpk(S[i][1], a.z, a.w);
                unpk(S[i][2], b.x, b.y); unpk(S[i][3], b.z, b.w);
                if (in0) *reinterpret_cast<float4*>(dst + c0) = a;
                if (in1) *reinterpret_cast<float4*>(dst + c1) = b;
            } else {
                __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.state_out) + base + state_offset(i);
                if (in0)
                    *reinterpret_cast<uint4*>(dst + c0) = make_uint4(pack2(S[i][0]), pack2(S[i][1]), pack2(S[i][2]), pack2(S[i][3]));
            }
        }
    };
    // one token's inputs, requested a token ahead of their use
    struct Token {
        uint2 q[2], k[2];
        unsigned short v[kIter];
        uint32_t g;
    };
    const __nv_bfloat16* const qp = p.q.ptr + batch * p.q.sb + static_cast<long long>(khead) * p.q.sh;
    const __nv_bfloat16* const kp = p.k.ptr + batch * p.k.sb + static_cast<long long>(khead) * p.k.sh;
    const __nv_bfloat16* const vp = p.v.ptr + batch * p.v.sb + static_cast<long long>(head) * p.v.sh;
    auto load_token = [&](long long t, Token& x) {
        const __nv_bfloat16 *qt = qp + t * p.q.st, *kt = kp + t * p.k.st, *vt = vp + t * p.v.st;
        const uint2 zero = make_uint2(0u, 0u);
        x.q[0] = in0 ? __ldg(reinterpret_cast<const uint2*>(qt + c0)) : zero;
        x.q[1] = in1 ? __ldg(reinterpret_cast<const uint2*>(qt + c1)) : zero;
        x.k[0] = in0 ? __ldg(reinterpret_cast<const uint2*>(kt + c0)) : zero;
        x.k[1] = in1 ? __ldg(reinterpret_cast<const uint2*>(kt + c1)) : zero;
#pragma unroll
        for (int i = 0; i < kIter; ++i) {
            const int row = row0 + kRowsAtOnce * i;
            x.v[i] = row < p.dv ? __ldg(reinterpret_cast<const unsigned short*>(vt) + row) : static_cast<unsigned short>(0);
        }
        x.g = p.gate.ptr ? p.gate.load_bits(batch, t, head) : 0u;
    };
    Token cur, next;
    if (tokens > 0) load_token(tok0, cur);
#pragma unroll 1
    for (long long t = 0; t < tokens; ++t) {
        if (t + 1 < tokens) load_token(tok0 + t + 1, next);
        const float decay = __expf(p.gate.value(cur.g));
        const f2 d2 = pk(decay, decay);
        f2 q[4], k[4];
        float o[kIter];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            q[2 * h] = pk(bf16_lo(cur.q[h].x), bf16_hi(cur.q[h].x));
            q[2 * h + 1] = pk(bf16_lo(cur.q[h].y), bf16_hi(cur.q[h].y));
            k[2 * h] = pk(bf16_lo(cur.k[h].x), bf16_hi(cur.k[h].x));
            k[2 * h + 1] = pk(bf16_lo(cur.k[h].y), bf16_hi(cur.k[h].y));
        }
#pragma unroll
        for (int i = 0; i < kIter; ++i) {
            const float vf = __uint_as_float(static_cast<uint32_t>(cur.v[i]) << 16);
            const f2 v2 = pk(vf, vf);
            f2 sum = 0ull;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                S[i][e] = fma2(S[i][e], d2, mul2(v2, k[e]));
                sum = fma2(S[i][e], q[e], sum);
            }
            float lo, hi;
            unpk(sum, lo, hi);
            o[i] = lo + hi;
        }
#pragma unroll
        for (int i = 0; i < kIter; ++i) {
#pragma unroll
            for (int m = LPR / 2; m > 0; m >>= 1) o[i] += __shfl_xor_sync(0xffffffffu, o[i], m);
        }
        __nv_bfloat16* const op = p.out.ptr + batch * p.out.sb + (tok0 + t) * p.out.st + static_cast<long long>(head) * p.out.sh;
#pragma unroll
        for (int i = 0; i < kIter; ++i) {
            const int row = row0 + kRowsAtOnce * i;
            if (l == 0 && row < p.dv) op[row] = __float2bfloat16(p.scale * o[i]);
        }
        if (p.store_step) store_state(step0 + t);
        cur = next;
    }
    if (!p.store_step && p.state_out) store_state(slot);
}

}  // namespace gdn
