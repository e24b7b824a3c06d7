// Linear attention with decay, token by token (decode, draft runs, wide heads).  Per token t of a sequence and v-head:
//     S <- e^g S + v k^T ,   o = scale S q          (S: dv x dk, rows independent of one another)
// One CTA per 32 rows of a state; the rows stay in registers over all tokens of the call, in fp32.
#pragma once
#include <cuda_bf16.h>

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

// LPR lanes share a row, 8 columns each: dk <= 8 LPR.  bf16 states: lane l holds columns 8 l .. 8 l + 7.  fp32 states: columns
// 4 l .. and 4 (LPR + l) .., so that a warp's 16-byte accesses are contiguous.
template <int LPR, bool kF32>
__global__ void __launch_bounds__(kLinThreads) gdn_linear_recurrent_kernel(const LinRecurrentParams p) {
    using namespace ptx;
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
    float S[kIter][8];
    if (p.state_in) {
        const long long base = static_cast<long long>(slot) * p.si_ss + static_cast<long long>(head) * p.si_sh;
#pragma unroll
        for (int i = 0; i < kIter; ++i) {
            const bool row_in = row0 + kRowsAtOnce * i < p.dv;
            if (kF32) {
                const float* src = static_cast<const float*>(p.state_in) + base + state_offset(i);
                const float4 a = row_in && in0 ? *reinterpret_cast<const float4*>(src + c0) : make_float4(0.f, 0.f, 0.f, 0.f);
                const float4 b = row_in && in1 ? *reinterpret_cast<const float4*>(src + c1) : make_float4(0.f, 0.f, 0.f, 0.f);
                S[i][0] = a.x; S[i][1] = a.y; S[i][2] = a.z; S[i][3] = a.w;
                S[i][4] = b.x; S[i][5] = b.y; S[i][6] = b.z; S[i][7] = b.w;
            } else {
                const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(p.state_in) + base + state_offset(i);
                const uint4 a = row_in && in0 ? *reinterpret_cast<const uint4*>(src + c0) : make_uint4(0u, 0u, 0u, 0u);
                S[i][0] = bf16_lo(a.x); S[i][1] = bf16_hi(a.x); S[i][2] = bf16_lo(a.y); S[i][3] = bf16_hi(a.y);
                S[i][4] = bf16_lo(a.z); S[i][5] = bf16_hi(a.z); S[i][6] = bf16_lo(a.w); S[i][7] = bf16_hi(a.w);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < kIter; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) S[i][e] = 0.f;
    }
    auto store_state = [&](long long where) {
        const long long base = where * p.so_ss + static_cast<long long>(head) * p.so_sh;
#pragma unroll
        for (int i = 0; i < kIter; ++i) {
            if (row0 + kRowsAtOnce * i >= p.dv) continue;
            if (kF32) {
                float* dst = static_cast<float*>(p.state_out) + base + state_offset(i);
                if (in0) *reinterpret_cast<float4*>(dst + c0) = make_float4(S[i][0], S[i][1], S[i][2], S[i][3]);
                if (in1) *reinterpret_cast<float4*>(dst + c1) = make_float4(S[i][4], S[i][5], S[i][6], S[i][7]);
            } else {
                __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.state_out) + base + state_offset(i);
                if (in0)
                    *reinterpret_cast<uint4*>(dst + c0) = make_uint4(pack_bf16(S[i][0], S[i][1]), pack_bf16(S[i][2], S[i][3]),
                                                                     pack_bf16(S[i][4], S[i][5]), pack_bf16(S[i][6], S[i][7]));
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
        float q[8], k[8], o[kIter];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            q[4 * h] = bf16_lo(cur.q[h].x); q[4 * h + 1] = bf16_hi(cur.q[h].x);
            q[4 * h + 2] = bf16_lo(cur.q[h].y); q[4 * h + 3] = bf16_hi(cur.q[h].y);
            k[4 * h] = bf16_lo(cur.k[h].x); k[4 * h + 1] = bf16_hi(cur.k[h].x);
            k[4 * h + 2] = bf16_lo(cur.k[h].y); k[4 * h + 3] = bf16_hi(cur.k[h].y);
        }
#pragma unroll
        for (int i = 0; i < kIter; ++i) {
            const float v = __uint_as_float(static_cast<uint32_t>(cur.v[i]) << 16);
            o[i] = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                S[i][e] = fmaf(S[i][e], decay, v * k[e]);
                o[i] = fmaf(S[i][e], q[e], o[i]);
            }
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
