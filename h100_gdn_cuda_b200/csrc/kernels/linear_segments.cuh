// What a segment of a sequence adds to the state of linear attention, for few long sequences (see linear_chunked.cuh): from a state of zero,
//     D = sum over the segment's tokens of e^{G_end - G_j} v_j k_j^T ,
// and the segment's whole decay; then the states that enter the segments, S <- e^{G} S + D from segment to segment.  The chunks are taken last to first,
// so that every factor is a decay to the segment's end (at most one), the products simply accumulate, and what was read last, the
// segment's beginning, is what the run over the chunks asks for first.
// One CTA per segment but the last of a sequence, v-head and 128 columns of dv; two CTAs fit an SM.  HBM-bound (K and V once, 32 KB a chunk at d = 128).  Values
// come in two parts as there.
#pragma once
#include "linear_chunked.cuh"

namespace gdn {

template <int DK, int DV>
struct LinSegSmem {
    static constexpr int kStages = 3;
    static constexpr int kTileK = kChunk * DK * 2, kTileV = kChunk * DV * 2, kOffV = kTileK, kStage = kTileK + kTileV;
    static constexpr int kOffGate = kStages * kStage;  // 4 x factors of the values [64]
    static constexpr int kOffBar = kOffGate + 4 * 256;
    static constexpr int kBytes = kOffBar + 256 + 1024;
};

namespace lin {
constexpr int kSegThreads = 224;   // 4 value warps, producer, issuer, gates
constexpr uint32_t kTmSegF = 0;    // fp32 increment, 128 columns
constexpr uint32_t kTmSegV = 128;  // 2 x bf16 values times factors, 32 columns; 2 x what is left of them
}  // namespace lin

template <int DK, int DV, bool kWhole>
__global__ void __launch_bounds__(lin::kSegThreads, 2)
    gdn_linear_segment_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const LinChunkedParams p) {
    using namespace ptx;
    using namespace lin;
    using L = LinSegSmem<DK, DV>;
    constexpr int kStages = L::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (ptx::smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kOffBar);
    uint64_t* bar_full = bars;                // [stages] K and V of a stage have arrived
    uint64_t* bar_empty = bar_full + kStages; // [stages] the chunk's product is done
    uint64_t* bar_gate = bar_empty + kStages; // [4] factors of a chunk
    uint64_t* bar_gfree = bar_gate + 4;       // [4] and read
    uint64_t* bar_v = bar_gfree + 4;          // [2] values written
    uint64_t* bar_done = bar_v + 2;           // [2] and read: a chunk's product is done
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_done + 2);
    int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
    static_assert((2 * kStages + 12) * 8 + 8 <= 256, "room for the barriers");

    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    grid_dep_wait();
    grid_dep_launch();
    LinWalker walker;
    LinItem it;
    if (!walker.locate(p, p.whole + blockIdx.x, it) || it.segment == it.segments - 1) return;  // (the same for all threads)
    const int chunks = __shfl_sync(0xffffffffu, it.chunks, 0);
    if (tid == 0) {
        *abort_flag = 0;
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&bar_full[i], 1);
            mbar_init(&bar_empty[i], 1);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&bar_gate[i], 1);
            mbar_init(&bar_gfree[i], 4);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar_v[i], 4);
            mbar_init(&bar_done[i], 1);
        }
        mbar_fence_init();
    }
    if (warp == 0) tmem_alloc(tmem_slot, 256);
    fence_proxy_async_smem();
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    auto factors = [&](uint32_t n) { return reinterpret_cast<float*>(smem + L::kOffGate + (n & 3) * 256); };

    if (warp < 4) {
        // =============================================================== value warps (as in gdn_linear_chunked_kernel)
        const int lq = warp;
        const uint32_t tm_lane = static_cast<uint32_t>(32 * lq) << 16;
        const uint32_t vlane = static_cast<uint32_t>((lq >> 1) * 8192 + (8 * (lane >> 4) + (lane & 7)) * 128);
        const uint32_t vchunk = static_cast<uint32_t>(4 * (lq & 1) + ((lane >> 3) & 1));
        const uint32_t vsw0 = vlane + ((vchunk ^ (lane & 7)) << 4), vsw1 = vlane + (((vchunk + 2) ^ (lane & 7)) << 4);
#pragma unroll 1
        for (uint32_t n = 0; n < static_cast<uint32_t>(chunks); ++n) {
            const uint32_t s = n % kStages;
            mbar_wait_short(&bar_gate[n & 3], (n >> 2) & 1, abort_flag);
            if (n > 1) mbar_wait_short(&bar_done[n & 1], ((n >> 1) + 1) & 1, abort_flag);
            mbar_wait_short(&bar_full[s], (n / kStages) & 1, abort_flag);
            tc_fence_after_sync();
            const uint2* const fv = reinterpret_cast<const uint2*>(factors(n)) + (lane & 3);
            const uint32_t sV = smem_u32(smem + s * L::kStage + L::kOffV);
            if (DV == 128 || lq < 2) {
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {  // 32 tokens
                    uint32_t v[2][2][4];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        ldmatrix_x4_trans(sV + vsw0 + 4096 * hf + 2048 * j, v[0][j]);
                        ldmatrix_x4_trans(sV + vsw1 + 4096 * hf + 2048 * j, v[1][j]);
                    }
                    const uint32_t to = tmem + kTmSegV + tm_lane + 32 * (n & 1) + 16 * hf;
                    uint32_t u[2][2][4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint2 f = fv[16 * hf + 4 * i];
#pragma unroll
                        for (int a = 0; a < 2; ++a) {
                            times_factors(v[0][i >> 1][2 * (i & 1) + a], u[0][i >> 1][2 * (i & 1) + a], f);
                            times_factors(v[1][i >> 1][2 * (i & 1) + a], u[1][i >> 1][2 * (i & 1) + a], f);
                        }
                    }
                    tmem_st_frag16(to + 64, u[0][0]);
                    tmem_st_frag16(to + 64 + (16u << 16), u[1][0]);
                    tmem_st_frag16(to, v[0][0]);
                    tmem_st_frag16(to + (16u << 16), v[1][0]);
                }
            }
            tmem_wait_st();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&bar_v[n & 1]);
                mbar_arrive(&bar_gfree[n & 3]);
            }
        }
        mbar_wait_short(&bar_done[(chunks - 1) & 1], ((chunks - 1) >> 1) & 1, abort_flag);
        tc_fence_after_sync();
        if (*static_cast<volatile int*>(abort_flag) == 0 && (DV == 128 || lq < 2)) {
            uint4* dst = reinterpret_cast<uint4*>(p.seg_state + static_cast<long long>(it.mine) * (128 * DK) + (32 * lq + lane) * DK);
#pragma unroll 1
            for (int q = 0; q < DK; q += 16) {
                uint32_t r[16];
                tmem_ld16(tmem + kTmSegF + tm_lane + q, r);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 4; ++e) dst[q / 4 + e] = *reinterpret_cast<const uint4*>(r + 4 * e);
            }
        }
    } else if (warp == 4) {
        // =============================================================== producer
        const int khead = __shfl_sync(0xffffffffu, it.khead, 0), head = __shfl_sync(0xffffffffu, it.head, 0), batch = __shfl_sync(0xffffffffu, it.batch, 0);
        const int tok0 = __shfl_sync(0xffffffffu, it.tok0, 0), dvt = __shfl_sync(0xffffffffu, it.dvt, 0);
#pragma unroll 1
        for (int n = 0; n < chunks; ++n) {
            const int s = n % kStages;
            mbar_wait_short(&bar_empty[s], ((n / kStages) + 1) & 1, abort_flag);
            uint8_t* st = smem + s * L::kStage;
            const int tok = tok0 + (chunks - 1 - n) * kChunk;
            if (elect_one()) {
                mbar_arrive_expect_tx(&bar_full[s], L::kStage);
                if (kWhole) {
                    tma_load_5d(st, &tmK, &bar_full[s], 0, tok, 0, khead, batch);
                    tma_load_5d(st + L::kOffV, &tmV, &bar_full[s], 0, tok, 2 * dvt, head, batch);
                } else {
#pragma unroll 1
                    for (int a = 0; a < DK / 64; ++a) tma_load_4d(st + a * 8192, &tmK, &bar_full[s], a * 64, khead, tok, batch);
#pragma unroll 1
                    for (int a = 0; a < DV / 64; ++a) tma_load_4d(st + L::kOffV + a * 8192, &tmV, &bar_full[s], dvt * 128 + a * 64, head, tok, batch);
                }
            }
            __syncwarp();
        }
        if (*static_cast<volatile int*>(abort_flag) != 0) {  // a wait has given up: the copies in flight land before the CTA goes
            for (int n = max(chunks - kStages, 0); n < chunks; ++n) {
                int none = 0;
                mbar_wait_limit(&bar_full[n % kStages], (n / kStages) & 1, &none, 1ll << 28);
            }
        }
    } else if (warp == 5) {
        // =============================================================== products
        constexpr uint32_t id_d = make_idesc_bf16(128, DK, false, true);
        const uint64_t dK = make_smem_desc_sw128(smem_u32(smem), 8192, 1024);  // read MN-major
#pragma unroll 1
        for (int n = 0; n < chunks; ++n) {
            const int s = n % kStages, b = n & 1;
            mbar_wait_short(&bar_full[s], (n / kStages) & 1, abort_flag);
            mbar_wait_short(&bar_v[b], (n >> 1) & 1, abort_flag);
            tc_fence_after_sync();
            const uint32_t tV = tmem + kTmSegV + 32 * b;
            if (n == 0) mma_ts_k64_w<false, 128>(tmem + kTmSegF, tV, desc_advance(dK, s * L::kStage), id_d);
            else mma_ts_k64_w<true, 128>(tmem + kTmSegF, tV, desc_advance(dK, s * L::kStage), id_d);
            mma_ts_k64_w<true, 128>(tmem + kTmSegF, tV + 64, desc_advance(dK, s * L::kStage), id_d);
            mma_commit_w(&bar_done[b]);
            mma_commit_w(&bar_empty[s]);
        }
    } else {
        // =============================================================== gates
        float suffix = 0.f, suffix_rest = 0.f;  // of the chunks behind, log2
        auto load = [&](int c, uint32_t& a0, uint32_t& a1) {
            a0 = a1 = 0u;
            if (c >= 0 && p.gate.ptr) {  // (segments in front of the last one are whole chunks)
                a0 = p.gate.load_bits(it.batch, it.tok0 + c * kChunk + 2 * lane, it.head);
                a1 = p.gate.load_bits(it.batch, it.tok0 + c * kChunk + 2 * lane + 1, it.head);
            }
        };
        uint32_t a0, a1, b0, b1, c0, c1;  // the gates of this chunk and the two in front of it: DRAM answers later than a chunk takes
        load(chunks - 1, a0, a1);
        load(chunks - 2, b0, b1);
        load(chunks - 3, c0, c1);
#pragma unroll 1
        for (int n = 0; n < chunks; ++n) {
            float g0 = lin_gate_log2(p.gate.value(a0)), g1 = lin_gate_log2(p.gate.value(a1));
            a0 = b0; a1 = b1;
            b0 = c0; b1 = c1;
            load(chunks - 4 - n, c0, c1);
            const float all = scan64_behind(g0, g1, lane);
            mbar_wait_short(&bar_gfree[n & 3], ((n >> 2) + 1) & 1, abort_flag);
            reinterpret_cast<uint2*>(factors(n))[lane] = factor_pair(ex2(suffix + (suffix_rest + g0)), ex2(suffix + (suffix_rest + g1)));
            add_kept(suffix, suffix_rest, all);
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar_gate[n & 3]);
        }
        if (lane == 0) p.seg_decay[it.mine] = suffix + suffix_rest;
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem, 256);
    if (tid == 0 && *abort_flag) {
        p.seg_decay[it.mine] = __int_as_float(0x7FFFFFFF);  // what is made of it is a NaN, not a guess
        if (p.status) atomicExch(p.status, 4);
    }
}

// The states behind the segments, in the place of what the segments add: one CTA per (sequence, v-head, 128 columns of dv) and part of the
// state; four values a thread, segment after segment, what they add asked for ahead.
constexpr int kLinCombineThreads = 256;

__global__ void __launch_bounds__(kLinCombineThreads) gdn_linear_combine_kernel(const LinChunkedParams p, int dk_tile) {
    __shared__ int first_slot, segments;
    ptx::grid_dep_wait();
    ptx::grid_dep_launch();
    const int per = p.vh * p.dv_tiles, chain = p.whole + blockIdx.x, seq = chain / per, rest = chain % per, head = rest / p.dv_tiles, dvt = rest % p.dv_tiles;
    int place = blockIdx.x * p.num_segments, stride = 1, n = p.num_segments - 1;  // of the chain's first segment; from one to the next
    bool keep = p.in_place != 0;
    if (p.cu_seqlens) {
        if (threadIdx.x < 32) {  // the segments of the sequences in front
            int mine = 0;
            for (int s = threadIdx.x; s <= seq; s += 32) {
                const int b = min(max(p.cu_seqlens[s], 0), p.total_tokens), e = min(max(p.cu_seqlens[s + 1], b), p.total_tokens);
                const int k = max(1, ((e - b + kChunk - 1) / kChunk + p.seg_chunks - 1) / p.seg_chunks);
                if (s < seq) mine += k;
                else segments = k;
            }
#pragma unroll
            for (int m = 16; m > 0; m >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, m);
            if (threadIdx.x == 0) first_slot = mine;
        }
        __syncthreads();
        place = first_slot * per + rest;
        stride = per;
        n = min(segments - 1, p.num_items / per - first_slot);  // (offsets that are not in order may ask for more slots than there are)
        keep = keep && first_slot + segments <= p.num_items / per;
    }
    if (n <= 0) return;
    const int at = (blockIdx.y * kLinCombineThreads + threadIdx.x) * 4, row = at / dk_tile, col = at % dk_tile;
    const long long drow = dvt * 128 + row;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (p.state_in && drow < p.dv && col < p.dk) {
        const long long o = seq * p.si_ss + head * p.si_sh + drow * p.dk + col;
        if (p.state_f32) {
            s = *reinterpret_cast<const float4*>(static_cast<const float*>(p.state_in) + o);
        } else {
            const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(p.state_in) + o);
            s = make_float4(ptx::bf16_lo(v.x), ptx::bf16_hi(v.x), ptx::bf16_lo(v.y), ptx::bf16_hi(v.y));
        }
    }
    const long long step = static_cast<long long>(stride) * 128 * dk_tile;
    float* from = p.seg_state + static_cast<long long>(place) * 128 * dk_tile + at;
    const float* decay = p.seg_decay + place;
    if (keep) *reinterpret_cast<float4*>(from + n * step) = s;
    constexpr int kAhead = 8;
    float4 d[kAhead];
    float g[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
        if (i < n) {
            d[i] = __ldcg(reinterpret_cast<const float4*>(from + i * step));
            g[i] = __ldcg(decay + static_cast<long long>(i) * stride);
        }
    for (int i0 = 0; i0 < n; i0 += kAhead) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (i0 + i < n) {
                const float e = lin::ex2(g[i]);
                s.x = fmaf(s.x, e, d[i].x);
                s.y = fmaf(s.y, e, d[i].y);
                s.z = fmaf(s.z, e, d[i].z);
                s.w = fmaf(s.w, e, d[i].w);
                *reinterpret_cast<float4*>(from + (i0 + i) * step) = s;
                if (i0 + i + kAhead < n) {
                    d[i] = __ldcg(reinterpret_cast<const float4*>(from + (i0 + i + kAhead) * step));
                    g[i] = __ldcg(decay + static_cast<long long>(i0 + i + kAhead) * stride);
                }
            }
        }
    }
}

}  // namespace gdn
