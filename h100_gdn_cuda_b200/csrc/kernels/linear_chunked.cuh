// Linear attention with decay over whole prompts, 64 tokens at a time.  With G the running sum of a chunk's log-decays and S the
// state that enters it (dv x dk),
//     O = scale * ( e^{G_i} Q S^T  +  (Q K^T .* e^{G_i - G_j}, j <= i) V )
//     S <- e^{G_L} S + V^T (e^{G_L - G_j} K) .
// The increment of the state does not depend on the state, so nothing but a multiplication and an addition per element
// runs from chunk to chunk, and all products of a chunk can be issued ahead of it.
//
// A persistent CTA takes work items (sequence segment, v-head, 128 columns of dv) one after the other; its roles run over the same
// items and chunks, handing tiles on through mbarriers:
//   warps 0-7   state warps: the fp32 state in registers (lane = dv row, half of the columns each), its bf16 copy into tensor memory
//   warps 8-11  output warps: both parts of O scaled and added, transposed through shared memory, stored
//   warps 12-15 score warps: e^{G_L - G_j} K as bf16 tile; the scores with their decay as bf16 tile
//   warp 16     producer: tensor copies of Q, K, V into a ring of stages
//   warp 17     issues every tcgen05.mma
//   warp 18     the gates' running sums and the factors made of them
// All accumulators that feed the output are transposed (128 dv rows = M): S is an A operand in tensor memory, V one read MN-major
// from the tile as it was copied, Q and the scores are B operands.
#pragma once
#include <cuda.h>

#include "prefill_common.cuh"

namespace gdn {

struct LinChunkedParams {
    TokenView out;
    ScalarView gate;  // log-decay; ptr == NULL: none
    const void* state_in;
    void* state_out;
    long long si_ss, si_sh, so_ss, so_sh;
    const int* cu_seqlens;
    long long total_tokens;
    int num_seqs, seq_len, kh, vh, dk, dv, dv_tiles;
    int state_f32;
    float scale;
    int* status;
    // segments of `seg_chunks` chunks: a sequence of c chunks has max(1, ceil(c / seg_chunks)) of them; slots are numbered through the
    // sequences.  num_items: slots (an upper bound in packed mode) x vh x dv_tiles.
    int seg_chunks, num_segments, num_items;
    float* seg_state;  // per item: what the segment adds to the state (gdn_linear_segment_kernel), then the state behind it
    float* seg_decay;  // per slot and head: the segment's sum of log2-decays
};

// Decays are handled as powers of two; anything below 2^-160 is zero in fp32, and sums of 64 such stay exact enough to tell G_i - G_j
// where a chunk forgets several times over (64 x 160 has a spacing of 2^-10).  A NaN stays one.
__device__ __forceinline__ float lin_gate_log2(float g) {
    const float x = g * 1.4426950408889634f;
    return x < -160.f ? -160.f : x;
}

struct LinItem {
    int seq, head, dvt, batch, segment, segments;
    long long slot, tok0, tokens;  // of the segment
    int chunks;
};

// Walks the items of a CTA in rising order; warp-collective (every warp keeps its own).
struct LinWalker {
    int base = 0;         // packed mode: first sequence of the 32 that were looked at last
    long long first = 0;  // its first slot
    // false: a surplus item
    __device__ __forceinline__ bool locate(const LinChunkedParams& p, long long it, LinItem& o) {
        const int per = p.vh * p.dv_tiles;
        o.slot = it / per;
        const int r = static_cast<int>(it - o.slot * per);
        o.head = r / p.dv_tiles;
        o.dvt = r - o.head * p.dv_tiles;
        long long bos = 0, len = p.seq_len;
        if (!p.cu_seqlens) {
            o.seq = static_cast<int>(o.slot / p.num_segments);
            o.segment = static_cast<int>(o.slot - static_cast<long long>(o.seq) * p.num_segments);
            o.segments = p.num_segments;
            o.batch = o.seq;
        } else {
            const int lane = threadIdx.x & 31;
            o.batch = 0;
            while (true) {
                if (base >= p.num_seqs) return false;
                const int s = base + lane;
                long long b = 0, e = 0;
                int n = 0;
                if (s < p.num_seqs) {
                    b = min(max(static_cast<long long>(p.cu_seqlens[s]), 0ll), p.total_tokens);
                    e = min(max(static_cast<long long>(p.cu_seqlens[s + 1]), b), p.total_tokens);
                    const long long chunks = (e - b + kChunk - 1) / kChunk;
                    n = max(1, static_cast<int>((chunks + p.seg_chunks - 1) / p.seg_chunks));
                }
                int incl = n;
#pragma unroll
                for (int m = 1; m < 32; m <<= 1) {
                    const int y = __shfl_up_sync(0xffffffffu, incl, m);
                    if (lane >= m) incl += y;
                }
                const int total = __shfl_sync(0xffffffffu, incl, 31);
                if (o.slot >= first + total) {
                    base += 32;
                    first += total;
                    continue;
                }
                const int mine = __ffs(__ballot_sync(0xffffffffu, o.slot < first + incl)) - 1;
                o.seq = base + mine;
                o.segments = __shfl_sync(0xffffffffu, n, mine);
                o.segment = static_cast<int>(o.slot - first) - (__shfl_sync(0xffffffffu, incl, mine) - o.segments);
                bos = __shfl_sync(0xffffffffu, b, mine);
                len = __shfl_sync(0xffffffffu, e, mine) - bos;
                break;
            }
        }
        const long long t0 = static_cast<long long>(o.segment) * p.seg_chunks * kChunk;
        o.tok0 = bos + t0;
        o.tokens = min(len - t0, static_cast<long long>(p.seg_chunks) * kChunk);
        o.chunks = static_cast<int>((o.tokens + kChunk - 1) / kChunk);
        return true;
    }
};

template <int DK, int DV>
struct LinSmem {
    static constexpr int kStages = 3;
    static constexpr int kTileK = kChunk * DK * 2, kTileV = kChunk * DV * 2;
    static constexpr int kOffQ = 0, kOffK = kTileK, kOffV = 2 * kTileK, kStage = 2 * kTileK + kTileV;
    static constexpr int kOffKT = kStages * kStage;        // 2 x decayed K
    static constexpr int kOffP = kOffKT + 2 * kTileK;      // 2 x scores, 64 x 64
    static constexpr int kOffO = kOffP + 2 * 8192;         // output staging
    static constexpr int kOffGate = kOffO + kTileV;        // 4 x { G[64], e^{G_L - G_j}[64], scale e^{G_i}[64], e^{G_L} }
    static constexpr int kGateStride = (3 * 64 + 4) * 4;
    static constexpr int kOffBar = kOffGate + 4 * kGateStride;
    static constexpr int kBytes = kOffBar + 256 + 1024;
};

namespace lin {
constexpr int kThreads = 640;  // 5 warpgroups: 2 x state, output, scores, the rest
constexpr uint32_t kTmS = 0;     // bf16 state, 64 columns
constexpr uint32_t kTmP = 64;    // fp32 Q K^T of even (lanes +0) and odd chunks (lanes +16), 64 columns
constexpr uint32_t kTmD = 128;   // fp32 state increment, 128 columns
constexpr uint32_t kTmO1 = 256;  // 2 x fp32 S Q^T, 64 columns
constexpr uint32_t kTmO2 = 384;  // 2 x fp32 V^T P^T, 64 columns
template <int N>
__device__ __forceinline__ void reg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void reg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
__device__ __forceinline__ void named_bar_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// the running sums of 64 log2-decays, lane l: tokens l and l + 32
__device__ __forceinline__ void scan64(float& g0, float& g1, int lane) {
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        const float y0 = __shfl_up_sync(0xffffffffu, g0, m), y1 = __shfl_up_sync(0xffffffffu, g1, m);
        if (lane >= m) {
            g0 += y0;
            g1 += y1;
        }
    }
    g1 += __shfl_sync(0xffffffffu, g0, 31);
}
// 16 bytes of K times a factor
__device__ __forceinline__ uint4 scale8(uint4 v, float f) {
    using namespace ptx;
    v.x = pack_bf16(bf16_lo(v.x) * f, bf16_hi(v.x) * f);
    v.y = pack_bf16(bf16_lo(v.y) * f, bf16_hi(v.y) * f);
    v.z = pack_bf16(bf16_lo(v.z) * f, bf16_hi(v.z) * f);
    v.w = pack_bf16(bf16_lo(v.w) * f, bf16_hi(v.w) * f);
    return v;
}
}  // namespace lin

template <int DK, int DV>
__global__ void __launch_bounds__(lin::kThreads, 1)
    gdn_linear_chunked_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                              const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmO, const LinChunkedParams p) {
    using namespace ptx;
    using namespace lin;
    using L = LinSmem<DK, DV>;
    constexpr int kStages = L::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (ptx::smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kOffBar);
    // (no barrier may run two phases ahead of somebody who waits on it: each one's next phase needs what its waiters do after theirs)
    uint64_t* bar_qk = bars;          // [3] Q and K of a stage have arrived
    uint64_t* bar_v = bars + 3;       // [3] V
    uint64_t* bar_empty = bars + 6;   // [3] the products of the stage's chunk are done
    uint64_t* bar_gate = bars + 9;    // [4] gate factors of a chunk
    uint64_t* bar_gfree = bars + 13;  // [4] read by state and output warps
    uint64_t* bar_score = bars + 17;  // [2] Q K^T done
    uint64_t* bar_p = bars + 19;      // [2] scores written
    uint64_t* bar_kt = bars + 21;     // [2] decayed K written (and rows of V past the end cleared)
    uint64_t* bar_ktfree = bars + 23; // [2] and read
    uint64_t* bar_o = bars + 25;      // [2] both parts of O done
    uint64_t* bar_ofree = bars + 27;  // [2] and read
    uint64_t* bar_d = bars + 29;      // state increment done
    uint64_t* bar_dfree = bars + 30;  // and read
    uint64_t* bar_s = bars + 31;      // the state a chunk reads is in tensor memory; (256 bytes of barriers end here)
    __shared__ uint64_t bar_sq;       // and has been read
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    int* abort_flag = &abort_word;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        *abort_flag = 0;
        for (int i = 0; i < 3; ++i) {
            mbar_init(&bar_qk[i], 1);
            mbar_init(&bar_v[i], 1);
            mbar_init(&bar_empty[i], 1);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&bar_gate[i], 1);
            mbar_init(&bar_gfree[i], 12);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar_score[i], 1);
            mbar_init(&bar_p[i], 4);
            mbar_init(&bar_kt[i], 4);
            mbar_init(&bar_ktfree[i], 1);
            mbar_init(&bar_o[i], 1);
            mbar_init(&bar_ofree[i], 4);
        }
        mbar_init(bar_d, 1);
        mbar_init(bar_dfree, 8);
        mbar_init(bar_s, 8);
        mbar_init(&bar_sq, 1);
        mbar_fence_init();
    }
    if (warp == 0) tmem_alloc(&tmem_slot, 512);
    fence_proxy_async_smem();
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = tmem_slot;
    grid_dep_wait();
    grid_dep_launch();

    auto gate_buf = [&](uint32_t gc) { return reinterpret_cast<float*>(smem + L::kOffGate + (gc & 3) * L::kGateStride); };
    LinWalker walker;
    LinItem it;
    uint32_t gc = 0;  // chunks so far, the same count in every role

    if (warp < 8) {
        // =============================================================== state warps
        // registers of the CTA: 640 x 96; 8 warps at 112, 8 at 96, 4 at 56
        static_assert(32 * (8 * 112 + 8 * 96 + 4 * 56) <= kThreads * 96, "register pool of the CTA");
        reg_inc<112>();
        constexpr int kCols = DK / 2;  // of a thread
        const int lq = warp & 3, hf = warp >> 2;
        const uint32_t tm_lane = static_cast<uint32_t>(32 * lq) << 16;
        float S[kCols];
        for (long long i = blockIdx.x; i < p.num_items; i += gridDim.x) {
            if (!walker.locate(p, i, it)) continue;
            const int row = it.dvt * 128 + 32 * lq + lane;
            const bool row_in = 32 * lq + lane < DV && row < p.dv;
            const int c0 = kCols * hf;
            // ---- the state that enters the segment
            const bool from_seg = it.segment > 0;
            if (from_seg) {
                const float* src = p.seg_state + (i - static_cast<long long>(p.vh) * p.dv_tiles) * (DV * DK) + (32 * lq + lane) * DK + c0;
#pragma unroll
                for (int q = 0; q < kCols / 4; ++q) {
                    const float4 v = 32 * lq + lane < DV ? __ldcg(reinterpret_cast<const float4*>(src) + q) : make_float4(0.f, 0.f, 0.f, 0.f);
                    S[4 * q] = v.x; S[4 * q + 1] = v.y; S[4 * q + 2] = v.z; S[4 * q + 3] = v.w;
                }
            } else if (p.state_in && p.state_f32) {
                const float* src = static_cast<const float*>(p.state_in) + it.seq * p.si_ss + it.head * p.si_sh + static_cast<long long>(row) * p.dk + c0;
#pragma unroll
                for (int q = 0; q < kCols / 4; ++q) {
                    const float4 v = row_in && c0 + 4 * q < p.dk ? *(reinterpret_cast<const float4*>(src) + q) : make_float4(0.f, 0.f, 0.f, 0.f);
                    S[4 * q] = v.x; S[4 * q + 1] = v.y; S[4 * q + 2] = v.z; S[4 * q + 3] = v.w;
                }
            } else if (p.state_in) {
                const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(p.state_in) + it.seq * p.si_ss + it.head * p.si_sh + static_cast<long long>(row) * p.dk + c0;
#pragma unroll
                for (int q = 0; q < kCols / 8; ++q) {
                    const uint4 v = row_in && c0 + 8 * q < p.dk ? *(reinterpret_cast<const uint4*>(src) + q) : make_uint4(0u, 0u, 0u, 0u);
                    S[8 * q] = bf16_lo(v.x); S[8 * q + 1] = bf16_hi(v.x); S[8 * q + 2] = bf16_lo(v.y); S[8 * q + 3] = bf16_hi(v.y);
                    S[8 * q + 4] = bf16_lo(v.z); S[8 * q + 5] = bf16_hi(v.z); S[8 * q + 6] = bf16_lo(v.w); S[8 * q + 7] = bf16_hi(v.w);
                }
            } else {
#pragma unroll
                for (int q = 0; q < kCols; ++q) S[q] = 0.f;
            }
            // the bf16 copy that chunk `n` reads (rounded for the product only: the state itself stays in fp32)
            auto publish = [&](uint32_t n) {
                if (n > 0) mbar_wait(&bar_sq, (n - 1) & 1, abort_flag);  // the copy of the chunk before has been read
                tc_fence_after_sync();
#pragma unroll
                for (int q = 0; q < kCols / 32; ++q) {
                    uint32_t w[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) w[e] = pack_bf16(S[q * 32 + 2 * e], S[q * 32 + 2 * e + 1]);
                    tmem_st16(tmem + kTmS + tm_lane + kCols / 2 * hf + 16 * q, w);
                }
                tmem_wait_st();
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_s);
            };
            if (it.chunks > 0) publish(gc);
            for (int c = 0; c < it.chunks; ++c, ++gc) {
                mbar_wait(&bar_gate[gc & 3], (gc >> 2) & 1, abort_flag);
                const float eg = gate_buf(gc)[192];
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar_gfree[gc & 3]);
                mbar_wait(bar_d, gc & 1, abort_flag);
                tc_fence_after_sync();
#pragma unroll
                for (int q = 0; q < kCols / 32; ++q) {
                    uint32_t r[32];
                    tmem_ld32(tmem + kTmD + tm_lane + kCols * hf + 32 * q, r);
                    tmem_wait_ld();
                    if (q == kCols / 32 - 1) {
                        tc_fence_before_sync();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(bar_dfree);
                    }
#pragma unroll
                    for (int e = 0; e < 32; ++e) S[32 * q + e] = fmaf(S[32 * q + e], eg, __uint_as_float(r[e]));
                }
                if (c + 1 < it.chunks) publish(gc + 1);
            }
            // ---- the state behind the sequence
            if (it.segment == it.segments - 1 && p.state_out && row_in && *abort_flag == 0) {
                const long long at = it.seq * p.so_ss + it.head * p.so_sh + static_cast<long long>(row) * p.dk + c0;
                if (p.state_f32) {
                    float4* dst = reinterpret_cast<float4*>(static_cast<float*>(p.state_out) + at);
#pragma unroll
                    for (int q = 0; q < kCols / 4; ++q)
                        if (c0 + 4 * q < p.dk) dst[q] = make_float4(S[4 * q], S[4 * q + 1], S[4 * q + 2], S[4 * q + 3]);
                } else {
                    uint4* dst = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.state_out) + at);
#pragma unroll
                    for (int q = 0; q < kCols / 8; ++q)
                        if (c0 + 8 * q < p.dk)
                            dst[q] = make_uint4(pack_bf16(S[8 * q], S[8 * q + 1]), pack_bf16(S[8 * q + 2], S[8 * q + 3]),
                                                pack_bf16(S[8 * q + 4], S[8 * q + 5]), pack_bf16(S[8 * q + 6], S[8 * q + 7]));
                }
            }
        }
    } else if (warp < 12) {
        // =============================================================== output warps
        const int lq = warp & 3, otid = tid - 256;
        const uint32_t tm_lane = static_cast<uint32_t>(32 * lq) << 16;
        // transposing matrix stores into the swizzled staging tile: lane 8m + r addresses token r of block m
        const uint32_t olane = static_cast<uint32_t>((lq >> 1) * 8192 + (8 * (lane >> 4) + (lane & 7)) * 128);
        const uint32_t ochunk = static_cast<uint32_t>(4 * (lq & 1) + ((lane >> 3) & 1));
        const uint32_t osw0 = olane + ((ochunk ^ (lane & 7)) << 4), osw1 = olane + (((ochunk + 2) ^ (lane & 7)) << 4);
        const bool packed = p.cu_seqlens != nullptr;
        uint8_t* const sO = smem + L::kOffO;
        const uint32_t sOa = smem_u32(sO);
        for (long long i = blockIdx.x; i < p.num_items; i += gridDim.x) {
            if (!walker.locate(p, i, it)) continue;
            for (int c = 0; c < it.chunks; ++c, ++gc) {
                const int n = static_cast<int>(min(it.tokens - static_cast<long long>(c) * kChunk, static_cast<long long>(kChunk)));
                const float* gb = gate_buf(gc) + 128;
                const uint32_t tO1 = tmem + kTmO1 + 64 * (gc & 1) + tm_lane, tO2 = tmem + kTmO2 + 64 * (gc & 1) + tm_lane;
                mbar_wait(&bar_gate[gc & 3], (gc >> 2) & 1, abort_flag);
                mbar_wait(&bar_o[gc & 1], (gc >> 1) & 1, abort_flag);
                tc_fence_after_sync();
                if (otid == 0) bulk_wait_read<0>();  // the store before has finished reading the staging tile
                named_bar_sync(1, 128);
#pragma unroll
                for (int b = 0; b < 2; ++b) {  // 32 tokens
                    float2 gv[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) gv[j] = *reinterpret_cast<const float2*>(gb + 32 * b + 8 * j + 2 * (lane & 3));
#pragma unroll
                    for (int h = 0; h < 2; ++h) {  // 16 rows
                        uint32_t r1[16], r2[16], w[8];
                        const uint32_t at = (static_cast<uint32_t>(16 * h) << 16) + 32 * b;
                        tmem_ld_frag32(tO1 + at, r1);
                        tmem_ld_frag32(tO2 + at, r2);
                        tmem_wait_ld();
                        if (b == 1 && h == 1) {
                            tc_fence_before_sync();
                            __syncwarp();
                            if (lane == 0) {
                                mbar_arrive(&bar_ofree[gc & 1]);
                                mbar_arrive(&bar_gfree[gc & 3]);
                            }
                        }
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            w[j] = pack_bf16(fmaf(gv[j >> 1].x, __uint_as_float(r1[2 * j]), p.scale * __uint_as_float(r2[2 * j])),
                                             fmaf(gv[j >> 1].y, __uint_as_float(r1[2 * j + 1]), p.scale * __uint_as_float(r2[2 * j + 1])));
                        if (DV == 128 || lq < 2) {
                            const uint32_t so = sOa + (h ? osw1 : osw0) + 4096 * b;
                            stmatrix_x4_trans(so, w[0], w[1], w[2], w[3]);
                            stmatrix_x4_trans(so + 2048, w[4], w[5], w[6], w[7]);
                        }
                    }
                }
                fence_proxy_async_smem();
                named_bar_sync(1, 128);
                const long long tok0 = it.tok0 + static_cast<long long>(c) * kChunk;
                const int left = p.dv - it.dvt * 128;  // columns from this tile on
                if (*abort_flag != 0) {
                    // a wait has given up: the tile is garbage and stays on chip
                } else if (!packed || n == kChunk) {
                    if (otid == 0) {
#pragma unroll
                        for (int a = 0; a < DV / 64; ++a)  // columns past dv and tokens past the end are clipped
                            if (64 * a < left) tma_store_4d(&tmO, sO + 8192 * a, it.dvt * 128 + 64 * a, it.head, static_cast<int>(tok0), it.batch);
                        bulk_commit();
                    }
                } else {  // a whole box would reach into the next sequence
                    __nv_bfloat16* base = p.out.ptr + it.batch * p.out.sb + tok0 * p.out.st + static_cast<long long>(it.head) * p.out.sh + it.dvt * 128;
                    const int pieces = min(left, DV) >> 3;
                    for (int idx = otid; idx < n * 16; idx += 128) {
                        const int row = idx >> 4, c16 = idx & 15;
                        if (c16 < pieces) *reinterpret_cast<uint4*>(base + row * p.out.st + c16 * 8) = *reinterpret_cast<const uint4*>(sO + tile_off(row, c16));
                    }
                }
            }
        }
        if (otid == 0) bulk_wait_read<0>();
    } else if (warp < 16) {
        // =============================================================== score warps
        const int lq = warp & 3, stid = tid - 384;
        const bool packed = p.cu_seqlens != nullptr;
        for (long long i = blockIdx.x; i < p.num_items; i += gridDim.x) {
            if (!walker.locate(p, i, it)) continue;
            for (int c = 0; c < it.chunks; ++c, ++gc) {
                const int n = static_cast<int>(min(it.tokens - static_cast<long long>(c) * kChunk, static_cast<long long>(kChunk)));
                const uint32_t s = gc % kStages, sp = (gc / kStages) & 1;
                uint8_t* stage = smem + s * L::kStage;
                const float* gb = gate_buf(gc);
                mbar_wait(&bar_gate[gc & 3], (gc >> 2) & 1, abort_flag);
                mbar_wait(&bar_qk[s], sp, abort_flag);
                // ---- decayed K (rounded to bf16 as an operand)
                mbar_wait(&bar_ktfree[gc & 1], ((gc >> 1) + 1) & 1, abort_flag);
                uint8_t* kt = smem + L::kOffKT + (gc & 1) * L::kTileK;
#pragma unroll
                for (int u = 0; u < L::kTileK / 16 / 128; ++u) {
                    const int at = stid + 128 * u, row = (at & 511) >> 3;
                    const uint4 v = *reinterpret_cast<const uint4*>(stage + L::kOffK + at * 16);
                    *reinterpret_cast<uint4*>(kt + at * 16) = row < n ? scale8(v, gb[64 + row]) : make_uint4(0u, 0u, 0u, 0u);
                }
                if (packed && n < kChunk) {  // rows of the next sequence meet zeros, but zero times its NaN is one
                    mbar_wait(&bar_v[s], sp, abort_flag);
                    for (int at = n * (DV / 8) + stid; at < kChunk * (DV / 8); at += 128)
                        *reinterpret_cast<uint4*>(stage + L::kOffV + (at % (DV / 64)) * 8192 + at / (DV / 64) * 16) = make_uint4(0u, 0u, 0u, 0u);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar_kt[gc & 1]);
                // ---- scores with their decay, row i = 16 lq + l/4 (+ 8), columns j
                float2 gj[8];
                const int i0 = 16 * lq + (lane >> 2);
                const float g0 = gb[i0], g1 = gb[i0 + 8];
                mbar_wait(&bar_score[gc & 1], (gc >> 1) & 1, abort_flag);
                tc_fence_after_sync();
                const uint32_t tP = tmem + kTmP + (static_cast<uint32_t>(32 * lq + ((gc & 1) ? 16 : 0)) << 16);
                const uint32_t sP = smem_u32(smem + L::kOffP + (gc & 1) * 8192);
#pragma unroll
                for (int h = 0; h < 2; ++h) {  // 32 columns
                    uint32_t r[16], w[8];
                    tmem_ld_frag32(tP + 32 * h, r);
#pragma unroll
                    for (int j = 0; j < 4; ++j) gj[j] = *reinterpret_cast<const float2*>(gb + 32 * h + 8 * j + 2 * (lane & 3));
                    tmem_wait_ld();
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int col = 32 * h + 8 * j + 2 * (lane & 3);
                        // (chosen, not multiplied by zero: what lies above the diagonal may be anything)
                        w[j] = pack_bf16(col <= i0 ? __uint_as_float(r[4 * j]) * ex2(g0 - gj[j].x) : 0.f,
                                         col + 1 <= i0 ? __uint_as_float(r[4 * j + 1]) * ex2(g0 - gj[j].y) : 0.f);
                        w[4 + j] = pack_bf16(col <= i0 + 8 ? __uint_as_float(r[4 * j + 2]) * ex2(g1 - gj[j].x) : 0.f,
                                             col + 1 <= i0 + 8 ? __uint_as_float(r[4 * j + 3]) * ex2(g1 - gj[j].y) : 0.f);
                    }
#pragma unroll
                    for (int a = 0; a < 2; ++a) {  // 8 rows; lane 8m + r: row r, columns 8 (4 h + m)
                        const int row = 16 * lq + 8 * a + (lane & 7);
                        stmatrix_x4(sP + row * 128 + (((4 * h + (lane >> 3)) ^ (row & 7)) << 4), w[4 * a], w[4 * a + 1], w[4 * a + 2], w[4 * a + 3]);
                    }
                }
                fence_proxy_async_smem();
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar_p[gc & 1]);
            }
        }
    } else {
        reg_dec<56>();
    }
    if (warp == 16) {
        // =============================================================== producer
        for (long long i = blockIdx.x; i < p.num_items; i += gridDim.x) {
            if (!walker.locate(p, i, it)) continue;
            const int khead = it.head / (p.vh / p.kh);
            for (int c = 0; c < it.chunks; ++c, ++gc) {
                const uint32_t s = gc % kStages;
                mbar_wait(&bar_empty[s], ((gc / kStages) + 1) & 1, abort_flag);
                uint8_t* st = smem + s * L::kStage;
                const int tok = static_cast<int>(it.tok0 + static_cast<long long>(c) * kChunk);
                mbar_arrive_expect_tx_w(&bar_qk[s], 2 * L::kTileK);
#pragma unroll
                for (int a = 0; a < DK / 64; ++a) {
                    tma_load_4d_w(st + L::kOffK + a * 8192, &tmK, &bar_qk[s], a * 64, khead, tok, it.batch);
                    tma_load_4d_w(st + L::kOffQ + a * 8192, &tmQ, &bar_qk[s], a * 64, khead, tok, it.batch);
                }
                mbar_arrive_expect_tx_w(&bar_v[s], L::kTileV);
#pragma unroll
                for (int a = 0; a < DV / 64; ++a) tma_load_4d_w(st + L::kOffV + a * 8192, &tmV, &bar_v[s], it.dvt * 128 + a * 64, it.head, tok, it.batch);
            }
        }
    } else if (warp == 17) {
        // =============================================================== MMA issuer
        constexpr uint32_t id_qk = make_idesc_bf16(64, 64, false, false);
        constexpr uint32_t id_d = make_idesc_bf16(128, DK, true, true);
        constexpr uint32_t id_sq = make_idesc_bf16(128, 64, false, false);
        constexpr uint32_t id_vp = make_idesc_bf16(128, 64, true, false);
        // dv rows 64 .. 127 of V^T: the second atom; where a head has none the first one again (those lanes are not looked at)
        constexpr uint32_t kLboV = DV == 128 ? 8192 : 0;
        const uint64_t dQ = make_smem_desc_sw128(smem_u32(smem + L::kOffQ), 0, 1024), dK = make_smem_desc_sw128(smem_u32(smem + L::kOffK), 0, 1024);
        const uint64_t dV = make_smem_desc_sw128(smem_u32(smem + L::kOffV), kLboV, 1024);
        const uint64_t dKT = make_smem_desc_sw128(smem_u32(smem + L::kOffKT), 8192, 1024), dP = make_smem_desc_sw128(smem_u32(smem + L::kOffP), 0, 1024);
        // Q K^T of chunk n, which the scores of the chunk wait for, goes out a chunk ahead
        auto issue_qk = [&](uint32_t n) {
            const uint32_t s = n % kStages;
            mbar_wait(&bar_qk[s], (n / kStages) & 1, abort_flag);
            tc_fence_after_sync();
            const uint32_t tP = tmem + kTmP + ((n & 1) ? (16u << 16) : 0u);
            const uint64_t q = desc_advance(dQ, s * L::kStage), k = desc_advance(dK, s * L::kStage);
            mma_ss_w<false>(tP, q, k, id_qk);
#pragma unroll
            for (int ks = 1; ks < DK / 16; ++ks) mma_ss_w<true>(tP, desc_advance(q, kmajor_step(ks, 8192)), desc_advance(k, kmajor_step(ks, 8192)), id_qk);
            mma_commit_w(&bar_score[n & 1]);
        };
        long long total = 0;  // chunks of this CTA
        for (long long i = blockIdx.x; i < p.num_items; i += gridDim.x)
            if (walker.locate(p, i, it)) total += it.chunks;
        if (total > 0) issue_qk(0);
        for (long long left = total; left > 0; --left, ++gc) {
            const uint32_t s = gc % kStages, b = gc & 1;
            // (the accumulator of chunk gc + 1 is that of gc - 1, whose scores have been written: its second product is issued)
            if (left > 1) issue_qk(gc + 1);
            const uint64_t v = desc_advance(dV, s * L::kStage), kt = desc_advance(dKT, b * L::kTileK), pp = desc_advance(dP, b * 8192), q = desc_advance(dQ, s * L::kStage);
            // D = V^T (decayed K)
            mbar_wait(&bar_v[s], (gc / kStages) & 1, abort_flag);
            mbar_wait(&bar_kt[b], (gc >> 1) & 1, abort_flag);
            if (gc > 0) mbar_wait(bar_dfree, (gc - 1) & 1, abort_flag);
            tc_fence_after_sync();
            mma_ss_w<false>(tmem + kTmD, v, kt, id_d);
#pragma unroll
            for (int ks = 1; ks < 4; ++ks) mma_ss_w<true>(tmem + kTmD, desc_advance(v, ks * 2048), desc_advance(kt, ks * 2048), id_d);
            mma_commit_w(bar_d);
            mma_commit_w(&bar_ktfree[b]);
            // S Q^T
            mbar_wait(bar_s, gc & 1, abort_flag);
            if (gc > 1) mbar_wait(&bar_ofree[b], ((gc >> 1) + 1) & 1, abort_flag);
            tc_fence_after_sync();
            if (DK == 128) mma_ts_k128_w<false>(tmem + kTmO1 + 64 * b, tmem + kTmS, q, id_sq);
            else mma_ts_k64_w<false, 2>(tmem + kTmO1 + 64 * b, tmem + kTmS, q, id_sq);
            mma_commit_w(&bar_sq);
            // V^T P^T
            mbar_wait(&bar_p[b], (gc >> 1) & 1, abort_flag);
            tc_fence_after_sync();
            mma_ss_w<false>(tmem + kTmO2 + 64 * b, v, pp, id_vp);
#pragma unroll
            for (int ks = 1; ks < 4; ++ks) mma_ss_w<true>(tmem + kTmO2 + 64 * b, desc_advance(v, ks * 2048), desc_advance(pp, ks * 32), id_vp);
            mma_commit_w(&bar_o[b]);
            mma_commit_w(&bar_empty[s]);
        }
    } else if (warp == 18) {
        // =============================================================== gates
        for (long long i = blockIdx.x; i < p.num_items; i += gridDim.x) {
            if (!walker.locate(p, i, it)) continue;
            auto load = [&](int c, uint32_t& a0, uint32_t& a1) {
                const long long t = static_cast<long long>(c) * kChunk + lane;
                a0 = p.gate.ptr && t < it.tokens ? p.gate.load_bits(it.batch, it.tok0 + t, it.head) : 0u;
                a1 = p.gate.ptr && t + 32 < it.tokens ? p.gate.load_bits(it.batch, it.tok0 + t + 32, it.head) : 0u;
            };
            uint32_t a0, a1;
            load(0, a0, a1);
            for (int c = 0; c < it.chunks; ++c, ++gc) {
                float g0 = lin_gate_log2(p.gate.value(a0)), g1 = lin_gate_log2(p.gate.value(a1));
                load(c + 1, a0, a1);
                scan64(g0, g1, lane);  // (tokens past the end have no decay: they carry the last one's sum)
                const float last = __shfl_sync(0xffffffffu, g1, 31);
                mbar_wait(&bar_gfree[gc & 3], ((gc >> 2) + 1) & 1, abort_flag);
                float* gb = gate_buf(gc);
                gb[lane] = g0;
                gb[lane + 32] = g1;
                gb[64 + lane] = ex2(last - g0);
                gb[96 + lane] = ex2(last - g1);
                gb[128 + lane] = p.scale * ex2(g0);
                gb[160 + lane] = p.scale * ex2(g1);
                if (lane == 0) gb[192] = ex2(last);
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar_gate[gc & 3]);
            }
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem, 512);
    if (tid == 0 && *abort_flag && p.status) atomicExch(p.status, 4);
}

}  // namespace gdn
