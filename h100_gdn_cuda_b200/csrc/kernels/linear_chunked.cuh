// Linear attention with decay over whole prompts, 64 tokens at a time.  With G the running sum of a chunk's log-decays and S the
// state that enters it (dv x dk),
//     O = scale * ( e^{G_i} Q S^T  +  (Q K^T .* e^{G_i - G_j}, j <= i) V )
//     S <- e^{G_L} S + (e^{G_L - G_j} V)^T K .
// The state's increment does not depend on the state, so all products of a chunk can be issued ahead of it.  Where no decay of the chunk is
// below 2^-120 it is a factor w_j = e^{-G_j} of the values alone,
//     O = scale e^{G_i} * ( Q S^T + (Q K^T w_j, j <= i) V ) ,   S <- e^{G_L} (S + (w_j V)^T K) ,
// so that the scores take one factor a column, have to be cut off above the diagonal, and both parts of O are one accumulation ("plain"
// chunks).  The factor e^{G_L} is not applied either but kept as an exponent c of the whole state, which joins the factors of the chunks that follow,
//     S = 2^c S' ,   w_j = e^{-G_j} 2^{-c} ,   O = scale e^{G_i} 2^c * ( ... ) ,
// until it leaves 2^-60 .. 2^60: S' is an accumulator in tensor memory that the increments are added to by the products themselves.  (That leaves
// 2^60 and more for the values in fp32.)  Other chunks form every decay as it stands in the first form, which cannot overflow: the scores take
// e^{G_i - G_j}, the rows of Q are scaled where they lie, the values of the increment take e^{G_L - G_j} and the state is scaled between its read
// and its increment.
// Roundings: scores, the copy of the state that Q meets, and Q where it is scaled are bf16, once each.  Values of the increment come in two parts, bf16
// and what that leaves, by a second product: with one part fp32 states are 2.3e-3 off and with two 5e-6, outputs with bf16 states 2.8e-3 and 2.35e-3
// (4 x 4096 tokens from DRAM 88 and 92 us, 2 x 131072 on 4 v-heads, back to back under the power cap, 256 and 285).  The tensor cores cut the state's sums off, eight a chunk: some 2e-9 of
// it for each token that a head remembers (131072 tokens without a decay 2.7e-4).
//
// A persistent CTA takes work items (sequence segment, v-head, 128 columns of dv) one after the other; its roles run over the same
// items and chunks, handing tiles on through mbarriers:
//   warps 0-7   state warps: a bf16 copy of the fp32 state for the products with Q (lane = dv row, half of the columns each); its scaling
//   warps 8-11  output warps: O scaled, transposed into Q's tile, stored
//   warps 12-15 score warps: the scores as bf16 tile
//   warps 16-19 value warps: V^T times its factors into tensor memory, for the increment
//   warp 20     producer: tensor copies of Q, K, V into a ring of stages
//   warp 21     issues the state's increment (w V)^T K, which the next chunk waits for, then the products of the output, S Q^T and V^T P^T
//   warp 22     issues the scores Q K^T
//   warp 23     finds the items; the gates' running sums and the factors made of them
// All products that feed output and state are transposed (128 dv rows = M): S and w V are A operands in tensor memory, V one in shared memory as it
// came; Q, K and the scores are B operands.
// What bounds it: HBM allows 2750 cycles a chunk at d = 128 on all SMs (2080 where two v-heads share Q and K), shared memory 1600 (208 KB of
// copies, operands and tiles), the tensor pipe 1150; a warp of each role needs 1000 to 1700 for its part, a few hundred instructions one behind the
// other.  None of that is the 2300 to 2550 that a chunk takes on 128 SMs: a chain alone on the GPU takes 2000, since S Q^T is issued behind the wait for
// the scores, these wait for the output before to be through with their one tile, and the state's next copy waits for S Q^T.
// 4 x 4096 tokens from DRAM: 91 us on 32 v-heads with 16 k-heads; the same copies in and out and nothing else take 69.  Where chunks forget by more than 2^-120, 116 to 125.
// The ring has four stages, and a fifth tile for Q and the output (three stages: 95 us where four took 92).
// The instruction cache counts: the waits are the short form, the item search is one warp's, the state's type is the kernel's (104 KB of code took 5200
// cycles a chunk with both SMs of a pair at work, 2900 with one).
#pragma once
#include <cuda.h>

#include "pairs.cuh"
#include "prefill_common.cuh"

namespace gdn {

struct LinChunkedParams {
    TokenView out;
    ScalarView gate;  // log-decay; ptr == NULL: none
    const void* state_in;
    void* state_out;
    long long si_ss, si_sh, so_ss, so_sh;
    const int* cu_seqlens;
    int total_tokens, num_seqs, seq_len, kh, vh, dk, dv, dv_tiles;
    int state_f32;
    float scale;
    int* status;
    // Work items.  Chains are (sequence, v-head, dv tile); a segment is `seg_chunks` chunks of one.
    //   padded: the first `whole` chains are an item each, every other one `num_segments` of them, one behind the other;
    //   packed: slots x vh x dv_tiles, where a sequence of c chunks has max(1, ceil(c / seg_chunks)) slots, numbered through the sequences
    //           (`by_length`: one each, in falling order of length).  num_items is an upper bound there.
    int whole, seg_chunks, num_segments, num_items, by_length;
    float* seg_state;  // per item behind `whole`: what the segment adds to the state (gdn_linear_segment_kernel), then the state behind it
    float* seg_decay;  // and its sum of log2-decays
    // state_out is state_in: a cut chain's last segment may write it before the first one has read it, which so finds it in the place of
    // the last one, where nothing is added (gdn_linear_combine_kernel puts it there)
    int in_place;
};

// Decays are handled as powers of two; anything below 2^-160 is zero in fp32, and sums of 64 such stay exact enough to tell G_i - G_j
// where a chunk forgets several times over (64 x 160 has a spacing of 2^-10, less than the scores' bf16).  A NaN stays one.
__device__ __forceinline__ float lin_gate_log2(float g) {
    const float x = g * 1.4426950408889634f;
    return x < -160.f ? -160.f : x;
}

struct alignas(16) LinItem {
    int seq, head, khead, dvt;
    int batch, segment, segments, mine;  // mine: the item's place among the segments' states (packed, padded behind `whole`)
    int before, tok0, tokens, chunks;    // before: where the state that enters the segment is, -1: state_in; tokens of the segment; chunks < 0: no more items
};

constexpr int kLinRankedSeqs = 32;  // packed sequences that are ordered by length, a lane each

// Finds items; warp-collective.
struct LinWalker {
    int base = 0;   // packed mode: first sequence of the 32 that were looked at last
    int first = 0;  // its first slot
    // false: a surplus item
    __device__ __forceinline__ bool locate(const LinChunkedParams& p, int it, LinItem& o) {
        int bos = 0, len = p.seq_len, chain = it;
        const int per = p.vh * p.dv_tiles;
        o.segment = 0;
        o.segments = 1;
        if (!p.cu_seqlens) {
            o.mine = it - p.whole;
            o.before = -1;
            if (o.mine >= 0) {
                const int r = o.mine / p.num_segments;
                chain = p.whole + r;
                o.segment = o.mine - r * p.num_segments;
                o.segments = p.num_segments;
                if (o.segment > 0) o.before = o.mine - 1;
                else if (p.in_place) o.before = o.mine + o.segments - 1;
            }
            o.seq = chain / per;
            o.batch = o.seq;
        } else {
            const int lane = threadIdx.x & 31, slot = it / per;
            o.batch = 0;
            o.mine = it;
            o.before = -1;
            auto offset = [&](int s) { return min(max(p.cu_seqlens[s], 0), p.total_tokens); };
            if (p.by_length) {
                if (slot >= p.num_seqs) return false;
                // order: more tokens first, of equally many the one in front first
                const int b = lane < p.num_seqs ? offset(lane) : 0, mine = lane < p.num_seqs ? max(offset(lane + 1) - b, 0) : -1;
                int rank = 0;
#pragma unroll 1
                for (int j = 0; j < p.num_seqs; ++j) {
                    const int other = __shfl_sync(0xffffffffu, mine, j);
                    rank += other > mine || (other == mine && j < lane);
                }
                o.seq = __ffs(__ballot_sync(0xffffffffu, lane < p.num_seqs && rank == slot)) - 1;
                bos = __shfl_sync(0xffffffffu, b, o.seq);
                len = __shfl_sync(0xffffffffu, mine, o.seq);
            } else {
                if (slot < first) base = first = 0;
#pragma unroll 1
                while (true) {
                    if (base >= p.num_seqs) return false;
                    const int s = base + lane;
                    int b = 0, e = 0, n = 0;
                    if (s < p.num_seqs) {
                        b = offset(s);
                        e = max(offset(s + 1), b);
                        n = max(1, ((e - b + kChunk - 1) / kChunk + p.seg_chunks - 1) / p.seg_chunks);
                    }
                    int incl = n;
#pragma unroll
                    for (int m = 1; m < 32; m <<= 1) {
                        const int y = __shfl_up_sync(0xffffffffu, incl, m);
                        if (lane >= m) incl += y;
                    }
                    const int total = __shfl_sync(0xffffffffu, incl, 31);
                    if (slot >= first + total) {
                        base += 32;
                        first += total;
                        continue;
                    }
                    const int mine = __ffs(__ballot_sync(0xffffffffu, slot < first + incl)) - 1;
                    o.seq = base + mine;
                    o.segments = __shfl_sync(0xffffffffu, n, mine);
                    o.segment = slot - first - (__shfl_sync(0xffffffffu, incl, mine) - o.segments);
                    bos = __shfl_sync(0xffffffffu, b, mine);
                    len = __shfl_sync(0xffffffffu, e, mine) - bos;
                    if (o.segment > 0) o.before = it - per;
                    else if (p.in_place && o.segments > 1 && slot + o.segments <= p.num_items / per) o.before = it + (o.segments - 1) * per;
                    break;
                }
            }
        }
        const int r = chain % per;
        o.head = r / p.dv_tiles;
        o.dvt = r - o.head * p.dv_tiles;
        o.khead = o.head / (p.vh / p.kh);
        if (o.segments > 1) {
            const int t0 = o.segment * p.seg_chunks * kChunk;
            bos += t0;
            len = min(len - t0, p.seg_chunks * kChunk);
        }
        o.tok0 = bos;
        o.tokens = len;
        o.chunks = (len + kChunk - 1) / kChunk;
        return true;
    }
};

template <int DK, int DV>
struct LinSmem {
    static constexpr int kStages = DK == 64 && DV == 64 ? 6 : 4, kStagesQ = kStages + 1;  // (the output is staged in Q's tile, which so lasts longer)
    static constexpr int kTileK = kChunk * DK * 2, kTileV = kChunk * DV * 2, kTileQ = kTileK > kTileV ? kTileK : kTileV;
    static constexpr int kOffV = kStages * kTileK;
    static constexpr int kOffQ = kOffV + kStages * kTileV;
    static constexpr int kOffP = kOffQ + kStagesQ * kTileQ;  // scores, 64 x 64
    // 4 x gate factors, fp32: of the scores [64]; of the output [64]; not plain: G[64] (log2), e^{G_i}[64]; of the state in front of its copy
    // and behind it; 2^c behind the chunk; plain or not; of the values [64] (see factor_pair).  Beside them, from the value warps: whether any of 32 columns
    // has a value that is not finite [4]; the first token of it in each column [128], a byte each
    static constexpr int kOffGate = kOffP + 8192;
    static constexpr int kGateOdd = 5 * 64 + 4, kGateStride = (kGateOdd + 4) * 4 + 128;
    static constexpr int kOffBar = kOffGate + 4 * kGateStride;
    static constexpr int kBytes = kOffBar + 640 + 1024;
};

namespace lin {
constexpr int kThreads = 768;  // 24 warps
constexpr uint32_t kTmS = 0;     // its bf16 copy, 64 columns
constexpr uint32_t kTmP = 64;    // fp32 Q K^T of even (lanes +0) and odd chunks (lanes +16), 64 columns
constexpr uint32_t kTmF = 128;   // fp32 state, 128 columns
constexpr uint32_t kTmO = 256;   // 2 x fp32 S Q^T + V^T P^T, 64 columns
constexpr uint32_t kTmV = 384;   // 2 x bf16 (w V)^T (not plain: (e^{G_L - G_j} V)^T), 32 columns
constexpr uint32_t kTmVlo = 448; // 2 x bf16: what is left of it
constexpr float kPlainLog2 = 60.f;
__device__ __forceinline__ void named_bar_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
using namespace pairs;
// the running sums of 64 log2-decays, lane l: tokens 2l and 2l + 1
__device__ __forceinline__ void scan64(float& g0, float& g1, int lane) {
    float sum = g0 + g1;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        const float y = __shfl_up_sync(0xffffffffu, sum, m);
        if (lane >= m) sum += y;
    }
    sum = __shfl_up_sync(0xffffffffu, sum, 1);
    if (lane > 0) g0 += sum;
    g1 += g0;
}
// The same for what lies behind each token; returns the sum of all 64.  A difference of two sums from the front has the spacing of the larger one, 2^-10
// where a chunk forgets 64 times over; these are off by half steps of their own size, and count where they are small.
__device__ __forceinline__ float scan64_behind(float& g0, float& g1, int lane) {
    float sum = g0 + g1;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        const float y = __shfl_down_sync(0xffffffffu, sum, m);
        if (lane + m < 32) sum += y;
    }
    const float all = __shfl_sync(0xffffffffu, sum, 0), behind = __shfl_down_sync(0xffffffffu, sum, 1);
    g0 = lane < 31 ? behind + g1 : g1;
    g1 = lane < 31 ? behind : 0.f;
    return all;
}
// x += y for a sum of many terms, kept as two numbers: x, and what it leaves of the exact sum (`rest`, which enters with y).  With one number
// the rounding of a sum that wanders up to 60 has the same sign chunk after chunk where a head's decay is slow: a state alone, decayed over
// 131072 tokens at g = -1e-4, was 2.5e-4 off, at -3e-4 5.3e-4; with two 8e-7 and 1.3e-7.
__device__ __forceinline__ void add_kept(float& x, float& rest, float y) {
    y += rest;
    const float sum = x + y, part = sum - x;
    rest = (x - (sum - part)) + (y - part);
    x = sum;
}
// 16 bytes of K times a factor (rounded to bf16 once, as an operand)
__device__ __forceinline__ uint4 scale8(uint4 v, float f) {
    using namespace ptx;
    const f2 w = pk(f, f);
    v.x = pack2(mul2(pk(bf16_lo(v.x), bf16_hi(v.x)), w));
    v.y = pack2(mul2(pk(bf16_lo(v.y), bf16_hi(v.y)), w));
    v.z = pack2(mul2(pk(bf16_lo(v.z), bf16_hi(v.z)), w));
    v.w = pack2(mul2(pk(bf16_lo(v.w), bf16_hi(v.w)), w));
    return v;
}
// Factors of values as two bf16 numbers each, which is 2^-16 of them; those of tokens 2t and 2t + 1, a pair each.
__device__ __forceinline__ uint2 factor_pair(float f0, float f1) {
    using namespace ptx;
    const uint32_t head = pack2(pk(f0, f1));
    return make_uint2(head, pack2(pk(f0 - bf16_lo(head), f1 - bf16_hi(head))));
}
// A pair of values times its factors in two parts: v, rounded to bf16, and what that leaves, to 2^-16 of it (v times a factor's head is exact in the
// difference).
__device__ __forceinline__ void times_factors(uint32_t& v, uint32_t& rest, uint2 f) {
    const __nv_bfloat162 x = *reinterpret_cast<const __nv_bfloat162*>(&v), head = *reinterpret_cast<const __nv_bfloat162*>(&f.x), tail = *reinterpret_cast<const __nv_bfloat162*>(&f.y);
    const __nv_bfloat162 y = __hmul2_rn(x, head), r = __hfma2(x, tail, __hfma2(x, head, __hneg2(y)));
    v = *reinterpret_cast<const uint32_t*>(&y);
    rest = *reinterpret_cast<const uint32_t*>(&r);
}
}  // namespace lin

// kWhole: head dims are multiples of 64, so that one copy fetches all columns of a tile (maps of rank 5: 64 columns, tokens, column blocks, heads,
// batch); otherwise every 64 columns are a copy of their own, which leaves out the columns that the next head begins with.
template <int DK, int DV, bool kWhole, bool kF32>
__global__ void __launch_bounds__(lin::kThreads, 1)
    gdn_linear_chunked_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                              const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmO, const LinChunkedParams p) {
    using namespace ptx;
    using namespace lin;
    using L = LinSmem<DK, DV>;
    constexpr int kStages = L::kStages, kStagesQ = L::kStagesQ;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (ptx::smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kOffBar);
    // No barrier may run two phases ahead of somebody who waits on it: each one's next phase but one needs what its waiters do after
    // theirs.  Barriers of two are those of even and of odd chunks.
    uint64_t* bar_full = bars;                    // [stages] Q, K, V of a chunk have arrived
    uint64_t* bar_empty = bar_full + kStages;     // [stages] the products of the stage's chunk are done
    uint64_t* bar_qempty = bar_empty + kStages;   // [Q's stages] the output that was staged there has been read
    uint64_t* bar_gate = bar_qempty + kStagesQ;  // [4] gate factors of a chunk
    uint64_t* bar_gfree = bar_gate + 4;         // [4] read by state and output warps
    uint64_t* bar_score = bar_gfree + 4;        // [2] Q K^T done
    uint64_t* bar_p = bar_score + 2;            // [2] scores written (and Q scaled)
    uint64_t* bar_dgo = bar_p + 2;              // [2] values written and the state copied
    uint64_t* bar_ofree = bar_dgo + 2;          // [2] O read
    uint64_t* bar_s = bar_ofree + 2;            // [2] the copy of the state read
    uint64_t* bar_o = bar_s + 2;                // [2] O done
    uint64_t* bar_d = bar_o + 2;                // [2] increment added
    uint64_t* bar_item = bar_d + 2;             // [2] an item is there
    uint64_t* bar_itemfree = bar_item + 2;      // [2] and every warp has it
    uint64_t* bar_next = bar_itemfree + 2;      // the answer to a request for another item is there
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_next + 1);
    int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
    LinItem* items = reinterpret_cast<LinItem*>(smem + L::kOffBar + 640 - 2 * sizeof(LinItem));
    uint8_t* next = smem + L::kOffBar + 640 - 2 * sizeof(LinItem) - 16;  // the answer
    static_assert((2 * kStages + kStagesQ + 27) * 8 + 8 + 16 + 2 * sizeof(LinItem) <= 640, "room for the barriers");
    static_assert(L::kBytes <= 232448, "room in shared memory");

    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    if (tid == 0) {
        *abort_flag = 0;
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&bar_full[i], 1);
            mbar_init(&bar_empty[i], 1);
        }
        for (int i = 0; i < kStagesQ; ++i) mbar_init(&bar_qempty[i], 1);
        for (int i = 0; i < 4; ++i) {
            mbar_init(&bar_gate[i], 1);
            mbar_init(&bar_gfree[i], 12);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar_score[i], 1);
            mbar_init(&bar_p[i], 4);
            mbar_init(&bar_ofree[i], 4);
            mbar_init(&bar_s[i], 1);
            mbar_init(&bar_dgo[i], 12);
            mbar_init(&bar_o[i], 1);
            mbar_init(&bar_d[i], 1);
            mbar_init(&bar_item[i], 1);
            mbar_init(&bar_itemfree[i], 23);
        }
        mbar_init(bar_next, 1);
        mbar_fence_init();
    }
    // the scores' blocks above the diagonal stay zero: nobody writes them
    for (int i = tid; i < 8192 / 16; i += kThreads) *reinterpret_cast<uint4*>(smem + L::kOffP + 16 * i) = make_uint4(0u, 0u, 0u, 0u);
    if (warp == 0) tmem_alloc(tmem_slot, 512);
    fence_proxy_async_smem();
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    if (warp == 20 && lane < 4) prefetch_tmap(lane == 0 ? &tmQ : lane == 1 ? &tmK : lane == 2 ? &tmV : &tmO);
    grid_dep_wait();
    grid_dep_launch();

    auto gate_buf = [&](uint32_t gc) { return reinterpret_cast<float*>(smem + L::kOffGate + (gc & 3) * L::kGateStride); };
    LinItem it;
    uint32_t gc = 0, taken = 0;  // chunks and items so far, the same counts in every role
    auto next_item = [&]() {
        const uint32_t s = taken & 1;
        mbar_wait_short(&bar_item[s], (taken >> 1) & 1, abort_flag);
        it = items[s];
        ++taken;
        // (the count by way of a shuffle, so that the compiler knows it to be the same in all lanes: loop counters, addresses and descriptors
        // made of it then live in uniform registers)
        it.chunks = __shfl_sync(0xffffffffu, *static_cast<volatile int*>(abort_flag) == 0 ? it.chunks : -1, 0);
        if (lane == 0) mbar_arrive(&bar_itemfree[s]);
        return it.chunks >= 0;
    };
    if (warp < 8) {
        // =============================================================== state warps
        const int lq = warp & 3, hf = warp >> 2;
        constexpr int kCols = DK / 2;  // of a thread
        const int c0 = kCols * hf;
        const uint32_t tm_lane = static_cast<uint32_t>(32 * lq) << 16;
        const uint32_t tF = tmem + kTmF + tm_lane + c0, tS = tmem + kTmS + tm_lane + c0 / 2;
        while (next_item()) {
            const int row = it.dvt * 128 + 32 * lq + lane;
            const bool row_in = 32 * lq + lane < DV && row < p.dv;
            // ---- the state that enters the segment (the increments of the item before have been read at its end)
#pragma unroll 2
            for (int q = 0; q < kCols; q += 16) {
                uint32_t r[16];
                const int cols = row_in ? p.dk - c0 - q : 0;  // columns that are there from this one on
                if (it.before >= 0) {
                    const uint4* src = reinterpret_cast<const uint4*>(p.seg_state + static_cast<long long>(it.before) * (128 * DK) + (32 * lq + lane) * DK + c0 + q);
#pragma unroll
                    for (int e = 0; e < 4; ++e) *reinterpret_cast<uint4*>(r + 4 * e) = __ldcg(src + e);
                } else if (kF32) {
                    const uint4* src = reinterpret_cast<const uint4*>(static_cast<const float*>(p.state_in) + it.seq * p.si_ss + it.head * p.si_sh + static_cast<long long>(row) * p.dk + c0 + q);
#pragma unroll
                    for (int e = 0; e < 4; ++e) *reinterpret_cast<uint4*>(r + 4 * e) = p.state_in && 4 * e < cols ? src[e] : make_uint4(0u, 0u, 0u, 0u);
                } else {
                    const uint4* src = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.state_in) + it.seq * p.si_ss + it.head * p.si_sh + static_cast<long long>(row) * p.dk + c0 + q);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const uint4 v = p.state_in && 8 * e < cols ? src[e] : make_uint4(0u, 0u, 0u, 0u);
                        r[8 * e] = v.x << 16; r[8 * e + 1] = v.x & 0xFFFF0000u;
                        r[8 * e + 2] = v.y << 16; r[8 * e + 3] = v.y & 0xFFFF0000u;
                        r[8 * e + 4] = v.z << 16; r[8 * e + 5] = v.z & 0xFFFF0000u;
                        r[8 * e + 6] = v.w << 16; r[8 * e + 7] = v.w & 0xFFFF0000u;
                    }
                }
                tmem_st16(tF + q, r);
            }
            tmem_wait_st();
            float pow_c = 1.f;  // 2^c
#pragma unroll 1
            for (int c = 0; c < it.chunks; ++c, ++gc) {
                mbar_wait_short(&bar_gate[gc & 3], (gc >> 2) & 1, abort_flag);
                const float before = gate_buf(gc)[256], behind = gate_buf(gc)[257];
                pow_c = gate_buf(gc)[258];
                const bool scaled = before != 1.f || behind != 1.f;  // (a NaN is)
                const f2 before2 = pk(before, before), behind2 = pk(behind, behind);
                if (gc > 0) mbar_wait_short(&bar_d[(gc - 1) & 1], ((gc - 1) >> 1) & 1, abort_flag);
                tc_fence_after_sync();
                uint32_t w[kCols / 2];  // (rounded to bf16 as an operand: the state itself stays in fp32)
#pragma unroll
                for (int q = 0; q < kCols; q += 32) {
                    uint32_t r[32];
                    tmem_ld32(tF + q, r);
                    tmem_wait_ld();
                    if (__builtin_expect(scaled, 0)) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            float x, y;
                            const f2 v = mul2(pk(r[2 * e], r[2 * e + 1]), before2);
                            w[q / 2 + e] = pack2(v);
                            unpk(mul2(v, behind2), x, y);
                            r[2 * e] = __float_as_uint(x);
                            r[2 * e + 1] = __float_as_uint(y);
                        }
                        tmem_st16(tF + q, r);
                        tmem_st16(tF + q + 16, r + 16);
                    } else {
#pragma unroll
                        for (int e = 0; e < 16; ++e) w[q / 2 + e] = pack2(pk(r[2 * e], r[2 * e + 1]));
                    }
                }
                if (gc > 0) mbar_wait_short(&bar_s[(gc - 1) & 1], ((gc - 1) >> 1) & 1, abort_flag);  // the copy before has been read
                tc_fence_after_sync();
#pragma unroll
                for (int q = 0; q < kCols / 2; q += 16) tmem_st16(tS + q, w + q);
                tmem_wait_st();
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&bar_dgo[gc & 1]);
                    mbar_arrive(&bar_gfree[gc & 3]);
                }
            }
            // ---- the state behind the sequence
            if (it.chunks > 0) mbar_wait_short(&bar_d[(gc - 1) & 1], ((gc - 1) >> 1) & 1, abort_flag);
            tc_fence_after_sync();
            if (it.segment == it.segments - 1 && p.state_out && *static_cast<volatile int*>(abort_flag) == 0) {
                const long long at = it.seq * p.so_ss + it.head * p.so_sh + static_cast<long long>(row) * p.dk + c0;
#pragma unroll 1
                for (int q = 0; q < kCols; q += 16) {
                    uint32_t r[16];
                    tmem_ld16(tF + q, r);
                    tmem_wait_ld();
                    const int cols = row_in ? p.dk - c0 - q : 0;
#pragma unroll
                    for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * pow_c);
                    if (kF32) {
                        uint4* dst = reinterpret_cast<uint4*>(static_cast<float*>(p.state_out) + at + q);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (4 * e < cols) dst[e] = *reinterpret_cast<const uint4*>(r + 4 * e);
                    } else {
                        uint4* dst = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.state_out) + at + q);
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            if (8 * e < cols)
                                dst[e] = make_uint4(pack2(pk(r[8 * e], r[8 * e + 1])), pack2(pk(r[8 * e + 2], r[8 * e + 3])),
                                                    pack2(pk(r[8 * e + 4], r[8 * e + 5])), pack2(pk(r[8 * e + 6], r[8 * e + 7])));
                    }
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
        while (next_item()) {
#pragma unroll 1
            for (int c = 0; c < it.chunks; ++c, ++gc) {
                const int n = min(it.tokens - c * kChunk, kChunk);
                const float* gb = gate_buf(gc) + 64;
                uint8_t* const sO = smem + L::kOffQ + gc % kStagesQ * L::kTileQ;
                const uint32_t sOa = smem_u32(sO), tO = tmem + kTmO + 64 * (gc & 1) + tm_lane;
                mbar_wait_short(&bar_gate[gc & 3], (gc >> 2) & 1, abort_flag);
                mbar_wait_short(&bar_o[gc & 1], (gc >> 1) & 1, abort_flag);
                tc_fence_after_sync();
                const bool odd = (DV == 128 || lq < 2) && gate_buf(gc)[L::kGateOdd + lq] != 0.f;
#pragma unroll 1
                for (int i = 0; i < 4; ++i) {  // 16 rows, 32 tokens
                    const int h = i & 1, b = i >> 1;
                    uint32_t r[16], w[8];
                    tmem_ld_frag32(tO + (static_cast<uint32_t>(16 * h) << 16) + 32 * b, r);
                    f2 gv[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) gv[j] = *reinterpret_cast<const f2*>(gb + 32 * b + 8 * j + 2 * (lane & 3));
                    tmem_wait_ld();
#pragma unroll
                    for (int j = 0; j < 8; ++j) w[j] = pack2(mul2(gv[j >> 1], pk(r[2 * j], r[2 * j + 1])));
                    if (__builtin_expect(odd, 0)) {  // NaN from the first token on whose value is not finite
                        const uint8_t* const first = reinterpret_cast<const uint8_t*>(gate_buf(gc) + L::kGateOdd + 4) + 32 * lq + 16 * h + (lane >> 2);
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const int t = 32 * b + 8 * (j >> 1) + 2 * (lane & 3), f = first[8 * (j & 1)];
                            w[j] |= (t >= f ? 0x7FFFu : 0u) | (t + 1 >= f ? 0x7FFF0000u : 0u);
                        }
                    }
                    if (DV == 128 || lq < 2) {
                        const uint32_t so = sOa + (h ? osw1 : osw0) + 4096 * b;
                        stmatrix_x4_trans(so, w[0], w[1], w[2], w[3]);
                        stmatrix_x4_trans(so + 2048, w[4], w[5], w[6], w[7]);
                    }
                }
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&bar_ofree[gc & 1]);
                    mbar_arrive(&bar_gfree[gc & 3]);
                }
                fence_proxy_async_smem();
                named_bar_sync(1, 128);
                const int tok0 = it.tok0 + c * kChunk;
                const int left = p.dv - it.dvt * 128;  // columns from this tile on
                if (__builtin_expect(*static_cast<volatile int*>(abort_flag) != 0, 0)) {
                    // a wait has given up: the tile is garbage and stays on chip
                } else if (__builtin_expect(!packed || n == kChunk, 1)) {
                    if (otid == 0) {
#pragma unroll
                        for (int a = 0; a < DV / 64; ++a)  // columns past dv and tokens past the end are clipped
                            if (64 * a < left) tma_store_4d(&tmO, sO + 8192 * a, it.dvt * 128 + 64 * a, it.head, tok0, it.batch);
                    }
                } else {  // a whole box would reach into the next sequence
                    __nv_bfloat16* base = p.out.ptr + it.batch * p.out.sb + tok0 * p.out.st + static_cast<long long>(it.head) * p.out.sh + it.dvt * 128;
                    const int pieces = min(left, DV) >> 3;
#pragma unroll 1
                    for (int idx = otid; idx < n * 16; idx += 128) {
                        const int row = idx >> 4, c16 = idx & 15;
                        if (c16 < pieces) *reinterpret_cast<uint4*>(base + row * p.out.st + c16 * 8) = *reinterpret_cast<const uint4*>(sO + tile_off(row, c16));
                    }
                }
                if (otid == 0) {
                    bulk_commit();
                    if (gc > 0) {
                        bulk_wait_read<1>();  // the tile of the chunk before has been read
                        mbar_arrive(&bar_qempty[(gc - 1) % kStagesQ]);
                    }
                }
            }
        }
        if (otid == 0) bulk_wait_read<0>();
    } else if (warp < 16) {
        // =============================================================== score warps
        // Rows i = 16 lq + l/4 and + 8; columns up to the diagonal blocks, 32 at a time.
        const int lq = warp & 3, stid = tid - 384;
        const int i0 = 16 * lq + (lane >> 2);
        // the columns 2 (l%4), + 1 of an 8 x 8 block on the diagonal that row l/4 keeps (cut off as bits: what lies above may be anything)
        const uint32_t keep = (2 * (lane & 3) <= (lane >> 2) ? 0xFFFFu : 0u) | (2 * (lane & 3) + 1 <= (lane >> 2) ? 0xFFFF0000u : 0u);
        while (next_item()) {
#pragma unroll 1
            for (int c = 0; c < it.chunks; ++c, ++gc) {
                const float* gb = gate_buf(gc);
                mbar_wait_short(&bar_gate[gc & 3], (gc >> 2) & 1, abort_flag);
                const bool plain = gb[259] != 0.f;
                mbar_wait_short(&bar_score[gc & 1], (gc >> 1) & 1, abort_flag);
                tc_fence_after_sync();
                const uint32_t tP = tmem + kTmP + (static_cast<uint32_t>(32 * lq + ((gc & 1) ? 16 : 0)) << 16);
                const uint32_t sP = smem_u32(smem + L::kOffP) + (16 * lq + (lane & 7)) * 128;
#pragma unroll 1
                for (int h = 0; h <= lq >> 1; ++h) {
                    uint32_t r[16], w[8];
                    tmem_ld_frag32(tP + 32 * h, r);
                    tmem_wait_ld();
                    if (__builtin_expect(plain, 1)) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {  // (rounded to bf16 as an operand)
                            const f2 f = *reinterpret_cast<const f2*>(gb + 32 * h + 8 * j + 2 * (lane & 3));
                            w[j] = pack2(mul2(pk(r[4 * j], r[4 * j + 1]), f));
                            w[4 + j] = pack2(mul2(pk(r[4 * j + 2], r[4 * j + 3]), f));
                        }
                    } else {
                        const float g0 = gb[128 + i0], g1 = gb[128 + i0 + 8];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float2 gj = *reinterpret_cast<const float2*>(gb + 128 + 32 * h + 8 * j + 2 * (lane & 3));
                            w[j] = pack2(pk(__uint_as_float(r[4 * j]) * ex2(g0 - gj.x), __uint_as_float(r[4 * j + 1]) * ex2(g0 - gj.y)));
                            w[4 + j] = pack2(pk(__uint_as_float(r[4 * j + 2]) * ex2(g1 - gj.x), __uint_as_float(r[4 * j + 3]) * ex2(g1 - gj.y)));
                        }
                    }
                    if (h == lq >> 1) {  // the diagonal blocks and what is above them
                        if (lq & 1) {
                            w[2] &= keep;
                            w[3] = 0u;
                            w[7] &= keep;
                        } else {
                            w[0] &= keep;
                            w[5] &= keep;
                            w[1] = w[2] = w[3] = w[6] = w[7] = 0u;
                        }
                    }
                    if (h == 0 && gc > 0) mbar_wait_short(&bar_o[(gc - 1) & 1], ((gc - 1) >> 1) & 1, abort_flag);  // the chunk before is through with the tile
                    const uint32_t to = sP + (((4 * h + (lane >> 3)) ^ (lane & 7)) << 4);  // lane 8m + r: row r (of 8), columns 8 (4 h + m)
                    stmatrix_x4(to, w[0], w[1], w[2], w[3]);
                    stmatrix_x4(to + 1024, w[4], w[5], w[6], w[7]);
                }
                if (__builtin_expect(!plain, 0)) {  // Q, which Q K^T has been through with, takes its decay where it lies
                    mbar_wait_short(&bar_full[gc % kStages], (gc / kStages) & 1, abort_flag);
                    uint8_t* q = smem + L::kOffQ + gc % kStagesQ * L::kTileQ;
#pragma unroll 1
                    for (int at = stid; at < L::kTileK / 16; at += 128)
                        *reinterpret_cast<uint4*>(q + at * 16) = scale8(*reinterpret_cast<const uint4*>(q + at * 16), gb[192 + ((at & 511) >> 3)]);
                }
                fence_proxy_async_smem();
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar_p[gc & 1]);
            }
        }
    } else if (warp < 20) {
        // =============================================================== value warps
        // V^T comes by transposing matrix loads: lane 8m + r addresses token r of block m (8 rows x 8 tokens), block m = rows 8 (m & 1) ..
        // of 16, tokens 8 (m >> 1) .. of 16.
        const int lq = warp & 3, vtid = tid - 512;
        const uint32_t tm_lane = static_cast<uint32_t>(32 * lq) << 16;
        const uint32_t vlane = static_cast<uint32_t>((lq >> 1) * 8192 + (8 * (lane >> 4) + (lane & 7)) * 128);
        const uint32_t vchunk = static_cast<uint32_t>(4 * (lq & 1) + ((lane >> 3) & 1));  // 16-byte piece of the first 16 rows
        const uint32_t vsw0 = vlane + ((vchunk ^ (lane & 7)) << 4), vsw1 = vlane + (((vchunk + 2) ^ (lane & 7)) << 4);
        const bool packed = p.cu_seqlens != nullptr;
        while (next_item()) {
#pragma unroll 1
            for (int c = 0; c < it.chunks; ++c, ++gc) {
                const int n = min(it.tokens - c * kChunk, kChunk);
                const uint32_t s = gc % kStages;
                uint8_t *tk = smem + s * L::kTileK, *tv = smem + L::kOffV + s * L::kTileV;
                const float* const gb = gate_buf(gc);
                mbar_wait_short(&bar_gate[gc & 3], (gc >> 2) & 1, abort_flag);
                if (gc > 1) mbar_wait_short(&bar_d[gc & 1], ((gc >> 1) + 1) & 1, abort_flag);  // the values of two chunks before have been read
                mbar_wait_short(&bar_full[s], (gc / kStages) & 1, abort_flag);
                tc_fence_after_sync();
                const uint32_t sV = smem_u32(tv);
                // What rounding leaves of a value that is not finite is a NaN, and so are sums of products with it (others only where they overflow, which
                // a look at the values tells apart).
                __nv_bfloat162 nan[2];
                nan[0] = nan[1] = __float2bfloat162_rn(0.f);
                if (DV == 128 || lq < 2) {
#pragma unroll 1
                    for (int hf = 0; hf < 2; ++hf) {  // 32 tokens
                        const int t0 = 32 * hf + 2 * (lane & 3);  // first token of this lane's first pair; the others are 8 further on each
                        uint32_t v[2][2][4];  // [16 rows][16 tokens][block]
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            ldmatrix_x4_trans(sV + vsw0 + 4096 * hf + 2048 * j, v[0][j]);
                            ldmatrix_x4_trans(sV + vsw1 + 4096 * hf + 2048 * j, v[1][j]);
                        }
                        if (__builtin_expect(n < kChunk, 0)) {  // tokens past the end (of the next sequence, maybe)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const uint32_t keep = (t0 + 8 * i < n ? 0xFFFFu : 0u) | (t0 + 8 * i + 1 < n ? 0xFFFF0000u : 0u);
#pragma unroll
                                for (int a = 0; a < 2; ++a) {
                                    v[0][i >> 1][2 * (i & 1) + a] &= keep;
                                    v[1][i >> 1][2 * (i & 1) + a] &= keep;
                                }
                            }
                        }
                        const uint32_t to = tmem + tm_lane + 32 * (gc & 1) + 16 * hf;
                        const uint2* const fv = reinterpret_cast<const uint2*>(gb + 260) + t0 / 2;
                        uint32_t u[2][2][4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint2 f = fv[4 * i];
#pragma unroll
                            for (int a = 0; a < 2; ++a) {
                                times_factors(v[0][i >> 1][2 * (i & 1) + a], u[0][i >> 1][2 * (i & 1) + a], f);
                                times_factors(v[1][i >> 1][2 * (i & 1) + a], u[1][i >> 1][2 * (i & 1) + a], f);
                                nan[a] = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&u[0][i >> 1][2 * (i & 1) + a]),
                                                 *reinterpret_cast<const __nv_bfloat162*>(&u[1][i >> 1][2 * (i & 1) + a]), nan[a]);
                            }
                        }
                        tmem_st_frag16(to + kTmVlo, u[0][0]);
                        tmem_st_frag16(to + kTmVlo + (16u << 16), u[1][0]);
                        tmem_st_frag16(to + kTmV, v[0][0]);
                        tmem_st_frag16(to + kTmV + (16u << 16), v[1][0]);
                    }
                }
                nan[0] = __hadd2(nan[0], nan[1]);
                if (__builtin_expect(__any_sync(0xffffffffu, !__hbeq2(nan[0], nan[0])), 0)) {
                    // The state takes such values as they are.  For the output a zero score would still make a NaN of them in the tokens in front: they are
                    // taken out, and the output warps write NaN from the first one on.  (A lane has a column.)
                    uint8_t* const at = tv + (lq >> 1) * 8192 + (lane & 7) * 2;
                    int first = kChunk;
#pragma unroll 1
                    for (int t = n - 1; t >= 0; --t) {
                        unsigned short* const x = reinterpret_cast<unsigned short*>(at + t * 128 + (((4 * (lq & 1) + (lane >> 3)) ^ (t & 7)) << 4));
                        if ((*x & 0x7F80) == 0x7F80) {
                            first = t;
                            *x = 0;
                        }
                    }
                    reinterpret_cast<uint8_t*>(gate_buf(gc) + L::kGateOdd + 4)[32 * lq + lane] = static_cast<uint8_t>(first);
                    if (lane == 0) gate_buf(gc)[L::kGateOdd + lq] = 1.f;
                    fence_proxy_async_smem();
                }
                if (__builtin_expect(packed && n < kChunk, 0)) {  // zero scores and values meet what the next sequence has there, but zero times its NaN is one
#pragma unroll 1
                    for (int at = n * (DK / 8) + vtid; at < kChunk * (DK / 8); at += 128)
                        *reinterpret_cast<uint4*>(tk + (at % (DK / 64)) * 8192 + at / (DK / 64) * 16) = make_uint4(0u, 0u, 0u, 0u);
                    __syncwarp();
                    if (DV == 128 || lq < 2) {  // the columns of V that this warp has read itself
#pragma unroll 1
                        for (int at = n * 4 + lane; at < kChunk * 4; at += 32)
                            *reinterpret_cast<uint4*>(tv + (lq >> 1) * 8192 + (at >> 2) * 128 + (((4 * (lq & 1) + (at & 3)) ^ ((at >> 2) & 7)) << 4)) =
                                make_uint4(0u, 0u, 0u, 0u);
                    }
                    fence_proxy_async_smem();
                }
                tmem_wait_st();
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar_dgo[gc & 1]);
            }
        }
    } else if (warp == 20) {
        // =============================================================== producer
        // (A stage's loads are issued two chunks before their use.  Asking L2 for chunks further ahead costs more than it brings: 4 x 4096 tokens 89
        // -> 99 us, 148 heads of 4096 111 -> 164, from DRAM.)
        while (next_item()) {
            const int khead = __shfl_sync(0xffffffffu, it.khead, 0), head = __shfl_sync(0xffffffffu, it.head, 0), batch = __shfl_sync(0xffffffffu, it.batch, 0);
            const int tok0 = __shfl_sync(0xffffffffu, it.tok0, 0), dvt = __shfl_sync(0xffffffffu, it.dvt, 0);
#pragma unroll 1
            for (int c = 0; c < it.chunks; ++c, ++gc) {
                const uint32_t s = gc % kStages, sq = gc % kStagesQ;
                uint8_t *tk = smem + s * L::kTileK, *tq = smem + L::kOffQ + sq * L::kTileQ, *tv = smem + L::kOffV + s * L::kTileV;
                const int tok = tok0 + c * kChunk;
                mbar_wait_short(&bar_empty[s], ((gc / kStages) + 1) & 1, abort_flag);
                mbar_wait_short(&bar_qempty[sq], ((gc / kStagesQ) + 1) & 1, abort_flag);
                if (elect_one()) {
                    mbar_arrive_expect_tx(&bar_full[s], 2 * L::kTileK + L::kTileV);
                    if (kWhole) {
                        tma_load_5d(tk, &tmK, &bar_full[s], 0, tok, 0, khead, batch);
                        tma_load_5d(tq, &tmQ, &bar_full[s], 0, tok, 0, khead, batch);
                        tma_load_5d(tv, &tmV, &bar_full[s], 0, tok, 2 * dvt, head, batch);
                    } else {
#pragma unroll 1
                        for (int a = 0; a < DK / 64; ++a) {
                            tma_load_4d(tk + a * 8192, &tmK, &bar_full[s], a * 64, khead, tok, batch);
                            tma_load_4d(tq + a * 8192, &tmQ, &bar_full[s], a * 64, khead, tok, batch);
                        }
#pragma unroll 1
                        for (int a = 0; a < DV / 64; ++a) tma_load_4d(tv + a * 8192, &tmV, &bar_full[s], dvt * 128 + a * 64, head, tok, batch);
                    }
                }
                __syncwarp();
            }
        }
        if (*static_cast<volatile int*>(abort_flag) != 0) {  // a wait has given up: the copies in flight land before the CTA goes
            for (uint32_t n = gc > kStages ? gc - kStages : 0; n < gc; ++n) {
                int none = 0;
                mbar_wait_limit(&bar_full[n % kStages], (n / kStages) & 1, &none, 1ll << 28);
            }
        }
    } else if (warp == 21) {
        // =============================================================== products of state and output
        constexpr uint32_t id_d = make_idesc_bf16(128, DK, false, true), id_o = make_idesc_bf16(128, 64, false, false), id_v = make_idesc_bf16(128, 64, true, false);
        // read MN-major (DV == 64: rows 64 on are what follows V's tile, and reach rows of O that nobody looks at)
        const uint64_t dK = make_smem_desc_sw128(smem_u32(smem), 8192, 1024), dV = make_smem_desc_sw128(smem_u32(smem + L::kOffV), 8192, 1024);
        const uint64_t dQ = make_smem_desc_sw128(smem_u32(smem + L::kOffQ), 0, 1024), dP = make_smem_desc_sw128(smem_u32(smem + L::kOffP), 0, 1024);
        while (next_item()) {
#pragma unroll 1
            for (int c = 0; c < it.chunks; ++c, ++gc) {
                const uint32_t s = gc % kStages, b = gc & 1;
                mbar_wait_short(&bar_full[s], (gc / kStages) & 1, abort_flag);
                mbar_wait_short(&bar_dgo[b], (gc >> 1) & 1, abort_flag);
                tc_fence_after_sync();
                const uint64_t k = desc_advance(dK, s * L::kTileK), q = desc_advance(dQ, gc % kStagesQ * L::kTileQ);
                mma_ts_k64_w<true, 128>(tmem + kTmF, tmem + kTmV + 32 * b, k, id_d);
                mma_ts_k64_w<true, 128>(tmem + kTmF, tmem + kTmVlo + 32 * b, k, id_d);
                mma_commit_w(&bar_d[b]);
                if (gc > 1) mbar_wait_short(&bar_ofree[b], ((gc >> 1) + 1) & 1, abort_flag);  // O of two chunks before
                mbar_wait_short(&bar_p[b], (gc >> 1) & 1, abort_flag);
                tc_fence_after_sync();
                if (DK == 128) mma_ts_k128_w<false>(tmem + kTmO + 64 * b, tmem + kTmS, q, id_o);
                else mma_ts_k64_w<false, 2>(tmem + kTmO + 64 * b, tmem + kTmS, q, id_o);
                mma_commit_w(&bar_s[b]);
                mma_ss_k64_w<true, 128, 2>(tmem + kTmO + 64 * b, desc_advance(dV, s * L::kTileV), dP, id_v);
                mma_commit_w(&bar_o[b]);
                mma_commit_w(&bar_empty[s]);
            }
        }
    } else if (warp == 22) {
        // =============================================================== scores
        constexpr uint32_t id_qk = make_idesc_bf16(64, 64, false, false);
        const uint64_t dQ = make_smem_desc_sw128(smem_u32(smem + L::kOffQ), 0, 1024), dK = make_smem_desc_sw128(smem_u32(smem), 0, 1024);
        while (next_item()) {
#pragma unroll 1
            for (int c = 0; c < it.chunks; ++c, ++gc) {
                const uint32_t s = gc % kStages, b = gc & 1;
                mbar_wait_short(&bar_full[s], (gc / kStages) & 1, abort_flag);
                if (gc > 1) mbar_wait_short(&bar_p[b], ((gc >> 1) + 1) & 1, abort_flag);  // the scores of two chunks before have been read
                tc_fence_after_sync();
                const uint32_t tP = tmem + kTmP + (b << 20);  // (16 lanes on for odd chunks)
                const uint64_t q = desc_advance(dQ, gc % kStagesQ * L::kTileQ), k = desc_advance(dK, s * L::kTileK);
                mma_ss_k64_w<false, 2, 2>(tP, q, k, id_qk);
                if (DK == 128) mma_ss_k64_w<true, 2, 2>(tP, desc_advance(q, 8192), desc_advance(k, 8192), id_qk);
                mma_commit_w(&bar_score[b]);
            }
        }
    } else if (warp == 23) {
        // =============================================================== items and gates
        LinWalker walker;
        uint32_t n = 0;
        auto hand_out = [&]() {
            mbar_wait_short(&bar_itemfree[n & 1], ((n >> 1) + 1) & 1, abort_flag);
            if (lane == 0) {
                items[n & 1] = it;
                mbar_arrive(&bar_item[n & 1]);
            }
            __syncwarp();
            ++n;
        };
        const int size_log2 = p.gate.is_f32 ? 2 : 1;
        const char* from = nullptr;  // the next chunk's gates of this lane
        auto load1 = [&](const char* at, bool there) {  // as bits, converted where it is used
            uint32_t bits = 0u;
            if (there) bits = size_log2 == 2 ? __ldg(reinterpret_cast<const uint32_t*>(at)) : static_cast<uint32_t>(__ldg(reinterpret_cast<const unsigned short*>(at))) << 16;
            return bits;
        };
        auto load = [&](int c, uint32_t& a0, uint32_t& a1) {
            const int t = c * kChunk + 2 * lane, end = p.gate.ptr ? it.tokens : 0;
            a0 = load1(from, t < end);
            a1 = load1(from + (p.gate.st << size_log2), t + 1 < end);
            from += p.gate.st << (6 + size_log2);
        };
        // The launch has a block for every item.  A block that runs asks for the next one that has not started and takes it over.
        uint32_t asked = 0;
        int i = blockIdx.x;
#pragma unroll 1
        while (i >= 0) {
            if (!walker.locate(p, i, it)) break;  // (surplus items are the last ones)
            hand_out();
            uint32_t a0, a1, b0, b1, c0, c1;  // the gates of this chunk and the two behind it: DRAM answers later than a chunk takes
            float expo = 0.f, expo_rest = 0.f;  // c
            from = static_cast<const char*>(p.gate.ptr) + ((it.batch * p.gate.sb + (it.tok0 + 2 * lane) * p.gate.st + it.head * p.gate.sh) << size_log2);
            load(0, a0, a1);
            load(1, b0, b1);
            load(2, c0, c1);
#pragma unroll 1
            for (int c = 0; c < it.chunks; ++c, ++gc) {
                float g0 = lin_gate_log2(__uint_as_float(a0)), g1 = lin_gate_log2(__uint_as_float(a1)), r0 = g0, r1 = g1;
                a0 = b0; a1 = b1;
                b0 = c0; b1 = c1;
                load(c + 3, c0, c1);
                scan64(g0, g1, lane);  // (tokens past the end have no decay: they carry the last one's sum)
                const float last = __shfl_sync(0xffffffffu, g1, 31);
                // (a NaN is not plain, neither are gates that grow)
                auto within = [&](float c, float rest) { return __all_sync(0xffffffffu, fabsf(g0 + rest + c) <= kPlainLog2 && fabsf(g1 + rest + c) <= kPlainLog2); };
                float before = 1.f, behind = 1.f;
                bool plain = within(expo, expo_rest);
                if (__builtin_expect(!plain, 0)) {  // the state takes another exponent, the largest one if that does
                    plain = within(kPlainLog2, 0.f);
                    const float other = plain ? kPlainLog2 : 0.f;
                    if (!plain) plain = within(0.f, 0.f);
                    before = ex2(expo - other + expo_rest);
                    expo = other;
                    expo_rest = 0.f;
                }
                mbar_wait_short(&bar_gfree[gc & 3], ((gc >> 2) + 1) & 1, abort_flag);
                float* gb = gate_buf(gc);
                float2* const gb2 = reinterpret_cast<float2*>(gb);
                uint2* const factors = reinterpret_cast<uint2*>(gb + 260);
                if (__builtin_expect(plain, 1)) {
                    g0 = g0 + expo_rest + expo;
                    g1 = g1 + expo_rest + expo;
                    const float f0 = ex2(-g0), f1 = ex2(-g1);
                    gb2[lane] = make_float2(f0, f1);
                    gb2[32 + lane] = make_float2(p.scale * ex2(g0), p.scale * ex2(g1));
                    factors[lane] = factor_pair(f0, f1);
                    add_kept(expo, expo_rest, last);
                } else {
                    behind = ex2(last);
                    scan64_behind(r0, r1, lane);
                    factors[lane] = factor_pair(ex2(r0), ex2(r1));
                    gb2[32 + lane] = make_float2(p.scale, p.scale);
                    gb2[64 + lane] = make_float2(g0, g1);
                    gb2[96 + lane] = make_float2(ex2(g0), ex2(g1));
                }
                if (lane == 0) *reinterpret_cast<float4*>(gb + 256) = make_float4(before, behind, ex2(expo + expo_rest), plain ? 1.f : 0.f);
                if (lane == 1) *reinterpret_cast<float4*>(gb + L::kGateOdd) = make_float4(0.f, 0.f, 0.f, 0.f);
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar_gate[gc & 3]);
            }
            if (lane == 0) {
                fence_proxy_async_smem();
                mbar_arrive_expect_tx(bar_next, 16);
                next_block_request(next, bar_next);
            }
            __syncwarp();
            mbar_wait_short(bar_next, asked & 1, abort_flag);
            ++asked;
            i = *static_cast<volatile int*>(abort_flag) == 0 ? next_block_answer(next) : -1;
        }
        it.chunks = -1;
        hand_out();
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem, 512);
    if (tid == 0 && *abort_flag && p.status) atomicExch(p.status, 4);
}

}  // namespace gdn
