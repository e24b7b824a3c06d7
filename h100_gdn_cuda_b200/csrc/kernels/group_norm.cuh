// Group norm, channels last.  x is (N, L, C): N samples of L rows of C channels; the channels are G groups of W = C / G.  With the
// mean m and the variance s^2 of a sample's L W values of a group,
//     u = (x - m) / sqrt(s^2 + eps) * weight[c] + bias[c] ,    y = act(u)   or, with a gate z,   y = u act(z) ,
// act = SiLU or nothing.  Sums are fp32; the variance is the mean of squared distances from a mean that is already known, and parts of a
// group are joined by  n s^2 = sum_i n_i (s_i^2 + (m_i - m)^2), so that a large mean costs no digits.
#pragma once
#include <cuda_bf16.h>
#include <stdint.h>

#include "pairs.cuh"

namespace gdn {

struct GroupNormParams {
    const void* x;
    const void* z;  // gate or NULL, laid out by its own strides
    void* y;
    const void* weight;  // (C) or NULL
    const void* bias;    // (C) or NULL
    int param_f32;       // weight and bias are fp32 (otherwise bf16)
    long long n, l;      // samples, rows of a sample
    int channels, groups, width;
    long long x_sn, x_sl, z_sn, z_sl, y_sn, y_sl;  // strides of a sample and a row, in elements
    float eps;
    int silu;
    // long samples: rows of a part, parts of a sample, channels of a block (whole groups); (mean, sum of squared distances) of every
    // (sample, part, group)
    int part_rows, parts, block_channels;
    int split;  // groups of more channels than a CTA sweeps at once: the pieces of one, a block each, the last one shorter (otherwise 1)
    float2* partial;
    int apply_rows;  // rows of a CTA of the second launch
    // what that one joins: `join_parts` entries of `join_rows` rows each (the parts, or one of all rows where those are many)
    const float2* join;
    long long join_rows;
    int join_parts;
};

namespace gn {
// V values as they lie in memory
template <typename T, int V>
struct alignas(sizeof(T) * V) Raw {
    T v[V];
};
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> load(const T* p) { return *reinterpret_cast<const Raw<T, V>*>(p); }
template <typename T, int V>
__device__ __forceinline__ void widen(const Raw<T, V>& r, float* out) {
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] = to_f32(r.v[e]);
}
template <int V>
__device__ __forceinline__ Raw<float, V> narrow(const float* in, float) {
    Raw<float, V> r;
#pragma unroll
    for (int e = 0; e < V; ++e) r.v[e] = in[e];
    return r;
}
template <int V>
__device__ __forceinline__ Raw<__nv_bfloat16, V> narrow(const float* in, __nv_bfloat16) {
    Raw<__nv_bfloat16, V> r;
#pragma unroll
    for (int e = 0; e + 1 < V; e += 2) *reinterpret_cast<__nv_bfloat162*>(&r.v[e]) = __floats2bfloat162_rn(in[e], in[e + 1]);
    if (V == 1) r.v[0] = __float2bfloat16(in[0]);
    return r;
}
template <typename T, int V>
__device__ __forceinline__ void store(T* p, const float* in) { *reinterpret_cast<Raw<T, V>*>(p) = narrow<V>(in, T()); }
__device__ __forceinline__ float param(const void* p, int f32, int c, float otherwise) {
    if (!p) return otherwise;
    return f32 ? __ldg(static_cast<const float*>(p) + c) : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[c]);
}
__device__ __forceinline__ float act(float u, bool silu) { return silu ? u * pairs::rcp(1.f + pairs::ex2(u * -1.4426950408889634f)) : u; }

// V values as (V + 1) / 2 pairs (V = 1: the upper one is zero)
template <int V>
constexpr int kPairs = (V + 1) / 2;
template <typename T, int V>
__device__ __forceinline__ void widen2(const Raw<T, V>& r, pairs::f2* out) {
#pragma unroll
    for (int e = 0; e < kPairs<V>; ++e) {
        if (V == 1) {
            out[0] = pairs::pk(to_f32(r.v[0]), 0.f);
        } else if (sizeof(T) == 2) {
            const uint32_t w = reinterpret_cast<const uint32_t*>(r.v)[e];
            out[e] = pairs::pk(ptx::bf16_lo(w), ptx::bf16_hi(w));
        } else {
            out[e] = pairs::pk(to_f32(r.v[2 * e]), to_f32(r.v[2 * e + 1]));
        }
    }
}
template <typename T, int V>
__device__ __forceinline__ void store2(T* p, const pairs::f2* in) {
    float f[2 * kPairs<V>];
#pragma unroll
    for (int e = 0; e < kPairs<V>; ++e) pairs::unpk(in[e], f[2 * e], f[2 * e + 1]);
    store<T, V>(p, f);
}
}  // namespace gn

// Samples of one row (a norm per token): LPR lanes per group, a lane keeps its channels from row to row, and with them their weight and bias.  kUnroll rows
// are in flight, every load of theirs issued before the first is used.  HBM-bound.
template <int kPass>
constexpr int gn_unroll() { return kPass == 1 ? 2 : 1; }

template <typename T, int V, int LPR, int kPass, bool kGated>
__global__ void __launch_bounds__(256, kPass == 1 ? 4 : 2) gdn_group_norm_rows_kernel(const GroupNormParams p) {
    constexpr int kUnroll = gn_unroll<kPass>();
    ptx::grid_dep_wait();
    ptx::grid_dep_launch();
    using namespace pairs;
    constexpr int P = gn::kPairs<V>;
    const int l = threadIdx.x % LPR, group = blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
    const bool live = group < p.groups;
    const int c_first = (live ? group : 0) * p.width;
    f2 w[kPass][P], b[kPass][P];
    bool in[kPass];
#pragma unroll
    for (int i = 0; i < kPass; ++i) {
        in[i] = live && (i * LPR + l) * V < p.width;
#pragma unroll
        for (int e = 0; e < P; ++e) {
            const int c = c_first + (i * LPR + l) * V + 2 * e, c2 = V > 1 ? c + 1 : c;
            w[i][e] = in[i] ? pk(gn::param(p.weight, p.param_f32, c, 1.f), gn::param(p.weight, p.param_f32, c2, 1.f)) : 0ull;
            b[i][e] = in[i] ? pk(gn::param(p.bias, p.param_f32, c, 0.f), gn::param(p.bias, p.param_f32, c2, 0.f)) : 0ull;
        }
    }
    const float inv = 1.f / static_cast<float>(p.width);
    const bool silu = p.silu != 0;
    const long long first = static_cast<long long>(blockIdx.y) * kUnroll, step = static_cast<long long>(gridDim.y) * kUnroll;
    const T* x = static_cast<const T*>(p.x) + first * p.x_sn + c_first + l * V;
    const T* z = static_cast<const T*>(p.z) + first * p.z_sn + c_first + l * V;
    T* y = static_cast<T*>(p.y) + first * p.y_sn + c_first + l * V;
#pragma unroll 1
    for (long long r0 = first; r0 < p.n; r0 += step, x += step * p.x_sn, z += step * p.z_sn, y += step * p.y_sn) {
        gn::Raw<T, V> xr[kUnroll][kPass], zr[kUnroll][kPass];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
            for (int i = 0; i < kPass; ++i) {
                xr[u][i] = zr[u][i] = gn::Raw<T, V>{};
                if (in[i] && r0 + u < p.n) {
                    xr[u][i] = gn::load<T, V>(x + u * p.x_sn + i * LPR * V);
                    if (kGated) zr[u][i] = gn::load<T, V>(z + u * p.z_sn + i * LPR * V);
                }
            }
        }
        f2 v[kUnroll][kPass][P];
        float sum[kUnroll], sq[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            f2 s = 0ull;
#pragma unroll
            for (int i = 0; i < kPass; ++i) {
                gn::widen2<T, V>(xr[u][i], v[u][i]);
#pragma unroll
                for (int e = 0; e < P; ++e) s = add2(s, v[u][i][e]);  // (zero where there is nothing)
            }
            float lo, hi;
            unpk(s, lo, hi);
            sum[u] = lo + hi;
        }
#pragma unroll
        for (int m = LPR / 2; m > 0; m >>= 1)
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) sum[u] += __shfl_xor_sync(0xffffffffu, sum[u], m);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const float mean = -sum[u] * inv;
            f2 s = 0ull;
#pragma unroll
            for (int i = 0; i < kPass; ++i) {
                const f2 mean2 = in[i] ? pk(mean, V > 1 ? mean : 0.f) : 0ull;
#pragma unroll
                for (int e = 0; e < P; ++e) {
                    v[u][i][e] = add2(v[u][i][e], mean2);
                    s = fma2(v[u][i][e], v[u][i][e], s);
                }
            }
            float lo, hi;
            unpk(s, lo, hi);
            sq[u] = lo + hi;
        }
#pragma unroll
        for (int m = LPR / 2; m > 0; m >>= 1)
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) sq[u] += __shfl_xor_sync(0xffffffffu, sq[u], m);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const float rstd = rsqrtf(fmaf(sq[u], inv, p.eps));
            const f2 rstd2 = pk(rstd, rstd);
#pragma unroll
            for (int i = 0; i < kPass; ++i) {
                f2 g[P];
                if (kGated) gn::widen2<T, V>(zr[u][i], g);
#pragma unroll
                for (int e = 0; e < P; ++e) {
                    const f2 t = fma2(mul2(v[u][i][e], rstd2), w[i][e], b[i][e]);
                    if (kGated) v[u][i][e] = mul2(t, silu ? silu2(g[e]) : g[e]);
                    else v[u][i][e] = silu ? silu2(t) : t;
                }
                if (in[i] && r0 + u < p.n) gn::store2<T, V>(y + u * p.y_sn + i * LPR * V, v[u][i]);
            }
        }
    }
}

// Short groups of several rows (L W up to 512 values): LPR lanes per (sample, group), the values in registers.
template <typename T, int V, int LPR, int kPass>
__global__ void __launch_bounds__(256) gdn_group_norm_short_kernel(const GroupNormParams p) {
    ptx::grid_dep_wait();
    ptx::grid_dep_launch();
    const int lane = threadIdx.x & 31, l = lane % LPR;
    const long long unit = (static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5)) * (32 / LPR) + lane / LPR;
    const bool live = unit < p.n * p.groups;
    const long long n = live ? unit / p.groups : 0;
    const int c_first = static_cast<int>(live ? unit % p.groups : 0) * p.width;
    const int size = live ? static_cast<int>(p.l) * p.width : 0;
    const T* x = static_cast<const T*>(p.x) + n * p.x_sn + c_first;
    float v[kPass][V];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kPass; ++i) {
        const int at = (i * LPR + l) * V;
        if (at < size) {
            gn::widen<T, V>(gn::load<T, V>(x + (at / p.width) * p.x_sl + at % p.width), v[i]);
#pragma unroll
            for (int e = 0; e < V; ++e) sum += v[i][e];
        }
    }
#pragma unroll
    for (int m = LPR / 2; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
    const float mean = sum / static_cast<float>(size);
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < kPass; ++i) {
        if ((i * LPR + l) * V < size) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[i][e] -= mean;
                sq = fmaf(v[i][e], v[i][e], sq);
            }
        }
    }
#pragma unroll
    for (int m = LPR / 2; m > 0; m >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, m);
    const float rstd = rsqrtf(sq / static_cast<float>(size) + p.eps);
#pragma unroll
    for (int i = 0; i < kPass; ++i) {
        const int at = (i * LPR + l) * V;
        if (at < size) {
            const long long row = at / p.width;
            const int c = c_first + at % p.width;
            float z[V];
            if (p.z) gn::widen<T, V>(gn::load<T, V>(static_cast<const T*>(p.z) + n * p.z_sn + row * p.z_sl + c), z);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float u = v[i][e] * rstd * gn::param(p.weight, p.param_f32, c + e, 1.f) + gn::param(p.bias, p.param_f32, c + e, 0.f);
                v[i][e] = p.z ? u * gn::act(z[e], p.silu) : gn::act(u, p.silu);
            }
            gn::store<T, V>(static_cast<T*>(p.y) + n * p.y_sn + row * p.y_sl + c, v[i]);
        }
    }
}

// Groups that a CTA's shared memory holds: a CTA per (sample, group), x read once and y written in one launch.  Neighbouring groups' pieces of a row may
// share a sector: L2 joins them.  Large groups are bound by one SM's rate of copies and of SiLU's
// exponentials, one after the other (640 channels, 4 x 4095 rows, 128 CTAs: 18 us, of which 6 are DRAM's).
constexpr int kNormWholeBytes = 224 * 1024;
constexpr int kNormPartBytes = 72 * 1024;  // three CTAs share an SM (two of the long groups' first launch where its sums take 4 or 8 KB more)

// the sum over a CTA of `kWarps` warps; everybody gets it
template <int kWarps>
__device__ __forceinline__ float gn_block_sum(float v, float* part) {
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    float sum = static_cast<int>(threadIdx.x & 31) < kWarps ? part[threadIdx.x & 31] : 0.f;
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
    __syncthreads();
    return sum;
}

template <typename T, int V, int kThreads, bool kGated>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) gdn_group_norm_whole_kernel(const GroupNormParams p) {
    extern __shared__ __align__(16) uint8_t tile_raw[];
    __shared__ float part[kThreads / 32];
    ptx::grid_dep_wait();
    ptx::grid_dep_launch();
    using namespace pairs;
    constexpr int P = gn::kPairs<V>;
    const long long n = blockIdx.x / p.groups;
    const int c_first = static_cast<int>(blockIdx.x % p.groups) * p.width, rows = static_cast<int>(p.l);
    const int vecs = p.width / V, rstep = kThreads / vecs, t = threadIdx.x, vec = t % vecs, r0 = t / vecs;  // (r0 == rstep: an idle thread)
    const int mine = r0 < rstep && r0 < rows ? (rows - r0 + rstep - 1) / rstep : 0, c = c_first + vec * V;
    gn::Raw<T, V>* const tile = reinterpret_cast<gn::Raw<T, V>*>(tile_raw) + t;  // this thread's rows, kThreads apart
    {
        const T* x = static_cast<const T*>(p.x) + n * p.x_sn + r0 * p.x_sl + c;
        const long long step = rstep * p.x_sl;
        constexpr int kBytes = V * static_cast<int>(sizeof(T));
#pragma unroll 4
        for (int i = 0; i < mine; ++i, x += step) {
            if (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ptx::smem_u32(tile + i * kThreads)), "l"(x) : "memory");
            else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(ptx::smem_u32(tile + i * kThreads)), "l"(x), "n"(kBytes) : "memory");
        }
    }
    f2 w[P], b[P], s[P];
#pragma unroll
    for (int e = 0; e < P; ++e) {
        const int ca = c + 2 * e, cb = V > 1 ? ca + 1 : ca;
        w[e] = pk(gn::param(p.weight, p.param_f32, ca, 1.f), gn::param(p.weight, p.param_f32, cb, 1.f));
        b[e] = pk(gn::param(p.bias, p.param_f32, ca, 0.f), gn::param(p.bias, p.param_f32, cb, 0.f));
        s[e] = 0ull;
    }
    auto total = [&]() {
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < P; ++e) {
            float lo, hi;
            unpk(s[e], lo, hi);
            sum += V > 1 ? lo + hi : lo;
            s[e] = 0ull;
        }
        return gn_block_sum<kThreads / 32>(sum, part);
    };
    asm volatile("cp.async.wait_all;" ::: "memory");  // (a thread reads what it has copied itself)
#pragma unroll 4
    for (int i = 0; i < mine; ++i) {
        f2 v[P];
        gn::widen2<T, V>(tile[i * kThreads], v);
#pragma unroll
        for (int e = 0; e < P; ++e) s[e] = add2(s[e], v[e]);
    }
    const float count = static_cast<float>(rows) * static_cast<float>(p.width), mean = total() / count;
    const f2 m = pk(-mean, -mean);
#pragma unroll 4
    for (int i = 0; i < mine; ++i) {
        f2 v[P];
        gn::widen2<T, V>(tile[i * kThreads], v);
#pragma unroll
        for (int e = 0; e < P; ++e) {
            const f2 d = add2(v[e], m);
            s[e] = fma2(d, d, s[e]);
        }
    }
    const float rstd = rsqrtf(total() / count + p.eps);
    const f2 rstd2 = pk(rstd, rstd);
#pragma unroll
    for (int e = 0; e < P; ++e) w[e] = mul2(w[e], rstd2);
    const T* z = static_cast<const T*>(p.z) + n * p.z_sn + r0 * p.z_sl + c;
    T* y = static_cast<T*>(p.y) + n * p.y_sn + r0 * p.y_sl + c;
    const long long z_step = rstep * p.z_sl, y_step = rstep * p.y_sl;
    constexpr int kUnroll = 4;  // rows in flight
    const bool silu = p.silu != 0;
#pragma unroll 1
    for (int i = 0; i < mine; i += kUnroll) {
        gn::Raw<T, V> zr[kUnroll];
        if (kGated) {
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                if (i + u < mine) zr[u] = gn::load<T, V>(z);
                z += z_step;
            }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            if (i + u >= mine) break;
            f2 v[P], g[P];
            gn::widen2<T, V>(tile[(i + u) * kThreads], v);
            if (kGated) gn::widen2<T, V>(zr[u], g);
#pragma unroll
            for (int e = 0; e < P; ++e) {
                const f2 t2 = fma2(add2(v[e], m), w[e], b[e]);
                if (kGated) v[e] = mul2(t2, silu ? silu2(g[e]) : g[e]);
                else v[e] = silu ? silu2(t2) : t2;
            }
            gn::store2<T, V>(y, v);
            y += y_step;
        }
    }
}

// Long groups, in two launches: a CTA takes `part_rows` rows of `block_channels` channels (whole groups) of a sample, all of them asked for at once, and
// keeps them in shared memory, so that the mean is there before the distances are summed; it leaves both per group.  The second launch
// joins the parts of its sample and writes y; where they are more than a few, a small one between joins them.  x is read twice, from L2
// the second time where it fits.  (640 channels, 4 x 4095 rows: 25 us; with loops over memory and a division per value 62.  A cluster of CTAs
// that holds a sample in its shared memory reads x once, but took 48: the clusters of eight whole SMs do not all fit at once.)
constexpr int kNormThreads = 256;
constexpr int kNormMaxGroups = 64;           // groups of a block
constexpr int kNormJoinParts = 32;           // more parts than that are joined by a launch of their own (every CTA of the second one reads all of its sample's)

// The channels of block `b`, and how wide its groups are (a piece of one for a group).
struct NormBlock {
    int first, channels, width;
    __device__ __forceinline__ NormBlock(const GroupNormParams& p, int b) {
        if (p.split == 1) {
            first = b * p.block_channels;
            channels = min(p.block_channels, p.channels - first);
            width = p.width;
        } else {
            const int at = b % p.split * p.block_channels;
            first = b / p.split * p.width + at;
            width = channels = min(p.block_channels, p.width - at);
        }
    }
};

// From the sums of a thread's V channels (rows r0, r0 + rstep, ... of the part) to sums of groups, in `out`.  Everybody calls it.
template <int V>
__device__ __forceinline__ void gn_group_sums(const pairs::f2* s, int vecs, int rstep, int width, int groups, float* scratch, float* out) {
    const int t = threadIdx.x, channels = vecs * V;
    if (groups == 1) {  // (8 lanes would add up what 256 threads have: 5378 samples of 851 rows of one channel 480 us)
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < gn::kPairs<V>; ++e) {
            float lo, hi;
            pairs::unpk(s[e], lo, hi);
            sum += V > 1 ? lo + hi : lo;
        }
        sum = gn_block_sum<kNormThreads / 32>(sum, scratch);
        if (t == 0) out[0] = sum;
        __syncthreads();
        return;
    }
    __syncthreads();
    if (t < vecs * rstep) {
#pragma unroll
        for (int e = 0; e < gn::kPairs<V>; ++e) {  // row r0 = t / vecs, channels behind one another
            float lo, hi;
            pairs::unpk(s[e], lo, hi);
            scratch[t * V + 2 * e] = lo;
            if (V > 1) scratch[t * V + 2 * e + 1] = hi;
        }
    }
    __syncthreads();
    const int l = t & 7;
    for (int g = t >> 3; g < (groups + kNormThreads / 8 - 1) / (kNormThreads / 8) * (kNormThreads / 8); g += kNormThreads / 8) {
        float sum = 0.f;
        if (g < groups)
            for (int r = 0; r < rstep; ++r)
                for (int c = l; c < width; c += 8) sum += scratch[r * channels + g * width + c];
#pragma unroll
        for (int m = 4; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
        if (l == 0 && g < groups) out[g] = sum;
    }
    __syncthreads();
}

template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads) gdn_group_norm_stats_kernel(const GroupNormParams p) {
    extern __shared__ __align__(16) uint8_t tile_raw[];
    __shared__ float scratch[kNormThreads * V];
    __shared__ float mean[kNormMaxGroups], sq[kNormMaxGroups];
    ptx::grid_dep_wait();
    ptx::grid_dep_launch();
    const long long n = blockIdx.z, r_first = static_cast<long long>(blockIdx.x) * p.part_rows;
    const NormBlock block(p, blockIdx.y);
    const int c_first = block.first, channels = block.channels, groups = channels / block.width;
    const int rows = static_cast<int>(min(static_cast<long long>(p.part_rows), p.l - r_first));
    const int vecs = channels / V, rstep = kNormThreads / vecs, t = threadIdx.x;
    const int vec = t % vecs, r0 = t / vecs;  // (r0 == rstep: an idle thread)
    const bool live = r0 < rstep;
    gn::Raw<T, V>* const tile = reinterpret_cast<gn::Raw<T, V>*>(tile_raw);  // this thread's rows: t, t + 256, ...
    using namespace pairs;
    constexpr int P = gn::kPairs<V>;
    const T* x = static_cast<const T*>(p.x) + n * p.x_sn + (r_first + r0) * p.x_sl + c_first + vec * V;
    const long long x_step = rstep * p.x_sl;
    const int mine = live && rows > r0 ? (rows - r0 + rstep - 1) / rstep : 0;  // rows of this thread
    f2 s[P];
#pragma unroll
    for (int e = 0; e < P; ++e) s[e] = 0ull;
    constexpr int kBytes = V * static_cast<int>(sizeof(T));
    constexpr int kInFlight = kBytes >= 4 ? 1 : 8;  // loads, where a value is less than an asynchronous copy takes
    int i0 = 0;
    if (kBytes < 4) {
#pragma unroll 1
        for (; i0 + kInFlight <= mine; i0 += kInFlight) {
            gn::Raw<T, V> r[kInFlight];
#pragma unroll
            for (int u = 0; u < kInFlight; ++u, x += x_step) r[u] = gn::load<T, V>(x);
#pragma unroll
            for (int u = 0; u < kInFlight; ++u) tile[t + (i0 + u) * kNormThreads] = r[u];
        }
    }
#pragma unroll 4
    for (int i = i0; i < mine; ++i, x += x_step) {
        if (kBytes == 16)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ptx::smem_u32(tile + t + i * kNormThreads)), "l"(x) : "memory");
        else if (kBytes >= 4)
            asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(ptx::smem_u32(tile + t + i * kNormThreads)), "l"(x), "n"(kBytes >= 4 ? kBytes : 4) : "memory");
        else
            tile[t + i * kNormThreads] = gn::load<T, V>(x);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");  // (a thread reads what it has copied itself)
#pragma unroll 4
    for (int i = 0; i < mine; ++i) {
        f2 v[P];
        gn::widen2<T, V>(tile[t + i * kNormThreads], v);
#pragma unroll
        for (int e = 0; e < P; ++e) s[e] = add2(s[e], v[e]);
    }
    const float count = static_cast<float>(rows) * static_cast<float>(block.width);
    gn_group_sums<V>(s, vecs, rstep, block.width, groups, scratch, mean);
    f2 m[P];
#pragma unroll
    for (int e = 0; e < P; ++e) {
        const int c = vec * V + 2 * e;
        m[e] = pk(-mean[c / block.width] / count, V > 1 ? -mean[(c + 1) / block.width] / count : 0.f);
        s[e] = 0ull;
    }
#pragma unroll 4
    for (int i = 0; i < mine; ++i) {
        f2 v[P];
        gn::widen2<T, V>(tile[t + i * kNormThreads], v);
#pragma unroll
        for (int e = 0; e < P; ++e) {
            const f2 d = add2(v[e], m[e]);
            s[e] = fma2(d, d, s[e]);
        }
    }
    gn_group_sums<V>(s, vecs, rstep, block.width, groups, scratch, sq);
    float2* out = p.partial + (n * p.parts + blockIdx.x) * p.groups * p.split + (p.split == 1 ? c_first / p.width : blockIdx.y);
    for (int g = t; g < groups; g += kNormThreads) out[g] = make_float2(mean[g] / count, sq[g]);
}

// Many parts, or groups in pieces: (mean, sum of squared distances) of whole groups, a warp for each (sample, group), behind the parts' entries.
__global__ void __launch_bounds__(256) gdn_group_norm_join_kernel(const GroupNormParams p) {
    ptx::grid_dep_wait();
    ptx::grid_dep_launch();
    const long long unit = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const int entries = p.parts * p.split;  // of a group: parts one behind the other, of pieces
    if (unit >= p.n * p.groups) return;
    const long long stride = static_cast<long long>(p.groups) * p.split;
    const float2* in = p.partial + unit / p.groups * p.parts * stride + unit % p.groups * p.split;
    auto count = [&](int i) {  // values of an entry
        const long long rows = min(static_cast<long long>(p.part_rows), p.l - static_cast<long long>(i / p.split) * p.part_rows);
        const int width = p.split == 1 ? p.width : min(p.block_channels, p.width - i % p.split * p.block_channels);
        return static_cast<float>(rows) * static_cast<float>(width);
    };
    constexpr int kMine = 8;  // entries a lane has in flight, and keeps from the means to the distances where there are no more
    const int l = threadIdx.x & 31;
    float2 mine[kMine];
    float sum = 0.f, q = 0.f;
    auto fetch = [&](int i0) {
#pragma unroll
        for (int j = 0; j < kMine; ++j) {
            const int i = i0 + l + 32 * j;
            mine[j] = i < entries ? __ldcg(in + i / p.split * stride + i % p.split) : make_float2(0.f, 0.f);
        }
    };
    for (int i0 = 0; i0 < entries; i0 += 32 * kMine) {
        fetch(i0);
#pragma unroll
        for (int j = 0; j < kMine; ++j)
            if (i0 + l + 32 * j < entries) sum += count(i0 + l + 32 * j) * mine[j].x;
    }
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
    const float mu = sum / (static_cast<float>(p.l) * static_cast<float>(p.width));
    for (int i0 = 0; i0 < entries; i0 += 32 * kMine) {
        if (entries > 32 * kMine) fetch(i0);
#pragma unroll
        for (int j = 0; j < kMine; ++j) {
            if (i0 + l + 32 * j < entries) {
                const float d = mine[j].x - mu;
                q += mine[j].y + count(i0 + l + 32 * j) * d * d;
            }
        }
    }
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) q += __shfl_xor_sync(0xffffffffu, q, m);
    if ((threadIdx.x & 31) == 0) const_cast<float2*>(p.join)[unit] = make_float2(mu, q);
}

template <typename T, int V, bool kGated>
__global__ void __launch_bounds__(kNormThreads, 3) gdn_group_norm_apply_kernel(const GroupNormParams p) {
    __shared__ float mean[kNormMaxGroups], rstd[kNormMaxGroups];
    const long long n = blockIdx.z, r_first = static_cast<long long>(blockIdx.x) * p.apply_rows;
    const NormBlock block(p, blockIdx.y);
    const int c_first = block.first, channels = block.channels, groups = channels / block.width;
    const int rows = static_cast<int>(min(static_cast<long long>(p.apply_rows), p.l - r_first));
    const int vecs = channels / V, rstep = kNormThreads / vecs, t = threadIdx.x, vec = t % vecs, r0 = t / vecs;
    ptx::grid_dep_wait();
    ptx::grid_dep_launch();
    using namespace pairs;
    constexpr int P = gn::kPairs<V>;
    f2 w[P], b[P];
#pragma unroll
    for (int e = 0; e < P; ++e) {
        const int c = c_first + vec * V + 2 * e, c2 = V > 1 ? c + 1 : c;
        w[e] = pk(gn::param(p.weight, p.param_f32, c, 1.f), gn::param(p.weight, p.param_f32, c2, 1.f));
        b[e] = pk(gn::param(p.bias, p.param_f32, c, 0.f), gn::param(p.bias, p.param_f32, c2, 0.f));
    }
    const int l = t & 7;
    for (int g = t >> 3; g < (groups + 31) / 32 * 32; g += kNormThreads / 8) {
        const float2* in = p.join + n * p.join_parts * p.groups + c_first / p.width + g;
        constexpr int kMine = kNormJoinParts / 8;
        float sum = 0.f, q = 0.f;
        auto count = [&](int i) { return static_cast<float>(min(p.join_rows, p.l - i * p.join_rows)); };
        float2 mine[kMine];
#pragma unroll
        for (int j = 0; j < kMine; ++j) {
            const int i = l + 8 * j;
            mine[j] = g < groups && i < p.join_parts ? __ldcg(in + static_cast<long long>(i) * p.groups) : make_float2(0.f, 0.f);
        }
#pragma unroll
        for (int j = 0; j < kMine; ++j) sum += l + 8 * j < p.join_parts ? count(l + 8 * j) * mine[j].x : 0.f;
#pragma unroll
        for (int m = 4; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
        const float mu = sum / static_cast<float>(p.l);
#pragma unroll
        for (int j = 0; j < kMine; ++j) {
            const float d = mine[j].x - mu;
            if (l + 8 * j < p.join_parts) q += mine[j].y + count(l + 8 * j) * static_cast<float>(p.width) * d * d;
        }
#pragma unroll
        for (int m = 4; m > 0; m >>= 1) q += __shfl_xor_sync(0xffffffffu, q, m);
        if (l == 0 && g < groups) {
            mean[g] = mu;
            rstd[g] = rsqrtf(q / (static_cast<float>(p.l) * static_cast<float>(p.width)) + p.eps);
        }
    }
    __syncthreads();
    if (r0 >= rstep || r0 >= rows) return;
    f2 m[P];
#pragma unroll
    for (int e = 0; e < P; ++e) {
        const int g = (vec * V + 2 * e) / p.width, g2 = V > 1 ? (vec * V + 2 * e + 1) / p.width : g;
        w[e] = mul2(w[e], pk(rstd[g], rstd[g2]));
        m[e] = pk(-mean[g], -mean[g2]);
    }
    const T* x = static_cast<const T*>(p.x) + n * p.x_sn + (r_first + r0) * p.x_sl + c_first + vec * V;
    const T* z = static_cast<const T*>(p.z) + n * p.z_sn + (r_first + r0) * p.z_sl + c_first + vec * V;
    T* y = static_cast<T*>(p.y) + n * p.y_sn + (r_first + r0) * p.y_sl + c_first + vec * V;
    const long long x_step = rstep * p.x_sl, z_step = rstep * p.z_sl, y_step = rstep * p.y_sl;
    const int mine = (rows - r0 + rstep - 1) / rstep;
    constexpr int kUnroll = kGated ? 2 : 4;  // rows in flight
    const bool silu = p.silu != 0;
#pragma unroll 1
    for (int i = 0; i < mine; i += kUnroll) {
        gn::Raw<T, V> xr[kUnroll], zr[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            if (i + u < mine) {
                xr[u] = gn::load<T, V>(x);
                if (kGated) zr[u] = gn::load<T, V>(z);
            }
            x += x_step;
            z += z_step;
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            if (i + u >= mine) break;
            f2 v[P], g[P];
            gn::widen2<T, V>(xr[u], v);
            if (kGated) gn::widen2<T, V>(zr[u], g);
#pragma unroll
            for (int e = 0; e < P; ++e) {
                const f2 t2 = fma2(add2(v[e], m[e]), w[e], b[e]);
                if (kGated) v[e] = mul2(t2, silu ? silu2(g[e]) : g[e]);
                else v[e] = silu ? silu2(t2) : t2;
            }
            gn::store2<T, V>(y, v);
            y += y_step;
        }
    }
}

// Groups of more channels than a CTA has room for in one sweep (width > 256 V), where they are short or as many as fit the SMs: one CTA per (sample, group), in
// three passes over memory.
template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads) gdn_group_norm_wide_kernel(const GroupNormParams p) {
    __shared__ float part[8];
    ptx::grid_dep_wait();
    ptx::grid_dep_launch();
    const long long n = blockIdx.x / p.groups;
    const int c_first = static_cast<int>(blockIdx.x % p.groups) * p.width;
    const T* x = static_cast<const T*>(p.x) + n * p.x_sn + c_first;
    auto total = [&](float s) {
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
        __syncthreads();
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < kNormThreads / 32; ++i) t += part[i];
        return t;
    };
    auto each = [&](auto f) {
        for (long long r = 0; r < p.l; ++r)
            for (int c = threadIdx.x * V; c < p.width; c += kNormThreads * V) {
                float v[V];
                gn::widen<T, V>(gn::load<T, V>(x + r * p.x_sl + c), v);
                f(r, c, v);
            }
    };
    const float size = static_cast<float>(p.l) * static_cast<float>(p.width);
    float s = 0.f;
    each([&](long long, int, float* v) {
        float t = 0.f;  // (runs of V first: the long sum then has few terms)
#pragma unroll
        for (int e = 0; e < V; ++e) t += v[e];
        s += t;
    });
    const float mean = total(s) / size;
    s = 0.f;
    each([&](long long, int, float* v) {
        float t = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) t = fmaf(v[e] - mean, v[e] - mean, t);
        s += t;
    });
    const float rstd = rsqrtf(total(s) / size + p.eps);
    each([&](long long r, int c, float* v) {
        float zv[V];
        if (p.z) gn::widen<T, V>(gn::load<T, V>(static_cast<const T*>(p.z) + n * p.z_sn + r * p.z_sl + c_first + c), zv);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float u = fmaf((v[e] - mean) * rstd, gn::param(p.weight, p.param_f32, c_first + c + e, 1.f), gn::param(p.bias, p.param_f32, c_first + c + e, 0.f));
            v[e] = p.z ? u * gn::act(zv[e], p.silu) : gn::act(u, p.silu);
        }
        gn::store<T, V>(static_cast<T*>(p.y) + n * p.y_sn + r * p.y_sl + c_first + c, v);
    });
}

}  // namespace gdn
