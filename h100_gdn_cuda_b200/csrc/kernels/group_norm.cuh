// Group norm, channels last.  x is (N, L, C): N samples of L rows of C channels; the channels are G groups of W = C / G.  With the
// mean m and the variance s^2 of a sample's L W values of a group,
//     u = (x - m) / sqrt(s^2 + eps) * weight[c] + bias[c] ,    y = act(u)   or, with a gate z,   y = u act(z) ,
// act = SiLU or nothing.  Sums are fp32; the variance is the mean of squared distances from a mean that is already known, and parts of a
// group are joined by  n s^2 = sum_i n_i (s_i^2 + (m_i - m)^2), so that a large mean costs no digits.
#pragma once
#include <cuda_bf16.h>
#include <stdint.h>

#include "sm100_ptx.cuh"

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
    // long samples: rows of a part, parts of a sample, (mean, sum of squared distances) of every (sample, part, group)
    int part_rows, parts, block_channels;
    float2* partial;
};

namespace gn {
template <typename T, int V>
struct Vec {
    T v[V];
};
template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16(v); }

template <typename T, int V>
__device__ __forceinline__ void load(const T* p, float* out) {
    struct alignas(sizeof(T) * V) Raw { T v[V]; };
    const Raw r = *reinterpret_cast<const Raw*>(p);
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] = to_f32(r.v[e]);
}
template <typename T, int V>
__device__ __forceinline__ void store(T* p, const float* in) {
    struct alignas(sizeof(T) * V) Raw { T v[V]; };
    Raw r;
#pragma unroll
    for (int e = 0; e < V; ++e) r.v[e] = from_f32<T>(in[e]);
    *reinterpret_cast<Raw*>(p) = r;
}
__device__ __forceinline__ float param(const void* p, int f32, int c, float otherwise) {
    if (!p) return otherwise;
    return f32 ? __ldg(static_cast<const float*>(p) + c) : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[c]);
}
__device__ __forceinline__ float act(float u, int silu) { return silu ? __fdividef(u, 1.f + __expf(-u)) : u; }
}  // namespace gn

// Short groups (L W up to 1024 values): LPR lanes per (sample, group), the values in registers.
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
            gn::load<T, V>(x + (at / p.width) * p.x_sl + at % p.width, v[i]);
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
            if (p.z) gn::load<T, V>(static_cast<const T*>(p.z) + n * p.z_sn + row * p.z_sl + c, z);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float u = v[i][e] * rstd * gn::param(p.weight, p.param_f32, c + e, 1.f) + gn::param(p.bias, p.param_f32, c + e, 0.f);
                v[i][e] = p.z ? u * gn::act(z[e], p.silu) : gn::act(u, p.silu);
            }
            gn::store<T, V>(static_cast<T*>(p.y) + n * p.y_sn + row * p.y_sl + c, v[i]);
        }
    }
}

// Long groups: a CTA takes `part_rows` rows of `block_channels` channels (whole groups) of a sample.
constexpr int kNormThreads = 256;
constexpr int kNormMaxGroups = 64;  // groups of a block

// sums over a CTA's part, group by group: `value(row, c)` summed into `out[group]` (shared memory)
template <int V, typename F>
__device__ __forceinline__ void gn_part_sums(const GroupNormParams& p, long long rows, int channels, float* scratch, float* out, F value) {
    // a thread has V channels of its own and every `rstep`-th row; channels in shared memory, then groups
    const int vecs = channels / V;
    const int rstep = max(1, kNormThreads / vecs);
    for (int i = threadIdx.x; i < channels / p.width; i += kNormThreads) out[i] = 0.f;
    for (int v0 = 0; v0 < vecs; v0 += kNormThreads) {
        const int vec = v0 + threadIdx.x % min(vecs, kNormThreads), r0 = vecs < kNormThreads ? threadIdx.x / vecs : 0;
        float s[V];
#pragma unroll
        for (int e = 0; e < V; ++e) s[e] = 0.f;
        const bool live = vec < vecs && r0 < rstep;
        if (live)
            for (long long r = r0; r < rows; r += rstep) value(r, vec * V, s);
        __syncthreads();
#pragma unroll
        for (int e = 0; e < V; ++e) scratch[threadIdx.x * V + e] = s[e];
        __syncthreads();
        // channel c of this round: threads (c / V) + vecs r of the round
        const int here = min(vecs - v0, kNormThreads) * V;
        for (int g = (v0 * V) / p.width + threadIdx.x; g * p.width < v0 * V + here; g += kNormThreads) {
            float t = 0.f;
            for (int c = max(g * p.width - v0 * V, 0); c < min((g + 1) * p.width - v0 * V, here); ++c)
                for (int r = 0; r < (vecs < kNormThreads ? rstep : 1); ++r) t += scratch[(r * vecs) * V + c];
            out[g] += t;
        }
    }
    __syncthreads();
}

template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads) gdn_group_norm_stats_kernel(const GroupNormParams p) {
    __shared__ float scratch[kNormThreads * V];
    __shared__ float mean[kNormMaxGroups], sq[kNormMaxGroups];
    ptx::grid_dep_wait();
    ptx::grid_dep_launch();
    const long long n = blockIdx.z, r_first = static_cast<long long>(blockIdx.x) * p.part_rows;
    const int c_first = blockIdx.y * p.block_channels, channels = min(p.block_channels, p.channels - c_first), groups = channels / p.width;
    const long long rows = min(static_cast<long long>(p.part_rows), p.l - r_first);
    const T* x = static_cast<const T*>(p.x) + n * p.x_sn + r_first * p.x_sl + c_first;
    gn_part_sums<V>(p, rows, channels, scratch, mean, [&](long long r, int c, float* s) {
        float v[V];
        gn::load<T, V>(x + r * p.x_sl + c, v);
#pragma unroll
        for (int e = 0; e < V; ++e) s[e] += v[e];
    });
    const float count = static_cast<float>(rows * p.width);
    for (int g = threadIdx.x; g < groups; g += kNormThreads) mean[g] /= count;
    __syncthreads();
    gn_part_sums<V>(p, rows, channels, scratch, sq, [&](long long r, int c, float* s) {
        float v[V];
        gn::load<T, V>(x + r * p.x_sl + c, v);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float d = v[e] - mean[(c + e) / p.width];
            s[e] = fmaf(d, d, s[e]);
        }
    });
    float2* out = p.partial + (n * p.parts + blockIdx.x) * p.groups + c_first / p.width;
    for (int g = threadIdx.x; g < groups; g += kNormThreads) out[g] = make_float2(mean[g], sq[g]);
}

template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads) gdn_group_norm_apply_kernel(const GroupNormParams p) {
    __shared__ float mean[kNormMaxGroups], rstd[kNormMaxGroups];
    ptx::grid_dep_wait();
    ptx::grid_dep_launch();
    const long long n = blockIdx.z, r_first = static_cast<long long>(blockIdx.x) * p.part_rows;
    const int c_first = blockIdx.y * p.block_channels, channels = min(p.block_channels, p.channels - c_first), groups = channels / p.width;
    const long long rows = min(static_cast<long long>(p.part_rows), p.l - r_first);
    auto part_count = [&](int i) { return static_cast<float>(min(static_cast<long long>(p.part_rows), p.l - static_cast<long long>(i) * p.part_rows)); };
    for (int g = threadIdx.x >> 5; g < groups; g += kNormThreads / 32) {
        const float2* in = p.partial + n * p.parts * p.groups + c_first / p.width + g;
        float s = 0.f, q = 0.f;
        for (int i = threadIdx.x & 31; i < p.parts; i += 32) s += part_count(i) * __ldcg(in + static_cast<long long>(i) * p.groups).x;
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
        const float mu = s / static_cast<float>(p.l);
        for (int i = threadIdx.x & 31; i < p.parts; i += 32) {
            const float2 t = __ldcg(in + static_cast<long long>(i) * p.groups);
            const float d = t.x - mu;
            q += t.y + part_count(i) * p.width * d * d;
        }
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) q += __shfl_xor_sync(0xffffffffu, q, m);
        if ((threadIdx.x & 31) == 0) {
            mean[g] = mu;
            rstd[g] = rsqrtf(q / (static_cast<float>(p.l) * p.width) + p.eps);
        }
    }
    __syncthreads();
    const int vecs = channels / V;
    const int rstep = max(1, kNormThreads / vecs);
    const T* x = static_cast<const T*>(p.x) + n * p.x_sn + r_first * p.x_sl + c_first;
    const T* z = static_cast<const T*>(p.z) + n * p.z_sn + r_first * p.z_sl + c_first;
    T* y = static_cast<T*>(p.y) + n * p.y_sn + r_first * p.y_sl + c_first;
    for (int v0 = 0; v0 < vecs; v0 += kNormThreads) {
        const int vec = v0 + threadIdx.x % min(vecs, kNormThreads), r0 = vecs < kNormThreads ? threadIdx.x / vecs : 0;
        if (vec >= vecs || r0 >= rstep) continue;
        float a[V], m[V], b[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const int c = vec * V + e;
            a[e] = rstd[c / p.width] * gn::param(p.weight, p.param_f32, c_first + c, 1.f);
            m[e] = mean[c / p.width];
            b[e] = gn::param(p.bias, p.param_f32, c_first + c, 0.f);
        }
        for (long long r = r0; r < rows; r += rstep) {
            float v[V], zv[V];
            gn::load<T, V>(x + r * p.x_sl + vec * V, v);
            if (p.z) gn::load<T, V>(z + r * p.z_sl + vec * V, zv);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float u = fmaf(v[e] - m[e], a[e], b[e]);
                v[e] = p.z ? u * gn::act(zv[e], p.silu) : gn::act(u, p.silu);
            }
            gn::store<T, V>(y + r * p.y_sl + vec * V, v);
        }
    }
}

}  // namespace gdn
