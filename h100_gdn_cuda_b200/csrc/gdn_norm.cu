// C-ABI entry point of the channels-last group norm (see include/gdn_b200.h).
#include <type_traits>

#include "host_common.hpp"
#include "kernels/group_norm.cuh"
#include "token_host.hpp"

using namespace gdn;

namespace {

// How a long sample is cut: channels of a block (whole groups, up to 256 vectors, or one of the `split` pieces of a group that is wider), rows of a part.
struct NormPlan {
    int block_channels, blocks, part_rows, parts, split;
};

NormPlan norm_plan(int64_t samples, int64_t rows, int channels, int groups, int vec, int size) {
    const int width = channels / groups;
    NormPlan plan{};
    if (width > kNormThreads * vec) {  // (whole vectors: see widest())
        const int most = (width / vec + kNormThreads - 1) / kNormThreads;
        plan.block_channels = (width / vec + most - 1) / most * vec;
        plan.split = (width + plan.block_channels - 1) / plan.block_channels;
        plan.blocks = groups * plan.split;
    } else {
        int unit = 1;  // groups of a block come in multiples that are whole vectors
        while (unit * width % vec != 0) ++unit;
        const int per = std::min(kNormThreads * vec / (unit * width), kNormMaxGroups / unit) * unit;
        // blocks of about the same number of groups
        const int units = (groups + unit - 1) / unit, blocks = (groups + per - 1) / per;
        plan.block_channels = std::min((units + blocks - 1) / blocks * unit * width, channels);
        plan.split = 1;
        plan.blocks = (channels + plan.block_channels - 1) / plan.block_channels;
    }
    const int vecs = plan.block_channels / vec, rstep = kNormThreads / vecs;
    // three parts an SM, as far as rows go round; no more than the part's shared memory holds, no fewer than a few rows a thread
    const int64_t most = static_cast<int64_t>(kNormPartBytes / (kNormThreads * vec * size)) * rstep;
    const int64_t want = std::max<int64_t>(1, 3 * 148 / std::max<int64_t>(1, samples * plan.blocks));
    int64_t part = std::max<int64_t>((rows + want - 1) / want, 4 * rstep);
    plan.part_rows = static_cast<int>(std::min(part, most));
    plan.parts = static_cast<int>((rows + plan.part_rows - 1) / plan.part_rows);
    return plan;
}

constexpr int kShortValues = 512;  // values of a (sample, group) that stay in the registers of a warp (1024: 65536 groups 100 -> 150 us and more)
bool short_groups(int64_t rows, int width) { return rows * width <= kShortValues; }

template <typename T, int V>
int launch_rows(const GroupNormParams& p, cudaStream_t st) {
    int lpr = 1;
    while (lpr < 32 && lpr * V < p.width) lpr *= 2;
    const int passes = (p.width + lpr * V - 1) / (lpr * V);
    auto launch = [&](auto kernel, int unroll) -> int {
        // (a CTA goes on to further rows while weight and bias stay where they are: as many CTAs as fit the SMs at once)
        const long long bx = (p.groups + 256 / lpr - 1) / (256 / lpr), slots = std::max<long long>(1, (passes > 1 ? 2 : 4) * 148 / bx);
        const long long by = std::min<long long>(std::min<long long>((p.n + unroll - 1) / unroll, slots), 65535);
        GDN_CUDA(launch_dependent(kernel, dim3(static_cast<unsigned>(bx), static_cast<unsigned>(by)), 256, 0, st, p));
        return GDN_OK;
    };
    auto pick = [&](auto gated) -> int {
        constexpr bool kG = decltype(gated)::value;
        switch (passes > 1 ? 32 * passes : lpr) {
            case 1: return launch(gdn_group_norm_rows_kernel<T, V, 1, 1, kG>, 2);
            case 2: return launch(gdn_group_norm_rows_kernel<T, V, 2, 1, kG>, 2);
            case 4: return launch(gdn_group_norm_rows_kernel<T, V, 4, 1, kG>, 2);
            case 8: return launch(gdn_group_norm_rows_kernel<T, V, 8, 1, kG>, 2);
            case 16: return launch(gdn_group_norm_rows_kernel<T, V, 16, 1, kG>, 2);
            case 32: return launch(gdn_group_norm_rows_kernel<T, V, 32, 1, kG>, 2);
            case 64: return launch(gdn_group_norm_rows_kernel<T, V, 32, 2, kG>, 1);
            default: return launch(gdn_group_norm_rows_kernel<T, V, 32, 4, kG>, 1);
        }
    };
    return p.z ? pick(std::true_type{}) : pick(std::false_type{});
}

template <typename T, int V>
int launch_short(const GroupNormParams& p, cudaStream_t st) {
    const long long size = p.l * p.width;
    if (p.l == 1 && size <= 4 * 32 * V) return launch_rows<T, V>(p, st);
    int lpr = 4;
    while (lpr < 32 && lpr * V < size) lpr *= 2;
    const int passes = static_cast<int>((size + lpr * V - 1) / (lpr * V));
    const long long per_block = 8ll * (32 / lpr), blocks = (p.n * p.groups + per_block - 1) / per_block;
    GDN_REQUIRE(blocks < (1ll << 31), "gdn_group_norm: too many samples");
    auto launch = [&](auto kernel) { return launch_dependent(kernel, dim3(static_cast<unsigned>(blocks)), 256, 0, st, p); };
    if (lpr == 4) GDN_CUDA(launch(gdn_group_norm_short_kernel<T, V, 4, 1>));
    else if (lpr == 8) GDN_CUDA(launch(gdn_group_norm_short_kernel<T, V, 8, 1>));
    else if (lpr == 16) GDN_CUDA(launch(gdn_group_norm_short_kernel<T, V, 16, 1>));
    else if (passes <= 1) GDN_CUDA(launch(gdn_group_norm_short_kernel<T, V, 32, 1>));
    else if (passes <= 4) GDN_CUDA(launch(gdn_group_norm_short_kernel<T, V, 32, 4>));
    else GDN_CUDA(launch(gdn_group_norm_short_kernel<T, V, 32, 32>));
    return GDN_OK;
}

constexpr long long kMostSamples = 65535;  // of a launch in parts

template <typename T, int V>
int launch_parts(GroupNormParams p, const NormPlan& plan, cudaStream_t st) {
    GDN_REQUIRE(plan.blocks <= kMostSamples, "gdn_group_norm: too many channels");
    if (p.n > kMostSamples) {  // a grid's limit: in turn, with the same workspace
        for (long long first = 0; first < p.n; first += kMostSamples) {
            GroupNormParams q = p;
            q.n = std::min<long long>(p.n - first, kMostSamples);
            q.x = static_cast<const T*>(p.x) + first * p.x_sn;
            q.y = static_cast<T*>(p.y) + first * p.y_sn;
            if (p.z) q.z = static_cast<const T*>(p.z) + first * p.z_sn;
            if (int rc = launch_parts<T, V>(q, plan, st)) return rc;
        }
        return GDN_OK;
    }
    p.part_rows = plan.part_rows;
    p.parts = plan.parts;
    p.block_channels = plan.block_channels;
    p.split = plan.split;
    const dim3 grid(static_cast<unsigned>(plan.parts), static_cast<unsigned>(plan.blocks), static_cast<unsigned>(p.n));
    const int rstep = kNormThreads / (plan.block_channels / V), smem = (plan.part_rows + rstep - 1) / rstep * kNormThreads * V * static_cast<int>(sizeof(T));
    if (int rc = set_smem<gdn_group_norm_stats_kernel<T, V>>(kNormPartBytes)) return rc;
    GDN_CUDA(launch_dependent(gdn_group_norm_stats_kernel<T, V>, grid, kNormThreads, smem, st, p));
    p.join = p.partial;
    p.join_rows = p.part_rows;
    p.join_parts = p.parts;
    if (p.parts > kNormJoinParts || p.split > 1) {
        p.join = p.partial + static_cast<size_t>(p.n) * p.parts * p.groups * p.split;
        p.join_rows = p.l;
        p.join_parts = 1;
        const long long blocks = (p.n * p.groups + 7) / 8;
        GDN_REQUIRE(blocks < (1ll << 31), "gdn_group_norm: too many samples");
        GDN_CUDA(launch_dependent(gdn_group_norm_join_kernel, dim3(static_cast<unsigned>(blocks)), 256, 0, st, p));
    }
    // CTAs of the second launch: three fit an SM; no fewer than eight rows a thread
    const long long want = std::max<long long>(1, 3 * 148 / std::max<long long>(1, p.n * plan.blocks));
    p.apply_rows = static_cast<int>(std::min<long long>(std::max<long long>((p.l + want - 1) / want, 8 * rstep), 1 << 20));
    const dim3 apply(static_cast<unsigned>((p.l + p.apply_rows - 1) / p.apply_rows), static_cast<unsigned>(plan.blocks), static_cast<unsigned>(p.n));
    GDN_CUDA(launch_dependent(p.z ? gdn_group_norm_apply_kernel<T, V, true> : gdn_group_norm_apply_kernel<T, V, false>, apply, kNormThreads, 0, st, p));
    return GDN_OK;
}

// Groups that are too wide for a sweep of a CTA's threads.  A CTA each, in one launch, where that takes it few sweeps (24 groups of 4 sweeps 9 : 18 us in
// pieces, of 16 24 : 17, of 64 96 : 18), or not many and there are as many groups as CTAs fit the SMs (2500 groups of 16 sweeps 217 : 231, 4000 of 36 174 : 411, but 2500 of 32
// 450 : 287); otherwise in pieces (one group of 16384 sweeps 36600 : 69 us, 300 of 64 162 : 63, 3000 of 600 2980 : 1190).
bool wide_groups(long long count, int64_t rows, int width, int vec) {
    const int64_t sweeps = rows * ((width + kNormThreads * vec - 1) / (kNormThreads * vec));
    return sweeps <= 12 || (sweeps <= 64 && count >= 8 * 148);
}

template <typename T, int V>
int launch_long(GroupNormParams p, const NormPlan& plan, cudaStream_t st) {
    if (plan.split > 1 && wide_groups(p.n * p.groups, p.l, p.width, V)) {
        GDN_REQUIRE(p.n * p.groups < (1ll << 31), "gdn_group_norm: too many samples");
        GDN_CUDA(launch_dependent(gdn_group_norm_wide_kernel<T, V>, dim3(static_cast<unsigned>(p.n * p.groups)), kNormThreads, 0, st, p));
        return GDN_OK;
    }
    return launch_parts<T, V>(p, plan, st);
}

// Shared memory of a CTA of `threads` that keeps a (sample, group); 0: it does not fit.
int whole_bytes(int64_t rows, int width, int vec, int size, int threads) {
    if (vec * size < 4 || width % vec != 0 || width / vec > threads) return 0;
    const int rstep = threads / (width / vec);
    const int64_t bytes = (rows + rstep - 1) / rstep * threads * vec * size;
    return bytes <= kNormWholeBytes ? static_cast<int>(bytes) : 0;
}
// One launch that reads x once is faster than two or three that read it twice (4 x 32 groups of 16 KB 8.5 -> 2.8 us, of 64 KB 18 -> 7,
// of 150 KB 24 -> 14), except where
//  - very many groups are so small that the CTAs' turn-over shows (65536 groups of 2 KB, 32 a sample, 99 -> 280 us, 8 a sample 187 -> 276; with few a
//    sample the sums of a part are long instead: 4 378 -> 275, 2 915 -> 273; of few rows they are not, 4 rows of 4 x 256 channels 307 -> 496), or
//  - a group's piece of a row is not whole sectors of 32 bytes: copies of less than 16 bytes go through L1, of which the tile leaves little (20
//    channels, bf16, 32 groups of 200 KB 21 -> 30 us, of 150 KB 20 -> 16), and where CTAs come in several waves, or read a gate as well, the
//    sectors that groups share move twice (512 groups of 64 KB 33 -> 42 us, 256 of 40 KB 20 -> 14; gated, 512 of 48 KB 30 -> 42, of 16 KB 19 -> 11).
bool whole_groups(int64_t samples, int groups, int64_t rows, int width, int vec, int size, bool gated) {
    const int bytes = whole_bytes(rows, width, vec, size, 512);
    const int64_t count = samples * groups;
    if (bytes == 0 || (rows * width * size < 16 * 1024 && count > 2048 && (groups > 4 || rows < 32))) return false;
    return width * size % 32 == 0 || bytes <= (gated ? 24 : count > 148 ? 48 : 176) * 1024;
}

template <typename T, int V>
int launch_whole(const GroupNormParams& p, cudaStream_t st) {
    GDN_REQUIRE(p.n * p.groups < (1ll << 31), "gdn_group_norm: too many samples");
    auto launch = [&](auto gated) -> int {
        constexpr bool kG = decltype(gated)::value;
        const int small = whole_bytes(p.l, p.width, V, sizeof(T), 256);
        const unsigned grid = static_cast<unsigned>(p.n * p.groups);
        // (512 groups of 64 KB: 29 us with CTAs of 1024 threads, 20 with three of 256 on an SM; of 100 KB 41 with 1024 and 31 with two of 512; of 150 KB
        // 51 with either.  Copies that go through L1 are better few at a time: 128 groups of 160 KB, 20 channels, 20 us with 512, 19 with 256)
        if (small > 0 && (small <= kNormPartBytes || V * sizeof(T) < 16)) {
            if (int rc = set_smem<gdn_group_norm_whole_kernel<T, V, 256, kG>>(kNormWholeBytes)) return rc;
            GDN_CUDA(launch_dependent(gdn_group_norm_whole_kernel<T, V, 256, kG>, grid, 256, small, st, p));
        } else {
            if (int rc = set_smem<gdn_group_norm_whole_kernel<T, V, 512, kG>>(kNormWholeBytes)) return rc;
            GDN_CUDA(launch_dependent(gdn_group_norm_whole_kernel<T, V, 512, kG>, grid, 512, whole_bytes(p.l, p.width, V, sizeof(T), 512), st, p));
        }
        return GDN_OK;
    };
    return p.z ? launch(std::true_type{}) : launch(std::false_type{});
}

template <typename T, int V>
int launch_norm(const GroupNormParams& p, bool is_short, bool is_whole, const GdnGroupNormArgs& a, cudaStream_t st) {
    if (is_short) return launch_short<T, V>(p, st);
    if constexpr (V * sizeof(T) >= 4)
        if (is_whole) return launch_whole<T, V>(p, st);
    return launch_long<T, V>(p, norm_plan(a.samples, a.rows, a.channels, a.groups, V, sizeof(T)), st);
}

}  // namespace

extern "C" {

// An upper bound over the vector widths, which go by the type, pointers and strides.
size_t gdn_group_norm_workspace_bytes(int64_t samples, int64_t rows, int32_t channels, int32_t groups) {
    if (samples <= 0 || rows <= 0 || groups <= 0 || channels <= 0 || channels % groups != 0 || short_groups(rows, channels / groups)) return 0;
    size_t entries = 0;  // of a sample and group
    for (int size = 2; size <= 4; size *= 2)
        for (int v = 1; v * size <= 16; v *= 2)
            if ((channels / groups > kNormThreads ? channels / groups : channels) % v == 0) {
                const NormPlan plan = norm_plan(samples, rows, channels, groups, v, size);
                entries = std::max(entries, static_cast<size_t>(plan.parts) * plan.split);
            }
    return (entries + 1) * static_cast<size_t>(samples) * groups * sizeof(float2);  // (one more: the parts joined)
}

int gdn_group_norm(const GdnGroupNormArgs* a, gdn_stream_t stream) {
    GDN_REQUIRE(a != nullptr, "gdn_group_norm: args is NULL");
    GDN_REQUIRE(a->samples >= 0 && a->rows >= 0 && a->channels > 0 && a->groups > 0 && a->channels % a->groups == 0,
                "gdn_group_norm: channels (%d) must be a positive multiple of groups (%d)", a->channels, a->groups);
    GDN_REQUIRE(a->dtype == GDN_BF16 || a->dtype == GDN_F32, "gdn_group_norm: dtype must be bf16 or f32");
    GDN_REQUIRE(a->param_dtype == GDN_BF16 || a->param_dtype == GDN_F32, "gdn_group_norm: param_dtype must be bf16 or f32");
    DeviceInfo* d = nullptr;
    if (int rc = get_device_info(&d)) return rc;
    if (a->samples == 0 || a->rows == 0) return GDN_OK;
    GDN_REQUIRE(a->x && a->y, "gdn_group_norm: x and y are required");
    GroupNormParams p{};
    p.x = a->x; p.z = a->z; p.y = a->y; p.weight = a->weight; p.bias = a->bias;
    p.param_f32 = a->param_dtype == GDN_F32;
    p.n = a->samples; p.l = a->rows;
    p.channels = a->channels; p.groups = a->groups; p.width = a->channels / a->groups;
    p.x_sn = a->x_stride_sample; p.x_sl = a->x_stride_row;
    p.z_sn = a->z_stride_sample; p.z_sl = a->z_stride_row;
    p.y_sn = a->y_stride_sample; p.y_sl = a->y_stride_row;
    p.eps = a->eps; p.silu = a->silu != 0;
    const bool is_short = short_groups(a->rows, p.width);
    if (!is_short) {
        const size_t need = gdn_group_norm_workspace_bytes(a->samples, a->rows, a->channels, a->groups);
        if (need > 0 && (!a->workspace || a->workspace_bytes < need || !aligned16(a->workspace)))
            return fail(GDN_ERR_WORKSPACE, "gdn_group_norm: workspace of %zu bytes (16-byte aligned) required, got %zu", need, a->workspace_bytes);
        p.partial = static_cast<float2*>(a->workspace);
    }
    // the widest access, up to 16 bytes, that pointers, strides and (where lanes share a group) the group's width allow
    const int size = a->dtype == GDN_F32 ? 4 : 2;
    auto fits = [&](int v, bool lanes_share) {  // lanes of one group: its width is whole vectors
        auto whole = [&](const void* ptr, int64_t sn, int64_t sl) {
            return reinterpret_cast<uintptr_t>(ptr) % (static_cast<unsigned>(v * size)) == 0 && (a->samples == 1 || sn % v == 0) && (a->rows == 1 || sl % v == 0);
        };
        return (lanes_share ? p.width : p.channels) % v == 0 && whole(p.x, p.x_sn, p.x_sl) && whole(p.y, p.y_sn, p.y_sl) &&
               (!p.z || whole(p.z, p.z_sn, p.z_sl));
    };
    auto widest = [&](bool lanes_share) {
        int v = 16 / size;
        while (!fits(v, lanes_share)) v /= 2;
        return v;
    };
    const int shared = widest(true);
    const bool is_whole = !is_short && whole_groups(a->samples, a->groups, a->rows, p.width, shared, size, p.z != nullptr);
    const int v = is_short || is_whole || p.width > kNormThreads ? shared : widest(false);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a->dtype == GDN_F32) {
        if (v == 4) return launch_norm<float, 4>(p, is_short, is_whole, *a, st);
        if (v == 2) return launch_norm<float, 2>(p, is_short, is_whole, *a, st);
        return launch_norm<float, 1>(p, is_short, is_whole, *a, st);
    }
    if (v == 8) return launch_norm<__nv_bfloat16, 8>(p, is_short, is_whole, *a, st);
    if (v == 4) return launch_norm<__nv_bfloat16, 4>(p, is_short, is_whole, *a, st);
    if (v == 2) return launch_norm<__nv_bfloat16, 2>(p, is_short, is_whole, *a, st);
    return launch_norm<__nv_bfloat16, 1>(p, is_short, is_whole, *a, st);
}

}  // extern "C"
