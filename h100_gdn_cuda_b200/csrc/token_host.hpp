// Host-side pieces shared by the entry points that run tcgen05 kernels on token tensors: tensor maps, the views the kernels
// see, checks of states and per-token scalars, the shared-memory limit of a kernel.
#pragma once
#include <atomic>

#include "host_common.hpp"
#include "kernels/prefill_common.cuh"
#include "tma_host.hpp"

namespace gdn {

// 4-D map over a token tensor: (dim, head, token, batch), box 64 x 1 x 64 x 1, 128-byte swizzle.
// `dim` below 128 (a multiple of 8): loads fill the columns past it with zeros and stores leave them out,
// so a kernel built for 128 sees a zero-padded head without a padded copy in memory.
inline int make_token_map(CUtensorMap* out, const GdnTokenTensor& t, const GdnShape& s, int heads, const char* name, int dim = 128) {
    const bool packed = s.cu_seqlens != nullptr;
    const uint64_t tokens = packed ? static_cast<uint64_t>(s.total_tokens) : static_cast<uint64_t>(s.seq_len);
    const uint64_t batch = packed ? 1 : static_cast<uint64_t>(s.batch);
    uint64_t dims[4] = {static_cast<uint64_t>(dim), static_cast<uint64_t>(heads), tokens, batch};
    uint64_t sb = static_cast<uint64_t>(t.stride_batch) * 2;
    if (packed || sb == 0) sb = std::max<uint64_t>(16, tokens * static_cast<uint64_t>(t.stride_token) * 2);
    uint64_t strides[3] = {static_cast<uint64_t>(t.stride_head) * 2, static_cast<uint64_t>(t.stride_token) * 2, sb};
    if (heads == 1 && strides[0] == 0) strides[0] = static_cast<uint64_t>(dim) * 2;
    uint32_t box[4] = {64, 1, 64, 1};
    if (tokens == 0) return fail(GDN_ERR_INVALID, "%s: no tokens", name);
    if (!make_tmap_bf16(out, t.ptr, 4, dims, strides, box, true))
        return fail(GDN_ERR_CUDA, "could not encode the TMA descriptor of %s (strides %llu/%llu/%llu bytes)", name,
                    (unsigned long long)strides[0], (unsigned long long)strides[1], (unsigned long long)strides[2]);
    return GDN_OK;
}

inline ScalarView scalar_view(const GdnTokenScalar& t) {
    ScalarView v;
    v.ptr = t.ptr;
    v.is_f32 = t.dtype == GDN_F32;
    v.sb = t.stride_batch;
    v.st = t.stride_token;
    v.sh = t.stride_head;
    return v;
}
inline TokenView token_view(const GdnTokenTensor& t) {
    TokenView v;
    v.ptr = static_cast<__nv_bfloat16*>(t.ptr);
    v.sb = t.stride_batch;
    v.st = t.stride_token;
    v.sh = t.stride_head;
    return v;
}
// States are read and written with 16-byte accesses.
inline int check_state(const GdnState& t, const char* name) {
    if (!t.ptr) return GDN_OK;
    GDN_REQUIRE(aligned16(t.ptr) && t.stride_seq % 8 == 0 && t.stride_head % 8 == 0,
                "%s must be 16-byte aligned with strides that are multiples of 8 elements", name);
    return GDN_OK;
}
inline int check_scalar(const GdnTokenScalar& t, const char* name, bool required) {
    if (!t.ptr) {
        GDN_REQUIRE(!required, "%s is NULL", name);
        return GDN_OK;
    }
    GDN_REQUIRE(t.dtype == GDN_BF16 || t.dtype == GDN_F32, "%s dtype must be bf16 or f32", name);
    return GDN_OK;
}

// The kernel's dynamic shared-memory limit, raised once per device (the attribute call is a good part of a
// microsecond, and a short prompt's call lasts a few).
template <auto kKernel>
int set_smem(int bytes) {
    static std::atomic<bool> done[64];
    int dev = 0;
    GDN_CUDA(cudaGetDevice(&dev));
    if (dev >= 0 && dev < 64 && done[dev].load(std::memory_order_acquire)) return GDN_OK;
    GDN_CUDA(cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    if (dev >= 0 && dev < 64) done[dev].store(true, std::memory_order_release);
    return GDN_OK;
}

}  // namespace gdn
