// C-ABI entry points of linear attention with decay (see include/gdn_b200.h): argument checks and launches.
#include "kernels/linear_recurrent.cuh"
#include "token_host.hpp"

using namespace gdn;

namespace {

// Token tensors of this path: 16-byte accesses (tensor copies in prompts), so no axis longer than one may be broadcast.
int check_linear_tokens(const GdnTokenTensor& t, const GdnShape& s, int heads, int dim, const char* name) {
    if (int rc = check_token_tensor(t, name, dim)) return rc;
    const bool packed = s.cu_seqlens != nullptr;
    GDN_REQUIRE((heads == 1 || t.stride_head >= dim) && (packed || s.batch == 1 || t.stride_batch > 0) && ((packed ? s.total_tokens : s.seq_len) <= 1 || t.stride_token > 0),
                "%s: strides must be positive (broadcast axes are not supported)", name);
    return GDN_OK;
}

int check_linear_shape(const GdnShape& s, const char* who) {
    if (int rc = check_shape(s, false)) return rc;
    GDN_REQUIRE(s.head_dim_k % 8 == 0 && s.head_dim_k <= 256, "%s: dk must be a multiple of 8 up to 256 (got %d)", who, s.head_dim_k);
    GDN_REQUIRE(s.head_dim_v % 8 == 0, "%s: dv must be a multiple of 8 (got %d)", who, s.head_dim_v);
    return GDN_OK;
}

template <bool kF32>
int launch_linear_recurrent(const LinRecurrentParams& p, cudaStream_t st) {
    const long long grid = static_cast<long long>(p.batch) * p.vh * ((p.dv + kLinRows - 1) / kLinRows);
    GDN_REQUIRE(grid < (1ll << 31), "gdn_linear_recurrent: too many state tiles");
    const dim3 g(static_cast<unsigned>(grid));
    if (p.dk <= 64) GDN_CUDA(launch_dependent(gdn_linear_recurrent_kernel<8, kF32>, g, kLinThreads, 0, st, p));
    else if (p.dk <= 128) GDN_CUDA(launch_dependent(gdn_linear_recurrent_kernel<16, kF32>, g, kLinThreads, 0, st, p));
    else GDN_CUDA(launch_dependent(gdn_linear_recurrent_kernel<32, kF32>, g, kLinThreads, 0, st, p));
    return GDN_OK;
}

}  // namespace

extern "C" {

int gdn_linear_recurrent(const GdnLinearRecurrentArgs* a, gdn_stream_t stream) {
    GDN_REQUIRE(a != nullptr, "gdn_linear_recurrent: args is NULL");
    const GdnShape& s = a->shape;
    if (int rc = check_linear_shape(s, "gdn_linear_recurrent")) return rc;
    GDN_REQUIRE(a->state_dtype == GDN_BF16 || a->state_dtype == GDN_F32, "gdn_linear_recurrent: state_dtype must be bf16 or f32");
    if (s.cu_seqlens == nullptr || s.total_tokens > 0) {
        if (int rc = check_linear_tokens(a->q, s, s.num_k_heads, s.head_dim_k, "q")) return rc;
        if (int rc = check_linear_tokens(a->k, s, s.num_k_heads, s.head_dim_k, "k")) return rc;
        if (int rc = check_linear_tokens(a->v, s, s.num_v_heads, s.head_dim_v, "v")) return rc;
        if (int rc = check_linear_tokens(a->out, s, s.num_v_heads, s.head_dim_v, "out")) return rc;
    }
    if (int rc = check_scalar(a->gate, "gate", false)) return rc;
    if (int rc = check_state(a->state_in, "state_in")) return rc;
    if (int rc = check_state(a->state_out, "state_out")) return rc;
    GDN_REQUIRE(!(a->store_step_state && !a->state_out.ptr), "gdn_linear_recurrent: step states need state_out");
    GDN_REQUIRE(!(a->store_step_state && a->state_in.ptr && a->state_in.ptr == a->state_out.ptr),
                "gdn_linear_recurrent: state_out may not alias state_in when step states are stored");
    GDN_REQUIRE(!(a->state_indices && a->store_step_state), "gdn_linear_recurrent: state_indices cannot be combined with step states");
    GDN_REQUIRE(!a->state_indices || (a->state_in.ptr && a->num_slots > 0), "gdn_linear_recurrent: state_indices needs a state_in pool of num_slots slots");
    DeviceInfo* d = nullptr;
    if (int rc = get_device_info(&d)) return rc;
    LinRecurrentParams p{};
    p.q = token_view(a->q); p.k = token_view(a->k); p.v = token_view(a->v); p.out = token_view(a->out);
    p.gate = scalar_view(a->gate);
    p.state_in = a->state_in.ptr; p.si_ss = a->state_in.stride_seq; p.si_sh = a->state_in.stride_head;
    p.state_out = a->state_out.ptr; p.so_ss = a->state_out.stride_seq; p.so_sh = a->state_out.stride_head;
    p.cu_seqlens = s.cu_seqlens;
    p.num_accepted = a->num_accepted_tokens;
    p.state_idx = a->state_indices;
    p.total_tokens = s.total_tokens;
    p.batch = s.batch; p.seq_len = s.seq_len; p.kh = s.num_k_heads; p.vh = s.num_v_heads; p.dk = s.head_dim_k; p.dv = s.head_dim_v;
    p.num_slots = a->num_slots;
    p.store_step = a->store_step_state != 0;
    p.scale = a->scale;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return a->state_dtype == GDN_F32 ? launch_linear_recurrent<true>(p, st) : launch_linear_recurrent<false>(p, st);
}

size_t gdn_linear_chunked_workspace_bytes(const GdnShape*) { return 0; }

int gdn_linear_chunked(const GdnLinearChunkedArgs* a, gdn_stream_t stream) {
    GDN_REQUIRE(a != nullptr, "gdn_linear_chunked: args is NULL");
    GdnLinearRecurrentArgs r{};
    r.shape = a->shape;
    r.q = a->q; r.k = a->k; r.v = a->v; r.out = a->out;
    r.gate = a->gate;
    r.state_in = a->initial_state;
    r.state_out = a->final_state;
    r.scale = a->scale;
    r.state_dtype = a->state_dtype;
    return gdn_linear_recurrent(&r, stream);
}

}  // extern "C"
