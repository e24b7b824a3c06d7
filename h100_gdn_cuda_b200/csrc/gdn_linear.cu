// C-ABI entry points of linear attention with decay (see include/gdn_b200.h): argument checks and launches.
#include "heuristics.hpp"
#include "kernels/linear_chunked.cuh"
#include "kernels/linear_recurrent.cuh"
#include "kernels/linear_segments.cuh"
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

// One memory for the state that is read and the one that is written: a block of it is then the same (sequence, head) of both.
int check_in_place(const GdnState& in, const GdnState& out, const GdnShape& s, bool several, const char* who) {
    GDN_REQUIRE(!in.ptr || in.ptr != out.ptr || ((!several || in.stride_seq == out.stride_seq) && (s.num_v_heads == 1 || in.stride_head == out.stride_head)),
                "%s: the state may be updated in place only with the same strides", who);
    return GDN_OK;
}

template <bool kF32>
int launch_linear_recurrent(const LinRecurrentParams& p, cudaStream_t st) {
    const long long grid = static_cast<long long>(p.batch) * p.vh * ((p.dv + kLinRows - 1) / kLinRows);
    GDN_REQUIRE(grid < (1ll << 31), "gdn_linear_recurrent: too many state tiles");
    const dim3 g(static_cast<unsigned>(grid));
    if (!p.cu_seqlens && p.seq_len == 1 && !p.num_accepted) {  // (a state per token is then a state per sequence)
        if (p.dk <= 64) GDN_CUDA(launch_dependent(gdn_linear_decode_kernel<8, kF32>, g, kLinThreads, 0, st, p));
        else if (p.dk <= 128) GDN_CUDA(launch_dependent(gdn_linear_decode_kernel<16, kF32>, g, kLinThreads, 0, st, p));
        else GDN_CUDA(launch_dependent(gdn_linear_decode_kernel<32, kF32>, g, kLinThreads, 0, st, p));
        return GDN_OK;
    }
    if (p.dk <= 64) GDN_CUDA(launch_dependent(gdn_linear_recurrent_kernel<8, kF32>, g, kLinThreads, 0, st, p));
    else if (p.dk <= 128) GDN_CUDA(launch_dependent(gdn_linear_recurrent_kernel<16, kF32>, g, kLinThreads, 0, st, p));
    else GDN_CUDA(launch_dependent(gdn_linear_recurrent_kernel<32, kF32>, g, kLinThreads, 0, st, p));
    return GDN_OK;
}

// Tensor map of a token tensor; an axis of one token or head may come with any stride, the map wants a positive one.  `columns` > 0: of rank 5,
// (64 columns, tokens, column blocks, heads, batch), for boxes of `columns` columns and 64 tokens; otherwise as make_token_map has it.
int linear_map(CUtensorMap* out, GdnTokenTensor t, const GdnShape& s, int heads, int dim, const char* name, int columns = 0) {
    if (heads == 1) t.stride_head = dim;
    const int64_t tokens = s.cu_seqlens ? s.total_tokens : s.seq_len;
    if (tokens == 1) t.stride_token = std::max<int64_t>(t.stride_token, static_cast<int64_t>(heads) * t.stride_head);
    if (columns == 0) return make_token_map(out, t, s, heads, name, dim);
    const bool packed = s.cu_seqlens != nullptr;
    const uint64_t batch = packed ? 1 : static_cast<uint64_t>(s.batch);
    uint64_t sb = static_cast<uint64_t>(t.stride_batch) * 2;
    if (packed || sb == 0) sb = std::max<uint64_t>(16, static_cast<uint64_t>(tokens * t.stride_token) * 2);
    const uint64_t dims[5] = {64, static_cast<uint64_t>(tokens), static_cast<uint64_t>(dim / 64), static_cast<uint64_t>(heads), batch};
    const uint64_t strides[4] = {static_cast<uint64_t>(t.stride_token) * 2, 128, static_cast<uint64_t>(t.stride_head) * 2, sb};
    const uint32_t box[5] = {64, 64, static_cast<uint32_t>(columns / 64), 1, 1};
    if (!make_tmap_bf16(out, t.ptr, 5, dims, strides, box, true)) return fail(GDN_ERR_CUDA, "could not encode the TMA descriptor of %s", name);
    return GDN_OK;
}

bool wide_linear(const GdnShape& s) { return s.head_dim_k > 128; }

// Items of a problem (see LinChunkedParams), and where the segments' states lie in the workspace: [states][decays], one each per item behind `whole`.
struct LinearPlan {
    long long whole, items, cut_chains;  // cut_chains: chains in segments (packed: all, if any)
    int seg_chunks, num_segments, by_length;
    size_t states, bytes;  // 0: no segments
};
LinearPlan linear_plan(const GdnShape& s) {
    const bool packed = s.cu_seqlens != nullptr;
    const long long tokens = packed ? s.total_tokens : s.seq_len, chunks = std::max<long long>(1, (tokens + kChunk - 1) / kChunk);
    const long long per = static_cast<long long>(s.num_v_heads) * ((s.head_dim_v + 127) / 128), chains = s.batch * per;
    LinearPlan plan{};
    plan.whole = plan.items = chains;
    plan.num_segments = 1;
    plan.seg_chunks = static_cast<int>(chunks);
    plan.by_length = packed && s.batch > 1 && s.batch <= kLinRankedSeqs;
    const LinearCut cut = linear_cut(chains, packed ? (chunks + s.batch - 1) / s.batch : chunks, packed);
    if (cut.segments <= 1) return plan;
    plan.seg_chunks = static_cast<int>(cut.seg_chunks);
    if (packed) {
        plan.by_length = 0;
        plan.whole = 0;
        plan.cut_chains = chains;
        plan.items = (s.batch + tokens / (static_cast<long long>(kChunk) * plan.seg_chunks)) * per;
    } else {
        plan.num_segments = static_cast<int>(cut.segments);
        plan.whole = cut.whole;
        plan.cut_chains = chains - cut.whole;
        plan.items = cut.whole + plan.cut_chains * cut.segments;
    }
    const size_t places = static_cast<size_t>(plan.items - plan.whole);
    plan.states = places * 128 * (s.head_dim_k <= 64 ? 64 : 128) * sizeof(float);
    plan.bytes = plan.states + (places * sizeof(float) + 255) / 256 * 256;
    return plan;
}

template <int DK, int DV, bool kWhole, bool kF32>
int launch_linear_chunked(const GdnLinearChunkedArgs& a, const LinChunkedParams& p, long long cut_chains, cudaStream_t st) {
    using L = LinSmem<DK, DV>;
    using LS = LinSegSmem<DK, DV>;
    const GdnShape& s = a.shape;
    CUtensorMap tmQ, tmK, tmV, tmO;
    if (int rc = linear_map(&tmQ, a.q, s, s.num_k_heads, s.head_dim_k, "q", kWhole ? DK : 0)) return rc;
    if (int rc = linear_map(&tmK, a.k, s, s.num_k_heads, s.head_dim_k, "k", kWhole ? DK : 0)) return rc;
    if (int rc = linear_map(&tmV, a.v, s, s.num_v_heads, s.head_dim_v, "v", kWhole ? DV : 0)) return rc;
    if (int rc = linear_map(&tmO, a.out, s, s.num_v_heads, s.head_dim_v, "out")) return rc;
    if (int rc = set_smem<gdn_linear_chunked_kernel<DK, DV, kWhole, kF32>>(L::kBytes)) return rc;
    cudaLaunchConfig_t cfg{};
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (p.seg_state) {
        if (int rc = set_smem<gdn_linear_segment_kernel<DK, DV, kWhole>>(LS::kBytes)) return rc;
        cfg.gridDim = dim3(static_cast<unsigned>(p.num_items - p.whole));
        cfg.blockDim = dim3(lin::kSegThreads);
        cfg.dynamicSmemBytes = LS::kBytes;
        GDN_CUDA(cudaLaunchKernelEx(&cfg, gdn_linear_segment_kernel<DK, DV, kWhole>, tmK, tmV, p));
        cfg.gridDim = dim3(static_cast<unsigned>(cut_chains), 128 * DK / 4 / kLinCombineThreads);
        cfg.blockDim = dim3(kLinCombineThreads);
        cfg.dynamicSmemBytes = 0;
        GDN_CUDA(cudaLaunchKernelEx(&cfg, gdn_linear_combine_kernel, p, DK));
    }
    cfg.gridDim = dim3(static_cast<unsigned>(p.num_items));
    cfg.blockDim = dim3(lin::kThreads);
    cfg.dynamicSmemBytes = L::kBytes;
    GDN_CUDA(cudaLaunchKernelEx(&cfg, gdn_linear_chunked_kernel<DK, DV, kWhole, kF32>, tmQ, tmK, tmV, tmO, p));
    return GDN_OK;
}

template <bool kF32>
int launch_linear_shape(const GdnLinearChunkedArgs& a, const LinChunkedParams& p, long long cut_chains, cudaStream_t st) {
    // (a single column block needs no rank 5: its map clips what is missing)
    const bool whole = p.dk == 128 && p.dv % 128 == 0;
    if (p.dk <= 64 && p.dv <= 64) return launch_linear_chunked<64, 64, false, kF32>(a, p, cut_chains, st);
    if (p.dk <= 64) return launch_linear_chunked<64, 128, false, kF32>(a, p, cut_chains, st);
    if (p.dv <= 64) return launch_linear_chunked<128, 64, false, kF32>(a, p, cut_chains, st);
    return whole ? launch_linear_chunked<128, 128, true, kF32>(a, p, cut_chains, st) : launch_linear_chunked<128, 128, false, kF32>(a, p, cut_chains, st);
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
    if (int rc = check_in_place(a->state_in, a->state_out, s, s.batch > 1 || a->state_indices, "gdn_linear_recurrent")) return rc;
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

size_t gdn_linear_chunked_workspace_bytes(const GdnShape* s) {
    if (!s || wide_linear(*s) || check_linear_shape(*s, "gdn_linear_chunked_workspace_bytes") != GDN_OK) return 0;
    return linear_plan(*s).bytes;
}

int gdn_linear_chunked(const GdnLinearChunkedArgs* a, gdn_stream_t stream) {
    GDN_REQUIRE(a != nullptr, "gdn_linear_chunked: args is NULL");
    const GdnShape& s = a->shape;
    if (int rc = check_linear_shape(s, "gdn_linear_chunked")) return rc;
    const long long tokens = s.cu_seqlens ? s.total_tokens : static_cast<long long>(s.batch) * s.seq_len;
    if (wide_linear(s) || tokens == 0) {  // (no tokens: the states are handed through)
        GdnLinearRecurrentArgs r{};
        r.shape = s;
        r.q = a->q; r.k = a->k; r.v = a->v; r.out = a->out;
        r.gate = a->gate;
        r.state_in = a->initial_state;
        r.state_out = a->final_state;
        r.scale = a->scale;
        r.state_dtype = a->state_dtype;
        return gdn_linear_recurrent(&r, stream);
    }
    GDN_REQUIRE(a->state_dtype == GDN_BF16 || a->state_dtype == GDN_F32, "gdn_linear_chunked: state_dtype must be bf16 or f32");
    if (int rc = check_linear_tokens(a->q, s, s.num_k_heads, s.head_dim_k, "q")) return rc;
    if (int rc = check_linear_tokens(a->k, s, s.num_k_heads, s.head_dim_k, "k")) return rc;
    if (int rc = check_linear_tokens(a->v, s, s.num_v_heads, s.head_dim_v, "v")) return rc;
    if (int rc = check_linear_tokens(a->out, s, s.num_v_heads, s.head_dim_v, "out")) return rc;
    if (int rc = check_scalar(a->gate, "gate", false)) return rc;
    if (int rc = check_state(a->initial_state, "initial_state")) return rc;
    if (int rc = check_state(a->final_state, "final_state")) return rc;
    if (int rc = check_in_place(a->initial_state, a->final_state, s, s.batch > 1, "gdn_linear_chunked")) return rc;
    GDN_REQUIRE(tokens < (1ll << 31) - kChunk, "gdn_linear_chunked: too many tokens");
    DeviceInfo* d = nullptr;
    if (int rc = get_device_info(&d)) return rc;
    LinChunkedParams p{};
    p.out = token_view(a->out);
    p.gate = scalar_view(a->gate);
    p.state_in = a->initial_state.ptr; p.si_ss = a->initial_state.stride_seq; p.si_sh = a->initial_state.stride_head;
    p.state_out = a->final_state.ptr; p.so_ss = a->final_state.stride_seq; p.so_sh = a->final_state.stride_head;
    p.cu_seqlens = s.cu_seqlens;
    p.total_tokens = static_cast<int>(s.total_tokens);
    p.num_seqs = s.batch; p.seq_len = s.seq_len; p.kh = s.num_k_heads; p.vh = s.num_v_heads;
    p.dk = s.head_dim_k; p.dv = s.head_dim_v; p.dv_tiles = (s.head_dim_v + 127) / 128;
    p.state_f32 = a->state_dtype == GDN_F32;
    p.scale = a->scale;
    p.status = d->status;
    const LinearPlan plan = linear_plan(s);
    GDN_REQUIRE(plan.items < (1ll << 31), "gdn_linear_chunked: too many sequences and heads");
    p.whole = static_cast<int>(plan.whole);
    p.seg_chunks = plan.seg_chunks;
    p.num_segments = plan.num_segments;
    p.by_length = plan.by_length;
    p.num_items = static_cast<int>(plan.items);
    if (plan.bytes) {
        if (!a->workspace || a->workspace_bytes < plan.bytes || (reinterpret_cast<uintptr_t>(a->workspace) & 255u))
            return fail(GDN_ERR_WORKSPACE, "gdn_linear_chunked: workspace of %zu bytes (256-byte aligned) required, got %zu", plan.bytes, a->workspace_bytes);
        p.seg_state = static_cast<float*>(a->workspace);
        p.seg_decay = reinterpret_cast<float*>(static_cast<uint8_t*>(a->workspace) + plan.states);
        p.in_place = a->initial_state.ptr && a->initial_state.ptr == a->final_state.ptr;
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return a->state_dtype == GDN_F32 ? launch_linear_shape<true>(*a, p, plan.cut_chains, st) : launch_linear_shape<false>(*a, p, plan.cut_chains, st);
}

}  // extern "C"
