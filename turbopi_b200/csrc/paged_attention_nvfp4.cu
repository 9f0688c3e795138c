// Attention of one new token per sequence on a cache of pages held in 4 bits (E2M1 values with an E4M3 scale for every 16), over all keys or over
// a window and the first few: the kernel of paged_decode.cuh on tiles of 16 tokens.
#include "paged_decode.cuh"

namespace tpb {
namespace {

template <typename T, int DP, int NT>
__global__ void __launch_bounds__(kThreads, Shape<Nvfp4, DP, NT>::kCtas) paged_attention_nvfp4_kernel(const __grid_constant__ DecodeParams P) {
    pdl_wait_prior_grids();
    pdl_launch_dependents();
    attend_pages<Nvfp4, T, DP, NT, true, true>(P);
}
template <typename T, int kLanes, int kLoads>
__global__ void __launch_bounds__(kJoinThreads) paged_attention_nvfp4_join_kernel(const __grid_constant__ DecodeParams P) {
    pdl_wait_prior_grids();
    pdl_launch_dependents();
    join_parts<Nvfp4, T, kLanes, kLoads>(P);
}

// query heads that go through together: eight, or sixteen where a group has more and their sums leave registers for the rest
int decode_rows4(int group, int head_dim) { return group <= 8 || head_dim > 128 ? 8 : 16; }

template <typename T, int DP, int NT>
int launch_tiles(const DecodeParams& P, int ctas, cudaStream_t stream) {
    return launch_decode<Nvfp4, DP, NT, paged_attention_nvfp4_kernel<T, DP, NT>>(P, ctas, stream);
}
template <typename T>
int launch_tiles(const DecodeParams& P, int ctas, cudaStream_t stream) {
    const int D = P.cache.head_dim;
    if (D > 128) return launch_tiles<T, 256, 1>(P, ctas, stream);
    if (D > 64) return P.rows > 8 ? launch_tiles<T, 128, 2>(P, ctas, stream) : launch_tiles<T, 128, 1>(P, ctas, stream);
    return P.rows > 8 ? launch_tiles<T, 64, 2>(P, ctas, stream) : launch_tiles<T, 64, 1>(P, ctas, stream);
}
int ctas_per_sm4(int rows, int head_dim) {
    if (head_dim > 128) return Shape<Nvfp4, 256, 1>::kCtas;
    if (head_dim > 64) return rows > 8 ? Shape<Nvfp4, 128, 2>::kCtas : Shape<Nvfp4, 128, 1>::kCtas;
    return rows > 8 ? Shape<Nvfp4, 64, 2>::kCtas : Shape<Nvfp4, 64, 1>::kCtas;
}

}  // namespace

int device_error_paged_attention_nvfp4(int clear) { return read_device_error(clear); }

}  // namespace tpb

extern "C" size_t tpb200_paged_attention_nvfp4_workspace_size(int q_heads, int kv_heads, int head_dim) {
    using namespace tpb;
    if (q_heads < 1 || kv_heads < 1 || q_heads % kv_heads != 0 || head_dim < 8 || head_dim > 256) return 0;
    const int group = q_heads / kv_heads, rows = std::min(group, decode_rows4(group, head_dim));
    const int ctas = decode_ctas(ctas_per_sm4(rows, head_dim));
    return ctas < 1 ? 0 : decode_scratch(ctas, rows, head_dim).bytes;
}

extern "C" int tpb200_paged_attention_nvfp4(const tpb200_paged_attention_nvfp4_args* a, tpb200_stream_t stream) {
    using namespace tpb;
    TPB_REQUIRE(a != nullptr, TPB200_ERR_NULL);
    DecodeParams P = {};
    const int st = paged_view_nvfp4(a->cache, &P.cache);
    if (st != TPB200_OK) return st;
    TPB_REQUIRE(a->dtype == TPB200_BF16 || a->dtype == TPB200_F16, TPB200_ERR_ENUM);
    TPB_REQUIRE(a->window >= 0 && a->sinks >= 0 && (a->window > 0 || a->sinks == 0), TPB200_ERR_SHAPE);
    const DecodeCall call = {a->q, a->out, a->q_stride, a->o_stride, a->q_heads, a->scale, a->workspace, a->workspace_bytes, a->flags, a->window, a->sinks};
    const int D = P.cache.head_dim, group = a->q_heads / P.cache.kv_heads, rows = decode_rows4(group, D);
    const int ctas = decode_ctas(ctas_per_sm4(std::min(group, rows), D));
    const int ready = prepare_decode(call, rows, D <= 64 ? 128 : (D <= 128 ? 64 : 32), ctas, &P);
    if (ready != TPB200_OK || P.cache.seqs == 0) return ready;
    P.scale2 *= a->cache.k_scale;
    TPB_REQUIRE(std::isfinite(P.scale2), TPB200_ERR_SHAPE);
    P.out_scale = a->cache.v_scale;
    const bool bf = a->dtype == TPB200_BF16;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const int done = bf ? launch_tiles<__nv_bfloat16>(P, ctas, s) : launch_tiles<__half>(P, ctas, s);
    if (done != TPB200_OK) return done;
    return bf ? launch_join(P, paged_attention_nvfp4_join_kernel<__nv_bfloat16, 8, 8>, paged_attention_nvfp4_join_kernel<__nv_bfloat16, 2, 4>, ctas, s)
              : launch_join(P, paged_attention_nvfp4_join_kernel<__half, 8, 8>, paged_attention_nvfp4_join_kernel<__half, 2, 4>, ctas, s);
}
