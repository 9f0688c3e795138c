// Attention of one new token per sequence on a cache of pages: softmax(scale q K^T) V with grouped heads, sequences of any
// lengths, bf16 or fp16.
//
// The work is the bytes of the cache (every key and value row once; 4 g flops per byte pair with g query heads to a key head), so
// the kernel is a stream from HBM with the arithmetic hung into it:
//
//   * The keys of all (sequence, key head) items form one line of slots of 8 KB; each resident warp takes an equal piece of it,
//     whatever the sequences' lengths.  A CTA reads the lengths and finds its warps' pieces itself: the host plans nothing and the call
//     can be captured while lengths and table change under it.  An item that crosses warps leaves partial sums (fp32 sums relative
//     to a reference, the reference, the sum of the weights) in the workspace, at most two to a warp, and a second kernel joins
//     them in order: the result does not depend on who came first.  A CTA inside one item leaves one part: long sequences
//     have few.
//   * A warp works on its own: rows of keys, then rows of values, come through a ring of three slots of its own by 16-byte
//     asynchronous copies, with two slots on their way while it works on the third; no barrier in a piece, nor from one item
//     to the next.  8 warps an SM keep 128 KB on their way, three times what latency times bandwidth needs.
//   * The products are turned round: S^T = K Q^T and O^T = V^T P^T put the keys and the columns of V on the 16-row side of
//     mma.sync and the g query heads that share a key head on its 8-column side, so that up to eight heads cost one tile and each byte
//     of the cache crosses the SM once.  P^T comes out of S^T by one 8x8 transposition in registers.  tcgen05 wants 128
//     rows or columns of queries; this issues in 30 % of the cycles.  (With the queries on the 16-row
//     side, eight of its rows zeros, 16 KB of cache took 1043 warp instructions and 48 ragged sequences 55 us instead of 45.)
//
// What bounds it: inside a piece the stream runs at 6.2-6.6 TB/s, the measured copy rate; around it lie 2 us until a warp knows its piece,
// SMs that get 5-10 % less of the bandwidth (the same ones in every run), and 3-5 us for the second kernel.  Calls in a CUDA graph: 3 sequences, 260 k keys, fp16, 8 on 1 heads
// of 256 (267 MB) 54 us = 4.9 TB/s; 48 sequences of 1 to 4096, 32 on 8 of 128 (160 MB) 38 us = 4.2, with pages of 24 39; 128 of 16 to 2000, 16 on 16 of
// 64 (215 MB) 50 us = 4.3; one sequence of 762 keys 9.6 us, all latency.  Equal pieces per CTA, items not weighed, took 45 and 69 us for
// the two batches: CTAs with many short items were done last.
#include "paged_decode.cuh"

namespace tpb {
namespace {

template <typename T, int DP, int NT, bool kAligned, bool kWindow>
__global__ void __launch_bounds__(Shape<Rows16, DP, NT>::kThreads, Shape<Rows16, DP, NT>::kCtas) paged_attention_kernel(const __grid_constant__ DecodeParams P) {
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), D = P.cache.head_dim;
    pdl_wait_prior_grids();
    pdl_launch_dependents();
    attend_rows<T, DP, NT, kAligned, kWindow>(P, warp, D);
}
template <typename T, int kLanes, int kLoads>
__global__ void __launch_bounds__(kJoinThreads) paged_attention_join_kernel(const __grid_constant__ DecodeParams P) {
    pdl_wait_prior_grids();
    pdl_launch_dependents();
    join_parts<Rows16, T, kLanes, kLoads>(P);
}

// query heads that go through together: eight, or sixteen where a group has more; larger groups read the cache once per sixteen (48 sequences of 1 to
// 4096, 4 key heads of 128, 80 MB: groups of 8 21 us, of 16 28, of 32 47)
int decode_rows(int group) { return group <= 8 ? 8 : 16; }

constexpr int kCtasPerSm = Shape<Rows16, 64, 1>::kCtas;

template <typename T, int DP, bool kWindow>
int launch_rows(const DecodeParams& P, int ctas, cudaStream_t stream) {
    static_assert(Shape<Rows16, DP, 1>::kCtas == kCtasPerSm && Shape<Rows16, DP, 2>::kCtas == kCtasPerSm, "the workspace is cut for them");
    const bool aligned = P.cache.page_size % 16 == 0;
    if (P.group <= 8) {
        return aligned ? launch_decode<Rows16, DP, 1, paged_attention_kernel<T, DP, 1, true, kWindow>>(P, ctas, stream)
                       : launch_decode<Rows16, DP, 1, paged_attention_kernel<T, DP, 1, false, kWindow>>(P, ctas, stream);
    }
    return aligned ? launch_decode<Rows16, DP, 2, paged_attention_kernel<T, DP, 2, true, kWindow>>(P, ctas, stream)
                   : launch_decode<Rows16, DP, 2, paged_attention_kernel<T, DP, 2, false, kWindow>>(P, ctas, stream);
}
template <typename T, bool kWindow>
int launch_rows(const DecodeParams& P, int ctas, cudaStream_t stream) {
    const int D = P.cache.head_dim;
    return D <= 64 ? launch_rows<T, 64, kWindow>(P, ctas, stream)
                   : (D <= 128 ? launch_rows<T, 128, kWindow>(P, ctas, stream) : launch_rows<T, 256, kWindow>(P, ctas, stream));
}

// window 0: all keys
int attend(const tpb200_paged_attention_args* a, int window, int sinks, cudaStream_t stream) {
    TPB_REQUIRE(a != nullptr, TPB200_ERR_NULL);
    DecodeParams P = {};
    const int st = paged_view(a->cache, &P.cache);
    if (st != TPB200_OK) return st;
    const DecodeCall call = {a->q, a->out, a->q_stride, a->o_stride, a->q_heads, a->scale, a->workspace, a->workspace_bytes, a->flags, window, sinks};
    const int group = a->q_heads / P.cache.kv_heads, slot_keys = P.cache.head_dim <= 64 ? 64 : (P.cache.head_dim <= 128 ? 32 : 16);
    const int ctas = decode_ctas(kCtasPerSm);
    const int ready = prepare_decode(call, decode_rows(group), slot_keys, Rows16::kItemUnits, ctas, &P);
    if (ready != TPB200_OK || P.cache.seqs == 0) return ready;
    const bool bf = a->cache.dtype == TPB200_BF16;
    // a window that no sequence of the table passes hides nothing
    const bool hides = window > 0 && window < P.cache.page_size * P.cache.table_width;
    const int done = hides ? (bf ? launch_rows<__nv_bfloat16, true>(P, ctas, stream) : launch_rows<__half, true>(P, ctas, stream))
                           : (bf ? launch_rows<__nv_bfloat16, false>(P, ctas, stream) : launch_rows<__half, false>(P, ctas, stream));
    if (done != TPB200_OK) return done;
    return bf ? launch_join(P, nullptr, paged_attention_join_kernel<__nv_bfloat16, 8, 8>, paged_attention_join_kernel<__nv_bfloat16, 2, 4>, ctas, stream)
              : launch_join(P, nullptr, paged_attention_join_kernel<__half, 8, 8>, paged_attention_join_kernel<__half, 2, 4>, ctas, stream);
}

}  // namespace

int device_error_paged_attention(int clear) { return read_device_error(clear); }

}  // namespace tpb

extern "C" size_t tpb200_paged_attention_workspace_size(int q_heads, int kv_heads, int head_dim) {
    if (q_heads < 1 || kv_heads < 1 || q_heads % kv_heads != 0 || head_dim < 8 || head_dim > 256) return 0;
    const int ctas = tpb::decode_ctas(tpb::kCtasPerSm);
    if (ctas < 1) return 0;
    const int group = q_heads / kv_heads;
    return tpb::decode_scratch(static_cast<size_t>(ctas) * tpb::kCtaWarps, std::min(group, tpb::decode_rows(group)), head_dim).bytes;
}

extern "C" int tpb200_paged_attention(const tpb200_paged_attention_args* a, tpb200_stream_t stream) {
    return tpb::attend(a, 0, 0, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int tpb200_paged_attention_window(const tpb200_paged_attention_args* a, int window, int sinks, tpb200_stream_t stream) {
    TPB_REQUIRE(window >= 1 && sinks >= 0, TPB200_ERR_SHAPE);
    return tpb::attend(a, window, sinks, reinterpret_cast<cudaStream_t>(stream));
}
