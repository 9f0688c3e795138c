// Writes into a cache of pages and moves of its pages.
//
//   append   the new tokens' keys and values go to the rows the page table names, keys (and the queries beside them) rotated to
//            their positions on the way: one launch where the parts would be two rotations, a gather of row addresses and two
//            scattered writes.  Bound by HBM for prompts; for a decode step by the chain offsets -> length -> page id -> store.
//   copy     pages of every layer, keys and values, moved for a fork or a compaction.  Bound by HBM: 900 pages of 16 x 256 in 18 layers
//            (531 MB read and written) take 87 us = 6.1 TB/s = 0.93 of the measured copy rate.
#include <stdlib.h>

#include <algorithm>

#include "paged.cuh"

namespace tpb {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kAppendLoads = 2;          // tokens whose unit a thread has in flight: 32 bytes each, 80 KB on an SM with five blocks
constexpr int kMaxTokensPerBlock = 4;

struct AppendParams {
    PagedView cache;
    const uint16_t *k, *v, *q;
    uint16_t* q_out;
    long long k_stride[2], v_stride[2], q_stride[2], o_stride[2];
    const int* cu;
    const void *cos, *sin;
    int rope_dtype, rope_positions;      // rope_positions 0: nothing is rotated
    int tokens, q_heads, tokens_per_block;
    int units_q, units_k, units_v;       // units per token of the queries, the keys, the values
};

// A unit is V values of a row and the V values half a row further on (rotated, or a plain copy of both), so that a rotation
// needs one thread.  V = 8 where half a row is a multiple of 8, else 4.  A thread keeps its unit (which tensor, head and columns) for all
// tokens of the block: one division per thread and not per token: 77 -> 54 us for the prompts of six sequences (10.5 k tokens, 32 on 8 heads of 128,
// 265 MB), and 48 us = 5.5 TB/s = 0.85 of the measured copy rate with five blocks on an SM that take four tokens each (three blocks of
// eight: 53; sixteen tokens: 60; six blocks, which spill: 61).
template <typename T, int V>
__global__ void __launch_bounds__(kAppendThreads, 5) paged_append_kernel(const __grid_constant__ AppendParams P) {
    __shared__ int seq[kMaxTokensPerBlock];
    __shared__ int position[kMaxTokensPerBlock];
    __shared__ long long row_at[kMaxTokensPerBlock];     // element offset of the token's row in the pages, -1: not written
    pdl_wait_prior_grids();
    pdl_launch_dependents();
    const int t0 = blockIdx.x * P.tokens_per_block;
    const int count = min(P.tokens_per_block, P.tokens - t0);
    const int per_token = P.units_q + P.units_k + P.units_v;
    const int half = P.cache.head_dim / 2, per_row = half / V;
    bool placed = false;
    for (int base = 0; base < per_token; base += kAppendThreads) {
        const int u = base + threadIdx.x;
        const bool mine = u < per_token;
        const int kind = u < P.units_q ? 0 : (u < P.units_q + P.units_k ? 1 : 2);        // queries, keys, values
        const int r = u - (kind == 0 ? 0 : (kind == 1 ? P.units_q : P.units_q + P.units_k)), head = r / per_row, at = (r - head * per_row) * V;
        const long long* st = kind == 0 ? P.q_stride : (kind == 1 ? P.k_stride : P.v_stride);
        const long long step = st[0];
        const uint16_t* src = (kind == 0 ? P.q : (kind == 1 ? P.k : P.v)) + t0 * step + head * st[1] + at;
        const bool turn = P.rope_positions > 0 && kind < 2;
        uint16_t* dst = kind == 0 ? P.q_out + t0 * P.o_stride[0] + head * P.o_stride[1] + at
                                  : static_cast<uint16_t*>(kind == 1 ? P.cache.k_pages : P.cache.v_pages) + head * P.cache.head_stride + at;
        for (int first = 0; first < count; first += kAppendLoads) {
            Vec<V> a[kAppendLoads], b[kAppendLoads];
#pragma unroll
            for (int i = 0; i < kAppendLoads; ++i) {
                if (mine && first + i < count) {
                    a[i] = load_vec<V>(src + (first + i) * step);
                    b[i] = load_vec<V>(src + (first + i) * step + half);
                }
            }
            if (!placed) {
                // the tokens' rows, behind the first loads: which sequence, which position, which page
                placed = true;
                if (threadIdx.x < kMaxTokensPerBlock) seq[threadIdx.x] = 0x7fffffff;
                __syncthreads();
                for (int s = threadIdx.x; s < P.cache.seqs; s += kAppendThreads) {
                    const int lo = max(P.cu[s], t0), hi = min(P.cu[s + 1], t0 + count);
                    for (int t = lo; t < hi; ++t) atomicMin(&seq[t - t0], s);
                }
                __syncthreads();
                if (threadIdx.x < count) {
                    const int s = seq[threadIdx.x];
                    long long row = -1;
                    int pos = -1;
                    if (s != 0x7fffffff) {               // tokens behind the last sequence belong to nobody
                        pos = P.cache.lengths[s] - (P.cu[s + 1] - (t0 + static_cast<int>(threadIdx.x)));
                        row = P.cache.row_offset(s, pos);
                        if (row >= 0 && P.rope_positions > 0 && pos >= P.rope_positions) row = -1;
                        if (row < 0) record_error(kErrPagedIndex);
                    }
                    row_at[threadIdx.x] = row;
                    position[threadIdx.x] = pos;
                }
                __syncthreads();
            }
#pragma unroll
            for (int i = 0; i < kAppendLoads; ++i) {
                if (!mine || first + i >= count) continue;
                const long long row = row_at[first + i];
                if (row < 0) continue;
                if (turn) {
                    float c[V], s[V];
                    const size_t e = static_cast<size_t>(position[first + i]) * half + at;
                    load_table<V>(P.cos, P.rope_dtype, e, c);
                    load_table<V>(P.sin, P.rope_dtype, e, s);
#pragma unroll
                    for (int j = 0; j < V / 2; ++j) {    // in fp32, rounded once
                        const float2 x = Half16<T>::unpack(a[i].w[j]), y = Half16<T>::unpack(b[i].w[j]);
                        a[i].w[j] = Half16<T>::pack(x.x * c[2 * j] - y.x * s[2 * j], x.y * c[2 * j + 1] - y.y * s[2 * j + 1]);
                        b[i].w[j] = Half16<T>::pack(y.x * c[2 * j] + x.x * s[2 * j], y.y * c[2 * j + 1] + x.y * s[2 * j + 1]);
                    }
                }
                uint16_t* to = dst + (kind == 0 ? (first + i) * P.o_stride[0] : row);
                store_vec<V>(to, a[i]);
                store_vec<V>(to + half, b[i]);
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ copies of pages
constexpr int kPairsPerLaunch = 480;      // by value: no copy of the list to the device, nothing to keep alive behind the call
constexpr int kCopyWarps = 8;
constexpr int kCopyLoads = 8;             // 16-byte loads a lane has in flight; a warp moves 4 KB of a page
constexpr int kCopyPart = kCopyLoads * 32 * 16;

struct CopyParams {
    uint8_t* base;
    long long slab_bytes;                 // from one layer's keys (or values) to the next
    long long page_bytes;
    int parts;                            // of kCopyPart bytes in a page, the last one ragged
    int slabs;
    long long units;
    int pair[2 * kPairsPerLaunch];        // (from, to)
};

__global__ void __launch_bounds__(kCopyWarps * 32) copy_pages_kernel(const __grid_constant__ CopyParams P) {
    pdl_wait_prior_grids();
    pdl_launch_dependents();
    const long long unit = static_cast<long long>(blockIdx.x) * kCopyWarps + (threadIdx.x >> 5);
    if (unit >= P.units) return;
    const int per_pair = P.slabs * P.parts;
    const int p = static_cast<int>(unit / per_pair), r = static_cast<int>(unit - static_cast<long long>(p) * per_pair);
    const int slab = r / P.parts, part = r - slab * P.parts;
    const long long in_page = static_cast<long long>(part) * kCopyPart + (threadIdx.x & 31) * 16;
    const int most = static_cast<int>(min(static_cast<long long>(kCopyLoads), (P.page_bytes - in_page + 511) / 512));
    uint8_t* at = P.base + slab * P.slab_bytes + in_page;
    const uint4* src = reinterpret_cast<const uint4*>(at + P.pair[2 * p] * P.page_bytes);
    uint4* dst = reinterpret_cast<uint4*>(at + P.pair[2 * p + 1] * P.page_bytes);
    uint4 x[kCopyLoads];
#pragma unroll
    for (int i = 0; i < kCopyLoads; ++i) {
        if (i < most) x[i] = __ldcs(src + i * 32);
    }
#pragma unroll
    for (int i = 0; i < kCopyLoads; ++i) {
        if (i < most) __stcs(dst + i * 32, x[i]);
    }
}

}  // namespace

int device_error_paged_cache(int clear) { return read_device_error(clear); }

}  // namespace tpb

extern "C" int tpb200_paged_append(const tpb200_paged_append_args* a, tpb200_stream_t stream) {
    using namespace tpb;
    TPB_REQUIRE(a != nullptr, TPB200_ERR_NULL);
    AppendParams P = {};
    const int st = paged_view(a->cache, &P.cache);
    if (st != TPB200_OK) return st;
    TPB_REQUIRE(a->tokens == 0 || (a->k && a->v && a->cu), TPB200_ERR_NULL);      // tensors of no tokens have no memory
    TPB_REQUIRE((a->flags & ~TPB200_FLAG_PDL) == 0, TPB200_ERR_ENUM);
    TPB_REQUIRE(a->tokens >= 0, TPB200_ERR_SHAPE);
    const bool rope = a->cos != nullptr || a->sin != nullptr;
    if (rope) {
        TPB_REQUIRE(a->cos && a->sin, TPB200_ERR_NULL);
        TPB_REQUIRE(a->rope_positions >= 1, TPB200_ERR_SHAPE);
        TPB_REQUIRE(tpb_valid_dtype(a->rope_dtype), TPB200_ERR_ENUM);
        TPB_REQUIRE(tpb_aligned16(a->cos) && tpb_aligned16(a->sin), TPB200_ERR_ALIGN);
    }
    if (a->q != nullptr) {
        TPB_REQUIRE(a->q_out != nullptr, TPB200_ERR_NULL);
        TPB_REQUIRE(a->q_heads >= 1 && rope, TPB200_ERR_SHAPE);          // queries that are not rotated stay where they are
    }
    TPB_REQUIRE(tpb_aligned16(a->k) && tpb_aligned16(a->v) && tpb_aligned16(a->q) && tpb_aligned16(a->q_out), TPB200_ERR_ALIGN);
    for (int i = 0; i < 2; ++i) {
        const int n = i == 0 ? a->tokens : P.cache.kv_heads, qn = a->q == nullptr ? 0 : (i == 0 ? a->tokens : a->q_heads);
        for (const int st : {paged_stride(a->k_stride[i], n, P.cache.head_dim), paged_stride(a->v_stride[i], n, P.cache.head_dim),
                             paged_stride(a->q_stride[i], qn, P.cache.head_dim), paged_stride(a->o_stride[i], qn, P.cache.head_dim)}) {
            if (st != TPB200_OK) return st;
        }
        P.k_stride[i] = a->k_stride[i];
        P.v_stride[i] = a->v_stride[i];
        P.q_stride[i] = a->q_stride[i];
        P.o_stride[i] = a->o_stride[i];
    }
    if (a->tokens == 0 || P.cache.seqs == 0) return TPB200_OK;
    TPB_REQUIRE(a->cache.k_pages != a->cache.v_pages, TPB200_ERR_SHAPE);
    if (a->q != nullptr) {               // other threads read what lies there
        const int D = P.cache.head_dim, H = P.cache.kv_heads;
        const RowSet out(a->q_out, a->o_stride, a->tokens, a->q_heads, D);
        TPB_REQUIRE(output_fits(out, RowSet(a->q, a->q_stride, a->tokens, a->q_heads, D)), TPB200_ERR_SHAPE);
        TPB_REQUIRE(!rows_meet(out, RowSet(a->k, a->k_stride, a->tokens, H, D)) && !rows_meet(out, RowSet(a->v, a->v_stride, a->tokens, H, D)),
                    TPB200_ERR_SHAPE);
    }
    P.k = static_cast<const uint16_t*>(a->k);
    P.v = static_cast<const uint16_t*>(a->v);
    P.q = static_cast<const uint16_t*>(a->q);
    P.q_out = static_cast<uint16_t*>(a->q_out);
    P.cu = a->cu;
    P.cos = a->cos;
    P.sin = a->sin;
    P.rope_dtype = a->rope_dtype;
    P.rope_positions = rope ? a->rope_positions : 0;
    P.tokens = a->tokens;
    P.q_heads = a->q != nullptr ? a->q_heads : 0;
    const int half = P.cache.head_dim / 2, V = half % 8 == 0 ? 8 : 4;
    const long long per_head = half / V, units = per_head * (P.q_heads + 2ll * P.cache.kv_heads);
    TPB_REQUIRE(units <= (1 << 24), TPB200_ERR_SHAPE);
    P.units_q = static_cast<int>(per_head * P.q_heads);
    P.units_k = P.units_v = static_cast<int>(per_head * P.cache.kv_heads);
    // four tokens share a block's look-up, fewer where that would leave SMs without a block
    P.tokens_per_block = std::max(1, std::min(kMaxTokensPerBlock, a->tokens / 444));
    const unsigned blocks = static_cast<unsigned>((a->tokens - 1) / P.tokens_per_block + 1);
    const bool bf = a->cache.dtype == TPB200_BF16;
    auto kernel = bf ? (V == 8 ? paged_append_kernel<__nv_bfloat16, 8> : paged_append_kernel<__nv_bfloat16, 4>)
                     : (V == 8 ? paged_append_kernel<__half, 8> : paged_append_kernel<__half, 4>);
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = paged_config(blocks, kAppendThreads, 0, &attr, reinterpret_cast<cudaStream_t>(stream));
    return cudaLaunchKernelEx(&cfg, kernel, P) == cudaSuccess ? TPB200_OK : TPB200_ERR_CUDA;
}

extern "C" int tpb200_copy_pages(void* pages, long long slab_bytes, int slabs, long long page_bytes, int num_pages, const int* src,
                                 const int* dst, int count, int flags, tpb200_stream_t stream) {
    using namespace tpb;
    TPB_REQUIRE(count >= 0 && slabs >= 1 && num_pages >= 1 && page_bytes >= 16, TPB200_ERR_SHAPE);
    TPB_REQUIRE((flags & ~TPB200_FLAG_PDL) == 0, TPB200_ERR_ENUM);
    if (count == 0) return TPB200_OK;
    TPB_REQUIRE(pages && src && dst, TPB200_ERR_NULL);
    TPB_REQUIRE(tpb_aligned16(pages) && page_bytes % 16 == 0 && slab_bytes % 16 == 0, TPB200_ERR_ALIGN);
    TPB_REQUIRE(slabs == 1 || slab_bytes >= page_bytes * num_pages, TPB200_ERR_SHAPE);
    const long long parts = (page_bytes + kCopyPart - 1) / kCopyPart;
    TPB_REQUIRE(parts * slabs <= (1 << 22), TPB200_ERR_SHAPE);
    // every index in range, no page written twice, none read that another pair writes: the pairs may then run in any order
    int* sorted = static_cast<int*>(malloc(sizeof(int) * static_cast<size_t>(count)));
    if (sorted == nullptr) return TPB200_ERR_WORKSPACE;
    std::copy(dst, dst + count, sorted);
    std::sort(sorted, sorted + count);
    bool fine = sorted[0] >= 0 && sorted[count - 1] < num_pages && std::adjacent_find(sorted, sorted + count) == sorted + count;
    for (int i = 0; i < count && fine; ++i) {
        fine = src[i] >= 0 && src[i] < num_pages && !std::binary_search(sorted, sorted + count, src[i]);
    }
    free(sorted);
    TPB_REQUIRE(fine, TPB200_ERR_SHAPE);
    CopyParams P;
    P.base = static_cast<uint8_t*>(pages);
    P.slab_bytes = slab_bytes;
    P.page_bytes = page_bytes;
    P.parts = static_cast<int>(parts);
    P.slabs = slabs;
    for (int first = 0; first < count; first += kPairsPerLaunch) {
        const int n = std::min(kPairsPerLaunch, count - first);
        for (int i = 0; i < n; ++i) {
            P.pair[2 * i] = src[first + i];
            P.pair[2 * i + 1] = dst[first + i];
        }
        P.units = parts * slabs * n;
        cudaLaunchAttribute attr;
        const cudaLaunchConfig_t cfg = paged_config(static_cast<unsigned>((P.units + kCopyWarps - 1) / kCopyWarps), kCopyWarps * 32, 0,
                                                    &attr, reinterpret_cast<cudaStream_t>(stream));
        if (cudaLaunchKernelEx(&cfg, copy_pages_kernel, P) != cudaSuccess) return TPB200_ERR_CUDA;
    }
    return TPB200_OK;
}
