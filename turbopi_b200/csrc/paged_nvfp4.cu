// A cache of pages held in 4 bits: new tokens quantised as they are written, and tokens read back (also out of 16-bit pages).
//
//   append   keys rotated to their positions and rounded to 16 bits, as a 16-bit cache would hold them, then 16 values x at a time:
//            s = e4m3(max |x| / 6), code = e2m1(x / s).  Queries are rotated beside them.  One launch.
//   read     rows of the last tokens of each sequence, one sequence behind the other: values out of 4 bits, or copies out of 16.
//
// Both are bound by HBM for prompts and by the chain offsets -> length -> page id -> row for a decode step.
#include <algorithm>

#include "paged.cuh"

namespace tpb {
namespace {

constexpr int kThreads = 256;            // of a block at most
constexpr int kAppendLoads = 2;          // tokens whose unit a thread has in flight
constexpr int kAppendTokens = 4;         // of a block at most
constexpr int kReadLoads = 4;
constexpr int kReadTokens = 16;

// Where the tokens [t0, t0 + count) of a packed batch stand: their positions, and the offsets of their rows (16-bit pages) or tiles (kTiles), -1 where
// the cache has no place for one, -2 for a token behind the last sequence.  All threads of the block call it; kMax >= count places.
template <bool kTiles, int kMax>
__device__ __forceinline__ void place_tokens(const PagedView& c, const int* cu, int t0, int count, int rope_positions, int* seq, int* position,
                                             long long* row_at) {
    for (int i = threadIdx.x; i < kMax; i += blockDim.x) seq[i] = 0x7fffffff;
    __syncthreads();
    for (int s = threadIdx.x; s < c.seqs; s += blockDim.x) {
        const int lo = max(cu[s], t0), hi = min(cu[s + 1], t0 + count);
        for (int t = lo; t < hi; ++t) atomicMin(&seq[t - t0], s);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < count; i += blockDim.x) {
        const int s = seq[i];
        long long row = -2;
        int pos = -1;
        if (s != 0x7fffffff) {
            pos = c.lengths[s] - (cu[s + 1] - (t0 + i));
            row = -1;
            if (pos >= 0 && (rope_positions == 0 || pos < rope_positions)) {
                const int page = pos / c.page_size, in = pos - page * c.page_size;
                if (page < c.table_width) {
                    const int id = c.table[s * c.table_stride + page];
                    if (static_cast<unsigned>(id) < static_cast<unsigned>(c.num_pages)) {
                        row = id * c.page_stride + (kTiles ? in / 16 : in) * c.row_stride;
                    }
                }
            }
            if (row < 0) record_error(kErrPagedIndex);
        }
        row_at[i] = row;
        position[i] = pos;
    }
    __syncthreads();
}

// ------------------------------------------------------------------------------------------------ append
struct AppendParams {
    PagedView cache;
    const uint16_t *k, *v, *q;
    uint16_t* q_out;
    long long k_stride[2], v_stride[2], q_stride[2], o_stride[2];
    const int* cu;
    const void *cos, *sin;
    int rope_dtype, rope_positions;      // rope_positions 0: nothing is rotated
    int tokens, tokens_per_block;
    int units_q, units_kv;               // units per token of the queries, and of the keys (as many of the values)
    float k_inv, v_inv;                  // 1 / k_scale, 1 / v_scale
};

// x * c - y * s and x * c + y * s, each operation rounded: the sums that elementary operations give, whatever else is compiled around them
__device__ __forceinline__ float turn_first(float x, float y, float c, float s) { return __fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s)); }
__device__ __forceinline__ float turn_second(float x, float y, float c, float s) { return __fadd_rn(__fmul_rn(x, c), __fmul_rn(y, s)); }

// 16 values -> a scale and 16 codes.  The quotient is x times the rounded inverse of s, off by 2^-22 at most for |x / s| <= 6.  Ties are common (s has four
// bits, x eight or eleven) and have to stay ties: the sum with 128 rounds the quotient to a multiple of 2^-17 or 2^-16.  A quotient that is no tie is 2^-13 from one
// at least, since x differs from a tie times s, which the type of x holds, by a step of that type.
__device__ __forceinline__ void quantise16(const float (&x)[16], float inv, uint2& codes, uint8_t& scale) {
    float top = 0.0f, odd = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        top = fmaxf(top, fabsf(x[i]));
        odd = fmaf(x[i], 0.0f, odd);     // NaN from the first infinity or NaN on
    }
    codes = make_uint2(0, 0);
    if (odd != 0.0f || isnan(odd)) {
        scale = 0x7f;                    // NaN
        return;
    }
    scale = encode_e4m3(__fdiv_rn(top * inv, 6.0f));
    if (scale == 0) return;
    const float r = __frcp_rn(decode_e4m3(scale));
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float y[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            // (x * inv is exact: a power of two.  Past 6 the conversion saturates.)
            y[j] = __fmul_rn(__fmul_rn(x[2 * i + j], inv), r);
            y[j] = __fsub_rn(__fadd_rn(y[j], 128.0f), 128.0f);
        }
        w[i >> 2] |= encode_e2m1x2(y[0], y[1]) << ((i & 3) * 8);
    }
    codes = make_uint2(w[0], w[1]);
}

// A unit of the queries is V values and the V values half a row further on, V = 8 where half a row is a multiple of 8, else 4; a unit of
// the keys or values is a block of 16, for keys with the 16 values half a row away beside it.  A thread keeps its unit for all tokens of the block.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads, 3) append_nvfp4_kernel(const __grid_constant__ AppendParams P) {
    __shared__ int seq[kAppendTokens];
    __shared__ int position[kAppendTokens];
    __shared__ long long row_at[kAppendTokens];
    constexpr int kVecs = 16 / V;
    pdl_wait_prior_grids();
    pdl_launch_dependents();
    const int t0 = blockIdx.x * P.tokens_per_block;
    const int count = min(P.tokens_per_block, P.tokens - t0);
    const int per_token = P.units_q + 2 * P.units_kv;
    const int D = P.cache.head_dim, half = D / 2, per_row = half / V, groups = (D + 31) / 32;
    bool placed = false;
    for (int base = 0; base < per_token; base += blockDim.x) {
        const int u = base + threadIdx.x;
        const bool mine = u < per_token;
        const int kind = u < P.units_q ? 0 : (u < P.units_q + P.units_kv ? 1 : 2);       // queries, keys, values
        const int r = u - (kind == 0 ? 0 : (kind == 1 ? P.units_q : P.units_q + P.units_kv));
        const int head = kind == 0 ? r / per_row : r / (2 * groups), in = kind == 0 ? r - head * per_row : r - head * 2 * groups;
        const int at = kind == 0 ? in * V : in * 16;     // first column; the partners of column c stand at c + half or c - half
        const long long* st = kind == 0 ? P.q_stride : (kind == 1 ? P.k_stride : P.v_stride);
        const long long step = st[0];
        const uint16_t* src = (kind == 0 ? P.q : (kind == 1 ? P.k : P.v)) + t0 * step + head * st[1];
        const bool turn = P.rope_positions > 0 && kind < 2;
        for (int first = 0; first < count; first += kAppendLoads) {
            Vec<V> x[kAppendLoads][kVecs], y[kAppendLoads][kVecs];
#pragma unroll
            for (int i = 0; i < kAppendLoads; ++i) {
                if (!mine || first + i >= count) continue;
                const uint16_t* row = src + (first + i) * step;
#pragma unroll
                for (int n = 0; n < kVecs; ++n) {
                    const int c = at + n * V;
                    x[i][n] = y[i][n] = Vec<V>{};
                    if ((kind == 0 && n > 0) || c >= D) continue;
                    x[i][n] = load_vec<V>(row + c);
                    if (turn) y[i][n] = load_vec<V>(row + (c < half ? c + half : c - half));
                }
            }
            if (!placed) {               // the tokens' rows, behind the first loads
                placed = true;
                place_tokens<true, kAppendTokens>(P.cache, P.cu, t0, count, P.rope_positions, seq, position, row_at);
            }
#pragma unroll
            for (int i = 0; i < kAppendLoads; ++i) {
                if (!mine || first + i >= count) continue;
                const long long row = row_at[first + i];
                if (row < 0) continue;
                const int pos = position[first + i];
                if (kind == 0) {
                    float c[V], s[V];
                    const size_t e = static_cast<size_t>(pos) * half + at;
                    load_table<V>(P.cos, P.rope_dtype, e, c);
                    load_table<V>(P.sin, P.rope_dtype, e, s);
                    Vec<V> a, b;
#pragma unroll
                    for (int j = 0; j < V / 2; ++j) {    // in fp32, rounded once
                        const float2 p = Half16<T>::unpack(x[i][0].w[j]), q = Half16<T>::unpack(y[i][0].w[j]);
                        a.w[j] = Half16<T>::pack(turn_first(p.x, q.x, c[2 * j], s[2 * j]), turn_first(p.y, q.y, c[2 * j + 1], s[2 * j + 1]));
                        b.w[j] = Half16<T>::pack(turn_second(q.x, p.x, c[2 * j], s[2 * j]), turn_second(q.y, p.y, c[2 * j + 1], s[2 * j + 1]));
                    }
                    uint16_t* to = P.q_out + (t0 + first + i) * P.o_stride[0] + head * P.o_stride[1] + at;
                    store_vec<V>(to, a);
                    store_vec<V>(to + half, b);
                    continue;
                }
                float f[16];
#pragma unroll
                for (int n = 0; n < kVecs; ++n) {
                    const int col = at + n * V;
                    if (turn && col < D) {
                        float c[V], s[V];
                        const bool low = col < half;
                        const size_t e = static_cast<size_t>(pos) * half + (low ? col : col - half);
                        load_table<V>(P.cos, P.rope_dtype, e, c);
                        load_table<V>(P.sin, P.rope_dtype, e, s);
#pragma unroll
                        for (int j = 0; j < V / 2; ++j) {
                            const float2 p = Half16<T>::unpack(x[i][n].w[j]), q = Half16<T>::unpack(y[i][n].w[j]);
                            const float s0 = low ? -s[2 * j] : s[2 * j], s1 = low ? -s[2 * j + 1] : s[2 * j + 1];
                            x[i][n].w[j] = Half16<T>::pack(turn_second(p.x, q.x, c[2 * j], s0), turn_second(p.y, q.y, c[2 * j + 1], s1));
                        }
                    }
#pragma unroll
                    for (int j = 0; j < V / 2; ++j) {
                        const float2 p = Half16<T>::unpack(x[i][n].w[j]);
                        f[n * V + 2 * j] = p.x;
                        f[n * V + 2 * j + 1] = p.y;
                    }
                }
                uint2 codes;
                uint8_t scale;
                quantise16(f, kind == 1 ? P.k_inv : P.v_inv, codes, scale);
                uint8_t* tile = static_cast<uint8_t*>(kind == 1 ? P.cache.k_pages : P.cache.v_pages) + row + head * P.cache.head_stride;
                *reinterpret_cast<uint2*>(tile + (pos & 15) * 16 * groups + in * 8) = codes;
                tile[256 * groups + (pos & 15) * 2 * groups + in] = scale;
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ read
struct ReadParams {
    PagedView cache;
    uint16_t *k, *v;
    long long k_stride[2], v_stride[2];
    const int* cu;
    int tokens, tokens_per_block;
    int units;                           // of eight values, per token of keys, and of values
    float k_scale, v_scale;
};

// A thread has eight columns of a head's keys or values (16 bytes to write, whole warps write whole lines) of every kLanes-th token of the block.
template <typename T, bool kTiles>
__global__ void __launch_bounds__(kThreads) read_kernel(const __grid_constant__ ReadParams P) {
    __shared__ int seq[kReadTokens];
    __shared__ int position[kReadTokens];
    __shared__ long long row_at[kReadTokens];
    pdl_wait_prior_grids();
    pdl_launch_dependents();
    const int t0 = blockIdx.x * P.tokens_per_block;
    const int count = min(P.tokens_per_block, P.tokens - t0);
    place_tokens<kTiles, kReadTokens>(P.cache, P.cu, t0, count, 0, seq, position, row_at);
    const int D = P.cache.head_dim, per_row = D / 8, groups = (D + 31) / 32;
    const int all = 2 * P.units, lanes = max(1, static_cast<int>(blockDim.x) / all), lane = all <= static_cast<int>(blockDim.x) ? threadIdx.x / all : 0;
    if (lane >= lanes) return;
    for (int u = threadIdx.x - lane * all; u < all; u += blockDim.x) {
        const bool keys = u < P.units;
        const int r = keys ? u : u - P.units, head = r / per_row, in = r - head * per_row;
        const uint8_t* pages = static_cast<const uint8_t*>(keys ? P.cache.k_pages : P.cache.v_pages);
        const long long* st = keys ? P.k_stride : P.v_stride;
        uint16_t* to = (keys ? P.k : P.v) + t0 * st[0] + head * st[1] + in * 8;
        const float factor = keys ? P.k_scale : P.v_scale;
        for (int first = lane; first < count; first += lanes * kReadLoads) {
            uint4 x[kReadLoads];
            uint32_t scale[kReadLoads];
#pragma unroll
            for (int i = 0; i < kReadLoads; ++i) {
                const int t = first + i * lanes;
                x[i] = make_uint4(0, 0, 0, 0);
                scale[i] = 0;
                if (t >= count || row_at[t] < 0) continue;
                if constexpr (kTiles) {
                    const uint8_t* tile = pages + row_at[t] + head * P.cache.head_stride;
                    const int row = position[t] & 15;
                    x[i].x = __ldg(reinterpret_cast<const uint32_t*>(tile + row * 16 * groups + in * 4));
                    scale[i] = __ldg(tile + 256 * groups + row * 2 * groups + in / 2);
                } else {
                    x[i] = __ldg(reinterpret_cast<const uint4*>(pages + 2 * (row_at[t] + head * P.cache.head_stride + in * 8)));
                }
            }
#pragma unroll
            for (int i = 0; i < kReadLoads; ++i) {
                const int t = first + i * lanes;
                if (t >= count || row_at[t] == -2) continue;
                if constexpr (kTiles) {
                    __half2 h[4];
                    uint32_t w[4];
                    decode_e2m1x8(x[i].x, h);
                    const float s = decode_e4m3(static_cast<uint8_t>(scale[i])) * factor;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {        // exact but for an overflow of fp16 or a factor's underflow
                        const float2 f = __half22float2(h[j]);
                        w[j] = Half16<T>::pack(f.x * s, f.y * s);
                    }
                    x[i] = make_uint4(w[0], w[1], w[2], w[3]);
                }
                *reinterpret_cast<uint4*>(to + t * st[0]) = x[i];
            }
        }
    }
}

// a block's threads for `units` a token: as few passes over them as kThreads allows, and those even
int threads_for(long long units) {
    const long long passes = (units + kThreads - 1) / kThreads;
    return static_cast<int>(((units + passes - 1) / passes + 31) / 32 * 32);
}

// bytes from the first to behind the last of a cache's pages
long long pool_bytes(const PagedView& c, long long row_bytes, int rows, int element) {
    return ((c.num_pages - 1) * c.page_stride + (rows - 1) * c.row_stride + (c.kv_heads - 1) * c.head_stride) * element + row_bytes;
}

int read_rows(const PagedView& cache, int dtype, bool tiles, float k_scale, float v_scale, const tpb200_paged_rows* a, cudaStream_t stream) {
    TPB_REQUIRE(a->tokens >= 0, TPB200_ERR_SHAPE);
    TPB_REQUIRE((a->flags & ~TPB200_FLAG_PDL) == 0 && (a->dtype == TPB200_BF16 || a->dtype == TPB200_F16) && (tiles || a->dtype == dtype), TPB200_ERR_ENUM);
    ReadParams P = {};
    P.cache = cache;
    for (int i = 0; i < 2; ++i) {
        const int n = i == 0 ? a->tokens : cache.kv_heads;
        for (const long long st : {a->k_stride[i], a->v_stride[i]}) {
            const int fine = paged_stride(st, n, cache.head_dim);
            if (fine != TPB200_OK) return fine;
        }
        P.k_stride[i] = n > 1 ? a->k_stride[i] : 0;
        P.v_stride[i] = n > 1 ? a->v_stride[i] : 0;
    }
    if (a->tokens == 0 || cache.seqs == 0) return TPB200_OK;
    TPB_REQUIRE(a->k && a->v && a->cu, TPB200_ERR_NULL);
    TPB_REQUIRE(tpb_aligned16(a->k) && tpb_aligned16(a->v), TPB200_ERR_ALIGN);
    // rows that meet one another, or the pages that other threads read
    const RowSet k(a->k, P.k_stride, a->tokens, cache.kv_heads, cache.head_dim), v(a->v, P.v_stride, a->tokens, cache.kv_heads, cache.head_dim);
    TPB_REQUIRE(!rows_cross(k) && !rows_cross(v) && !rows_meet(k, v), TPB200_ERR_SHAPE);
    const long long bytes = tiles ? pool_bytes(cache, 288ll * ((cache.head_dim + 31) / 32), cache.page_size / 16, 1)
                                  : pool_bytes(cache, 2ll * cache.head_dim, cache.page_size, 2);
    for (const RowSet& rows : {k, v}) {
        for (const void* pages : {cache.k_pages, cache.v_pages}) {
            const long long at = static_cast<long long>(reinterpret_cast<uintptr_t>(pages));
            TPB_REQUIRE(2 * rows.end() <= at || at + bytes <= 2 * rows.at, TPB200_ERR_SHAPE);
        }
    }
    P.k = static_cast<uint16_t*>(a->k);
    P.v = static_cast<uint16_t*>(a->v);
    P.cu = a->cu;
    P.tokens = a->tokens;
    P.k_scale = k_scale;
    P.v_scale = v_scale;
    const long long units = static_cast<long long>(cache.head_dim / 8) * cache.kv_heads;
    TPB_REQUIRE(units <= (1 << 24), TPB200_ERR_SHAPE);
    P.units = static_cast<int>(units);
    const int threads = 2 * units <= kThreads ? kThreads : threads_for(2 * units), lanes = std::max(1, static_cast<int>(threads / (2 * units)));
    // a block's look-up serves up to a tile of tokens, fewer where that would leave SMs without a block, but at least one for each lane
    P.tokens_per_block = std::max(std::min(lanes, kReadTokens), std::min(kReadTokens, a->tokens / 592));
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = paged_config(static_cast<unsigned>((a->tokens - 1) / P.tokens_per_block + 1), threads, 0, &attr, stream);
    const bool bf = a->dtype == TPB200_BF16;
    const auto kernel = tiles ? (bf ? read_kernel<__nv_bfloat16, true> : read_kernel<__half, true>) : read_kernel<__half, false>;
    return cudaLaunchKernelEx(&cfg, kernel, P) == cudaSuccess ? TPB200_OK : TPB200_ERR_CUDA;
}

}  // namespace

int device_error_paged_nvfp4(int clear) { return read_device_error(clear); }

}  // namespace tpb

extern "C" int tpb200_paged_read(const tpb200_paged_cache* cache, const tpb200_paged_rows* rows, tpb200_stream_t stream) {
    using namespace tpb;
    TPB_REQUIRE(cache != nullptr && rows != nullptr, TPB200_ERR_NULL);
    PagedView view;
    const int st = paged_view(*cache, &view);
    if (st != TPB200_OK) return st;
    return read_rows(view, cache->dtype, false, 1.0f, 1.0f, rows, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int tpb200_paged_read_nvfp4(const tpb200_paged_nvfp4_cache* cache, const tpb200_paged_rows* rows, tpb200_stream_t stream) {
    using namespace tpb;
    TPB_REQUIRE(cache != nullptr && rows != nullptr, TPB200_ERR_NULL);
    PagedView view;
    const int st = paged_view_nvfp4(*cache, &view);
    if (st != TPB200_OK) return st;
    return read_rows(view, 0, true, cache->k_scale, cache->v_scale, rows, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int tpb200_paged_append_nvfp4(const tpb200_paged_append_nvfp4_args* a, tpb200_stream_t stream) {
    using namespace tpb;
    TPB_REQUIRE(a != nullptr, TPB200_ERR_NULL);
    AppendParams P = {};
    const int st = paged_view_nvfp4(a->cache, &P.cache);
    if (st != TPB200_OK) return st;
    TPB_REQUIRE(a->tokens == 0 || (a->k && a->v && a->cu), TPB200_ERR_NULL);      // tensors of no tokens have no memory
    TPB_REQUIRE((a->flags & ~TPB200_FLAG_PDL) == 0 && (a->dtype == TPB200_BF16 || a->dtype == TPB200_F16), TPB200_ERR_ENUM);
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
    const int D = P.cache.head_dim, H = P.cache.kv_heads;
    if (a->q != nullptr) {               // other threads read what lies there
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
    P.k_inv = 1.0f / a->cache.k_scale;
    P.v_inv = 1.0f / a->cache.v_scale;
    const int half = D / 2, V = half % 8 == 0 ? 8 : 4;
    const long long units_q = a->q != nullptr ? static_cast<long long>(half / V) * a->q_heads : 0, units_kv = 2ll * ((D + 31) / 32) * H;
    TPB_REQUIRE(units_q + 2 * units_kv <= (1 << 24), TPB200_ERR_SHAPE);
    P.units_q = static_cast<int>(units_q);
    P.units_kv = static_cast<int>(units_kv);
    // four tokens share a block's look-up, fewer where that would leave SMs without a block
    P.tokens_per_block = std::max(1, std::min(kAppendTokens, a->tokens / 444));
    const unsigned blocks = static_cast<unsigned>((a->tokens - 1) / P.tokens_per_block + 1);
    const bool bf = a->dtype == TPB200_BF16;
    const auto kernel = bf ? (V == 8 ? append_nvfp4_kernel<__nv_bfloat16, 8> : append_nvfp4_kernel<__nv_bfloat16, 4>)
                           : (V == 8 ? append_nvfp4_kernel<__half, 8> : append_nvfp4_kernel<__half, 4>);
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = paged_config(blocks, threads_for(units_q + 2 * units_kv), 0, &attr, reinterpret_cast<cudaStream_t>(stream));
    return cudaLaunchKernelEx(&cfg, kernel, P) == cudaSuccess ? TPB200_OK : TPB200_ERR_CUDA;
}
