// A cache of pages held in 4 bits: new tokens quantised as they are written, and tokens read back (also out of 16-bit pages).
//
//   append   keys rotated to their positions and rounded to 16 bits, as a 16-bit cache would hold them, then 16 values x at a time:
//            s = e4m3(max |x| / 6), code = e2m1(x / s).  Queries are rotated beside them.  One launch.
//   read     rows of the last tokens of each sequence, one sequence behind the other: values out of 4 bits, or copies out of 16.
//
// A decode step is the chain offsets -> length -> page id -> row.  Prompts, calls in a CUDA graph: 14.4 k tokens of six sequences, 32 on 8 heads of 128, turned and
// written (312 MB) 66 us = 4.7 TB/s: what a block waits for (its look-up, then each token's loads) and 70 instructions for 16 values; keys and values alone 30 (floor 12.6), not turned
// 19.6 (11.5).  The same tokens into 16 bits (354 MB): 63.  25 k tokens of 8 heads of 128 read back (132 MB) 26.2 us = 5.0 TB/s, 0.77 of the measured copy rate;
// out of 16 bits (206 MB) 39 = 5.3.
#include <algorithm>
#include <type_traits>

#include "paged.cuh"

namespace tpb {
namespace {

constexpr int kAppendThreads = 256;      // of a block at most
constexpr int kPairThreads = 256, kPairBlocks = 4;
constexpr int kReadThreads = 256;
constexpr int kAppendTokens = 6;         // of a block at most
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

// Two floats an instruction, each result rounded by itself
__device__ __forceinline__ uint64_t two(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 one_by_one(uint64_t p) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
template <typename T>
__device__ __forceinline__ uint64_t unpack2(uint32_t w) {
    const float2 f = Half16<T>::unpack(w);
    return two(f.x, f.y);
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(uint64_t p) {
    const float2 f = one_by_one(p);
    return Half16<T>::pack(f.x, f.y);
}

// 16 values of a type as eight words -> a scale and 16 codes.  The quotient is x times the rounded inverse of s, off by |x / s| 2^-24: less than 2^-21 up to
// 6 (s may have been rounded down, so that quotients pass 6; there the conversion saturates).
// Ties are common (s has four bits, x eight or eleven) and have to stay ties: the sum with 128 rounds the quotient to a multiple of 2^-17 or 2^-16, half a
// step of which, 2^-18, is more than that error.  A quotient that is no tie is 2^-13 from one at least, since x differs from a tie times s, which the type
// of x holds, by a step of that type.  (Powers of two in `inv` change nothing of this.)
template <typename T>
__device__ __forceinline__ void quantise16(const uint32_t (&x)[8], float inv, uint2& codes, uint32_t& scale) {
    constexpr uint32_t kInf = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    uint32_t both = 0;                   // the largest size in the low halves and in the high ones: sizes are ordered as their bits are
#pragma unroll
    for (int i = 0; i < 8; ++i) both = __vmaxu2(both, x[i] & 0x7fff7fffu);
    const uint32_t top = max(both & 0xffffu, both >> 16);
    codes = make_uint2(0, 0);
    scale = 0x7f;                        // NaN
    if (top >= kInf) return;
    scale = encode_e4m3(__fdiv_rn(Half16<T>::unpack(top).x * inv, 6.0f));
    if (scale == 0) return;
    const float inverse = __frcp_rn(decode_e4m3(static_cast<uint8_t>(scale))) * inv;
    const uint64_t f = two(inverse, inverse), up = two(128.0f, 128.0f), down = two(-128.0f, -128.0f);
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float y[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 q = one_by_one(add2(fma2(unpack2<T>(x[i * 4 + j]), f, up), down));
            y[2 * j] = q.x;
            y[2 * j + 1] = q.y;
        }
        asm("{\n .reg .b8 a, b, c, d;\n cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
            " cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n mov.b32 %0, {a, b, c, d};\n}\n"
            : "=r"(w[i]) : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
    }
    codes = make_uint2(w[0], w[1]);
}

// Turns V values and the V values half a row further on: x c - y s and y c + x s in fp32, each operation rounded, as elementary operations give
// them whatever else is compiled around them, then rounded to the type
template <typename T, int V>
__device__ __forceinline__ void turn_pair(Vec<V>& a, Vec<V>& b, const AppendParams& P, int pos, int at) {
    float c[V], s[V];
    const size_t e = static_cast<size_t>(pos) * (P.cache.head_dim / 2) + at;
    load_table<V>(P.cos, P.rope_dtype, e, c);
    load_table<V>(P.sin, P.rope_dtype, e, s);
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
        const uint64_t x = unpack2<T>(a.w[j]), y = unpack2<T>(b.w[j]), c2 = two(c[2 * j], c[2 * j + 1]), s2 = two(s[2 * j], s[2 * j + 1]);
        a.w[j] = pack2<T>(fma2(mul2(y, s2), two(-1.0f, -1.0f), mul2(x, c2)));
        // (a packed sum of packed products would become a product and a fused sum)
        const float2 p = one_by_one(mul2(y, c2)), q = one_by_one(mul2(x, s2));
        b.w[j] = Half16<T>::pack(__fadd_rn(p.x, q.x), __fadd_rn(p.y, q.y));
    }
}

// Head sizes that are multiples of 32.  A unit of the queries is 8 values and the 8 values half a row further on; of the keys and values two blocks of
// 16, half a row apart for keys that are turned, else side by side.  A thread keeps its unit for all tokens of the block, and has 64 bytes on their way:
// two tokens of the queries, or one of the keys or values.
template <typename T>
__global__ void __launch_bounds__(kPairThreads, kPairBlocks) append_pairs_kernel(const __grid_constant__ AppendParams P) {
    __shared__ int seq[kAppendTokens];
    __shared__ int position[kAppendTokens];
    __shared__ long long row_at[kAppendTokens];
    pdl_wait_prior_grids();
    pdl_launch_dependents();
    const int t0 = blockIdx.x * P.tokens_per_block;
    const int count = min(P.tokens_per_block, P.tokens - t0);
    const int per_token = P.units_q + 2 * P.units_kv;
    const int D = P.cache.head_dim, half = D / 2, per_row = half / 8, groups = D / 32;
    bool placed = false;
    for (int base = 0; base < per_token; base += blockDim.x) {
        const int u = base + threadIdx.x;
        const bool mine = u < per_token;
        const int kind = u < P.units_q ? 0 : (u < P.units_q + P.units_kv ? 1 : 2);       // queries, keys, values
        const int r = u - (kind == 0 ? 0 : (kind == 1 ? P.units_q : P.units_q + P.units_kv));
        const int head = kind == 0 ? r / per_row : r / groups, in = kind == 0 ? r - head * per_row : r - head * groups;
        const bool turn = P.rope_positions > 0 && kind < 2;
        const int at = kind == 0 ? in * 8 : (turn ? in * 16 : in * 32), at2 = turn ? at + half : at + 16;        // first columns of the two blocks
        const long long* st = kind == 0 ? P.q_stride : (kind == 1 ? P.k_stride : P.v_stride);
        const long long step = st[0];
        const uint16_t* src = (kind == 0 ? P.q : (kind == 1 ? P.k : P.v)) + t0 * step + head * st[1] + at;
        const int apart = at2 - at;
        const int tokens = kind == 0 ? 2 : 1;
        Vec<8> a, b, a2, b2;             // of the queries: a, b of a token, a2, b2 of the next; else the first and second halves of two blocks
        auto load = [&](int first) {
            const uint16_t* row = src + first * step;
            if (!mine || first >= count) return;
            a = load_vec<8>(row);
            b = load_vec<8>(row + apart);
            row += kind == 0 ? step : 8;
            if (kind == 0 && first + 1 >= count) return;
            a2 = load_vec<8>(row);
            b2 = load_vec<8>(row + apart);
        };
        load(0);
        if (!placed) {                   // the tokens' rows, behind the first loads
            placed = true;
            place_tokens<true, kAppendTokens>(P.cache, P.cu, t0, count, P.rope_positions, seq, position, row_at);
        }
        for (int first = 0; mine && first < count; first += tokens) {
            if (kind == 0) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (first + i >= count || row_at[first + i] < 0) continue;
                    Vec<8>&x = i == 0 ? a : a2, &y = i == 0 ? b : b2;
                    turn_pair<T, 8>(x, y, P, position[first + i], at);
                    uint16_t* to = P.q_out + (t0 + first + i) * P.o_stride[0] + head * P.o_stride[1] + at;
                    store_vec<8>(to, x);
                    store_vec<8>(to + half, y);
                }
            } else if (row_at[first] >= 0) {
                const int pos = position[first];
                if (turn) {
                    turn_pair<T, 8>(a, b, P, pos, at);
                    turn_pair<T, 8>(a2, b2, P, pos, at + 8);
                }
                uint8_t* tile = static_cast<uint8_t*>(kind == 1 ? P.cache.k_pages : P.cache.v_pages) + row_at[first] + head * P.cache.head_stride;
                const float inv = kind == 1 ? P.k_inv : P.v_inv;
                uint8_t* codes_at = tile + (pos & 15) * 16 * groups;
                uint8_t* scales_at = tile + 256 * groups + (pos & 15) * 2 * groups;
                const uint32_t x[8] = {a.w[0], a.w[1], a.w[2], a.w[3], a2.w[0], a2.w[1], a2.w[2], a2.w[3]};
                const uint32_t y[8] = {b.w[0], b.w[1], b.w[2], b.w[3], b2.w[0], b2.w[1], b2.w[2], b2.w[3]};
                uint2 codes, codes2;
                uint32_t scale, scale2;
                quantise16<T>(x, inv, codes, scale);
                quantise16<T>(y, inv, codes2, scale2);
                if (turn) {
                    *reinterpret_cast<uint2*>(codes_at + at / 2) = codes;
                    *reinterpret_cast<uint2*>(codes_at + at2 / 2) = codes2;
                    scales_at[at / 16] = static_cast<uint8_t>(scale);
                    scales_at[at2 / 16] = static_cast<uint8_t>(scale2);
                } else {
                    *reinterpret_cast<uint4*>(codes_at + at / 2) = make_uint4(codes.x, codes.y, codes2.x, codes2.y);
                    *reinterpret_cast<uint16_t*>(scales_at + at / 16) = static_cast<uint16_t>(scale | scale2 << 8);
                }
            }
            load(first + tokens);
        }
    }
}

// Other head sizes.  A unit of the queries is V values and the V values half a row further on, V = 8 where half a row is a multiple of 8, else 4; a unit of
// the keys or values is a block of 16, for keys that are turned with the 16 values half a row away beside it.  A thread keeps its unit for all tokens of the
// block.
template <typename T, int V>
__global__ void __launch_bounds__(kAppendThreads, 4) append_blocks_kernel(const __grid_constant__ AppendParams P) {
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
        const bool turn = P.rope_positions > 0 && kind < 2;
        const int at = kind == 0 ? in * V : in * 16;     // first column; the partners of column c stand at c + half or c - half
        const long long* st = kind == 0 ? P.q_stride : (kind == 1 ? P.k_stride : P.v_stride);
        const long long step = st[0];
        const uint16_t* src = (kind == 0 ? P.q : (kind == 1 ? P.k : P.v)) + t0 * step + head * st[1];
        for (int t = 0; t < count; ++t) {
            Vec<V> x[kVecs], y[kVecs];
            if (mine) {
                const uint16_t* row = src + t * step;
#pragma unroll
                for (int n = 0; n < kVecs; ++n) {
                    const int c = at + n * V;
                    x[n] = y[n] = Vec<V>{};
                    if ((kind == 0 && n > 0) || c >= D) continue;
                    x[n] = load_vec<V>(row + c);
                    if (turn) y[n] = load_vec<V>(row + (c < half ? c + half : c - half));
                }
            }
            if (!placed) {               // the tokens' rows, behind the first loads
                placed = true;
                place_tokens<true, kAppendTokens>(P.cache, P.cu, t0, count, P.rope_positions, seq, position, row_at);
            }
            const long long row = row_at[t];
            if (!mine || row < 0) continue;
            const int pos = position[t];
            if (kind == 0) {
                turn_pair<T, V>(x[0], y[0], P, pos, at);
                uint16_t* to = P.q_out + (t0 + t) * P.o_stride[0] + head * P.o_stride[1] + at;
                store_vec<V>(to, x[0]);
                store_vec<V>(to + half, y[0]);
                continue;
            }
            if (turn) {
#pragma unroll
                for (int n = 0; n < kVecs; ++n) {
                    const int c = at + n * V;
                    if (c < half) turn_pair<T, V>(x[n], y[n], P, pos, c);
                    else if (c < D) turn_pair<T, V>(y[n], x[n], P, pos, c - half);
                }
            }
            uint8_t* tile = static_cast<uint8_t*>(kind == 1 ? P.cache.k_pages : P.cache.v_pages) + row + head * P.cache.head_stride;
            const float inv = kind == 1 ? P.k_inv : P.v_inv;
            uint8_t* codes_at = tile + (pos & 15) * 16 * groups;
            uint8_t* scales_at = tile + 256 * groups + (pos & 15) * 2 * groups;
            uint2 codes;
            uint32_t scale;
            quantise16<T>(reinterpret_cast<const uint32_t(&)[8]>(x), inv, codes, scale);
            *reinterpret_cast<uint2*>(codes_at + in * 8) = codes;
            scales_at[in] = static_cast<uint8_t>(scale);
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
    int units;                           // per token of keys, and of values
    float k_scale, v_scale;
};

// A thread has a unit, 16 columns of a head's keys or values (8 of 16-bit pages), of every kLanes-th token of the block.  kWide: the rows it writes begin
// on 32 bytes, and a unit leaves in one store.
template <typename T, bool kTiles, bool kWide>
__global__ void __launch_bounds__(kReadThreads) read_kernel(const __grid_constant__ ReadParams P) {
    __shared__ int seq[kReadTokens];
    __shared__ int position[kReadTokens];
    __shared__ long long row_at[kReadTokens];
    pdl_wait_prior_grids();
    pdl_launch_dependents();
    const int t0 = blockIdx.x * P.tokens_per_block;
    const int count = min(P.tokens_per_block, P.tokens - t0);
    const int named = blockIdx.x == 0 && threadIdx.x == 0 ? P.cu[P.cache.seqs] : 0;       // rows that the offsets name
    place_tokens<kTiles, kReadTokens>(P.cache, P.cu, t0, count, 0, seq, position, row_at);
    constexpr int kColumns = kTiles ? 16 : 8;
    const int D = P.cache.head_dim, per_row = (D + kColumns - 1) / kColumns, groups = (D + 31) / 32;
    const int all = 2 * P.units, lanes = max(1, static_cast<int>(blockDim.x) / all), lane = all <= static_cast<int>(blockDim.x) ? threadIdx.x / all : 0;
    if (lane >= lanes) return;
    for (int u = threadIdx.x - lane * all; u < all; u += blockDim.x) {
        const bool keys = u < P.units;
        const int r = keys ? u : u - P.units, head = r / per_row, in = r - head * per_row;
        const uint8_t* from = static_cast<const uint8_t*>(keys ? P.cache.k_pages : P.cache.v_pages) + head * P.cache.head_stride * (kTiles ? 1 : 2);
        const long long* st = keys ? P.k_stride : P.v_stride;
        const long long step = lanes * st[0];
        uint16_t* to = (keys ? P.k : P.v) + (t0 + lane) * st[0] + head * st[1] + in * kColumns;
        const float factor = keys ? P.k_scale : P.v_scale;
        const bool whole = kWide || in * kColumns + kColumns <= D;       // of 16 columns the last 8 may be past the head's
        for (int first = lane; first < count; first += lanes * kReadLoads) {
            uint4 x[kReadLoads];
            long long row[kReadLoads];
#pragma unroll
            for (int i = 0; i < kReadLoads; ++i) {
                const int t = first + i * lanes;
                x[i] = make_uint4(0, 0, 0, 0);
                row[i] = t < count ? row_at[t] : -2;
                if (row[i] < 0) continue;
                if constexpr (kTiles) {
                    const uint8_t* tile = from + row[i];
                    const int line = (position[t] & 15) * 2 * groups;
                    const uint2 codes = __ldg(reinterpret_cast<const uint2*>(tile + line * 8 + in * 8));
                    x[i] = make_uint4(codes.x, codes.y, __ldg(tile + 256 * groups + line + in), 0);
                } else {
                    x[i] = __ldg(reinterpret_cast<const uint4*>(from + 2 * row[i] + in * 16));
                }
            }
#pragma unroll
            for (int i = 0; i < kReadLoads; ++i, to += step) {
                if (row[i] == -2) continue;
                if constexpr (kTiles) {
                    const float s = decode_e4m3(static_cast<uint8_t>(x[i].z)) * factor;
                    uint32_t w[8];
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        __half2 h[4];
                        decode_e2m1x8(half == 0 ? x[i].x : x[i].y, h);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {    // exact but for an overflow of fp16 or a factor's underflow
                            const float2 f = __half22float2(h[j]);
                            w[half * 4 + j] = Half16<T>::pack(f.x * s, f.y * s);
                        }
                    }
                    if constexpr (kWide) {
                        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                                     "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
                    } else {
                        *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
                        if (whole) *reinterpret_cast<uint4*>(to + 8) = make_uint4(w[4], w[5], w[6], w[7]);
                    }
                } else {
                    *reinterpret_cast<uint4*>(to) = x[i];
                }
            }
        }
    }
    // A captured call whose offsets have grown: what a caller goes on to use lacks tokens
    if (named > P.tokens) record_error(kErrPagedIndex);
}

// a block's threads for `units` a token: as few passes over them as `most` threads allow, and those even
int threads_for(long long units, int most) {
    const long long passes = (units + most - 1) / most;
    return static_cast<int>(((units + passes - 1) / passes + 31) / 32 * 32);
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
    const long long bytes = tiles ? nvfp4_pool_bytes(cache) : pool_bytes(cache, 2ll * cache.head_dim, cache.page_size, 2);
    TPB_REQUIRE(!rows_in_pools(k, cache, bytes) && !rows_in_pools(v, cache, bytes), TPB200_ERR_SHAPE);
    P.k = static_cast<uint16_t*>(a->k);
    P.v = static_cast<uint16_t*>(a->v);
    P.cu = a->cu;
    P.tokens = a->tokens;
    P.k_scale = k_scale;
    P.v_scale = v_scale;
    const long long units = static_cast<long long>(tiles ? (cache.head_dim + 15) / 16 : cache.head_dim / 8) * cache.kv_heads;
    TPB_REQUIRE(units <= (1 << 24), TPB200_ERR_SHAPE);
    P.units = static_cast<int>(units);
    const int threads = 2 * units <= kReadThreads ? kReadThreads : threads_for(2 * units, kReadThreads), lanes = std::max(1, static_cast<int>(threads / (2 * units)));
    // a block's look-up serves up to a tile of tokens, fewer where that would leave SMs without a block, but at least one for each lane
    P.tokens_per_block = std::max(std::min(lanes, kReadTokens), std::min(kReadTokens, a->tokens / 592));
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = paged_config(static_cast<unsigned>((a->tokens - 1) / P.tokens_per_block + 1), threads, 0, &attr, stream);
    bool wide = cache.head_dim % 16 == 0 && (reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v)) % 32 == 0;
    for (const long long st : {P.k_stride[0], P.k_stride[1], P.v_stride[0], P.v_stride[1]}) wide = wide && st % 16 == 0;
    auto pick = [&](auto type) { return wide ? read_kernel<decltype(type), true, true> : read_kernel<decltype(type), true, false>; };
    const auto kernel = !tiles ? read_kernel<__half, false, false> : (a->dtype == TPB200_BF16 ? pick(__nv_bfloat16()) : pick(__half()));
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
    // tiles that are written twice, and rows in the pages that other threads write
    TPB_REQUIRE(!nvfp4_tiles_meet(P.cache), TPB200_ERR_SHAPE);
    const int D = P.cache.head_dim, H = P.cache.kv_heads;
    const long long bytes = nvfp4_pool_bytes(P.cache);
    const RowSet k_rows(a->k, a->k_stride, a->tokens, H, D), v_rows(a->v, a->v_stride, a->tokens, H, D);
    TPB_REQUIRE(!rows_in_pools(k_rows, P.cache, bytes) && !rows_in_pools(v_rows, P.cache, bytes), TPB200_ERR_SHAPE);
    if (a->q != nullptr) {               // other threads read what lies there
        const RowSet in(a->q, a->q_stride, a->tokens, a->q_heads, D), out(a->q_out, a->o_stride, a->tokens, a->q_heads, D);
        TPB_REQUIRE(output_fits(out, in) && !rows_meet(out, k_rows) && !rows_meet(out, v_rows), TPB200_ERR_SHAPE);
        TPB_REQUIRE(!rows_in_pools(in, P.cache, bytes) && !rows_in_pools(out, P.cache, bytes), TPB200_ERR_SHAPE);
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
    const long long units_q = a->q != nullptr ? static_cast<long long>(half / V) * a->q_heads : 0, units_kv = (D % 32 == 0 ? 1ll : 2ll) * ((D + 31) / 32) * H;
    TPB_REQUIRE(units_q + 2 * units_kv <= (1 << 24), TPB200_ERR_SHAPE);
    P.units_q = static_cast<int>(units_q);
    P.units_kv = static_cast<int>(units_kv);
    // Six tokens share a block's look-up, of other head sizes four, fewer where that would leave SMs without a block (the prompts of six sequences 66 us, with four
    // 68, eight 73; heads of 72, 4800 tokens, 37 with four, 46 with six)
    const bool pairs = D % 32 == 0;
    P.tokens_per_block = std::max(1, std::min(pairs ? kAppendTokens : kAppendTokens - 2, a->tokens / 444));
    const unsigned blocks = static_cast<unsigned>((a->tokens - 1) / P.tokens_per_block + 1);
    const bool bf = a->dtype == TPB200_BF16;
    auto pick = [&](auto type) {
        using T = decltype(type);
        return pairs ? append_pairs_kernel<T> : (V == 8 ? append_blocks_kernel<T, 8> : append_blocks_kernel<T, 4>);
    };
    const auto kernel = bf ? pick(__nv_bfloat16()) : pick(__half());
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = paged_config(blocks, threads_for(units_q + 2 * units_kv, pairs ? kPairThreads : kAppendThreads), 0, &attr,
                                                reinterpret_cast<cudaStream_t>(stream));
    return cudaLaunchKernelEx(&cfg, kernel, P) == cudaSuccess ? TPB200_OK : TPB200_ERR_CUDA;
}
