// What the kernels on a cache of pages share: the view of the cache, its checks, 16-bit pairs.
#pragma once

#include <algorithm>

#include "common.cuh"

namespace tpb {

// Pairs of a 16-bit type in a 32-bit word.  kLift: softmax weights, which are rounded to the type for their product with the values, are held
// 2^kLift times larger than against their reference, which the sum's division takes out again.  fp16 has no exponents below -14 and steps of
// 2^-24 there; a weight is at most 2^8 of its reference, so seven bits are free at the other end (2^15 < 65504), and weights keep their eleven bits
// down to 2^-21 and vanish below 2^-32.  bf16 has fp32's exponents.
template <typename T>
struct Half16;
template <>
struct Half16<__nv_bfloat16> {
    static constexpr float kLift = 0.0f;
    static __device__ __forceinline__ float2 unpack(uint32_t w) {
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    // x * 0 + sum: NaN from the first infinity or NaN on
    static __device__ __forceinline__ uint32_t add_zeros(uint32_t x, uint32_t sum) {
        const __nv_bfloat162 h = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&x), __nv_bfloat162(__float2bfloat16_rn(0.0f), __float2bfloat16_rn(0.0f)),
                                         *reinterpret_cast<const __nv_bfloat162*>(&sum));
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};
template <>
struct Half16<__half> {
    static constexpr float kLift = 7.0f;
    static __device__ __forceinline__ float2 unpack(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ uint32_t add_zeros(uint32_t x, uint32_t sum) {
        const __half2 h = __hfma2(*reinterpret_cast<const __half2*>(&x), __half2(__float2half_rn(0.0f), __float2half_rn(0.0f)),
                                  *reinterpret_cast<const __half2*>(&sum));
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};

// The cache as a kernel sees it.  Offsets are in elements and 64 bits wide: a pool of pages passes 2^31 elements at 4 GB.
struct PagedView {
    void *k_pages, *v_pages;
    long long page_stride, row_stride, head_stride;
    const int *table, *lengths;
    long long table_stride;
    int num_pages, page_size, kv_heads, head_dim, table_width, seqs;

    // offset of the row of `pos` of sequence s, -1 where the table has none
    __device__ __forceinline__ long long row_offset(int s, int pos) const {
        if (pos < 0) return -1;
        const int i = pos / page_size;
        if (i >= table_width) return -1;
        const int id = table[s * table_stride + i];
        if (static_cast<unsigned>(id) >= static_cast<unsigned>(num_pages)) return -1;
        return id * page_stride + (pos - i * page_size) * row_stride;
    }
};

// A stride between `n` rows of head_dim values: of one row it does not matter, else the rows lie apart, whole 16-byte groups
static inline int paged_stride(long long stride, int n, int head_dim) {
    TPB_REQUIRE(n <= 1 || stride % 8 == 0, TPB200_ERR_ALIGN);
    TPB_REQUIRE(stride >= 0 && (n <= 1 || stride >= head_dim), TPB200_ERR_SHAPE);
    return TPB200_OK;
}

// Rows of head_dim 16-bit values, [n0][n1] with element strides; where heads lie side by side a token is one run
struct RowSet {
    long long at, s0, s1;
    int n0, n1, width;
    RowSet(const void* p, const long long (&stride)[2], int tokens, int heads, int head_dim)
        : at(static_cast<long long>(reinterpret_cast<uintptr_t>(p) / 2)), s0(stride[0]), s1(stride[1]), n0(tokens), n1(heads), width(head_dim) {
        if (n1 > 1 && s1 == width) {
            width *= n1;
            n1 = 1;
        }
    }
    long long token() const { return (n1 - 1) * s1 + width; }
    long long end() const { return at + (n0 - 1) * s0 + token(); }
};

// Whether runs of `a` and `b` values, the second `d` behind the first, meet when the second moves on by t * s0 for a t in [first, last]
static inline bool runs_meet(long long d, int a, int b, long long s0, long long first, long long last) {
    const long long lo = 1 - b - d, hi = a - 1 - d;              // what t * s0 has to lie between
    const long long t_lo = lo > 0 ? (lo + s0 - 1) / s0 : -(-lo / s0), t_hi = hi >= 0 ? hi / s0 : -((-hi + s0 - 1) / s0);
    return std::max(t_lo, first) <= std::min(t_hi, last);
}
// Whether two sets share an element.  Views of one tensor (equal token strides) are compared row by row; sets of different
// strides whose ranges meet count as meeting.
static inline bool rows_meet(const RowSet& a, const RowSet& b) {
    if (a.n0 < 1 || b.n0 < 1 || a.at >= b.end() || b.at >= a.end()) return false;
    if (a.n0 > 1 && b.n0 > 1 && a.s0 != b.s0) return true;
    const long long s0 = a.n0 > 1 ? a.s0 : (b.n0 > 1 ? b.s0 : 1);
    for (int i = 0; i < a.n1; ++i) {
        for (int j = 0; j < b.n1; ++j) {
            if (runs_meet(b.at + j * b.s1 - a.at - i * a.s1, a.width, b.width, s0, 1ll - a.n0, b.n0 - 1ll)) return true;
        }
    }
    return false;
}
// Whether two rows of an output share an element
static inline bool rows_cross(const RowSet& a) {
    if (a.n0 < 2) return false;          // heads do not: their stride is at least a row
    if (a.s0 < a.width) return true;
    for (int i = 1; i < a.n1; ++i) {
        if (runs_meet(i * a.s1, a.width, a.width, a.s0, 1ll - a.n0, a.n0 - 1ll)) return true;
    }
    return false;
}
static inline bool rows_same(const RowSet& a, const RowSet& b) {
    return a.at == b.at && a.width == b.width && a.n1 == b.n1 && (a.n1 < 2 || a.s1 == b.s1) && (a.n0 < 2 || a.s0 == b.s0);
}
// An output may lie where its input lies, row on row, and else shares nothing with it or with itself
static inline bool output_fits(const RowSet& out, const RowSet& in) { return !rows_cross(out) && (rows_same(in, out) || !rows_meet(in, out)); }

static inline int paged_view(const tpb200_paged_cache& c, PagedView* v) {
    TPB_REQUIRE(c.seqs >= 0 && c.num_pages >= 1 && c.page_size >= 1 && c.kv_heads >= 1 && c.table_width >= 1, TPB200_ERR_SHAPE);
    TPB_REQUIRE(c.head_dim >= 8 && c.head_dim <= 256 && c.head_dim % 8 == 0, TPB200_ERR_SHAPE);
    TPB_REQUIRE(static_cast<long long>(c.page_size) * c.table_width <= 0x7fffffff, TPB200_ERR_SHAPE);   // positions are 32 bits
    TPB_REQUIRE(c.dtype == TPB200_BF16 || c.dtype == TPB200_F16, TPB200_ERR_ENUM);
    TPB_REQUIRE(c.k_pages && c.v_pages, TPB200_ERR_NULL);
    TPB_REQUIRE(c.seqs == 0 || (c.table && c.lengths), TPB200_ERR_NULL);
    TPB_REQUIRE(tpb_aligned16(c.k_pages) && tpb_aligned16(c.v_pages), TPB200_ERR_ALIGN);
    TPB_REQUIRE(c.seqs <= 1 || c.table_stride >= 0, TPB200_ERR_SHAPE);
    const long long strides[3] = {c.page_stride, c.row_stride, c.head_stride};
    const int sizes[3] = {c.num_pages, c.page_size, c.kv_heads};
    for (int i = 0; i < 3; ++i) {
        const int st = paged_stride(strides[i], sizes[i], c.head_dim);
        if (st != TPB200_OK) return st;
    }
    auto used = [](long long stride, int n) { return n > 1 ? stride : 0; };
    *v = {c.k_pages, c.v_pages, used(c.page_stride, c.num_pages), used(c.row_stride, c.page_size), used(c.head_stride, c.kv_heads), c.table,
          c.lengths, used(c.table_stride, c.seqs), c.num_pages, c.page_size, c.kv_heads, c.head_dim, c.table_width, c.seqs};
    return TPB200_OK;
}

// These kernels wait for the launch before them ahead of everything they read or write, so they are always launched as dependents
// (TPB200_FLAG_PDL or not): their CTAs start while it drains.  They let the next launch in behind that wait, not before it: what was
// enqueued ahead of one of them is complete when a launch behind it starts, as behind any launch without the flag.
static inline cudaLaunchConfig_t paged_config(unsigned blocks, int threads, size_t smem, cudaLaunchAttribute* attr, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks, 1, 1);
    cfg.blockDim = dim3(threads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    attr->id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr->val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cfg;
}

}  // namespace tpb
