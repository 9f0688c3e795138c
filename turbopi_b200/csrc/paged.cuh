// What the kernels on a cache of pages share: the view of the cache, its checks, 16-bit pairs.
#pragma once

#include "common.cuh"

namespace tpb {

// Pairs of a 16-bit type in a 32-bit word
template <typename T>
struct Half16;
template <>
struct Half16<__nv_bfloat16> {
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
