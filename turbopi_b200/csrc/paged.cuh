// What the kernels on a cache of pages share: the view of the cache, its checks, 16-bit pairs.
#pragma once

#include <algorithm>
#include <cmath>

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

// Weights 2^(scale S - m), the product fused into the sum, are off by the rounding of their reference m, the product of the largest score.  It cancels out
// with their sum, but from 2^24 on it may be a factor of two, which fp16 weights have no room for, and from 2^31 on all of them may be infinite, or zeros.
// Past this size (a quarter of a power of two) scores are rounded first, as the reference is, so that the largest weight is what it should be.  Asking costs
// short prompts most: 24 of 1 to 1200 tokens, 16 on 4 heads of 64, 26.0 -> 26.3 us; others up to 1 %.
constexpr float kFar = 4194304.0f;       // 2^22

// V values of a 16-bit type
template <int V>
struct Vec { uint32_t w[V / 2]; };

template <int V>
__device__ __forceinline__ Vec<V> load_vec(const uint16_t* p) {
    Vec<V> r;
    if constexpr (V == 8) {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        r.w[0] = u.x; r.w[1] = u.y; r.w[2] = u.z; r.w[3] = u.w;
    } else {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        r.w[0] = u.x; r.w[1] = u.y;
    }
    return r;
}
template <int V>
__device__ __forceinline__ void store_vec(uint16_t* p, const Vec<V>& r) {
    if constexpr (V == 8) *reinterpret_cast<uint4*>(p) = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
    else *reinterpret_cast<uint2*>(p) = make_uint2(r.w[0], r.w[1]);
}

// V consecutive table entries as floats
template <int V>
__device__ __forceinline__ void load_table(const void* p, int dtype, size_t at, float (&f)[V]) {
    if (dtype == TPB200_F32) {
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            const float4 t = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + at + i));
            f[i] = t.x; f[i + 1] = t.y; f[i + 2] = t.z; f[i + 3] = t.w;
        }
    } else {
        const Vec<V> t = load_vec<V>(static_cast<const uint16_t*>(p) + at);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            const float2 x = dtype == TPB200_F16 ? Half16<__half>::unpack(t.w[i]) : Half16<__nv_bfloat16>::unpack(t.w[i]);
            f[2 * i] = x.x;
            f[2 * i + 1] = x.y;
        }
    }
}

// Asynchronous copies of 16 bytes into shared memory, the bytes past `bytes` zero
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

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

// A cache of 4-bit values as a PagedView: strides in bytes, row_stride from one tile of 16 tokens to the next
static inline int paged_view_nvfp4(const tpb200_paged_nvfp4_cache& c, PagedView* v) {
    TPB_REQUIRE(c.seqs >= 0 && c.num_pages >= 1 && c.kv_heads >= 1 && c.table_width >= 1, TPB200_ERR_SHAPE);
    TPB_REQUIRE(c.page_size >= 16 && c.page_size % 16 == 0, TPB200_ERR_SHAPE);
    TPB_REQUIRE(c.head_dim >= 8 && c.head_dim <= 256 && c.head_dim % 8 == 0, TPB200_ERR_SHAPE);
    TPB_REQUIRE(static_cast<long long>(c.page_size) * c.table_width <= 0x7fffffff, TPB200_ERR_SHAPE);   // positions are 32 bits
    TPB_REQUIRE(c.k_pages && c.v_pages, TPB200_ERR_NULL);
    TPB_REQUIRE(c.seqs == 0 || (c.table && c.lengths), TPB200_ERR_NULL);
    TPB_REQUIRE(tpb_aligned16(c.k_pages) && tpb_aligned16(c.v_pages), TPB200_ERR_ALIGN);
    TPB_REQUIRE(c.seqs <= 1 || c.table_stride >= 0, TPB200_ERR_SHAPE);
    for (const float f : {c.k_scale, c.v_scale}) {           // powers of two: what is held stays exact in 16 bits
        int e = 0;
        TPB_REQUIRE(std::isfinite(f) && std::frexp(f, &e) == 0.5f && e >= -62 && e <= 65, TPB200_ERR_SHAPE);
    }
    const long long tile = 288ll * ((c.head_dim + 31) / 32), strides[3] = {c.page_stride, c.head_stride, c.tile_stride};
    const int sizes[3] = {c.num_pages, c.kv_heads, c.page_size / 16};
    for (int i = 0; i < 3; ++i) {
        TPB_REQUIRE(sizes[i] <= 1 || strides[i] % 16 == 0, TPB200_ERR_ALIGN);
        TPB_REQUIRE(strides[i] >= 0 && (sizes[i] <= 1 || strides[i] >= tile), TPB200_ERR_SHAPE);
    }
    auto used = [](long long stride, int n) { return n > 1 ? stride : 0; };
    *v = {c.k_pages, c.v_pages, used(c.page_stride, c.num_pages), used(c.tile_stride, c.page_size / 16), used(c.head_stride, c.kv_heads), c.table,
          c.lengths, used(c.table_stride, c.seqs), c.num_pages, c.page_size, c.kv_heads, c.head_dim, c.table_width, c.seqs};
    return TPB200_OK;
}

// bytes from the first to behind the last of a cache's keys, and of its values
static inline long long pool_bytes(const PagedView& c, long long row_bytes, int rows, int element) {
    return ((c.num_pages - 1) * c.page_stride + (rows - 1) * c.row_stride + (c.kv_heads - 1) * c.head_stride) * element + row_bytes;
}
static inline long long nvfp4_tile_bytes(const PagedView& c) { return 288ll * ((c.head_dim + 31) / 32); }
static inline long long nvfp4_pool_bytes(const PagedView& c) { return pool_bytes(c, nvfp4_tile_bytes(c), c.page_size / 16, 1); }
// whether rows reach into what lies between a pool's first and last byte
static inline bool rows_in_pools(const RowSet& rows, const PagedView& c, long long bytes) {
    for (const void* pages : {c.k_pages, c.v_pages}) {
        const long long at = static_cast<long long>(reinterpret_cast<uintptr_t>(pages));
        if (2 * rows.end() > at && at + bytes > 2 * rows.at) return true;
    }
    return false;
}
// Whether a tile of the keys shares bytes with one of the values (which may lie between the keys' pages, heads or tiles), or two of either do.  Dimensions whose
// strides reach over the ones below them, as those of any tensor do, have one place or two near a distance to look at; others count as meeting.
static inline bool nvfp4_tiles_meet(const PagedView& c) {
    const long long tile = nvfp4_tile_bytes(c);
    struct { long long stride; int n; } dim[3] = {{c.page_stride, c.num_pages}, {c.head_stride, c.kv_heads}, {c.row_stride, c.page_size / 16}};
    std::sort(dim, dim + 3, [](const auto& a, const auto& b) { return a.stride > b.stride; });       // of one: 0, and the last
    long long reach[4] = {0, 0, 0, tile};            // bytes of the dimensions from i on
    for (int i = 2; i >= 0; --i) {
        reach[i] = reach[i + 1] + (dim[i].n - 1) * dim[i].stride;
        if (dim[i].n > 1 && dim[i].stride < reach[i + 1]) return true;
    }
    long long d = static_cast<long long>(reinterpret_cast<uintptr_t>(c.v_pages)) - static_cast<long long>(reinterpret_cast<uintptr_t>(c.k_pages));
    if (d < 0) d = -d;
    auto near = [&](auto&& self, int i, long long off) -> bool {       // whether places `off` apart but for the dimensions before i may share bytes
        if (off <= -reach[i] || off >= reach[i]) return false;
        if (i == 3) return true;
        if (dim[i].n == 1) return self(self, i + 1, off);
        const long long s = dim[i].stride, t = off / s - (off % s < 0);             // rounded down
        for (const long long x : {t, t + 1}) {
            if (x > -dim[i].n && x < dim[i].n && self(self, i + 1, off - x * s)) return true;
        }
        return false;
    };
    return near(near, 0, d);
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
