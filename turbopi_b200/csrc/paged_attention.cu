// Attention of one new token per sequence on a cache of pages: softmax(scale q K^T) V with grouped heads, sequences of any
// lengths, bf16 or fp16.
//
// The work is the bytes of the cache (every key and value row once; 4 g flops per byte pair with g query heads to a key head), so
// the kernel is a stream from HBM with the arithmetic hung into it:
//
//   * The keys of all (sequence, key head) items form one line of chunks; each of the resident CTAs takes an equal piece of it,
//     whatever the sequences' lengths.  A CTA reads the lengths and finds its piece itself: the host plans nothing and the call
//     can be captured while lengths and table change under it.  An item that crosses CTAs leaves partial sums (fp32 sums relative
//     to their maximum, the maximum, the sum of the weights) in the workspace, at most two to a CTA, and a second kernel joins them
//     in order: the result does not depend on who came first.
//   * A warp works on its own: rows of keys, then rows of values, come through a ring of three 8 KB slots of its own by 16-byte
//     asynchronous copies, with two slots on their way while it works on the third; no barrier inside a piece, also from one item
//     to the next.  8 warps an SM keep 128 KB on their way, three times what latency times bandwidth needs.
//   * The products are turned round: S^T = K Q^T and O^T = V^T P^T put the keys and the columns of V on the 16-row side of
//     mma.sync and the g query heads that share a key head on its 8-column side, so that up to eight heads cost one tile and each byte
//     of the cache crosses the SM once.  P^T comes out of S^T by one 8x8 transposition in registers.  tcgen05 wants 128
//     rows or columns of queries; this needs a seventh of the instruction slots that an SM's share of the stream leaves (16 KB per 700 cycles).
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "paged.cuh"

namespace tpb {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kSlotBytes = 8192;
constexpr int kSlots = 3;
constexpr int kCtasPerSm = 2;

struct DecodeParams {
    PagedView cache;
    const uint16_t* q;
    uint16_t* out;
    long long q_stride[2], o_stride[2];
    int group;                           // query heads per key head
    int tiles;                           // tiles of query heads per key head
    int rows;                            // rows of a tile that are used at most
    int join_by_item;                    // joins[] has a place per item, else one per CTA
    float scale2;                        // scale * log2 e
    float* part_o;                       // [2 * CTAs][rows][head_dim]
    float* part_ml;                      // [2 * CTAs][rows][2]
    int4* joins;                         // (item or -1, parts, first slot, CTA it begins in)
};

// DP: head_dim rounded up to 64, 128 or 256.  NT: tiles of eight query heads that go through together.
template <int DP, int NT>
struct Shape {
    static constexpr int kKeys = kSlotBytes / (DP * 2);     // keys of a slot: 16, 32, 64
    static constexpr int kChunk = kKeys * kWarps;           // keys of a chunk: a slot for each warp
    static constexpr int kLanesRow = DP / 8;                // lanes that copy a row
    static constexpr int kRowsIter = 32 / kLanesRow;        // rows a warp copies at a time
    static constexpr int kCopies = kKeys / kRowsIter;
    static constexpr int kOwn = (kKeys + 31) / 32;          // rows a lane knows the place of
    static constexpr int kRows = 8 * NT;
    static constexpr bool kQueriesStay = NT * DP <= 256;    // in registers; else they are read again for every slot
    static constexpr int kSlab = NT == 1 ? 64 : 16;         // columns that pass through shared memory at a time when sums are joined
    static constexpr int kSlabPitch = kSlab + 4;            // the four query pairs of a store fall into different banks
};

template <int NT>
struct Control {
    int warp_sum[kWarps];
    int first_seq, first_before;         // the sequence of the CTA's first chunk, and the chunks before it
    float ml[kWarps][8 * NT][2];
};

template <int DP, int NT>
constexpr int smem_bytes() {
    using S = Shape<DP, NT>;
    return kWarps * kSlots * kSlotBytes + S::kRows * DP * 2 + kWarps * S::kRows * S::kSlabPitch * 4 + static_cast<int>(sizeof(Control<NT>));
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    } else {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// keys of a sequence that the cache can hold: a length beyond the table's pages is an error, not an address
__device__ __forceinline__ int keys_of(const PagedView& c, int s) {
    const int n = c.lengths[s], most = c.page_size * c.table_width;
    if (n > most) record_error(kErrPagedIndex);
    return max(0, min(n, most));
}

// A place in the line of chunks: chunk `ci` of item (sequence, tile of query heads)
template <int kChunk>
struct Place {
    int s, h, ci, n, len;                // n: chunks of the sequence's items
    __device__ __forceinline__ void enter(const DecodeParams& P, int seq) {
        for (s = seq; s < P.cache.seqs; ++s) {
            len = keys_of(P.cache, s);
            if (len > 0) break;
        }
        n = (len + kChunk - 1) / kChunk;
        h = ci = 0;
    }
    __device__ __forceinline__ void next(const DecodeParams& P) {
        if (++ci < n) return;
        ci = 0;
        if (++h < P.cache.kv_heads * P.tiles) return;
        enter(P, s + 1);
    }
};

// kAligned: the page size is a multiple of 16, so that 16 rows from a multiple of 16 on lie in one page and share an address
template <typename T, int DP, int NT, bool kAligned>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) paged_attention_kernel(const __grid_constant__ DecodeParams P) {
    using S = Shape<DP, NT>;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* sq = smem + kWarps * kSlots * kSlotBytes;                                  // queries of the item
    float* slab = reinterpret_cast<float*>(sq + S::kRows * DP * 2);
    Control<NT>* ctl = reinterpret_cast<Control<NT>*>(slab + kWarps * S::kRows * S::kSlabPitch);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int heads = P.cache.kv_heads * P.tiles;
    const int D = P.cache.head_dim;
    pdl_launch_dependents();
    pdl_wait_prior_grids();

    // ------------------------------------------------ this CTA's piece of the line
    // Chunks before each thread's run of sequences, then the sequence that holds the first chunk.
    const int run = (P.cache.seqs + kThreads - 1) / kThreads, s0 = min(P.cache.seqs, static_cast<int>(threadIdx.x) * run),
              s1 = min(P.cache.seqs, s0 + run);
    int mine = 0;
    for (int s = s0; s < s1; ++s) mine += (keys_of(P.cache, s) + S::kChunk - 1) / S::kChunk * heads;
    int before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += y;
    }
    if (lane == 31) ctl->warp_sum[warp] = before;
    __syncthreads();
    int total = 0;
    before -= mine;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += ctl->warp_sum[w];
        total += ctl->warp_sum[w];
    }
    const int ctas = min(static_cast<int>(gridDim.x), total), cta = blockIdx.x;
    const int share = ctas > 0 ? total / ctas : 0, more = ctas > 0 ? total - share * ctas : 0;
    const int begin = cta < ctas ? cta * share + min(cta, more) : total;
    const int end = cta < ctas ? begin + share + (cta < more ? 1 : 0) : total;
    if (begin < end && before <= begin && begin < before + mine) {
        int s = s0, at = before;
        for (;; ++s) {
            const int n = (keys_of(P.cache, s) + S::kChunk - 1) / S::kChunk * heads;
            if (begin < at + n) break;
            at += n;
        }
        ctl->first_seq = s;
        ctl->first_before = at;
    }
    // sequences without keys: zeros
    for (int s = cta; s < P.cache.seqs; s += gridDim.x) {
        if (keys_of(P.cache, s) > 0) continue;
        const int per_head = D / 8;
        for (int i = threadIdx.x; i < P.cache.kv_heads * P.group * per_head; i += kThreads) {
            const int hq = i / per_head, c = i - hq * per_head;
            *reinterpret_cast<uint4*>(P.out + s * P.o_stride[0] + hq * P.o_stride[1] + c * 8) = make_uint4(0, 0, 0, 0);
        }
        if (P.join_by_item) {
            for (int h = threadIdx.x; h < heads; h += kThreads) P.joins[s * heads + h] = make_int4(-1, 0, 0, 0);
        }
    }
    if (!P.join_by_item && threadIdx.x == 0) P.joins[cta] = make_int4(-1, 0, 0, 0);
    if (begin >= end) return;
    __syncthreads();

    Place<S::kChunk> load, work;
    load.enter(P, ctl->first_seq);
    {
        const int in = begin - ctl->first_before;
        load.h = in / load.n;
        load.ci = in - load.h * load.n;
    }
    work = load;

    // ------------------------------------------------ loads
    const uint32_t ring = smem_u32(smem) + warp * kSlots * kSlotBytes;
    const int lane_row = lane / S::kLanesRow, lane_col = lane % S::kLanesRow;
    const bool lane_in = lane_col * 8 < D;
    constexpr int kPlaces = kAligned ? 1 : S::kOwn;
    int left = end - begin;              // chunks the loads have still to enter
    int page_id[kPlaces];                // of this lane's rows of the next chunk to load
    long long row_at[kPlaces];           // of the chunk whose keys were asked for last: element offsets, -1: no such row
    int there = 0;                       // its keys in this warp's slot

    // the key whose place lane `lane` looks up: aligned, the first of a group of 16; else its own
    auto own_key = [&](int o) { return load.ci * S::kChunk + warp * S::kKeys + (kAligned ? (lane * 16) % S::kKeys : o * 32 + lane); };
    auto fetch_ids = [&]() {             // page ids of the chunk at `load`, asked for one chunk ahead of their use
#pragma unroll
        for (int o = 0; o < kPlaces; ++o) {
            const int key = own_key(o);
            page_id[o] = -1;
            if (left > 0 && key < load.len && (kAligned || o * 32 + lane < S::kKeys)) {
                page_id[o] = P.cache.table[load.s * P.cache.table_stride + key / P.cache.page_size];
            }
        }
    };
    auto enter_chunk = [&]() {           // places of the chunk at `load`; on to the next
        there = min(load.len - (load.ci * S::kChunk + warp * S::kKeys), S::kKeys);
#pragma unroll
        for (int o = 0; o < kPlaces; ++o) {
            const int key = own_key(o);
            row_at[o] = -1;
            if (key < load.len && (kAligned || o * 32 + lane < S::kKeys)) {
                if (static_cast<unsigned>(page_id[o]) < static_cast<unsigned>(P.cache.num_pages)) {
                    row_at[o] = page_id[o] * P.cache.page_stride + (key % P.cache.page_size) * P.cache.row_stride +
                                load.h / P.tiles * P.cache.head_stride;
                } else {
                    record_error(kErrPagedIndex);
                }
            }
        }
        --left;
        if (left > 0) load.next(P);
        fetch_ids();
    };
    auto copy_rows = [&](const uint16_t* base, uint32_t dst) {
        if constexpr (kAligned) {
            const long long lane_off = lane_row * P.cache.row_stride + lane_col * 8;
            const long long step = S::kRowsIter * P.cache.row_stride;
            const uint16_t* src = base;
            int rows = 0;
            if (there == S::kKeys && D == DP && __all_sync(0xffffffffu, row_at[0] >= 0)) {
#pragma unroll
                for (int i = 0; i < S::kCopies; ++i) {
                    if ((i * S::kRowsIter) % 16 == 0) src = base + __shfl_sync(0xffffffffu, row_at[0], i * S::kRowsIter / 16) + lane_off;
                    const int r = i * S::kRowsIter + lane_row;
                    cp_async16(dst + r * (DP * 2) + ((lane_col ^ (r & 7)) << 4), src);
                    src += step;
                }
                return;
            }
#pragma unroll 1
            for (int i = 0; i < S::kCopies; ++i) {
                if ((i * S::kRowsIter) % 16 == 0) {
                    const long long off = __shfl_sync(0xffffffffu, row_at[0], i * S::kRowsIter / 16);
                    rows = off >= 0 && lane_in ? there : 0;
                    src = base + (rows > 0 ? off + lane_off : 0);
                }
                const int r = i * S::kRowsIter + lane_row;
                cp_async16(dst + r * (DP * 2) + ((lane_col ^ (r & 7)) << 4), r < rows ? src : base, r < rows ? 16 : 0);
                src += step;
            }
        } else {
#pragma unroll 4
            for (int i = 0; i < S::kCopies; ++i) {
                const int r = i * S::kRowsIter + lane_row;
                long long off = __shfl_sync(0xffffffffu, row_at[0], r & 31);
                if (kPlaces > 1) {
                    const long long hi = __shfl_sync(0xffffffffu, row_at[kPlaces - 1], r & 31);
                    if (r >= 32) off = hi;
                }
                const bool in = off >= 0 && lane_in;
                cp_async16(dst + r * (DP * 2) + ((lane_col ^ (r & 7)) << 4), base + (in ? off + lane_col * 8 : 0), in ? 16 : 0);
            }
        }
    };

    // ------------------------------------------------ queries, as the B operand: rows past the end zero
    constexpr int kQueryVecs = (S::kRows * DP / 8 + kThreads - 1) / kThreads;
    uint4 q_next[kQueryVecs];
    auto ask_queries = [&](const Place<S::kChunk>& at) {
        const int kvh = at.h / P.tiles, row0 = (at.h - kvh * P.tiles) * S::kRows;
#pragma unroll
        for (int v = 0; v < kQueryVecs; ++v) {
            const int i = v * kThreads + threadIdx.x, r = i / (DP / 8), c = i - r * (DP / 8);
            q_next[v] = make_uint4(0, 0, 0, 0);
            if (r < S::kRows && row0 + r < P.group && c * 8 < D) {
                q_next[v] = *reinterpret_cast<const uint4*>(P.q + at.s * P.q_stride[0] + (kvh * P.group + row0 + r) * P.q_stride[1] + c * 8);
            }
        }
    };
    // byte offsets of a lane's row in a 16-row fragment, for the four positions of a 16-column step in 128 bytes: K (and V) as A
    // operand; the columns behind them are a constant further on
    uint32_t k_off[4], v_off[4];
    {
        const int kr = (lane & 7) + ((lane >> 3) & 1) * 8, kc = lane >> 4;          // matrices: keys 0-7, 8-15, then 8 columns on
        const int vr = (lane & 7) + (lane >> 4) * 8, vc = (lane >> 3) & 1;          // transposed: columns 0-7, 8-15, then 8 keys on
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            k_off[i] = kr * (DP * 2) + (((2 * i + kc) ^ (kr & 7)) << 4);
            v_off[i] = vr * (DP * 2) + (((2 * i + vc) ^ (vr & 7)) << 4);
        }
    }
    const uint32_t q_addr = smem_u32(sq) + (lane & 7) * (DP * 2);
    uint32_t qf[S::kQueriesStay ? DP / 16 : 1][NT][2];
    auto read_queries = [&](int kk, uint32_t (&f0)[NT][2], uint32_t (&f1)[NT][2]) {     // two 16-column steps
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            uint32_t r[4];
            ldsm4(r, q_addr + t * 8 * (DP * 2) + (((kk * 2 + (lane >> 3)) ^ (lane & 7)) << 4));
            f0[t][0] = r[0]; f0[t][1] = r[1];
            f1[t][0] = r[2]; f1[t][1] = r[3];
        }
    };
    float o[DP / 16][NT][4];             // O^T: columns of head_dim by query heads
    float m[NT][2], l[NT][2];            // reference and sum of the lane's two query heads of a tile; l over the lane's keys only
    auto start = [&]() {                 // an item's (or its piece's) beginning
#pragma unroll
        for (int i = 0; i < DP / 16; ++i)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[i][t][j] = 0.0f;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            m[t][0] = m[t][1] = -INFINITY;
            l[t][0] = l[t][1] = 0.0f;
        }
#pragma unroll
        for (int v = 0; v < kQueryVecs; ++v) {
            const int i = v * kThreads + threadIdx.x, r = i / (DP / 8), c = i - r * (DP / 8);
            if (r < S::kRows) *reinterpret_cast<uint4*>(sq + r * (DP * 2) + ((c ^ (r & 7)) << 4)) = q_next[v];
        }
        __syncthreads();
        if constexpr (S::kQueriesStay) {
#pragma unroll
            for (int kk = 0; kk < DP / 16; kk += 2) read_queries(kk, qf[kk], qf[kk + 1]);
        }
    };

    int parts = 0;                       // partial results this CTA has left
    int first_ci = work.ci;
    uint32_t p[S::kKeys / 16][NT][2];
    ask_queries(work);
    fetch_ids();
    // Uses of the ring: keys, values, keys, ... of consecutive chunks, use u in slot u % 3.  Round t works on use t - 3 and then asks
    // for use t in the same slot.
    const int uses = 2 * (end - begin);
    int slot = 0;
    for (int t = 0; t < uses + kSlots; ++t) {
        const uint32_t at = ring + slot * kSlotBytes;
        if (t >= kSlots) {
            cp_async_wait<kSlots - 1>();
            __syncwarp();
            const int valid = work.len - (work.ci * S::kChunk + warp * S::kKeys);     // keys of this warp's slot (may be none)
            if (((t - kSlots) & 1) == 0) {
                // ---- S^T = K Q^T: 16 keys x 8 query heads a tile
                float sc[S::kKeys / 16][NT][4];
#pragma unroll
                for (int b = 0; b < S::kKeys / 16; ++b) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int j = 0; j < 4; ++j) sc[b][n][j] = 0.0f;
                }
                if (valid > 0) {
#pragma unroll
                    for (int kk = 0; kk < DP / 16; kk += 2) {
                        uint32_t f[2][NT][2];
                        if constexpr (!S::kQueriesStay) read_queries(kk, f[0], f[1]);
#pragma unroll
                        for (int b = 0; b < S::kKeys / 16; ++b) {
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                uint32_t a[4];
                                ldsm4(a, at + k_off[(kk + h) & 3] + b * 16 * (DP * 2) + ((kk + h) >> 2) * 128);
#pragma unroll
                                for (int n = 0; n < NT; ++n) {
                                    if constexpr (S::kQueriesStay) mma16816<T>(sc[b][n], a, qf[kk + h][n][0], qf[kk + h][n][1]);
                                    else mma16816<T>(sc[b][n], a, f[h][n][0], f[h][n][1]);
                                }
                            }
                        }
                    }
                }
                // ---- a query head's scores lie in the lanes of equal lane % 4.  The reference is raised only when a score passes
                // it by 8 (weights stay below 2^8), so the maximum crosses the lanes hardly ever.
                float top[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) top[n][0] = top[n][1] = -INFINITY;
                if (valid < S::kKeys) {
#pragma unroll
                    for (int b = 0; b < S::kKeys / 16; ++b)
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                sc[b][n][j] = b * 16 + (lane >> 2) + (j >> 1) * 8 < valid ? sc[b][n][j] * P.scale2 : -INFINITY;
                            }
                } else {
#pragma unroll
                    for (int b = 0; b < S::kKeys / 16; ++b)
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int j = 0; j < 4; ++j) sc[b][n][j] *= P.scale2;
                }
                bool raise = false;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int b = 0; b < S::kKeys / 16; ++b) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) top[n][j & 1] = fmaxf(top[n][j & 1], sc[b][n][j]);
                    }
                    raise = raise || top[n][0] > m[n][0] + 8.0f || top[n][1] > m[n][1] + 8.0f;
                }
                if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
#pragma unroll
                            for (int x = 4; x < 32; x <<= 1) top[n][j] = fmaxf(top[n][j], __shfl_xor_sync(0xffffffffu, top[n][j], x));
                            const float now = fmaxf(m[n][j], top[n][j]);
                            const float shrink = now == m[n][j] ? 1.0f : ex2(m[n][j] - now);
#pragma unroll
                            for (int i = 0; i < DP / 16; ++i) {
                                o[i][n][j] *= shrink;
                                o[i][n][j + 2] *= shrink;
                            }
                            l[n][j] *= shrink;
                            m[n][j] = now;
                        }
                    }
                }
                // ---- weights, rounded to the values' type for the second product, transposed into its B operand
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float b0 = m[n][0] == -INFINITY ? 0.0f : m[n][0], b1 = m[n][1] == -INFINITY ? 0.0f : m[n][1];
#pragma unroll
                    for (int b = 0; b < S::kKeys / 16; ++b) {
                        float w[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) w[j] = ex2(sc[b][n][j] - (j & 1 ? b1 : b0));
                        l[n][0] += w[0] + w[2];
                        l[n][1] += w[1] + w[3];
                        p[b][n][0] = transpose8x8(Half16<T>::pack(w[0], w[1]));
                        p[b][n][1] = transpose8x8(Half16<T>::pack(w[2], w[3]));
                    }
                }
            } else if (valid > 0) {
                // ---- O^T += V^T P^T
#pragma unroll
                for (int i = 0; i < DP / 16; ++i) {
#pragma unroll
                    for (int b = 0; b < S::kKeys / 16; ++b) {
                        uint32_t a[4];
                        ldsm4_trans(a, at + v_off[i & 3] + b * 16 * (DP * 2) + (i >> 2) * 128);
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma16816<T>(o[i][n], a, p[b][n][0], p[b][n][1]);
                    }
                }
            }
            __syncwarp();
        }
        if (t < uses) {
            if ((t & 1) == 0) enter_chunk();
            copy_rows(static_cast<const uint16_t*>((t & 1) == 0 ? P.cache.k_pages : P.cache.v_pages), at);
        }
        cp_async_commit();
        slot = slot == kSlots - 1 ? 0 : slot + 1;
        if (t < kSlots) {
            if (t == kSlots - 1) start();                // the first loads are on their way
            continue;
        }
        if (((t - kSlots) & 1) == 0) continue;
        const bool item_done = work.ci + 1 == work.n, last = t == uses + kSlots - 1;
        if (!item_done && !last) {
            ++work.ci;
            continue;
        }
        // ------------------------------------------------ the four warps' sums -> the output, or a part of it
        Place<S::kChunk> then = work;
        if (!last) {
            then.next(P);
            ask_queries(then);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], x);
                if (lane < 4) *reinterpret_cast<float2*>(ctl->ml[warp][n * 8 + lane * 2 + j]) = make_float2(m[n][j], l[n][j]);
            }
        }
        __syncthreads();
        float f[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int row = n * 8 + (lane & 3) * 2 + j;
                float M = -INFINITY;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) M = fmaxf(M, ctl->ml[w][row][0]);
                f[n][j] = ex2(m[n][j] - (M == -INFINITY ? 0.0f : M));
            }
        }
        const bool whole = first_ci == 0 && item_done;
        const int kvh = work.h / P.tiles, row0 = (work.h - kvh * P.tiles) * S::kRows;
        constexpr int kQuads = S::kSlab / 4;
        const int orow = threadIdx.x / kQuads, ocol = (threadIdx.x % kQuads) * 4;
        const bool writes = orow < min(P.group - row0, S::kRows);
        float M = -INFINITY, L = 0.0f;
        if (writes) {
#pragma unroll
            for (int w = 0; w < kWarps; ++w) M = fmaxf(M, ctl->ml[w][orow][0]);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) L += ctl->ml[w][orow][1] * ex2(ctl->ml[w][orow][0] - (M == -INFINITY ? 0.0f : M));
        }
        const long long part = 2ll * cta + parts;
        if (!whole && writes && ocol == 0) *reinterpret_cast<float2*>(P.part_ml + (part * P.rows + orow) * 2) = make_float2(M, L);
        const float inv = 1.0f / L;
#pragma unroll
        for (int x = 0; x < DP / S::kSlab; ++x) {
#pragma unroll
            for (int i = 0; i < S::kSlab / 16; ++i) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        slab[(warp * S::kRows + n * 8 + (lane & 3) * 2 + (j & 1)) * S::kSlabPitch + i * 16 + (lane >> 2) + (j >> 1) * 8] =
                            o[x * (S::kSlab / 16) + i][n][j] * f[n][j & 1];
                    }
                }
            }
            __syncthreads();
            const int col = x * S::kSlab + ocol;
            if (writes && col < D) {
                float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float4 y = *reinterpret_cast<const float4*>(slab + (w * S::kRows + orow) * S::kSlabPitch + ocol);
                    sum.x += y.x; sum.y += y.y; sum.z += y.z; sum.w += y.w;
                }
                if (whole) {
                    uint16_t* to = P.out + work.s * P.o_stride[0] + (kvh * P.group + row0 + orow) * P.o_stride[1] + col;
                    *reinterpret_cast<uint2*>(to) = make_uint2(Half16<T>::pack(sum.x * inv, sum.y * inv), Half16<T>::pack(sum.z * inv, sum.w * inv));
                } else {
                    *reinterpret_cast<float4*>(P.part_o + (part * P.rows + orow) * D + col) = sum;
                }
            }
            __syncthreads();
        }
        if (threadIdx.x == 0 && first_ci == 0) {
            const int item = work.s * heads + work.h;
            if (whole) {
                if (P.join_by_item) P.joins[item] = make_int4(-1, 0, 0, 0);
            } else {
                // the item begins here and ends in a later CTA
                const int c = end - 1 + (work.n - 1 - work.ci);         // its last chunk in the line: this CTA's last is its chunk ci
                const int wide = more * (share + 1);
                const int last_cta = c < wide ? c / (share + 1) : more + (c - wide) / share;
                P.joins[P.join_by_item ? item : cta] = make_int4(item, last_cta - cta + 1, static_cast<int>(part), cta);
            }
        }
        if (!whole) ++parts;
        if (!last) {
            work = then;
            first_ci = 0;
            start();
        }
    }
    cp_async_wait<0>();
}

// One CTA per (item or CTA of the first kernel, row, 64 columns): where an item begins that ends in another CTA, its parts are joined.
// The first part is the last one the CTA left in which the item begins, the others are the first ones of the CTAs behind it.  A thread takes four
// columns of every eighth part, up to eight on their way at a time, with a running maximum of its own.
constexpr int kJoinQuads = 16, kJoinLanes = 8, kJoinThreads = kJoinQuads * kJoinLanes, kJoinLoads = 8;

template <typename T>
__global__ void __launch_bounds__(kJoinThreads) paged_attention_join_kernel(const __grid_constant__ DecodeParams P) {
    __shared__ float4 sums[kJoinLanes][kJoinQuads];
    __shared__ float2 mls[kJoinLanes];
    pdl_launch_dependents();
    pdl_wait_prior_grids();
    const int4 join = P.joins[blockIdx.x];
    if (join.x < 0) return;
    const int heads = P.cache.kv_heads * P.tiles, D = P.cache.head_dim;
    const int s = join.x / heads, h = join.x - s * heads;
    const int kvh = h / P.tiles, head = (h - kvh * P.tiles) * P.rows + blockIdx.y, parts = join.y;
    if (head >= P.group) return;
    const int lane = threadIdx.x / kJoinQuads, quad = threadIdx.x % kJoinQuads, col = blockIdx.z * 64 + quad * 4;
    float m = -INFINITY, l = 0.0f;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int i0 = lane; i0 < parts; i0 += kJoinLanes * kJoinLoads) {
        float2 ml[kJoinLoads];
        float4 x[kJoinLoads];
#pragma unroll
        for (int n = 0; n < kJoinLoads; ++n) {
            const int i = i0 + n * kJoinLanes;
            ml[n] = make_float2(-INFINITY, 0.0f);
            x[n] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (i < parts) {
                const long long at = (i == 0 ? join.z : 2ll * (join.w + i)) * P.rows + blockIdx.y;
                ml[n] = *reinterpret_cast<const float2*>(P.part_ml + at * 2);
                if (col < D) x[n] = *reinterpret_cast<const float4*>(P.part_o + at * D + col);
            }
        }
        float now = m;
#pragma unroll
        for (int n = 0; n < kJoinLoads; ++n) now = fmaxf(now, ml[n].x);
        const float base = now == -INFINITY ? 0.0f : now, shrink = ex2(m - base);
        l *= shrink;
        sum.x *= shrink; sum.y *= shrink; sum.z *= shrink; sum.w *= shrink;
#pragma unroll
        for (int n = 0; n < kJoinLoads; ++n) {
            const float w = ex2(ml[n].x - base);
            l += ml[n].y * w;
            sum.x += x[n].x * w; sum.y += x[n].y * w; sum.z += x[n].z * w; sum.w += x[n].w * w;
        }
        m = now;
    }
    sums[lane][quad] = sum;
    if (quad == 0) mls[lane] = make_float2(m, l);
    __syncthreads();
    if (lane == 0 && col < D) {
#pragma unroll
        for (int i = 1; i < kJoinLanes; ++i) m = fmaxf(m, mls[i].x);
        const float base = m == -INFINITY ? 0.0f : m;
        l = 0.0f;
        sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < kJoinLanes; ++i) {
            const float w = ex2(mls[i].x - base);
            const float4 x = sums[i][quad];
            l += mls[i].y * w;
            sum.x += x.x * w; sum.y += x.y * w; sum.z += x.z * w; sum.w += x.w * w;
        }
        const float inv = 1.0f / l;
        uint16_t* to = P.out + s * P.o_stride[0] + (kvh * P.group + head) * P.o_stride[1] + col;
        *reinterpret_cast<uint2*>(to) = make_uint2(Half16<T>::pack(sum.x * inv, sum.y * inv), Half16<T>::pack(sum.z * inv, sum.w * inv));
    }
}

int decode_ctas() {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    return sms * kCtasPerSm;
}

// places for joins: an item's where the items are fewer than the CTAs, else a CTA's
struct DecodeScratch { size_t part_ml, part_o, bytes; };

DecodeScratch decode_scratch(int ctas, int rows, int head_dim) {
    DecodeScratch d;
    d.part_ml = static_cast<size_t>(ctas) * sizeof(int4);
    d.part_o = d.part_ml + static_cast<size_t>(2) * ctas * rows * 2 * sizeof(float);
    d.part_o = (d.part_o + 255) / 256 * 256;
    d.bytes = d.part_o + static_cast<size_t>(2) * ctas * rows * head_dim * sizeof(float);
    return d;
}

// query heads that go through together: eight, or sixteen where a group has more
int decode_rows(int group) { return group <= 8 ? 8 : 16; }

template <typename T, int DP, int NT, bool kAligned>
int launch_decode(const DecodeParams& P, int ctas, int flags, cudaStream_t stream) {
    constexpr int smem = smem_bytes<DP, NT>();
    static_assert(kCtasPerSm * (smem + 1024) <= 228 * 1024, "two CTAs of an SM");
    static std::atomic<uint64_t> configured{0};
    int dev = 0;
    cudaGetDevice(&dev);
    const uint64_t bit = 1ull << (dev & 63);
    if (!(configured.load(std::memory_order_relaxed) & bit)) {
        if (cudaFuncSetAttribute(paged_attention_kernel<T, DP, NT, kAligned>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) {
            return TPB200_ERR_CUDA;
        }
        configured.fetch_or(bit, std::memory_order_relaxed);
    }
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = paged_config(static_cast<unsigned>(ctas), kThreads, smem, flags, &attr, stream);
    return cudaLaunchKernelEx(&cfg, paged_attention_kernel<T, DP, NT, kAligned>, P) == cudaSuccess ? TPB200_OK : TPB200_ERR_CUDA;
}

template <typename T, int DP>
int launch_decode(const DecodeParams& P, int ctas, int flags, cudaStream_t stream) {
    const bool aligned = P.cache.page_size % 16 == 0;
    if (P.group <= 8) return aligned ? launch_decode<T, DP, 1, true>(P, ctas, flags, stream) : launch_decode<T, DP, 1, false>(P, ctas, flags, stream);
    return aligned ? launch_decode<T, DP, 2, true>(P, ctas, flags, stream) : launch_decode<T, DP, 2, false>(P, ctas, flags, stream);
}

}  // namespace

int device_error_paged_attention(int clear) { return read_device_error(clear); }

}  // namespace tpb

extern "C" size_t tpb200_paged_attention_workspace_size(int q_heads, int kv_heads, int head_dim) {
    if (q_heads < 1 || kv_heads < 1 || q_heads % kv_heads != 0 || head_dim < 8 || head_dim > 256) return 0;
    const int ctas = tpb::decode_ctas();
    if (ctas < 1) return 0;
    const int group = q_heads / kv_heads;
    return tpb::decode_scratch(ctas, std::min(group, tpb::decode_rows(group)), head_dim).bytes;
}

extern "C" int tpb200_paged_attention(const tpb200_paged_attention_args* a, tpb200_stream_t stream) {
    using namespace tpb;
    TPB_REQUIRE(a != nullptr, TPB200_ERR_NULL);
    DecodeParams P = {};
    const int st = paged_view(a->cache, &P.cache);
    if (st != TPB200_OK) return st;
    TPB_REQUIRE(a->q && a->out, TPB200_ERR_NULL);
    TPB_REQUIRE((a->flags & ~TPB200_FLAG_PDL) == 0, TPB200_ERR_ENUM);
    TPB_REQUIRE(a->q_heads >= 1 && a->q_heads % P.cache.kv_heads == 0, TPB200_ERR_SHAPE);
    TPB_REQUIRE(tpb_aligned16(a->q) && tpb_aligned16(a->out), TPB200_ERR_ALIGN);
    for (int i = 0; i < 2; ++i) {
        TPB_REQUIRE(a->q_stride[i] % 8 == 0 && a->o_stride[i] % 8 == 0, TPB200_ERR_ALIGN);
        P.q_stride[i] = a->q_stride[i];
        P.o_stride[i] = a->o_stride[i];
    }
    if (P.cache.seqs == 0) return TPB200_OK;
    P.group = a->q_heads / P.cache.kv_heads;
    P.tiles = (P.group + decode_rows(P.group) - 1) / decode_rows(P.group);
    P.rows = std::min(P.group, decode_rows(P.group));
    // the line's length, at most one chunk of 64 keys per page slot, must fit an int
    const long long most = (static_cast<long long>(P.cache.page_size) * P.cache.table_width + 63) / 64;
    const long long items = static_cast<long long>(P.cache.kv_heads) * P.tiles * P.cache.seqs;
    TPB_REQUIRE(items <= 0x7fffffff && most * items <= 0x7fffffff, TPB200_ERR_SHAPE);
    const int ctas = decode_ctas();
    TPB_REQUIRE(ctas >= 2, TPB200_ERR_CUDA);
    const DecodeScratch d = decode_scratch(ctas, P.rows, P.cache.head_dim);
    TPB_REQUIRE(a->workspace != nullptr && a->workspace_bytes >= d.bytes, TPB200_ERR_WORKSPACE);
    TPB_REQUIRE(tpb_aligned16(a->workspace), TPB200_ERR_ALIGN);
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    P.joins = reinterpret_cast<int4*>(ws);
    P.part_ml = reinterpret_cast<float*>(ws + d.part_ml);
    P.part_o = reinterpret_cast<float*>(ws + d.part_o);
    P.join_by_item = items < ctas;
    P.q = static_cast<const uint16_t*>(a->q);
    P.out = static_cast<uint16_t*>(a->out);
    P.scale2 = a->scale * 1.4426950408889634f;
    const bool bf = a->cache.dtype == TPB200_BF16;
    const int D = P.cache.head_dim;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const int done = D <= 64 ? (bf ? launch_decode<__nv_bfloat16, 64>(P, ctas, a->flags, s) : launch_decode<__half, 64>(P, ctas, a->flags, s))
                   : D <= 128 ? (bf ? launch_decode<__nv_bfloat16, 128>(P, ctas, a->flags, s) : launch_decode<__half, 128>(P, ctas, a->flags, s))
                              : (bf ? launch_decode<__nv_bfloat16, 256>(P, ctas, a->flags, s) : launch_decode<__half, 256>(P, ctas, a->flags, s));
    if (done != TPB200_OK) return done;
    // always dependent: its launch hides behind the first kernel, which it waits for
    cudaLaunchAttribute attr;
    cudaLaunchConfig_t cfg = paged_config(P.join_by_item ? static_cast<unsigned>(items) : ctas - 1, kJoinThreads, 0, TPB200_FLAG_PDL, &attr, s);
    cfg.gridDim.y = static_cast<unsigned>(P.rows);
    cfg.gridDim.z = static_cast<unsigned>((D + 63) / 64);
    const auto join = bf ? paged_attention_join_kernel<__nv_bfloat16> : paged_attention_join_kernel<__half>;
    return cudaLaunchKernelEx(&cfg, join, P) == cudaSuccess ? TPB200_OK : TPB200_ERR_CUDA;
}
