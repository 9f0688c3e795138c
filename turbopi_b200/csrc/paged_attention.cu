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
//   * The g query heads that share a key head are the rows of one 16-row tile of mma.sync, so each byte of the cache
//     crosses the SM once.  The tile is at most half full for g <= 8, and needs no more: an SM's share of the stream is 16 KB per 700
//     cycles, in which four warps' worth of this work takes about a quarter of the issue slots.  tcgen05 wants 128 rows.
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
constexpr int kRowsTile = 16;            // query heads of a tile
constexpr int kSlab = 32;                // columns that pass through shared memory at a time when the warps' sums are joined
constexpr int kCtasPerSm = 2;

struct DecodeParams {
    PagedView cache;
    const uint16_t* q;
    uint16_t* out;
    long long q_stride[2], o_stride[2];
    int group;                           // query heads per key head
    int tiles;                           // 16-row tiles per key head
    int rows;                            // rows of a tile that are used at most
    float scale2;                        // scale * log2 e
    float* part_o;                       // [2 * CTAs][rows][head_dim]
    float* part_ml;                      // [2 * CTAs][rows][2]
    int4* joins;                         // per CTA: (item or -1, parts, first slot, 0)
};

template <int DP>
struct Shape {
    static constexpr int kKeys = kSlotBytes / (DP * 2);     // keys of a slot: 16, 32, 64
    static constexpr int kChunk = kKeys * kWarps;           // keys of a chunk: a slot for each warp
    static constexpr int kLanesRow = DP / 8;                // lanes that copy a row
    static constexpr int kRowsIter = 32 / kLanesRow;        // rows a warp copies at a time
    static constexpr int kOwn = (kKeys + 31) / 32;          // rows a lane knows the place of
};

struct Control {
    int warp_sum[kWarps];
    int first_seq, first_before;         // the sequence of the CTA's first chunk, and the chunks before it
    int total;
    float ml[kWarps][kRowsTile][2];
};

template <int DP>
constexpr int smem_bytes() {
    return kWarps * kSlots * kSlotBytes + kRowsTile * DP * 2 + kWarps * kRowsTile * kSlab * 4 + static_cast<int>(sizeof(Control));
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
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

// A place in the line of chunks: chunk `ci` of item (sequence, key head tile)
template <int DP>
struct Place {
    int s, h, ci, n, len;                // n: chunks of the sequence's items
    __device__ __forceinline__ void enter(const DecodeParams& P, int seq) {
        for (s = seq; s < P.cache.seqs; ++s) {
            len = keys_of(P.cache, s);
            if (len > 0) break;
        }
        n = (len + Shape<DP>::kChunk - 1) / Shape<DP>::kChunk;
        h = ci = 0;
    }
    __device__ __forceinline__ void next(const DecodeParams& P) {
        if (++ci < n) return;
        ci = 0;
        if (++h < P.cache.kv_heads * P.tiles) return;
        enter(P, s + 1);
    }
};

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) paged_attention_kernel(const __grid_constant__ DecodeParams P) {
    using S = Shape<DP>;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* sq = smem + kWarps * kSlots * kSlotBytes;                                  // queries of the item
    float* slab = reinterpret_cast<float*>(sq + kRowsTile * DP * 2);
    Control* ctl = reinterpret_cast<Control*>(slab + kWarps * kRowsTile * kSlab);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int heads = P.cache.kv_heads * P.tiles;
    const int D = P.cache.head_dim;
    pdl_launch_dependents();
    pdl_wait_prior_grids();

    // ------------------------------------------------ this CTA's piece of the line
    // Chunks before each thread's run of sequences, then the sequence that holds the first chunk.
    if (threadIdx.x == 0) ctl->first_seq = P.cache.seqs;
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
    }
    __syncthreads();
    if (threadIdx.x == 0) P.joins[cta] = make_int4(-1, 0, 0, 0);
    if (begin >= end) return;

    Place<DP> load, work;
    load.enter(P, ctl->first_seq);
    {
        const int in = begin - ctl->first_before;
        load.h = in / load.n;
        load.ci = in - load.h * load.n;
    }
    work = load;

    // ------------------------------------------------ the ring
    const uint32_t ring = smem_u32(smem) + warp * kSlots * kSlotBytes;
    const int lane_row = lane / S::kLanesRow, lane_col = lane % S::kLanesRow;
    int left = end - begin;              // chunks the loads have still to enter
    int page_id[S::kOwn];                // of this lane's rows of the next chunk to load
    long long row_at[S::kOwn];           // of the chunk whose keys were asked for last: element offsets, -1: no such row

    auto fetch_ids = [&]() {             // page ids of the chunk at `load`, asked for one chunk ahead of their use
#pragma unroll
        for (int o = 0; o < S::kOwn; ++o) {
            const int r = o * 32 + lane, key = load.ci * S::kChunk + warp * S::kKeys + r;
            page_id[o] = -1;
            if (left > 0 && r < S::kKeys && key < load.len) page_id[o] = P.cache.table[load.s * P.cache.table_stride + key / P.cache.page_size];
        }
    };
    auto copy_rows = [&](const uint16_t* base, uint32_t dst) {
#pragma unroll
        for (int i = 0; i < S::kKeys / S::kRowsIter; ++i) {
            const int r = i * S::kRowsIter + lane_row;
            const long long off = __shfl_sync(0xffffffffu, row_at[(i * S::kRowsIter) / 32], r & 31);
            const bool there = off >= 0 && lane_col * 8 < D;
            cp_async16(dst + r * (DP * 2) + ((lane_col ^ (r & 7)) << 4), base + (there ? off + lane_col * 8 : 0), there ? 16 : 0);
        }
    };
    auto load_keys = [&](int slot) {
        if (left > 0) {
#pragma unroll
            for (int o = 0; o < S::kOwn; ++o) {
                const int r = o * 32 + lane, key = load.ci * S::kChunk + warp * S::kKeys + r;
                row_at[o] = -1;
                if (r < S::kKeys && key < load.len) {
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
            copy_rows(static_cast<const uint16_t*>(P.cache.k_pages), ring + slot * kSlotBytes);
        }
        cp_async_commit();
    };
    int values_left = end - begin;
    auto load_values = [&](int slot) {
        if (values_left > 0) {
            --values_left;
            copy_rows(static_cast<const uint16_t*>(P.cache.v_pages), ring + slot * kSlotBytes);
        }
        cp_async_commit();
    };

    fetch_ids();
    load_keys(0);
    load_values(1);
    load_keys(2);                        // uses: keys, values, keys, ... of consecutive chunks, use u in slot u % 3
    int slot = 0;

    float o[DP / 8][4];
    float m[2], l[2];
    auto start = [&]() {                 // an item's (or its piece's) beginning
#pragma unroll
        for (int i = 0; i < DP / 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.0f;
        // queries -> shared memory, rows and columns past the end zero
        const int kvh = work.h / P.tiles, row0 = (work.h - kvh * P.tiles) * kRowsTile;
        for (int i = threadIdx.x; i < kRowsTile * (DP / 8); i += kThreads) {
            const int r = i / (DP / 8), c = i - r * (DP / 8);
            uint4 x = make_uint4(0, 0, 0, 0);
            if (row0 + r < P.group && c * 8 < D) {
                x = *reinterpret_cast<const uint4*>(P.q + work.s * P.q_stride[0] + (kvh * P.group + row0 + r) * P.q_stride[1] + c * 8);
            }
            *reinterpret_cast<uint4*>(sq + r * (DP * 2) + ((c ^ (r & 7)) << 4)) = x;
        }
        __syncthreads();
    };

    const uint32_t q_addr = smem_u32(sq);
    int parts = 0;                       // partial results this CTA has left
    int first_ci = work.ci;
    start();
    for (int c = begin; c < end; ++c) {
        const int key0 = work.ci * S::kChunk + warp * S::kKeys;
        const int valid = work.len - key0;               // keys of this warp's slot that exist (may be none)
        // ---- S = Q K^T: 16 rows x the slot's keys
        cp_async_wait<2>();
        __syncwarp();
        uint32_t p[S::kKeys / 16][4];
        if (valid > 0) {
            float sc[S::kKeys / 8][4];
#pragma unroll
            for (int i = 0; i < S::kKeys / 8; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) sc[i][j] = 0.0f;
            const uint32_t k_addr = ring + slot * kSlotBytes;
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk) {
                uint32_t a[4];
                const int qr = lane & 15, qc = kk * 2 + (lane >> 4);
                ldsm4(a, q_addr + qr * (DP * 2) + ((qc ^ (qr & 7)) << 4));
#pragma unroll
                for (int n = 0; n < S::kKeys / 16; ++n) {
                    uint32_t b[4];
                    const int kr = n * 16 + (lane & 7) + ((lane >> 4) << 3), kc = kk * 2 + ((lane >> 3) & 1);
                    ldsm4(b, k_addr + kr * (DP * 2) + ((kc ^ (kr & 7)) << 4));
                    mma16816<T>(sc[2 * n], a, b[0], b[1]);
                    mma16816<T>(sc[2 * n + 1], a, b[2], b[3]);
                }
            }
            // ---- running maximum and sum; a row is spread over the four lanes of a quad
            float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < S::kKeys / 8; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int key = i * 8 + (lane & 3) * 2 + (j & 1);
                    sc[i][j] = key < valid ? sc[i][j] * P.scale2 : -INFINITY;
                    top[j >> 1] = fmaxf(top[j >> 1], sc[i][j]);
                }
            }
            float base[2], shrink[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
                top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
                top[r] = fmaxf(top[r], m[r]);
                base[r] = top[r] == -INFINITY ? 0.0f : top[r];
                shrink[r] = ex2(m[r] - base[r]);
            }
            if (__any_sync(0xffffffffu, top[0] != m[0] || top[1] != m[1])) {
#pragma unroll
                for (int i = 0; i < DP / 8; ++i) {
                    o[i][0] *= shrink[0];
                    o[i][1] *= shrink[0];
                    o[i][2] *= shrink[1];
                    o[i][3] *= shrink[1];
                }
                l[0] *= shrink[0];
                l[1] *= shrink[1];
                m[0] = top[0];
                m[1] = top[1];
            }
            // weights rounded to the values' type for the second product; the sum is that of the rounded ones
#pragma unroll
            for (int i = 0; i < S::kKeys / 8; ++i) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const uint32_t w = Half16<T>::pack(ex2(sc[i][2 * r] - base[r]), ex2(sc[i][2 * r + 1] - base[r]));
                    const float2 f = Half16<T>::unpack(w);
                    l[r] += f.x + f.y;
                    p[i >> 1][(i & 1) * 2 + r] = w;
                }
            }
        }
        __syncwarp();
        load_values(slot);               // the slot of this chunk's keys takes the next chunk's values
        slot = slot == kSlots - 1 ? 0 : slot + 1;
        // ---- O += P V
        cp_async_wait<2>();
        __syncwarp();
        if (valid > 0) {
            const uint32_t v_addr = ring + slot * kSlotBytes;
#pragma unroll
            for (int kk = 0; kk < S::kKeys / 16; ++kk) {
#pragma unroll
                for (int n = 0; n < DP / 16; ++n) {
                    uint32_t b[4];
                    const int vr = kk * 16 + (lane & 15), vc = n * 2 + (lane >> 4);
                    ldsm4_trans(b, v_addr + vr * (DP * 2) + ((vc ^ (vr & 7)) << 4));
                    mma16816<T>(o[2 * n], p[kk], b[0], b[1]);
                    mma16816<T>(o[2 * n + 1], p[kk], b[2], b[3]);
                }
            }
        }
        __syncwarp();
        load_keys(slot);
        slot = slot == kSlots - 1 ? 0 : slot + 1;

        const bool item_done = work.ci + 1 == work.n;
        if (!item_done && c + 1 < end) {
            ++work.ci;
            continue;
        }
        // ------------------------------------------------ the four warps' sums -> the output, or a part of it
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            if ((lane & 3) == 0) {
                ctl->ml[warp][(lane >> 2) + 8 * r][0] = m[r];
                ctl->ml[warp][(lane >> 2) + 8 * r][1] = l[r];
            }
        }
        __syncthreads();
        float f[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = (lane >> 2) + 8 * r;
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) M = fmaxf(M, ctl->ml[w][row][0]);
            f[r] = ex2(m[r] - (M == -INFINITY ? 0.0f : M));
        }
        const bool whole = first_ci == 0 && item_done;
        const int kvh = work.h / P.tiles, row0 = (work.h - kvh * P.tiles) * kRowsTile;
        const int used = min(P.group - row0, kRowsTile);
        const int orow = threadIdx.x >> 3, ocol = (threadIdx.x & 7) * 4;
        float M = -INFINITY, L = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, ctl->ml[w][orow][0]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) L += ctl->ml[w][orow][1] * ex2(ctl->ml[w][orow][0] - (M == -INFINITY ? 0.0f : M));
        const long long part = 2ll * cta + parts;
        if (!whole && ocol == 0 && orow < used) {
            P.part_ml[(part * P.rows + orow) * 2] = M;
            P.part_ml[(part * P.rows + orow) * 2 + 1] = L;
        }
#pragma unroll
        for (int x = 0; x < DP / kSlab; ++x) {
#pragma unroll
            for (int n = 0; n < kSlab / 8; ++n) {
                const int i = x * (kSlab / 8) + n, col = n * 8 + (lane & 3) * 2;
                float* to = slab + (warp * kRowsTile + (lane >> 2)) * kSlab + col;
                *reinterpret_cast<float2*>(to) = make_float2(o[i][0] * f[0], o[i][1] * f[0]);
                *reinterpret_cast<float2*>(to + 8 * kSlab) = make_float2(o[i][2] * f[1], o[i][3] * f[1]);
            }
            __syncthreads();
            const int col = x * kSlab + ocol;
            if (orow < used && col < D) {
                float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float4 y = *reinterpret_cast<const float4*>(slab + (w * kRowsTile + orow) * kSlab + ocol);
                    sum.x += y.x; sum.y += y.y; sum.z += y.z; sum.w += y.w;
                }
                if (whole) {
                    uint16_t* to = P.out + work.s * P.o_stride[0] + (kvh * P.group + row0 + orow) * P.o_stride[1] + col;
                    *reinterpret_cast<uint2*>(to) = make_uint2(Half16<T>::pack(sum.x / L, sum.y / L), Half16<T>::pack(sum.z / L, sum.w / L));
                } else {
                    *reinterpret_cast<float4*>(P.part_o + (part * P.rows + orow) * D + col) = sum;
                }
            }
            __syncthreads();
        }
        if (!whole) {
            ++parts;
            if (first_ci == 0 && threadIdx.x == 0) {
                // the item begins here and ends in a later CTA: the chunk behind this CTA's last is in the next one, and so on
                const int last = c + (work.n - 1 - work.ci);            // the item's last chunk in the line
                const int wide = more * (share + 1);
                const int last_cta = last < wide ? last / (share + 1) : more + (last - wide) / share;
                P.joins[cta] = make_int4(work.s * heads + work.h, last_cta - cta + 1, static_cast<int>(part), 0);
            }
        }
        if (c + 1 < end) {
            work.next(P);
            first_ci = 0;
            start();
        }
    }
    cp_async_wait<0>();
}

// One CTA per (CTA of the first kernel, row): if an item begins there and ends elsewhere, its parts are joined.  Its first part
// is the last one that CTA left, the others are the first ones of the CTAs behind it.
constexpr int kJoinThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kJoinThreads) paged_attention_join_kernel(const __grid_constant__ DecodeParams P) {
    __shared__ float4 sums[kJoinThreads];
    __shared__ float weights[kJoinThreads / 2];
    pdl_launch_dependents();
    pdl_wait_prior_grids();
    const int4 join = P.joins[blockIdx.x];
    if (join.x < 0) return;
    const int heads = P.cache.kv_heads * P.tiles, D = P.cache.head_dim;
    const int s = join.x / heads, h = join.x - s * heads;
    const int kvh = h / P.tiles, row0 = (h - kvh * P.tiles) * kRowsTile, row = blockIdx.y;
    if (row0 + row >= P.group) return;
    const int parts = join.y;
    auto slot = [&](int i) { return i == 0 ? static_cast<long long>(join.z) : 2ll * (blockIdx.x + i); };
    float M = -INFINITY;
    for (int i = threadIdx.x; i < parts; i += kJoinThreads) M = fmaxf(M, P.part_ml[(slot(i) * P.rows + row) * 2]);
    M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, 16));
    M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, 8));
    M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, 4));
    M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, 2));
    M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, 1));
    if ((threadIdx.x & 31) == 0) weights[threadIdx.x >> 5] = M;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kJoinThreads / 32; ++w) M = fmaxf(M, weights[w]);
    if (M == -INFINITY) M = 0.0f;
    // a thread: four columns of every `lanes`-th part
    const int cols = D / 4, lanes = kJoinThreads / cols, lane = threadIdx.x / cols, col = (threadIdx.x - lane * cols) * 4;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float L = 0.0f;
    if (lane < lanes) {
#pragma unroll 8
        for (int i = lane; i < parts; i += lanes) {
            const long long at = slot(i) * P.rows + row;
            const float2 ml = *reinterpret_cast<const float2*>(P.part_ml + at * 2);
            const float4 x = *reinterpret_cast<const float4*>(P.part_o + at * D + col);
            const float w = ex2(ml.x - M);
            L += ml.y * w;
            sum.x += x.x * w; sum.y += x.y * w; sum.z += x.z * w; sum.w += x.w * w;
        }
        sums[threadIdx.x] = sum;
        if (col == 0) weights[lane] = L;
    }
    __syncthreads();
    if (threadIdx.x < cols) {
        L = 0.0f;
        sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int i = 0; i < lanes; ++i) {
            const float4 x = sums[i * cols + threadIdx.x];
            sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
            L += weights[i];
        }
        uint16_t* to = P.out + s * P.o_stride[0] + (kvh * P.group + row0 + row) * P.o_stride[1] + threadIdx.x * 4;
        *reinterpret_cast<uint2*>(to) = make_uint2(Half16<T>::pack(sum.x / L, sum.y / L), Half16<T>::pack(sum.z / L, sum.w / L));
    }
}

int decode_ctas() {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    return sms * kCtasPerSm;
}

struct DecodeScratch { size_t joins, part_ml, part_o, bytes; };

DecodeScratch decode_scratch(int ctas, int rows, int head_dim) {
    DecodeScratch d;
    d.joins = 0;
    d.part_ml = static_cast<size_t>(ctas) * sizeof(int4);
    d.part_o = d.part_ml + static_cast<size_t>(2) * ctas * rows * 2 * sizeof(float);
    d.part_o = (d.part_o + 255) / 256 * 256;
    d.bytes = d.part_o + static_cast<size_t>(2) * ctas * rows * head_dim * sizeof(float);
    return d;
}

template <typename T, int DP>
int launch_decode(const DecodeParams& P, int ctas, int flags, cudaStream_t stream) {
    constexpr int smem = smem_bytes<DP>();
    static_assert(kCtasPerSm * (smem + 1024) <= 228 * 1024, "two CTAs of an SM");
    static std::atomic<uint64_t> configured{0};
    int dev = 0;
    cudaGetDevice(&dev);
    const uint64_t bit = 1ull << (dev & 63);
    if (!(configured.load(std::memory_order_relaxed) & bit)) {
        if (cudaFuncSetAttribute(paged_attention_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) {
            return TPB200_ERR_CUDA;
        }
        configured.fetch_or(bit, std::memory_order_relaxed);
    }
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = paged_config(static_cast<unsigned>(ctas), kThreads, smem, flags, &attr, stream);
    return cudaLaunchKernelEx(&cfg, paged_attention_kernel<T, DP>, P) == cudaSuccess ? TPB200_OK : TPB200_ERR_CUDA;
}

}  // namespace

int device_error_paged_attention(int clear) { return read_device_error(clear); }

}  // namespace tpb

extern "C" size_t tpb200_paged_attention_workspace_size(int q_heads, int kv_heads, int head_dim) {
    if (q_heads < 1 || kv_heads < 1 || q_heads % kv_heads != 0 || head_dim < 8 || head_dim > 256) return 0;
    const int ctas = tpb::decode_ctas();
    if (ctas < 1) return 0;
    return tpb::decode_scratch(ctas, std::min(q_heads / kv_heads, tpb::kRowsTile), head_dim).bytes;
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
    P.tiles = (P.group + kRowsTile - 1) / kRowsTile;
    P.rows = std::min(P.group, kRowsTile);
    // the line's length, at most one chunk of 64 keys per page slot, must fit an int
    const long long most = (static_cast<long long>(P.cache.page_size) * P.cache.table_width + 63) / 64;
    TPB_REQUIRE(most * P.cache.kv_heads * P.tiles * P.cache.seqs <= 0x7fffffff, TPB200_ERR_SHAPE);
    const int ctas = decode_ctas();
    TPB_REQUIRE(ctas >= 1, TPB200_ERR_CUDA);
    const DecodeScratch d = decode_scratch(ctas, P.rows, P.cache.head_dim);
    TPB_REQUIRE(a->workspace != nullptr && a->workspace_bytes >= d.bytes, TPB200_ERR_WORKSPACE);
    TPB_REQUIRE(tpb_aligned16(a->workspace), TPB200_ERR_ALIGN);
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    P.joins = reinterpret_cast<int4*>(ws + d.joins);
    P.part_ml = reinterpret_cast<float*>(ws + d.part_ml);
    P.part_o = reinterpret_cast<float*>(ws + d.part_o);
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
    cudaLaunchConfig_t cfg = paged_config(static_cast<unsigned>(ctas - 1), kJoinThreads, 0, TPB200_FLAG_PDL, &attr, s);
    cfg.gridDim.y = static_cast<unsigned>(P.rows);
    if (ctas == 1) return TPB200_OK;
    const auto join = bf ? paged_attention_join_kernel<__nv_bfloat16> : paged_attention_join_kernel<__half>;
    return cudaLaunchKernelEx(&cfg, join, P) == cudaSuccess ? TPB200_OK : TPB200_ERR_CUDA;
}
