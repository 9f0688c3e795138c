// The bodies of the kernels of single-token attention on a cache of pages, for 16-bit rows (Rows16) and for tiles of 4-bit values (Nvfp4), over all keys or
// over the last ones and a few first ones (kWindow): softmax(scale q K^T) V.  The files that
// launch them say what bounds them; their kernels wait for the launch before them ahead of these bodies.
#pragma once

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "paged.cuh"

namespace tpb {
namespace {

constexpr int kCtaWarps = 4;
constexpr int kSlotUnits = 2;            // what a slot costs; an item besides, for queries, sums and the output: Src::kItemUnits
constexpr float kLowest = -FLT_MAX;      // the least reference of a row with a key

// What only the host or some calls read stands last: a small call of one that reads all from the front takes 0.05-0.1 us less
struct DecodeParams {
    PagedView cache;
    const uint16_t* q;
    uint16_t* out;
    long long q_stride[2], o_stride[2];
    int group;                           // query heads per key head
    int tiles;                           // tiles of query heads per key head
    int rows;                            // rows of a tile that are used at most
    int join_by_item;                    // joins[] has a place per item, else one per worker
    float scale2;                        // scale * log2 e, times the factor of the keys' scales
    float* part_o;                       // [2 * workers][rows][head_dim]
    float* part_ml;                      // [2 * workers][rows][2]
    int4* joins;                         // (item or -1, its first part, its last worker, 1: first CTA merged | 2: last CTA merged)
    long long items;                     // (sequence, tile of query heads)
    int workers;                         // warps of the grid
    float out_scale;                     // factor of the values' scales (Nvfp4)
    int window, sinks;                   // keys that are seen: the last `window` and the first `sinks` (kWindow)
};

// What a cache holds.  Rows16: rows of head_dim 16-bit values, strides in elements.  Nvfp4: tiles of 16 tokens of one head, strides in bytes
// (row_stride: from tile to tile).  A tile, with G = ceil(head_dim / 32): 16 rows of 16 G bytes of E2M1 codes, two to a byte, the even value in
// the low half, then 16 rows of 2 G E4M3 scales, one for 16 values.
struct Rows16 {
    static constexpr bool kQuant = false;
    static constexpr int kItemUnits = 1;
};
struct Nvfp4 {
    static constexpr bool kQuant = true;
    // With 2, 4, 5, 6, 7: 96 ragged sequences 47.7, 40.0, 39.4, 36.8, 36.4 us (heads of 128), windows of 64 sequences 38.9, 38.3, 39.0, 39.4, 39.0 (of 64),
    // five long ones 35.4, 34.6, 34.6, 34.6, 34.6 (of 256): medians, the first two of which move by 1 us from run to run
    static constexpr int kItemUnits = 6;
};

// DP: head_dim rounded up to 64, 128 or 256.  NT: tiles of eight query heads that go through together.
template <typename Src, int DP, int NT>
struct Shape {
    static constexpr int kKeys = !Src::kQuant || DP < 256 ? 4096 / DP : 32;                     // of a slot: 16 or 32, 32, 64
    static constexpr int kSlotBytes = Src::kQuant ? 2 * kKeys * (DP / 2 + DP / 16) : kKeys * DP * 2;     // tiles of keys and of values; rows of keys, or of values
    static constexpr int kSlots = 3;                        // of a warp's ring
    static constexpr int kCtas = Src::kQuant && DP < 256 ? 3 : 2;       // on an SM
    static constexpr int kWarps = kCtaWarps, kThreads = kWarps * 32;
    static constexpr int kLengths = 1024;                   // lengths kept in shared memory; with more sequences they are read where they lie
    static constexpr int kLanesRow = Src::kQuant ? DP / 32 : DP / 8;        // lanes that copy a row
    static constexpr int kRowsIter = 32 / kLanesRow;        // rows a warp copies at a time
    static constexpr int kCopies = kKeys / kRowsIter;
    static constexpr int kOwn = (kKeys + 31) / 32;          // rows a lane knows the place of
    static constexpr int kRows = 8 * NT;
    static constexpr int kChains = 1;    // 16-key blocks whose scores are summed in two chains of products, a latency each
    static constexpr bool kQueriesStay = NT * DP <= 256;    // in registers; else they are read again for every slot
    static constexpr bool kQueriesAhead = !Src::kQuant && kQueriesStay && NT * DP * NT <= 256;      // the next item's too, where registers are left
    static constexpr int kSlab = NT == 1 || Src::kQuant ? 64 : 16;          // columns of a warp's sums that pass through shared memory at a time
    static_assert(!Src::kQuant || kQueriesStay, "");
    static constexpr int kSlabPitch = kSlab + 4;            // the four query pairs of a store fall into different banks
    static constexpr int kSumPitch = DP + 4;
    static_assert(kRows * kSumPitch * 4 <= kSlots * kSlotBytes, "a warp's sums where its ring was");
    // Where a lane's sum j of tile i stands: in a row of the output, and in slab x's piece of it.  The tiles of Nvfp4 take two neighbouring columns from
    // each of the lanes' eight runs.
    static __device__ __forceinline__ int column(int i, int lane, int j) {
        return Src::kQuant ? (lane >> 2) * (DP / 8) + 2 * i + (j >> 1) : i * 16 + (lane >> 2) + (j >> 1) * 8;
    }
    static __device__ __forceinline__ int slab_column(int i, int lane, int j) {
        return Src::kQuant ? (lane >> 2) * (kSlab / 8) + 2 * i + (j >> 1) : i * 16 + (lane >> 2) + (j >> 1) * 8;
    }
    static __device__ __forceinline__ int column_of_slab(int x, int c) {
        return Src::kQuant ? c / (kSlab / 8) * (DP / 8) + x * (kSlab / 8) + c % (kSlab / 8) : x * kSlab + c;
    }
};

template <typename S>
struct Control {
    int lengths[S::kLengths];
    float ml[S::kWarps][S::kRows][2];
};

// 4-bit tiles: sums pass through the slot whose tiles were used last
template <typename Src, int DP, int NT>
constexpr int smem_bytes() {
    using S = Shape<Src, DP, NT>;
    static_assert(!Src::kQuant || S::kRows * S::kSlabPitch * 4 <= S::kSlotBytes, "");
    return S::kWarps * S::kSlots * S::kSlotBytes + (Src::kQuant ? 0 : S::kWarps * S::kRows * S::kSlabPitch * 4) + static_cast<int>(sizeof(Control<S>));
}

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

// 1 over the sum of the weights; a row without any key (its reference never left -infinity) gives zeros
__device__ __forceinline__ float inverse(float reference, float sum) { return reference == -INFINITY ? 0.0f : 1.0f / sum; }

// keys of a sequence that the cache can hold: a length beyond the table's pages is an error, not an address
__device__ __forceinline__ int keys_of(const PagedView& c, int s) {
    const int n = c.lengths[s], most = c.page_size * c.table_width;
    if (n > most) record_error(kErrPagedIndex);
    return max(0, min(n, most));
}

// Lengths go up to 2^31 - 1: a length rounded up to whole slots, and the place of a key behind the last one in its slot, are unsigned
template <int kKeys>
__device__ __forceinline__ int slots_of(int len) { return static_cast<int>((static_cast<unsigned>(len) + kKeys - 1) / kKeys); }

// The slots of a sequence that hold keys which are seen: the first `n` of its slots, or those of the sinks and, `skip` further on, those of the
// window (a slot in between holds no such key; each of the others does)
struct Extent { int n, skip; };
template <int kKeys, bool kWindow>
__device__ __forceinline__ Extent extent_of(const DecodeParams& P, int len) {
    const int n = slots_of<kKeys>(len);
    if (!kWindow) return {n, 0};
    const int skip = max(0, max(0, len - P.window) / kKeys - slots_of<kKeys>(P.sinks));
    return {n - skip, skip};
}

// A place in the line of slots: slot `ci` of item (sequence, tile of query heads)
template <typename Src, int kKeys, int kLengths, bool kWindow>
struct Place {
    int s, h, ci, n, len;                // n: slots of the sequence's items
    int skip;                            // slots of the sequence that are left out behind those of the sinks
    int units;                           // of the line before the item
    int step;                            // slots from one of the warp's to its next
    __device__ __forceinline__ void enter(const DecodeParams& P, const int* lengths, int seq) {
        for (s = seq; s < P.cache.seqs; ++s) {
            len = P.cache.seqs <= kLengths ? lengths[s] : keys_of(P.cache, s);
            if (len > 0) break;
        }
        set_extent(P);
        h = ci = 0;
    }
    __device__ __forceinline__ void set_extent(const DecodeParams& P) {
        const Extent e = extent_of<kKeys, kWindow>(P, len);
        n = e.n;
        skip = e.skip;
    }
    __device__ __forceinline__ int first_key(const DecodeParams& P) const {          // of the slot
        return (kWindow && ci >= slots_of<kKeys>(P.sinks) ? ci + skip : ci) * kKeys;
    }
    __device__ __forceinline__ void next(const DecodeParams& P, const int* lengths) {
        ci += step;
        if (ci < n) return;
        units += n * kSlotUnits + Src::kItemUnits;
        ci = 0;
        if (++h < P.cache.kv_heads * P.tiles) return;
        enter(P, lengths, s + 1);
    }
};

// The line cut into pieces of equal cost, over the CTAs and a CTA's over its warps, the first ones of each getting a unit more.  A
// slot belongs to the piece in which its first unit lies, behind the item's own; pieces are two units at least, so a warp between the
// first and the last of an item always has a slot of it.  A line shorter than that for four warps is one warp's.
template <int kItemUnits, int kWarps>
struct Share {
    // a CTA has at least as many units; one inside an item has a slot of it, since the item's own units are fewer
    static_assert(kItemUnits < kWarps * kSlotUnits, "a CTA inside an item leaves a part");
    int total, ctas, each, more;         // `more` CTAs of each + 1 units, the others of each
    __device__ __forceinline__ void cut(int units, int grid) {
        total = units;
        ctas = min(grid, max(1, units / (kWarps * kSlotUnits)));
        each = total / ctas;
        more = total - each * ctas;
    }
    __device__ __forceinline__ bool solo() const { return total < kWarps * kSlotUnits; }
    __device__ __forceinline__ int cta_begin(int c) const { return c * each + min(c, more); }
    __device__ __forceinline__ int begin(int c, int w) const {       // of warp w of CTA c, or the CTA's end
        const int b = cta_begin(c);
        if (w == 0) return b;
        if (solo()) return total;
        const unsigned n = cta_begin(c + 1) - b;
        return b + w * (n / kWarps) + min(w, n % kWarps);
    }
    __device__ __forceinline__ int worker_of(int unit) const {
        if (solo()) return 0;
        const int wide = more * (each + 1);
        const int c = unit < wide ? unit / (each + 1) : more + (unit - wide) / each;
        const unsigned n = cta_begin(c + 1) - cta_begin(c), at = unit - cta_begin(c), wq = n / kWarps, wr = n % kWarps;
        return c * kWarps + (at < wr * (wq + 1) ? at / (wq + 1) : wr + (at - wr * (wq + 1)) / wq);
    }
    // the worker of the last slot of an item of n slots, and whether its CTA lies inside the item and adds its warps' sums up itself
    __device__ __forceinline__ int last_worker(int item, int n) const { return worker_of(item + kItemUnits + (n - 1) * kSlotUnits); }
    __device__ __forceinline__ bool ends_merged(int item, int n, int last) const {
        return cta_begin(last / kWarps) >= item && cta_begin(last / kWarps + 1) <= item + kItemUnits + n * kSlotUnits;
    }
};

// A warp's piece of the line: where it begins, and its slots
template <typename Src, typename S, bool kWindow>
struct Piece {
    Place<Src, S::kKeys, S::kLengths, kWindow> work;
    Share<Src::kItemUnits, S::kWarps> line;
    static constexpr int kWarps = S::kWarps;
    int slots;
    bool merged, whole_item;             // the CTA lies inside one item; it is the whole of it

    // false: the CTA has none.  Sequences without keys get their zeros here.
    __device__ __forceinline__ bool find(const DecodeParams& P, int* lengths, int warp, int lane) {
        const int heads = P.cache.kv_heads * P.tiles, D = P.cache.head_dim;
        // Every warp for itself, without a barrier: slots and units before each lane's run of sequences, then the places where its piece
        // begins and ends.
        const bool staged = P.cache.seqs <= S::kLengths;     // all warps write the same lengths there, each reads its own
        const int run = (P.cache.seqs + 31) / 32, s0 = min(P.cache.seqs, lane * run), s1 = min(P.cache.seqs, s0 + run);
        int slots_here = 0, units_here = 0;
        bool empty = false;
        for (int s = s0; s < s1; ++s) {
            const int len = keys_of(P.cache, s), n = extent_of<S::kKeys, kWindow>(P, len).n;
            if (staged) lengths[s] = len;
            slots_here += n * heads;
            units_here += n > 0 ? (n * kSlotUnits + Src::kItemUnits) * heads : 0;
            empty = empty || n == 0;
        }
        __syncwarp();
        auto length = [&](int s) { return staged ? lengths[s] : keys_of(P.cache, s); };
        int slots_to = slots_here, units_to = units_here;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, slots_to, o), y = __shfl_up_sync(0xffffffffu, units_to, o);
            if (lane >= o) {
                slots_to += x;
                units_to += y;
            }
        }
        line.cut(__shfl_sync(0xffffffffu, units_to, 31), static_cast<int>(gridDim.x));
        const int cta = blockIdx.x, worker = cta * kWarps + warp;
        // sequences without keys: zeros
        if (__any_sync(0xffffffffu, empty)) {
            for (int s = worker; s < P.cache.seqs; s += gridDim.x * kWarps) {
                if (length(s) > 0) continue;
                const int per_head = D / 8;
                for (int i = lane; i < P.cache.kv_heads * P.group * per_head; i += 32) {
                    const int hq = i / per_head, c = i - hq * per_head;
                    *reinterpret_cast<uint4*>(P.out + s * P.o_stride[0] + hq * P.o_stride[1] + c * 8) = make_uint4(0, 0, 0, 0);
                }
                if (P.join_by_item) {
                    for (int h = lane; h < heads; h += 32) P.joins[s * heads + h] = make_int4(-1, 0, 0, 0);
                }
            }
        }
        if (!P.join_by_item && lane == 0) P.joins[worker] = make_int4(-1, 0, 0, 0);
        if (line.total == 0 || cta >= line.ctas) return false;

        // The place of the first slot that begins at `unit` or behind it, and the slots of the line before it.  A lane whose run holds the unit
        // finds the sequence, all lanes the rest.
        int item_first = 0;                  // units of the line before the item that holds the unit, and behind it
        int item_behind = 0;
        auto find = [&](int unit) {
            const bool here = unit >= units_to - units_here && unit < units_to;
            int s = s0, slots = slots_to - slots_here, units = units_to - units_here;
            if (here) {
                for (;; ++s) {
                    const int n = extent_of<S::kKeys, kWindow>(P, length(s)).n, more = n > 0 ? (n * kSlotUnits + Src::kItemUnits) * heads : 0;
                    if (unit < units + more) break;
                    slots += n * heads;
                    units += more;
                }
            }
            const int from = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
            s = __shfl_sync(0xffffffffu, s, from);
            slots = __shfl_sync(0xffffffffu, slots, from);
            units = __shfl_sync(0xffffffffu, units, from);
            work.s = s;
            work.len = length(s);
            work.set_extent(P);
            const int item = work.n * kSlotUnits + Src::kItemUnits;
            work.h = (unit - units) / item;
            work.units = item_first = units + work.h * item;
            item_behind = item_first + item;
            const int in = unit - item_first;
            work.ci = in <= Src::kItemUnits ? 0 : (in - Src::kItemUnits + kSlotUnits - 1) / kSlotUnits;
            const int before = slots + work.h * work.n + work.ci;
            if (work.ci == work.n) {         // behind the item's last slot
                work.ci = work.n - 1;
                work.step = 1;
                work.next(P, lengths);
            }
            return before;
        };
        const int cta_first = line.cta_begin(cta), cta_behind = line.cta_begin(cta + 1);
        const int unit_first = line.begin(cta, warp), unit_behind = line.begin(cta, warp + 1);
        slots = 0;
        merged = whole_item = false;
        if (unit_first < unit_behind) {
            if (unit_behind < line.total) slots = find(unit_behind);
            else slots = __shfl_sync(0xffffffffu, slots_to, 31);
            slots -= find(unit_first);
            work.step = 1;
            // A CTA inside one item adds its warps' sums up itself, and deals its slots to them in turn: neighbours are read together.
            merged = cta_first >= item_first && cta_behind <= item_behind;
        } else {                             // one warp's line
            find(cta_first);
            merged = cta_behind <= item_behind;
        }
        if (merged) {
            auto slot_of = [&](int unit) {
                const int in = unit - item_first;
                return in <= Src::kItemUnits ? 0 : min(work.n, (in - Src::kItemUnits + kSlotUnits - 1) / kSlotUnits);
            };
            const int first = slot_of(cta_first), behind = slot_of(cta_behind);
            whole_item = first == 0 && behind == work.n;
            slots = max(0, (behind - first - warp + kWarps - 1) / kWarps);
            work.ci = first + warp;
            work.step = kWarps;
        }
        return true;
    }
};

// A warp's sums of an item, or of its piece of one, to the output or to a part; through shared memory (`own`), so that rows leave in runs.
// Returns whether they were the whole item's.
template <typename Src, typename T, typename S, int DP, int NT, typename Work, typename Line>
__device__ __forceinline__ bool store_item(const DecodeParams& P, const Work& work, const Line& line, float* own, int cta, int worker, int lane, int parts,
                                           bool from_start, bool item_done, const float (&o)[DP / 16][NT][4], const float (&m)[NT][2], float (&l)[NT][2]) {
    const int heads = P.cache.kv_heads * P.tiles, D = P.cache.head_dim;
    const bool whole = from_start && item_done;
    const int kvh = work.h / P.tiles, row0 = (work.h - kvh * P.tiles) * S::kRows;
    const long long part = 2ll * worker + parts;
    float f[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], x);
            f[n][j] = whole ? inverse(m[n][j], l[n][j]) : 1.0f;
            if (Src::kQuant && whole) f[n][j] *= P.out_scale;
            const int row = n * 8 + (lane & 3) * 2 + j;
            if (!whole && lane < 4 && row < P.rows) {
                *reinterpret_cast<float2*>(P.part_ml + (part * P.rows + row) * 2) = make_float2(m[n][j], l[n][j]);
            }
        }
    }
    constexpr int kQuads = S::kSlab / 4;
#pragma unroll
    for (int x = 0; x < DP / S::kSlab; ++x) {
#pragma unroll
        for (int i = 0; i < S::kSlab / 16; ++i) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    own[(n * 8 + (lane & 3) * 2 + (j & 1)) * S::kSlabPitch + S::slab_column(i, lane, j)] =
                        o[x * (S::kSlab / 16) + i][n][j] * f[n][j & 1];
                }
            }
        }
        __syncwarp();
        for (int u = lane; u < min(P.group - row0, S::kRows) * kQuads; u += 32) {
            const int row = u / kQuads, col = S::column_of_slab(x, u % kQuads * 4);
            if (col >= D) continue;
            const float4 y = *reinterpret_cast<const float4*>(own + row * S::kSlabPitch + u % kQuads * 4);
            if (whole) {
                uint16_t* to = P.out + work.s * P.o_stride[0] + (kvh * P.group + row0 + row) * P.o_stride[1] + col;
                *reinterpret_cast<uint2*>(to) = make_uint2(Half16<T>::pack(y.x, y.y), Half16<T>::pack(y.z, y.w));
            } else {
                *reinterpret_cast<float4*>(P.part_o + (part * P.rows + row) * D + col) = y;
            }
        }
        __syncwarp();
    }
    if (lane == 0 && from_start) {
        const int item = work.s * heads + work.h;
        if (whole) {
            if (P.join_by_item) P.joins[item] = make_int4(-1, 0, 0, 0);
        } else {                     // it begins here and ends with a later warp
            const int by = line.last_worker(work.units, work.n);
            P.joins[P.join_by_item ? item : worker] =
                make_int4(item, static_cast<int>(part), by, by / S::kWarps != cta && line.ends_merged(work.units, work.n, by) ? 2 : 0);
        }
    }
    return whole;
}

// The sums of a CTA inside one item, each warp's where its ring was
template <typename Src, typename T, typename S, int DP, int NT, typename Work, typename Line>
__device__ __forceinline__ void merge_cta(const DecodeParams& P, const Work& work, const Line& line, uint8_t* smem, float (&ml)[S::kWarps][S::kRows][2], int cta,
                                          int warp, int lane, bool from_start, bool whole, const float (&o)[DP / 16][NT][4], const float (&m)[NT][2], float (&l)[NT][2]) {
    constexpr int kSlotBytes = S::kSlotBytes, kSlots = S::kSlots, kWarps = S::kWarps;
    const int heads = P.cache.kv_heads * P.tiles, D = P.cache.head_dim, worker = cta * kWarps;
    float* sums = reinterpret_cast<float*>(smem + warp * kSlots * kSlotBytes);
    __syncwarp();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], x);
            if (lane < 4) *reinterpret_cast<float2*>(ml[warp][n * 8 + lane * 2 + j]) = make_float2(m[n][j], l[n][j]);
        }
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                sums[(n * 8 + (lane & 3) * 2 + (j & 1)) * S::kSumPitch + S::column(i, lane, j)] = o[i][n][j];
            }
        }
    }
    __syncthreads();
    const int kvh = work.h / P.tiles, row0 = (work.h - kvh * P.tiles) * S::kRows;
    const long long part = 2ll * kWarps * cta;
    const int rows = min(P.group - row0, S::kRows);
#pragma unroll 4
    for (int u = threadIdx.x; u < S::kRows * (DP / 4); u += S::kThreads) {
        const int row = u / (DP / 4), col = u % (DP / 4) * 4;
        if (row >= rows || col >= D) continue;
        float M = -INFINITY, L = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, ml[w][row][0]);
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = ex2(ml[w][row][0] - (M == -INFINITY ? 0.0f : M));
            const float4 y = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem + w * kSlots * kSlotBytes) + row * S::kSumPitch + col);
            L += ml[w][row][1] * f;
            sum.x += y.x * f; sum.y += y.y * f; sum.z += y.z * f; sum.w += y.w * f;
        }
        if (whole) {
            const float inv = Src::kQuant ? inverse(M, L) * P.out_scale : inverse(M, L);
            uint16_t* to = P.out + work.s * P.o_stride[0] + (kvh * P.group + row0 + row) * P.o_stride[1] + col;
            *reinterpret_cast<uint2*>(to) = make_uint2(Half16<T>::pack(sum.x * inv, sum.y * inv), Half16<T>::pack(sum.z * inv, sum.w * inv));
        } else {
            *reinterpret_cast<float4*>(P.part_o + (part * P.rows + row) * D + col) = sum;
            if (col == 0) *reinterpret_cast<float2*>(P.part_ml + (part * P.rows + row) * 2) = make_float2(M, L);
        }
    }
    if (threadIdx.x == 0 && from_start) {
        const int item = work.s * heads + work.h;
        if (whole) {
            if (P.join_by_item) P.joins[item] = make_int4(-1, 0, 0, 0);
        } else {
            const int by = line.last_worker(work.units, work.n);
            P.joins[P.join_by_item ? item : worker] = make_int4(item, static_cast<int>(part), by, line.ends_merged(work.units, work.n, by) ? 3 : 1);
        }
    }
}

// kAligned: the page size is a multiple of 16, so that 16 rows from a multiple of 16 on lie in one page and share an address.  The warp and D are what its
// kernel has found out ahead of its wait for the launch before.
template <typename T, int DP, int NT, bool kAligned, bool kWindow>
__device__ __forceinline__ void attend_rows(const DecodeParams& P, int warp, int D) {
    using Src = Rows16;
    using S = Shape<Src, DP, NT>;
    constexpr int kSlotBytes = S::kSlotBytes, kSlots = S::kSlots, kWarps = S::kWarps;
    extern __shared__ __align__(128) uint8_t smem[];
    float* slab = reinterpret_cast<float*>(smem + kWarps * kSlots * kSlotBytes);
    auto* ctl = reinterpret_cast<Control<S>*>(slab + kWarps * S::kRows * S::kSlabPitch);
    const int lane = threadIdx.x & 31;

    Piece<Src, S, kWindow> piece;
    if (!piece.find(P, ctl->lengths, warp, lane)) return;
    auto& work = piece.work;
    const auto& line = piece.line;
    const int slots = piece.slots, cta = blockIdx.x, worker = cta * kWarps + warp;
    const bool merged = piece.merged, whole_item = piece.whole_item;
    auto load = work;

    // ------------------------------------------------ loads
    const uint32_t ring = smem_u32(smem) + warp * kSlots * kSlotBytes;
    const int lane_row = lane / S::kLanesRow, lane_col = lane % S::kLanesRow;
    const bool lane_in = lane_col * 8 < D;
    constexpr int kPlaces = kAligned ? 1 : S::kOwn;
    int left = slots;                    // that the loads have still to enter
    int page_id[kPlaces];                // of this lane's rows of the next slot to load
    long long row_at[kPlaces];           // of the slot whose keys were asked for last: element offsets, -1: no such row
    int there = 0;                       // its keys
    int hide_from = 0, hide_to = 0;      // of these, [hide_from, hide_to) are not seen (kWindow)
    // Keys whose page is not in the pool, a bit per group of 16 (aligned) or per key: of the slot whose keys were asked for last, and of the
    // one before it, which is the one that is worked on.
    constexpr int kKeysPerBit = kAligned ? 16 : 1;
    using Absent = std::conditional_t<(S::kKeys / kKeysPerBit > 32), uint64_t, uint32_t>;
    Absent absent_next = 0, absent = 0;

    // the key whose place lane `lane` looks up: aligned, the first of a group of 16; else its own
    auto own_key = [&](int o) { return static_cast<unsigned>(load.first_key(P)) + (kAligned ? (lane * 16) % S::kKeys : o * 32 + lane); };
    // whether that key, or one of its group, is seen
    auto own_seen = [&](int o, unsigned key) {
        if (key >= static_cast<unsigned>(load.len) || !(kAligned || o * 32 + lane < S::kKeys)) return false;
        if (!kWindow) return true;
        return key < static_cast<unsigned>(P.sinks) || static_cast<int>(min(key + (kAligned ? 16u : 1u), static_cast<unsigned>(load.len))) > load.len - P.window;
    };
    auto fetch_ids = [&]() {             // page ids of the slot at `load`, asked for one slot ahead of their use
#pragma unroll
        for (int o = 0; o < kPlaces; ++o) {
            const unsigned key = own_key(o);
            page_id[o] = -1;
            if (left > 0 && own_seen(o, key)) {
                page_id[o] = P.cache.table[load.s * P.cache.table_stride + key / P.cache.page_size];
            }
        }
    };
    auto enter_slot = [&]() {            // places of the slot at `load`; on to the next
        there = min(load.len - load.first_key(P), S::kKeys);
        if (kWindow) {
            hide_from = P.sinks - load.first_key(P);
            hide_to = load.len - P.window - load.first_key(P);
        }
#pragma unroll
        for (int o = 0; o < kPlaces; ++o) {
            const unsigned key = own_key(o);
            row_at[o] = -1;
            const bool in = own_seen(o, key);
            const bool known = static_cast<unsigned>(page_id[o]) < static_cast<unsigned>(P.cache.num_pages);
            if (in && known) {
                row_at[o] = page_id[o] * P.cache.page_stride + (key % P.cache.page_size) * P.cache.row_stride +
                            load.h / P.tiles * P.cache.head_stride;
            }
            const uint32_t gone = __ballot_sync(0xffffffffu, in && !known);
            if (gone != 0) {
                record_error(kErrPagedIndex);
                absent_next |= kAligned ? gone & ((1u << (S::kKeys / 16)) - 1) : static_cast<Absent>(gone) << (o * 32);
            }
        }
        --left;
        if (left > 0) load.next(P, ctl->lengths);
        fetch_ids();
    };
    auto copy_rows = [&](const uint16_t* base, uint32_t dst) {
        if constexpr (kAligned) {
            const long long lane_off = lane_row * P.cache.row_stride + lane_col * 8;
            const long long step = S::kRowsIter * P.cache.row_stride;
            const uint16_t* src = base;
            int rows = 0;
#pragma unroll
            for (int i = 0; i < S::kCopies; ++i) {
                if ((i * S::kRowsIter) % 16 == 0) {
                    const long long off = __shfl_sync(0xffffffffu, row_at[0], i * S::kRowsIter / 16);
                    rows = off >= 0 && lane_in ? there : 0;
                    src = rows > 0 ? base + off + lane_off : base;
                }
                const int r = i * S::kRowsIter + lane_row;
                const bool in = r < rows && !(kWindow && r >= hide_from && r < hide_to);
                cp_async16(dst + r * (DP * 2) + ((lane_col ^ (r & 7)) << 4), src, in ? 16 : 0);
                if (r < rows) src += step;
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
    // queries as the B operand: a lane's two pairs of a 16-column step, zero past the group and past head_dim
    uint32_t qf[S::kQueriesStay ? DP / 16 : 1][NT][2], q_ahead[S::kQueriesAhead ? DP / 16 : 1][NT][2];
    const uint16_t* q_row[NT];           // null: no such query head
    auto aim_queries = [&](const decltype(piece.work)& at) {
        const int kvh = at.h / P.tiles, row0 = (at.h - kvh * P.tiles) * S::kRows;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int r = row0 + t * 8 + (lane >> 2);
            q_row[t] = r < P.group ? P.q + at.s * P.q_stride[0] + (kvh * P.group + r) * P.q_stride[1] + (lane & 3) * 2 : nullptr;
        }
    };
    auto read_queries = [&](int kk, uint32_t (&f)[NT][2]) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int c = kk * 16 + j * 8;
                f[t][j] = q_row[t] != nullptr && c < D ? __ldg(reinterpret_cast<const uint32_t*>(q_row[t] + c)) : 0u;
            }
        }
    };
    float o[DP / 16][NT][4];             // O^T: columns of head_dim by query heads
    float m[NT][2], l[NT][2];            // reference and sum of the lane's two query heads of a tile; l over the lane's keys only
    auto clear = [&]() {
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
    };
    auto start = [&]() {                 // an item's (or its piece's) beginning
        clear();
        if constexpr (S::kQueriesAhead) {
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    qf[kk][n][0] = q_ahead[kk][n][0];
                    qf[kk][n][1] = q_ahead[kk][n][1];
                }
            }
        } else {
            aim_queries(work);
            if constexpr (S::kQueriesStay) {
#pragma unroll
                for (int kk = 0; kk < DP / 16; ++kk) read_queries(kk, qf[kk]);
            }
        }
    };
    auto ask_queries = [&](const decltype(piece.work)& at) {
        if constexpr (S::kQueriesAhead) {
            aim_queries(at);
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk) read_queries(kk, q_ahead[kk]);
        }
    };

    auto ask_next = [&]() {              // the queries of the item behind `work`
        if constexpr (S::kQueriesAhead) {
            auto then = work;
            then.ci = then.n - 1;
            then.next(P, ctl->lengths);
            ask_queries(then);
        }
    };
    int parts = 0;                       // partial results this warp has left
    int first_ci = work.ci;
    uint32_t p[S::kKeys / 16][NT][2];
    // Uses of the ring: keys, values, keys, ... of consecutive slots of the line, use u in slot u % 3.  Round t works on use t - 3 and then asks
    // for use t in the same slot.
    const int uses = 2 * slots;
    int slot = 0;
    if (slots == 0) clear();
    else fetch_ids(), ask_queries(work);
    for (int t = 0; t < (uses > 0 ? uses + kSlots : 0); ++t) {
        const uint32_t at = ring + slot * kSlotBytes;
        if (t >= kSlots) {
            cp_async_wait<kSlots - 1>();
            __syncwarp();
            const int key0 = work.first_key(P), valid = work.len - key0;               // keys of the slot, at least one
            const int hidden = P.sinks - key0, shown = valid - P.window;               // [hidden, shown) are not seen (kWindow)
            const bool some_hidden = kWindow && shown > 0 && hidden < S::kKeys && hidden < shown;
            if (((t - kSlots) & 1) == 0) {
                // ---- S^T = K Q^T: 16 keys x 8 query heads a tile
                float sc[S::kKeys / 16][NT][4], odd[S::kChains][NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
#pragma unroll
                        for (int b = 0; b < S::kKeys / 16; ++b) sc[b][n][j] = 0.0f;
#pragma unroll
                        for (int b = 0; b < S::kChains; ++b) odd[b][n][j] = 0.0f;
                    }
                }
#pragma unroll
                for (int kk = 0; kk < DP / 16; ++kk) {
                    uint32_t f[NT][2];
                    if constexpr (!S::kQueriesStay) read_queries(kk, f);
#pragma unroll
                    for (int b = 0; b < S::kKeys / 16; ++b) {
                        uint32_t a[4];
                        ldsm4(a, at + k_off[kk & 3] + b * 16 * (DP * 2) + (kk >> 2) * 128);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            float(&sum)[4] = kk % 2 == 1 && b < S::kChains ? odd[b % S::kChains][n] : sc[b][n];
                            if constexpr (S::kQueriesStay) mma16816<T>(sum, a, qf[kk][n][0], qf[kk][n][1]);
                            else mma16816<T>(sum, a, f[n][0], f[n][1]);
                        }
                    }
                }
#pragma unroll
                for (int b = 0; b < S::kKeys / 16 && b < S::kChains; ++b)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int j = 0; j < 4; ++j) sc[b][n][j] += odd[b][n][j];
                // ---- a query head's scores lie in the lanes of equal lane % 4.  The reference is raised only when a score passes
                // it by 8 (weights stay below 2^8), so the maximum crosses the lanes hardly ever.
                // A slot with a key has a finite reference, whatever the score: one of -infinity at the end means that there was no key.
                bool some = absent == 0 || __popcll(absent) < (min(valid, S::kKeys) + kKeysPerBit - 1) / kKeysPerBit;
                if (kWindow && absent != 0) {            // whether one that is seen is there
                    bool mine = false;
                    for (int key = lane; key < min(valid, S::kKeys); key += 32) {
                        mine = mine || (!(key >= hidden && key < shown) && ((absent >> (kAligned ? key / 16 : key)) & 1) == 0);
                    }
                    some = __any_sync(0xffffffffu, mine);
                }
                float top[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) top[n][0] = top[n][1] = some ? kLowest : -INFINITY;
                if (valid < S::kKeys || absent != 0 || some_hidden) {
#pragma unroll
                    for (int b = 0; b < S::kKeys / 16; ++b)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int key = b * 16 + (lane >> 2) + (j >> 1) * 8;
                            const bool seen = key < valid && ((absent >> (kAligned ? b : key)) & 1) == 0 && !(kWindow && key >= hidden && key < shown);
#pragma unroll
                            for (int n = 0; n < NT; ++n) sc[b][n][j] = seen ? sc[b][n][j] * P.scale2 : -INFINITY;
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
                // ---- weights, rounded to the values' type for the second product (their sum is that of the unrounded ones), transposed into
                // its B operand
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float b0 = (m[n][0] == -INFINITY ? 0.0f : m[n][0]) - Half16<T>::kLift, b1 = (m[n][1] == -INFINITY ? 0.0f : m[n][1]) - Half16<T>::kLift;
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
            } else {
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
        if ((t & 1) == 0) {
            absent = absent_next;
            absent_next = 0;
        }
        if (t < uses) {
            if ((t & 1) == 0) enter_slot();
            copy_rows(static_cast<const uint16_t*>((t & 1) == 0 ? P.cache.k_pages : P.cache.v_pages), at);
        }
        cp_async_commit();
        slot = slot == kSlots - 1 ? 0 : slot + 1;
        if (t < kSlots) {
            if (t == kSlots - 1) {                       // the first loads are on their way
                start();
                if (!merged && uses > 2 * (work.n - work.ci)) ask_next();
            }
            continue;
        }
        if (((t - kSlots) & 1) == 0) continue;
        const bool item_done = work.ci + work.step >= work.n, last = t == uses + kSlots - 1;
        if (merged || (!item_done && !last)) {
            work.ci += work.step;
            continue;
        }
        float* own = slab + warp * S::kRows * S::kSlabPitch;
        if (!store_item<Src, T, S, DP, NT>(P, work, line, own, cta, worker, lane, parts, first_ci == 0, item_done, o, m, l)) ++parts;
        if (!last) {
            work.next(P, ctl->lengths);
            first_ci = 0;
            start();
            if ((uses + kSlots - 1 - t) / 2 > work.n) ask_next();
        }
    }
    cp_async_wait<0>();
    if (!merged) return;
    merge_cta<Src, T, S, DP, NT>(P, work, line, smem, ctl->ml, cta, warp, lane, first_ci == 0, whole_item, o, m, l);
}

// Where an item begins that ends with another worker, its parts are joined.  Workers are warps; a CTA that lies inside the item has
// left one part, as its first worker, the item's other workers one each: the one it begins with its last part, those behind it their
// first.  blockIdx.x: the item, or the worker it begins with; a thread has four columns of a row (blockIdx.y: which ones) of every
// kLanes-th part, kLoads of them on their way at a time, with a running maximum of its own.
constexpr int kJoinThreads = 128;

template <typename Src, typename T, int kLanes, int kLoads>
__device__ __forceinline__ void join_parts(const DecodeParams& P) {
    constexpr int kWarps = kCtaWarps;
    constexpr int kQuads = kJoinThreads / kLanes;
    __shared__ float4 sums[kLanes][kQuads];
    __shared__ float2 mls[kLanes][kQuads];
    const int4 join = P.joins[blockIdx.x];
    if (join.x < 0) return;
    const int heads = P.cache.kv_heads * P.tiles, D = P.cache.head_dim;
    const int first_worker = join.y >> 1, first_cta = first_worker / kWarps, last_cta = join.z / kWarps;
    // parts of the first CTA, of the ones between (one each), of the last
    const int n_first = join.w & 1 ? 1 : min(join.z, first_cta * kWarps + kWarps - 1) - first_worker + 1;
    const int n_last = last_cta == first_cta ? 0 : (join.w & 2 ? 1 : join.z - last_cta * kWarps + 1);
    const int parts = n_first + max(0, last_cta - first_cta - 1) + n_last;
    auto part = [&](int i) {
        if (i == 0) return join.y;
        if (i < n_first) return 2 * (first_worker + i);
        const int c = first_cta + 1 + i - n_first;
        return c <= last_cta ? 2 * kWarps * c : 2 * (kWarps * last_cta + c - last_cta);
    };
    const int lane = threadIdx.x / kQuads, quad = threadIdx.x % kQuads, at = (blockIdx.y * kQuads + quad) * 4, row = at / D, col = at - row * D;
    const bool there = row < P.rows;
    float m = -INFINITY, l = 0.0f;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int i0 = lane; i0 < parts; i0 += kLanes * kLoads) {
        float2 ml[kLoads];
        float4 x[kLoads];
#pragma unroll
        for (int n = 0; n < kLoads; ++n) {
            const int i = i0 + n * kLanes;
            ml[n] = make_float2(-INFINITY, 0.0f);
            x[n] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (i < parts && there) {
                const size_t from = static_cast<size_t>(part(i)) * P.rows + row;
                ml[n] = *reinterpret_cast<const float2*>(P.part_ml + from * 2);
                x[n] = *reinterpret_cast<const float4*>(P.part_o + from * D + col);
            }
        }
        float now = m;
#pragma unroll
        for (int n = 0; n < kLoads; ++n) now = fmaxf(now, ml[n].x);
        const float base = now == -INFINITY ? 0.0f : now, shrink = ex2(m - base);
        l *= shrink;
        sum.x *= shrink; sum.y *= shrink; sum.z *= shrink; sum.w *= shrink;
#pragma unroll
        for (int n = 0; n < kLoads; ++n) {
            const float w = ex2(ml[n].x - base);
            l += ml[n].y * w;
            sum.x += x[n].x * w; sum.y += x[n].y * w; sum.z += x[n].z * w; sum.w += x[n].w * w;
        }
        m = now;
    }
    sums[lane][quad] = sum;
    mls[lane][quad] = make_float2(m, l);
    __syncthreads();
    const int s = join.x / heads, h = join.x - s * heads, kvh = h / P.tiles, head = (h - kvh * P.tiles) * P.rows + row;
    if (lane == 0 && there && head < P.group) {
#pragma unroll
        for (int i = 1; i < kLanes; ++i) m = fmaxf(m, mls[i][quad].x);
        const float base = m == -INFINITY ? 0.0f : m;
        l = 0.0f;
        sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < kLanes; ++i) {
            const float2 ml = mls[i][quad];
            const float w = ex2(ml.x - base);
            const float4 x = sums[i][quad];
            l += ml.y * w;
            sum.x += x.x * w; sum.y += x.y * w; sum.z += x.z * w; sum.w += x.w * w;
        }
        const float inv = Src::kQuant ? inverse(m, l) * P.out_scale : inverse(m, l);
        uint16_t* to = P.out + s * P.o_stride[0] + (kvh * P.group + head) * P.o_stride[1] + col;
        *reinterpret_cast<uint2*>(to) = make_uint2(Half16<T>::pack(sum.x * inv, sum.y * inv), Half16<T>::pack(sum.z * inv, sum.w * inv));
    }
}

int decode_ctas(int per_sm) {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    return sms * per_sm;
}

// places for joins: an item's where the items are fewer than the workers, else a worker's
struct DecodeScratch { size_t part_ml, part_o, bytes; };

DecodeScratch decode_scratch(size_t workers, int rows, int head_dim) {
    DecodeScratch d;
    d.part_ml = workers * sizeof(int4);
    d.part_o = d.part_ml + 2 * workers * rows * 2 * sizeof(float);
    d.part_o = (d.part_o + 255) / 256 * 256;
    d.bytes = d.part_o + 2 * workers * rows * head_dim * sizeof(float);
    return d;
}


// ------------------------------------------------------------------------------------------------ launches
using Kernel = void (*)(DecodeParams);

// Once per device: dynamic shared memory, and the whole of an SM's for shared memory (all_shared).  An SM that runs the joins of a call with a
// smaller share keeps it until it is idle, and takes fewer of the next call's CTAs; one that came to run a fourth then began 20 us late.
template <Kernel kernel>
bool configure(int smem, bool all_shared) {
    static std::atomic<uint64_t> configured{0};
    int dev = 0;
    cudaGetDevice(&dev);
    const uint64_t bit = 1ull << (dev & 63);
    if (configured.load(std::memory_order_relaxed) & bit) return true;
    if (smem > 0 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return false;
    if (all_shared && cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared) != cudaSuccess) return false;
    configured.fetch_or(bit, std::memory_order_relaxed);
    return true;
}

template <typename Src, int DP, int NT, Kernel kernel>
int launch_decode(const DecodeParams& P, int ctas, cudaStream_t stream) {
    constexpr int smem = smem_bytes<Src, DP, NT>();
    static_assert(Shape<Src, DP, NT>::kCtas * (smem + 1024) <= 228 * 1024, "shared memory of an SM");
    if (!configure<kernel>(smem, Src::kQuant)) return TPB200_ERR_CUDA;
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = paged_config(static_cast<unsigned>(ctas), Shape<Src, DP, NT>::kThreads, smem, &attr, stream);
    return cudaLaunchKernelEx(&cfg, kernel, P) == cudaSuccess ? TPB200_OK : TPB200_ERR_CUDA;
}

// A call but for its cache
struct DecodeCall {
    const void* q;
    void* out;
    const long long *q_stride, *o_stride;
    int q_heads;
    float scale;
    void* workspace;
    size_t workspace_bytes;
    int flags, window, sinks;            // window 0: all keys
    long long pool_bytes = 0;            // of the pages, which the output must not reach into; 0: not asked
};

// The checks of a call and its parameters, P->cache being set; group_rows: query heads that go through together
int prepare_decode(const DecodeCall& a, int group_rows, int slot_keys, int item_units, int ctas, DecodeParams* out) {
    DecodeParams& P = *out;
    TPB_REQUIRE(a.q && a.out, TPB200_ERR_NULL);
    TPB_REQUIRE((a.flags & ~TPB200_FLAG_PDL) == 0, TPB200_ERR_ENUM);
    TPB_REQUIRE(a.q_heads >= 1 && a.q_heads % P.cache.kv_heads == 0, TPB200_ERR_SHAPE);
    TPB_REQUIRE(tpb_aligned16(a.q) && tpb_aligned16(a.out), TPB200_ERR_ALIGN);
    P.scale2 = a.scale * 1.4426950408889634f;
    TPB_REQUIRE(std::isfinite(P.scale2), TPB200_ERR_SHAPE);
    long long q_stride[2], o_stride[2];
    for (int i = 0; i < 2; ++i) {
        const int n = i == 0 ? P.cache.seqs : a.q_heads;
        q_stride[i] = a.q_stride[i];
        o_stride[i] = a.o_stride[i];
        for (const long long stride : {q_stride[i], o_stride[i]}) {
            const int fine = paged_stride(stride, n, P.cache.head_dim);
            if (fine != TPB200_OK) return fine;
        }
        P.q_stride[i] = n > 1 ? q_stride[i] : 0;
        P.o_stride[i] = n > 1 ? o_stride[i] : 0;
    }
    if (P.cache.seqs == 0) return TPB200_OK;
    TPB_REQUIRE(output_fits(RowSet(a.out, o_stride, P.cache.seqs, a.q_heads, P.cache.head_dim),
                            RowSet(a.q, q_stride, P.cache.seqs, a.q_heads, P.cache.head_dim)), TPB200_ERR_SHAPE);
    TPB_REQUIRE(a.pool_bytes == 0 || !rows_in_pools(RowSet(a.out, o_stride, P.cache.seqs, a.q_heads, P.cache.head_dim), P.cache, a.pool_bytes),
                TPB200_ERR_SHAPE);
    P.group = a.q_heads / P.cache.kv_heads;
    P.tiles = (P.group + group_rows - 1) / group_rows;
    P.rows = std::min(P.group, group_rows);
    // the line's length must fit an int, were every sequence as long as the table
    const int positions = P.cache.page_size * P.cache.table_width;
    const long long most = (static_cast<long long>(positions) + slot_keys - 1) / slot_keys;
    P.items = static_cast<long long>(P.cache.kv_heads) * P.tiles * P.cache.seqs;
    TPB_REQUIRE(P.items <= 0x7fffffff && (most * kSlotUnits + item_units) * P.items <= 0x7fffffff, TPB200_ERR_SHAPE);
    P.window = a.window > 0 ? std::min(a.window, positions) : positions;
    P.sinks = a.window > 0 ? std::min(a.sinks, positions) : 0;
    P.out_scale = 1.0f;
    TPB_REQUIRE(ctas >= 2, TPB200_ERR_CUDA);
    P.workers = ctas * kCtaWarps;
    const DecodeScratch d = decode_scratch(P.workers, P.rows, P.cache.head_dim);
    TPB_REQUIRE(a.workspace != nullptr && a.workspace_bytes >= d.bytes, TPB200_ERR_WORKSPACE);
    TPB_REQUIRE(tpb_aligned16(a.workspace), TPB200_ERR_ALIGN);
    uint8_t* ws = static_cast<uint8_t*>(a.workspace);
    P.joins = reinterpret_cast<int4*>(ws);
    P.part_ml = reinterpret_cast<float*>(ws + d.part_ml);
    P.part_o = reinterpret_cast<float*>(ws + d.part_o);
    P.join_by_item = P.items < P.workers;
    P.q = static_cast<const uint16_t*>(a.q);
    P.out = static_cast<uint16_t*>(a.out);
    return TPB200_OK;
}

// The second kernel, given for items of a hundred parts, of many and of few.  Its launch hides behind the first, which it waits for.  Where items are
// few they have many parts each (eight lanes of eight loads, or 32), else few (two of four, so that the whole launch is resident at once).
int launch_join(const DecodeParams& P, Kernel most_parts, Kernel many_parts, Kernel few_parts, int ctas, cudaStream_t stream) {
    const bool few = P.items * 8 < P.workers, fewest = most_parts != nullptr && P.items * 32 < ctas;
    const int quads = kJoinThreads / (fewest ? 32 : (few ? 8 : 2));
    cudaLaunchAttribute attr;
    cudaLaunchConfig_t cfg = paged_config(static_cast<unsigned>(P.join_by_item ? P.items : P.workers - 1), kJoinThreads, 0, &attr, stream);
    cfg.gridDim.y = static_cast<unsigned>((P.rows * P.cache.head_dim / 4 + quads - 1) / quads);
    return cudaLaunchKernelEx(&cfg, fewest ? most_parts : (few ? many_parts : few_parts), P) == cudaSuccess ? TPB200_OK : TPB200_ERR_CUDA;
}

}  // namespace
}  // namespace tpb
