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
#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "paged.cuh"

namespace tpb {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kSlotBytes = 8192;
constexpr int kSlots = 3;
constexpr int kCtasPerSm = 2;
constexpr int kSlotUnits = 2, kItemUnits = 1;      // what a slot costs, and an item besides: queries, sums, the output
constexpr float kLowest = -FLT_MAX;      // the least reference of a row with a key
constexpr int kLengths = 1024;           // lengths kept in shared memory; with more sequences they are read where they lie

struct DecodeParams {
    PagedView cache;
    const uint16_t* q;
    uint16_t* out;
    long long q_stride[2], o_stride[2];
    int group;                           // query heads per key head
    int tiles;                           // tiles of query heads per key head
    int rows;                            // rows of a tile that are used at most
    int join_by_item;                    // joins[] has a place per item, else one per worker
    float scale2;                        // scale * log2 e
    float* part_o;                       // [2 * workers][rows][head_dim]
    float* part_ml;                      // [2 * workers][rows][2]
    int4* joins;                         // (item or -1, its first part, its last worker, 1: first CTA merged | 2: last CTA merged)
};

// DP: head_dim rounded up to 64, 128 or 256.  NT: tiles of eight query heads that go through together.
template <int DP, int NT>
struct Shape {
    static constexpr int kKeys = kSlotBytes / (DP * 2);     // keys of a slot: 16, 32, 64
    static constexpr int kLanesRow = DP / 8;                // lanes that copy a row
    static constexpr int kRowsIter = 32 / kLanesRow;        // rows a warp copies at a time
    static constexpr int kCopies = kKeys / kRowsIter;
    static constexpr int kOwn = (kKeys + 31) / 32;          // rows a lane knows the place of
    static constexpr int kRows = 8 * NT;
    static constexpr int kChains = 1;    // 16-key blocks whose scores are summed in two chains of products, a latency each
    static constexpr bool kQueriesStay = NT * DP <= 256;    // in registers; else they are read again for every slot
    static constexpr bool kQueriesAhead = kQueriesStay && NT * DP * NT <= 256;      // the next item's too, where registers are left
    static constexpr int kSlab = NT == 1 ? 64 : 16;         // columns of a warp's sums that pass through shared memory at a time
    static constexpr int kSlabPitch = kSlab + 4;            // the four query pairs of a store fall into different banks
    static constexpr int kSumPitch = DP + 4;
    static_assert(kRows * kSumPitch * 4 <= kSlots * kSlotBytes, "a warp's sums where its ring was");
};

template <int NT>
struct Control {
    int lengths[kLengths];
    float ml[kWarps][8 * NT][2];
};

template <int DP, int NT>
constexpr int smem_bytes() {
    using S = Shape<DP, NT>;
    return kWarps * kSlots * kSlotBytes + kWarps * S::kRows * S::kSlabPitch * 4 + static_cast<int>(sizeof(Control<NT>));
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

// A place in the line of slots: slot `ci` of item (sequence, tile of query heads)
template <int kKeys>
struct Place {
    int s, h, ci, n, len;                // n: slots of the sequence's items
    int units;                           // of the line before the item
    int step;                            // slots from one of the warp's to its next
    __device__ __forceinline__ void enter(const DecodeParams& P, const int* lengths, int seq) {
        for (s = seq; s < P.cache.seqs; ++s) {
            len = P.cache.seqs <= kLengths ? lengths[s] : keys_of(P.cache, s);
            if (len > 0) break;
        }
        n = slots_of<kKeys>(len);
        h = ci = 0;
    }
    __device__ __forceinline__ void next(const DecodeParams& P, const int* lengths) {
        ci += step;
        if (ci < n) return;
        units += n * kSlotUnits + kItemUnits;
        ci = 0;
        if (++h < P.cache.kv_heads * P.tiles) return;
        enter(P, lengths, s + 1);
    }
};

// The line cut into pieces of equal cost, over the CTAs and a CTA's over its warps, the first ones of each getting a unit more.  A
// slot belongs to the piece in which its first unit lies, behind the item's own; pieces are two units at least, so a warp between the
// first and the last of an item always has a slot of it.  A line shorter than that for four warps is one warp's.
struct Share {
    int total, ctas, each, more;         // `more` CTAs of each + 1 units, the others of each
    __device__ __forceinline__ Share(int units, int grid) : total(units), ctas(min(grid, max(1, units / (kWarps * kSlotUnits)))) {
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

// kAligned: the page size is a multiple of 16, so that 16 rows from a multiple of 16 on lie in one page and share an address
template <typename T, int DP, int NT, bool kAligned>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) paged_attention_kernel(const __grid_constant__ DecodeParams P) {
    using S = Shape<DP, NT>;
    extern __shared__ __align__(128) uint8_t smem[];
    float* slab = reinterpret_cast<float*>(smem + kWarps * kSlots * kSlotBytes);
    Control<NT>* ctl = reinterpret_cast<Control<NT>*>(slab + kWarps * S::kRows * S::kSlabPitch);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int heads = P.cache.kv_heads * P.tiles;
    const int D = P.cache.head_dim;
    pdl_wait_prior_grids();
    pdl_launch_dependents();

    // ------------------------------------------------ this warp's piece of the line
    // Every warp for itself, without a barrier: slots and units before each lane's run of sequences, then the places where its piece
    // begins and ends.
    const bool staged = P.cache.seqs <= kLengths;        // all warps write the same lengths there, each reads its own
    const int run = (P.cache.seqs + 31) / 32, s0 = min(P.cache.seqs, lane * run), s1 = min(P.cache.seqs, s0 + run);
    int slots_here = 0, units_here = 0;
    bool empty = false;
    for (int s = s0; s < s1; ++s) {
        const int len = keys_of(P.cache, s), n = slots_of<S::kKeys>(len);
        if (staged) ctl->lengths[s] = len;
        slots_here += n * heads;
        units_here += n > 0 ? (n * kSlotUnits + kItemUnits) * heads : 0;
        empty = empty || n == 0;
    }
    __syncwarp();
    auto length = [&](int s) { return staged ? ctl->lengths[s] : keys_of(P.cache, s); };
    int slots_to = slots_here, units_to = units_here;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, slots_to, o), y = __shfl_up_sync(0xffffffffu, units_to, o);
        if (lane >= o) {
            slots_to += x;
            units_to += y;
        }
    }
    const Share line(__shfl_sync(0xffffffffu, units_to, 31), static_cast<int>(gridDim.x));
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
    if (line.total == 0 || cta >= line.ctas) return;

    // The place of the first slot that begins at `unit` or behind it, and the slots of the line before it.  A lane whose run holds the unit
    // finds the sequence, all lanes the rest.
    Place<S::kKeys> work;
    int item_first = 0;                  // units of the line before the item that holds the unit, and behind it
    int item_behind = 0;
    auto find = [&](int unit) {
        const bool here = unit >= units_to - units_here && unit < units_to;
        int s = s0, slots = slots_to - slots_here, units = units_to - units_here;
        if (here) {
            for (;; ++s) {
                const int n = slots_of<S::kKeys>(length(s)), more = n > 0 ? (n * kSlotUnits + kItemUnits) * heads : 0;
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
        work.n = slots_of<S::kKeys>(work.len);
        const int item = work.n * kSlotUnits + kItemUnits;
        work.h = (unit - units) / item;
        work.units = item_first = units + work.h * item;
        item_behind = item_first + item;
        const int in = unit - item_first;
        work.ci = in <= kItemUnits ? 0 : (in - kItemUnits + kSlotUnits - 1) / kSlotUnits;
        const int before = slots + work.h * work.n + work.ci;
        if (work.ci == work.n) {         // behind the item's last slot
            work.ci = work.n - 1;
            work.step = 1;
            work.next(P, ctl->lengths);
        }
        return before;
    };
    const int cta_first = line.cta_begin(cta), cta_behind = line.cta_begin(cta + 1);
    const int unit_first = line.begin(cta, warp), unit_behind = line.begin(cta, warp + 1);
    int slots = 0;
    bool merged = false, whole_item = false;
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
            return in <= kItemUnits ? 0 : min(work.n, (in - kItemUnits + kSlotUnits - 1) / kSlotUnits);
        };
        const int first = slot_of(cta_first), behind = slot_of(cta_behind);
        whole_item = first == 0 && behind == work.n;
        slots = max(0, (behind - first - warp + kWarps - 1) / kWarps);
        work.ci = first + warp;
        work.step = kWarps;
    }
    Place<S::kKeys> load = work;

    // ------------------------------------------------ loads
    const uint32_t ring = smem_u32(smem) + warp * kSlots * kSlotBytes;
    const int lane_row = lane / S::kLanesRow, lane_col = lane % S::kLanesRow;
    const bool lane_in = lane_col * 8 < D;
    constexpr int kPlaces = kAligned ? 1 : S::kOwn;
    int left = slots;                    // that the loads have still to enter
    int page_id[kPlaces];                // of this lane's rows of the next slot to load
    long long row_at[kPlaces];           // of the slot whose keys were asked for last: element offsets, -1: no such row
    int there = 0;                       // its keys
    // Keys whose page is not in the pool, a bit per group of 16 (aligned) or per key: of the slot whose keys were asked for last, and of the
    // one before it, which is the one that is worked on.
    constexpr int kKeysPerBit = kAligned ? 16 : 1;
    using Absent = std::conditional_t<(S::kKeys / kKeysPerBit > 32), uint64_t, uint32_t>;
    Absent absent_next = 0, absent = 0;

    // the key whose place lane `lane` looks up: aligned, the first of a group of 16; else its own
    auto own_key = [&](int o) { return static_cast<unsigned>(load.ci * S::kKeys) + (kAligned ? (lane * 16) % S::kKeys : o * 32 + lane); };
    auto fetch_ids = [&]() {             // page ids of the slot at `load`, asked for one slot ahead of their use
#pragma unroll
        for (int o = 0; o < kPlaces; ++o) {
            const unsigned key = own_key(o);
            page_id[o] = -1;
            if (left > 0 && key < static_cast<unsigned>(load.len) && (kAligned || o * 32 + lane < S::kKeys)) {
                page_id[o] = P.cache.table[load.s * P.cache.table_stride + key / P.cache.page_size];
            }
        }
    };
    auto enter_slot = [&]() {            // places of the slot at `load`; on to the next
        there = min(load.len - load.ci * S::kKeys, S::kKeys);
#pragma unroll
        for (int o = 0; o < kPlaces; ++o) {
            const unsigned key = own_key(o);
            row_at[o] = -1;
            const bool in = key < static_cast<unsigned>(load.len) && (kAligned || o * 32 + lane < S::kKeys);
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
                cp_async16(dst + r * (DP * 2) + ((lane_col ^ (r & 7)) << 4), src, r < rows ? 16 : 0);
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
    auto aim_queries = [&](const Place<S::kKeys>& at) {
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
    auto ask_queries = [&](const Place<S::kKeys>& at) {
        if constexpr (S::kQueriesAhead) {
            aim_queries(at);
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk) read_queries(kk, q_ahead[kk]);
        }
    };

    auto ask_next = [&]() {              // the queries of the item behind `work`
        if constexpr (S::kQueriesAhead) {
            Place<S::kKeys> then = work;
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
            const int valid = work.len - work.ci * S::kKeys;                           // keys of the slot, at least one
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
                const bool some = absent == 0 || __popcll(absent) < (min(valid, S::kKeys) + kKeysPerBit - 1) / kKeysPerBit;
                float top[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) top[n][0] = top[n][1] = some ? kLowest : -INFINITY;
                if (valid < S::kKeys || absent != 0) {
#pragma unroll
                    for (int b = 0; b < S::kKeys / 16; ++b)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int key = b * 16 + (lane >> 2) + (j >> 1) * 8;
                            const bool seen = key < valid && ((absent >> (kAligned ? b : key)) & 1) == 0;
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
        // ------------------------------------------------ the warp's sums -> the output, or a part of it
        const bool whole = first_ci == 0 && item_done;
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
                const int row = n * 8 + (lane & 3) * 2 + j;
                if (!whole && lane < 4 && row < P.rows) {
                    *reinterpret_cast<float2*>(P.part_ml + (part * P.rows + row) * 2) = make_float2(m[n][j], l[n][j]);
                }
            }
        }
        float* own = slab + warp * S::kRows * S::kSlabPitch;
        constexpr int kQuads = S::kSlab / 4;
#pragma unroll
        for (int x = 0; x < DP / S::kSlab; ++x) {
#pragma unroll
            for (int i = 0; i < S::kSlab / 16; ++i) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        own[(n * 8 + (lane & 3) * 2 + (j & 1)) * S::kSlabPitch + i * 16 + (lane >> 2) + (j >> 1) * 8] =
                            o[x * (S::kSlab / 16) + i][n][j] * f[n][j & 1];
                    }
                }
            }
            __syncwarp();
            for (int u = lane; u < min(P.group - row0, S::kRows) * kQuads; u += 32) {
                const int row = u / kQuads, col = x * S::kSlab + u % kQuads * 4;
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
        if (lane == 0 && first_ci == 0) {
            const int item = work.s * heads + work.h;
            if (whole) {
                if (P.join_by_item) P.joins[item] = make_int4(-1, 0, 0, 0);
            } else {                     // it begins here and ends with a later warp
                const int by = line.last_worker(work.units, work.n);
                P.joins[P.join_by_item ? item : worker] =
                    make_int4(item, static_cast<int>(part), by, by / kWarps != cta && line.ends_merged(work.units, work.n, by) ? 2 : 0);
            }
        }
        if (!whole) ++parts;
        if (!last) {
            work.next(P, ctl->lengths);
            first_ci = 0;
            start();
            if ((uses + kSlots - 1 - t) / 2 > work.n) ask_next();
        }
    }
    cp_async_wait<0>();
    if (!merged) return;
    // ------------------------------------------------ the CTA's sums, each warp's where its ring was
    float* sums = reinterpret_cast<float*>(smem + warp * kSlots * kSlotBytes);
    __syncwarp();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], x);
            if (lane < 4) *reinterpret_cast<float2*>(ctl->ml[warp][n * 8 + lane * 2 + j]) = make_float2(m[n][j], l[n][j]);
        }
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                sums[(n * 8 + (lane & 3) * 2 + (j & 1)) * S::kSumPitch + i * 16 + (lane >> 2) + (j >> 1) * 8] = o[i][n][j];
            }
        }
    }
    __syncthreads();
    const bool whole = whole_item;
    const int kvh = work.h / P.tiles, row0 = (work.h - kvh * P.tiles) * S::kRows;
    const long long part = 2ll * kWarps * cta;
    const int rows = min(P.group - row0, S::kRows);
#pragma unroll 4
    for (int u = threadIdx.x; u < S::kRows * (DP / 4); u += kThreads) {
        const int row = u / (DP / 4), col = u % (DP / 4) * 4;
        if (row >= rows || col >= D) continue;
        float M = -INFINITY, L = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, ctl->ml[w][row][0]);
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = ex2(ctl->ml[w][row][0] - (M == -INFINITY ? 0.0f : M));
            const float4 y = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem + w * kSlots * kSlotBytes) + row * S::kSumPitch + col);
            L += ctl->ml[w][row][1] * f;
            sum.x += y.x * f; sum.y += y.y * f; sum.z += y.z * f; sum.w += y.w * f;
        }
        if (whole) {
            const float inv = inverse(M, L);
            uint16_t* to = P.out + work.s * P.o_stride[0] + (kvh * P.group + row0 + row) * P.o_stride[1] + col;
            *reinterpret_cast<uint2*>(to) = make_uint2(Half16<T>::pack(sum.x * inv, sum.y * inv), Half16<T>::pack(sum.z * inv, sum.w * inv));
        } else {
            *reinterpret_cast<float4*>(P.part_o + (part * P.rows + row) * D + col) = sum;
            if (col == 0) *reinterpret_cast<float2*>(P.part_ml + (part * P.rows + row) * 2) = make_float2(M, L);
        }
    }
    if (threadIdx.x == 0 && first_ci == 0) {
        const int item = work.s * heads + work.h;
        if (whole) {
            if (P.join_by_item) P.joins[item] = make_int4(-1, 0, 0, 0);
        } else {
            const int by = line.last_worker(work.units, work.n);
            P.joins[P.join_by_item ? item : worker] = make_int4(item, static_cast<int>(part), by, line.ends_merged(work.units, work.n, by) ? 3 : 1);
        }
    }
}

// Where an item begins that ends with another worker, its parts are joined.  Workers are warps; a CTA that lies inside the item has
// left one part, as its first worker, the item's other workers one each: the one it begins with its last part, those behind it their
// first.  blockIdx.x: the item, or the worker it begins with; a thread has four columns of a row (blockIdx.y: which ones) of every
// kLanes-th part, kLoads of them on their way at a time, with a running maximum of its own.
constexpr int kJoinThreads = 128;

template <typename T, int kLanes, int kLoads>
__global__ void __launch_bounds__(kJoinThreads) paged_attention_join_kernel(const __grid_constant__ DecodeParams P) {
    constexpr int kQuads = kJoinThreads / kLanes;
    __shared__ float4 sums[kLanes][kQuads];
    __shared__ float2 mls[kLanes][kQuads];
    pdl_wait_prior_grids();
    pdl_launch_dependents();
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
        const float inv = inverse(m, l);
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

// places for joins: an item's where the items are fewer than the workers, else a worker's
struct DecodeScratch { size_t part_ml, part_o, bytes; };

DecodeScratch decode_scratch(int ctas, int rows, int head_dim) {
    DecodeScratch d;
    const size_t workers = static_cast<size_t>(ctas) * kWarps;
    d.part_ml = workers * sizeof(int4);
    d.part_o = d.part_ml + 2 * workers * rows * 2 * sizeof(float);
    d.part_o = (d.part_o + 255) / 256 * 256;
    d.bytes = d.part_o + 2 * workers * rows * head_dim * sizeof(float);
    return d;
}

// query heads that go through together: eight, or sixteen where a group has more; larger groups read the cache once per sixteen (48 sequences of 1 to
// 4096, 4 key heads of 128, 80 MB: groups of 8 21 us, of 16 28, of 32 47)
int decode_rows(int group) { return group <= 8 ? 8 : 16; }

template <typename T, int DP, int NT, bool kAligned>
int launch_decode(const DecodeParams& P, int ctas, cudaStream_t stream) {
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
    const cudaLaunchConfig_t cfg = paged_config(static_cast<unsigned>(ctas), kThreads, smem, &attr, stream);
    return cudaLaunchKernelEx(&cfg, paged_attention_kernel<T, DP, NT, kAligned>, P) == cudaSuccess ? TPB200_OK : TPB200_ERR_CUDA;
}

template <typename T, int DP>
int launch_decode(const DecodeParams& P, int ctas, cudaStream_t stream) {
    const bool aligned = P.cache.page_size % 16 == 0;
    if (P.group <= 8) return aligned ? launch_decode<T, DP, 1, true>(P, ctas, stream) : launch_decode<T, DP, 1, false>(P, ctas, stream);
    return aligned ? launch_decode<T, DP, 2, true>(P, ctas, stream) : launch_decode<T, DP, 2, false>(P, ctas, stream);
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
    P.scale2 = a->scale * 1.4426950408889634f;
    TPB_REQUIRE(std::isfinite(P.scale2), TPB200_ERR_SHAPE);
    for (int i = 0; i < 2; ++i) {
        const int n = i == 0 ? P.cache.seqs : a->q_heads;
        for (const long long stride : {a->q_stride[i], a->o_stride[i]}) {
            const int fine = paged_stride(stride, n, P.cache.head_dim);
            if (fine != TPB200_OK) return fine;
        }
        P.q_stride[i] = n > 1 ? a->q_stride[i] : 0;
        P.o_stride[i] = n > 1 ? a->o_stride[i] : 0;
    }
    if (P.cache.seqs == 0) return TPB200_OK;
    TPB_REQUIRE(output_fits(RowSet(a->out, a->o_stride, P.cache.seqs, a->q_heads, P.cache.head_dim),
                            RowSet(a->q, a->q_stride, P.cache.seqs, a->q_heads, P.cache.head_dim)), TPB200_ERR_SHAPE);
    P.group = a->q_heads / P.cache.kv_heads;
    P.tiles = (P.group + decode_rows(P.group) - 1) / decode_rows(P.group);
    P.rows = std::min(P.group, decode_rows(P.group));
    // the line's length must fit an int, were every sequence as long as the table
    const int slot_keys = P.cache.head_dim <= 64 ? 64 : (P.cache.head_dim <= 128 ? 32 : 16);
    const long long most = (static_cast<long long>(P.cache.page_size) * P.cache.table_width + slot_keys - 1) / slot_keys;
    const long long items = static_cast<long long>(P.cache.kv_heads) * P.tiles * P.cache.seqs;
    TPB_REQUIRE(items <= 0x7fffffff && (most * kSlotUnits + kItemUnits) * items <= 0x7fffffff, TPB200_ERR_SHAPE);
    const int ctas = decode_ctas();
    TPB_REQUIRE(ctas >= 2, TPB200_ERR_CUDA);
    const DecodeScratch d = decode_scratch(ctas, P.rows, P.cache.head_dim);
    TPB_REQUIRE(a->workspace != nullptr && a->workspace_bytes >= d.bytes, TPB200_ERR_WORKSPACE);
    TPB_REQUIRE(tpb_aligned16(a->workspace), TPB200_ERR_ALIGN);
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    P.joins = reinterpret_cast<int4*>(ws);
    P.part_ml = reinterpret_cast<float*>(ws + d.part_ml);
    P.part_o = reinterpret_cast<float*>(ws + d.part_o);
    P.join_by_item = items < static_cast<long long>(ctas) * kWarps;
    P.q = static_cast<const uint16_t*>(a->q);
    P.out = static_cast<uint16_t*>(a->out);
    const bool bf = a->cache.dtype == TPB200_BF16;
    const int D = P.cache.head_dim;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const int done = D <= 64 ? (bf ? launch_decode<__nv_bfloat16, 64>(P, ctas, s) : launch_decode<__half, 64>(P, ctas, s))
                   : D <= 128 ? (bf ? launch_decode<__nv_bfloat16, 128>(P, ctas, s) : launch_decode<__half, 128>(P, ctas, s))
                              : (bf ? launch_decode<__nv_bfloat16, 256>(P, ctas, s) : launch_decode<__half, 256>(P, ctas, s));
    if (done != TPB200_OK) return done;
    // Its launch hides behind the first kernel, which it waits for.  Where items are few they have many parts each
    // (eight lanes of eight loads), else few (two of four, so that the whole launch is resident at once).
    const bool few = items * 8 < static_cast<long long>(ctas) * kWarps;
    const int quads = kJoinThreads / (few ? 8 : 2);
    cudaLaunchAttribute attr;
    cudaLaunchConfig_t cfg = paged_config(static_cast<unsigned>(P.join_by_item ? items : ctas * kWarps - 1), kJoinThreads, 0, &attr, s);
    cfg.gridDim.y = static_cast<unsigned>((P.rows * D / 4 + quads - 1) / quads);
    const auto join = few ? (bf ? paged_attention_join_kernel<__nv_bfloat16, 8, 8> : paged_attention_join_kernel<__half, 8, 8>)
                          : (bf ? paged_attention_join_kernel<__nv_bfloat16, 2, 4> : paged_attention_join_kernel<__half, 2, 4>);
    return cudaLaunchKernelEx(&cfg, join, P) == cudaSuccess ? TPB200_OK : TPB200_ERR_CUDA;
}
