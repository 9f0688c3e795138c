// Attention over whole prompts, packed one behind the other: softmax(scale Q K^T) V per sequence, causal or not, with
// grouped heads, queries behind keys that are already there, bf16 or fp16, on tcgen05.mma kind::f16.
//
// One pass over the keys per tile of 128 query rows, with the running reference m of a softmax:
//     S = Q K_j^T,  P = 2^(scale2 S - m),  O += P V_j,  l += rowsum P,      out = O / l
// m is raised (and O, l scaled by 2^(m_old - m_new)) only when a row's maximum passes m by 8, a published way to run a softmax: P stays below
// 2^8 and after the first tiles O is hardly ever touched between its products.  P is rounded to the tensors' type; fp16 holds it 2^7 times
// larger (Half16::kLift), so that small weights keep their bits.
//
// A row of a tile is a (token, head) pair: `pack` query heads of one key head, the largest power of two in the group, side by side,
// so that short prompts fill tiles and the heads of a group read their keys once.
//
// Roles (384 threads, one CTA an SM): warp 0 requests tiles of K and V by TMA into a ring of units, warp 1 issues the products, warps
// 2 and 3 look tiles with masked pairs over, two groups of four warps do the softmax, a thread per row, with registers moved over to
// them from the others (setmaxnreg).
// The products are a line of events e; event e computes S into tensor-memory buffer e & 1, group e & 1 turns it into P in the same
// columns, the product with V reads P from there, the first half of the keys while the weights of the second are computed:
//   head sizes up to 128  two tiles of 128 rows per CTA, one per group: event e is key tile e / 2 of row tile e & 1; each unit of K
//                         and V is read by both, which halves what comes through L2 (a row tile of its own needs 64 KB per
//                         1024 cycles of products, more than an SM gets);
//                         short sequences: one row tile and one group (256 threads), two CTAs on an SM;
//   above                 one row tile (its O alone is 256 columns), the groups take alternate key tiles and hand m on through
//                         shared memory.
// While one group works the other's products run.
//
// What bounds it, measured on one B200 (ten calls in a CUDA graph, before the board's power limit; calls one after the other reach it):
//   one sequence of 8191 tokens, causal, 8 on 1 heads of 256: 197 us = 1.40 PFLOP/s, 0.85 of the measured bf16 burst rate: hand-overs from product to
//   softmax and back.  Call after call 237 us = 1.16, 0.83 of the rate that lasts for seconds.
//   4 sequences, 24.6 k tokens, causal, 32 on 8 heads of 128: 1.38 ms = 1.23 PFLOP/s, 0.75, at 1965 MHz; after some 10 ms of it the board
//   is at its 1000 W, the clock goes to 1.6 GHz and the call to 1.56-1.62 ms.  At full clock two tiles take 3350 cycles, of which their products
//   need 2048 and so do their exponentials (16 a cycle and SM): a group's softmax takes 2000 (1300 to the first half of P) while the
//   other's runs too, then 1130 pass until its next scores are there.  About 6 us of each CTA's 60 pass in its first loads and its output.
//   One sequence of 200 tokens, 8 on 1 heads of 256: 10.7 us: look-up 0.6, tensor memory and barriers 0.3, loads 1-2, 1.1 of softmax per tile,
//   1.4 for the output, one after the other.
// One thread issues the products, from operands that the compiler knows to be the same in all lanes (uniform()), and tests barriers while
// products ahead of them run.  With operands it had to move over for every product, issuing took as long as running, and of an event's 1760
// cycles 690 went between products (one sequence 201 -> 195 us, four 1414 -> 1381 unthrottled, 1645 -> 1605 throttled).
// Tried without gain: an eighth to a half of the exponentials as polynomials on the FMA pipes (four sequences 1555 us without, 1585-1620 with:
// their energy); two threads issuing, one per row tile (1725 us: the two no longer alternate); four groups, two threads per row (1.75 -> 1.94 ms;
// sequences of 100 tokens gain 7 %, those of 1 to 1200 lose 6 %); pairs of CTAs on one product (cta_group::2, M = 256: 2.47 ms, the single
// sequence 250 us, each hand-over crosses the cluster).
//
// Sliding windows (kWindow): tiles without a visible pair are not visited.  One sequence of 8191 tokens, 8 on 1 heads of 256, window 1024, four sinks: 86.4 us
// (all keys: 197), 9 tiles a CTA for 8.03 of visible pairs; 512 CTAs of 21 us, 5 of them look-up, first loads and output, in four waves.  24 ragged sequences of 1 to 1200, 16 on 4 heads
// of 64, window 200: 26.1; four long ones, 32 on 8 of 128, window 1500: 281, 0.55 of the measured bf16 burst rate.  With whole tiles left out instead of keys: 93, 27.8, 291.
//
// What may stand in masked places does not matter: scores are selected, not biased.  Rows of V behind a sequence's end are zeroed in
// shared memory, and in tiles that hold masked pairs V is searched for infinities and NaN (weight 0 times those would be NaN): they are
// taken out and added to the rows that do see them at the end.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "paged.cuh"
#include "tcgen05.cuh"

namespace tpb {
namespace {

constexpr int kTile = 128;               // rows of a query tile, keys of a key tile
constexpr int kHalf = kTile / 2;         // keys of a request where a window may leave out keys between two of them
constexpr int kBlockBytes = kTile * 128; // 128 rows x 64 columns of 16 bits
constexpr long long kWait = 200000000LL; // about 0.1 s: the bound of each wait
constexpr float kRaise = 8.0f;
constexpr int kMaxTokens = 0x7fffffff - 1023;        // positions are 32 bits, and up to four tiles' rows behind the last one are counted
constexpr int kBadTiles = 4;             // key tiles with masked pairs at most: 256 rows on the diagonal and the sequence's end

struct PackedParams {
    CUtensorMap q, k, v;
    uint16_t* out;
    const uint16_t* v_rows;
    long long o_stride[2], v_stride[2];
    const int *cu, *cu_keys;
    int seqs, q_tokens, k_tokens;
    int head_dim;
    int pack, pack_shift, head_groups;   // query heads of a tile; tiles' worth of heads
    int groups_per_kv;                   // head groups that share a key head
    float scale2;                        // |scale| log2 e
    uint32_t idesc_s, idesc_o;
    int causal;
    int window, sinks;                   // a query sees the last `window` keys up to its own and the first `sinks` (kWindow)
};

// DP: head_dim rounded up to 64, 128 or 256; R: tiles of 128 rows per CTA, two only up to 128
template <int DP, int R>
struct Layout {
    static constexpr bool kOwn = DP <= 128;                        // every row tile has a group, a buffer of scores and an O of its own
    static constexpr int kGroups = kOwn ? R : 2;
    static constexpr int kThreads = 128 + 128 * kGroups;
    static constexpr int kCtas = kOwn && R == 1 ? 2 : 1;           // on an SM
    static constexpr uint32_t kTmemCols = kCtas == 2 ? 256 : 512, kColO = kGroups * kTile;
    // Where tensor memory has room for P beside S, the next scores are computed while the exponentials of these are: 8192 tokens, 16 heads
    // of 64, 203 -> 194 us.  With one row tile the other CTA fills the gaps: 16 sequences of 512 36.0 us, ahead 36.4.
    static constexpr bool kAhead = DP == 64 && R == 2;
    static constexpr uint32_t kColP = kAhead ? kColO + kGroups * DP : 0, kStepP = kAhead ? kTile / 2 : kTile;
    static constexpr int kBlocks = DP / 64;                        // 64-column blocks of a row
    static constexpr int kUnitBlocks = DP < 128 ? 1 : 2;           // a unit: 128 keys x up to 128 columns
    static constexpr int kHalves = kBlocks / kUnitBlocks;          // units of a tile
    static constexpr int kUnitBytes = kUnitBlocks * kBlockBytes;
    static constexpr int kUnits = kCtas == 2 ? (DP < 128 ? 4 : 2) : (DP < 128 ? 8 : 4);
    static constexpr int kQBytes = R * kBlocks * kBlockBytes;
    // registers move over to the softmax: threads x registers at launch (168 or 128 each) on both sides
    static constexpr int kFewRegs = kCtas == 2 ? 56 : 64, kManyRegs = kCtas == 2 ? 200 : 216;
    static_assert(R == 1 || kOwn, "");
};

struct PackedControl {
    uint64_t q_full;
    uint64_t full[8], empty[8];
    uint64_t s_ready[2], p_ready[2][2], o_done[2];       // p_ready: by half of the tile's keys
    uint64_t s_read[2];                  // scores are in registers, the next ones may take their place (kAhead)
    uint64_t ref_ready[2][4];            // one row tile: the reference of event e, by quarter of the rows
    uint64_t v_landed[2 * kBadTiles];    // V of a tile with masked pairs, which is looked over before its units count as full
    uint32_t tmem_base;
    int failed;
    int seq, tile, q0, nq, k0, nk;       // the CTA's work
    int bad_any;
    uint32_t bad[2 * kBadTiles][4];      // keys of masked tiles with infinities or NaN in V
    float ref[kTile];
    float part_l[2][kTile], part_m[2][kTile];
};

template <int DP, int R>
constexpr int packed_smem() {
    using L = Layout<DP, R>;
    return std::max(L::kQBytes + L::kUnits * L::kUnitBytes + static_cast<int>(sizeof(PackedControl)) + 1024, min_smem_of_columns(L::kTmemCols));
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a),
        "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a),
        "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};\n" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
// Waits for the loads into r, which nothing may read before: the operands keep the compiler from moving a use up
__device__ __forceinline__ void tmem_ld_wait_for(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_st_x8(uint32_t addr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
                 "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ void tmem_st_done() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Pairs of floats in one instruction
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity) {
    return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, kWait));
}

// The value all lanes hold, where the compiler knows that they do: operands of products live in uniform registers
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __reduce_or_sync(0xffffffffu, x); }

// Warps 2 and 3 meet, and learn whether both are fine
__device__ __forceinline__ bool meet_and(bool ok) {
    uint32_t all;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.u32 q, %1, 0;\n barrier.cta.red.and.pred p, 2, 64, q;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(all)
        : "r"(static_cast<uint32_t>(ok))
        : "memory");
    return all != 0;
}

// The keys a query row sees: [0, limit)
__device__ __forceinline__ int row_limit(const PackedParams& P, int nq, int nk, int token) {
    if (token >= nq) return 0;
    return P.causal ? max(0, min(nk, nk - nq + token + 1)) : nk;
}

template <int kRegs>
__device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs)); }
template <int kRegs>
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs)); }

template <typename T, int DP, int R, bool kWindow>
__global__ void __launch_bounds__(Layout<DP, R>::kThreads, Layout<DP, R>::kCtas) packed_attention_kernel(const __grid_constant__ PackedParams P) {
    using L = Layout<DP, R>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sQ = smem;
    uint8_t* ring = smem + L::kQBytes;
    PackedControl* ctl = reinterpret_cast<PackedControl*>(ring + L::kUnits * L::kUnitBytes);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int head_group = blockIdx.x % P.head_groups;
    constexpr int kRowsCta = R * kTile;
    const int tokens_cta = kRowsCta >> P.pack_shift;

    pdl_wait_prior_grids();              // the offsets may come from the previous kernel too
    if (warp == 0) {
        // which tile of which sequence: tiles are dealt from the last one back, so that within a sequence the long rows come first
        const int want = static_cast<int>(gridDim.x / P.head_groups - 1 - blockIdx.x / P.head_groups);
        int before = 0;
        if (lane == 0) ctl->seq = -1;
        __syncwarp();
        for (int s0 = 0; s0 < P.seqs; s0 += 32) {
            const int s = s0 + lane;
            int n = 0, a = 0, b = 0, ka = 0, kb = 0;
            if (s < P.seqs) {
                a = min(max(P.cu[s], 0), P.q_tokens);
                b = min(max(P.cu[s + 1], a), P.q_tokens);
                ka = min(max(P.cu_keys[s], 0), P.k_tokens);
                kb = min(max(P.cu_keys[s + 1], ka), P.k_tokens);
                n = (b - a + tokens_cta - 1) / tokens_cta;
            }
            int upto = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += y;
            }
            const bool mine = want >= before + upto - n && want < before + upto;
            if (mine) {
                ctl->seq = s;
                ctl->tile = want - before - (upto - n);
                ctl->q0 = a;
                ctl->nq = b - a;
                ctl->k0 = ka;
                ctl->nk = kb - ka;
            }
            if (__any_sync(0xffffffffu, mine)) break;
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
    }
    if (threadIdx.x == 32) {
        mbar_init(&ctl->q_full, 1);
        for (int i = 0; i < L::kUnits; ++i) {
            mbar_init(&ctl->full[i], 1);
            mbar_init(&ctl->empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&ctl->s_ready[i], 1);
            for (int h = 0; h < 2; ++h) mbar_init(&ctl->p_ready[i][h], 4);
            mbar_init(&ctl->o_done[i], 1);
            mbar_init(&ctl->s_read[i], 4);
            for (int w = 0; w < 4; ++w) mbar_init(&ctl->ref_ready[i][w], 1);
        }
        for (int i = 0; i < (kWindow ? 2 : 1) * kBadTiles; ++i) mbar_init(&ctl->v_landed[i], L::kHalves);
        fence_mbar_init();
        ctl->failed = 0;
        ctl->bad_any = 0;
        for (int i = 0; i < (kWindow ? 2 : 1) * kBadTiles * 4; ++i) ctl->bad[i >> 2][i & 3] = 0;
        tc::prefetch_tensormap(&P.q);
        if (P.k_tokens > 0) {
            tc::prefetch_tensormap(&P.k);
            tc::prefetch_tensormap(&P.v);
        }
    }
    if (warp == 2) {
        tc::tmem_alloc(&ctl->tmem_base, L::kTmemCols);
        tc::tmem_relinquish();
    }
    tc::fence_before_thread_sync();
    __syncthreads();
    tc::fence_after_thread_sync();
    pdl_launch_dependents();
    const uint32_t tmem = ctl->tmem_base;
    if (ctl->seq < 0) {                  // more tiles were launched than there are
        if (warp == 2) tc::tmem_dealloc(tmem, L::kTmemCols);
        return;
    }
    const int nq = ctl->nq, nk = ctl->nk, q0 = ctl->q0, k0 = ctl->k0;
    const int token0 = ctl->tile * tokens_cta;
    const int tokens_tile = kTile >> P.pack_shift;
    // key tiles of each row tile: up to the last row's limit; the second row tile of a CTA never has fewer than the first
    int tiles[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int first = token0 + x * tokens_tile, last = min(first + tokens_tile, nq) - 1;
        tiles[x] = (x < R && last >= first) ? (row_limit(P, nq, nk, last) + kTile - 1) / kTile : 0;
    }
    if (!L::kOwn) tiles[1] = 0;
    // With a window, the keys between those of the sinks (whole halves of a tile) and the first one that the first row's window reaches are left out:
    // the CTA's keys are numbered without these `gap` keys, and so are the rows' limits.  Whatever is left between the sinks and a row's window is one
    // range for each row.  Tiles from left_begin to left_end hold pairs of it, kBadTiles at most: the windows of 256 rows begin within
    // 256 keys, behind at most 64 of the sinks' last half.
    int gap = 0, sink_keys = 0, left_begin = 0, left_end = 0;
    const int first_limit = row_limit(P, nq, nk, token0);
    if (kWindow) {
        const int last = row_limit(P, nq, nk, min(token0 + tokens_cta, nq) - 1);
        sink_keys = static_cast<int>(min((static_cast<unsigned>(P.sinks) + kHalf - 1) / kHalf * kHalf, 0x7fffff00u));
        const int reach = max(0, first_limit - P.window);        // the first row's first key in its window
        gap = reach > sink_keys ? reach - sink_keys : 0;
        const int behind = last - gap - P.window;        // of the keys that some row does not see, but for the sinks
        if (behind > P.sinks) {
            left_begin = min(P.sinks, first_limit - gap) / kTile;
            left_end = (behind + kTile - 1) / kTile;
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int first = token0 + x * tokens_tile, end = min(first + tokens_tile, nq) - 1;
            if (tiles[x] > 0) tiles[x] = (row_limit(P, nq, nk, end) - gap + kTile - 1) / kTile;
        }
    }
    auto real = [&](int key) { return kWindow && key >= sink_keys ? key + gap : key; };      // of its sequence
    const int n_tiles = max(tiles[0], tiles[1]);
    const int first_masked = (first_limit - gap) / kTile;                // tiles from here on hold masked pairs: kBadTiles at most
    const int right_begin = kWindow ? max(first_masked, left_end) : first_masked;
    // the places of tiles with masked pairs in v_landed and bad
    auto looked_over = [&](int j) { return j >= first_masked || (kWindow && j >= left_begin && j < left_end); };
    auto place = [&](int j) { return kWindow ? (j < left_end ? j - left_begin : kBadTiles + j - right_begin) : j - first_masked; };
    auto tile_at = [&](int place) { return kWindow ? (place < kBadTiles ? left_begin + place : right_begin + place - kBadTiles) : first_masked + place; };
    const int events = L::kOwn ? 2 * n_tiles : n_tiles;
    // the order of the line of events: which are computed, and where the tiles of K and V stand in the ring
    auto active = [&](int e) { return L::kOwn ? (e >> 1) < tiles[e & 1] : true; };
    auto key_tile = [&](int e) { return L::kOwn ? e >> 1 : e; };
    auto k_unit = [&](int j) { return L::kHalves * (L::kOwn ? 2 * j : (j < 2 ? j : 2 * j - 1)); };
    auto v_unit = [&](int j) { return L::kHalves * (L::kOwn ? 2 * j + 1 : (j == n_tiles - 1 ? 2 * j + 1 : 2 * j + 2)); };

    if (warp < 4) {
        fewer_registers<L::kFewRegs>();
        if (warp == 0 && n_tiles > 0) {
            // -------------------------------------------------------- producer
            const int kv_head = head_group / P.groups_per_kv;
            if (tc::elect_one()) {
                bool ok = true;
                mbar_expect_tx(&ctl->q_full, (tiles[1] > 0 ? 2 : 1) * L::kBlocks * kBlockBytes);
                for (int x = 0; x < (tiles[1] > 0 ? 2 : 1); ++x) {
                    for (int b = 0; b < L::kBlocks; ++b) {
                        tma_load_3d(sQ + (x * L::kBlocks + b) * kBlockBytes, &P.q, b * 64, head_group << P.pack_shift,
                                    q0 + token0 + x * tokens_tile, &ctl->q_full);
                    }
                }
                int u = 0;
                auto request = [&](const CUtensorMap* map, int j, bool values = false) {
                    for (int h = 0; h < L::kHalves; ++h, ++u) {
                        const int slot = u % L::kUnits;
                        if (!mbar_wait_bounded(&ctl->empty[slot], ((u / L::kUnits) & 1) ^ 1, kWait)) return false;
                        uint64_t* bar = values && looked_over(j) ? &ctl->v_landed[place(j)] : &ctl->full[slot];
                        mbar_expect_tx(bar, L::kUnitBytes);
                        for (int b = 0; b < L::kUnitBlocks; ++b) {
                            uint8_t* to = ring + slot * L::kUnitBytes + b * kBlockBytes;
                            const int column = (h * L::kUnitBlocks + b) * 64;
                            tma_load_3d(to, map, column, kv_head, k0 + real(j * kTile), bar);
                            if (kWindow) tma_load_3d(to + kBlockBytes / 2, map, column, kv_head, k0 + real(j * kTile + kHalf), bar);
                        }
                    }
                    return true;
                };
                if (L::kOwn) {
                    for (int j = 0; j < n_tiles && ok; ++j) ok = request(&P.k, j) && request(&P.v, j, true);
                } else {
                    ok = request(&P.k, 0);
                    for (int j = 1; j < n_tiles && ok; ++j) ok = request(&P.k, j) && request(&P.v, j - 1, true);
                    ok = ok && request(&P.v, n_tiles - 1, true);
                }
                if (!ok) {
                    record_error(kErrPackedBarrierTimeout);
                    ctl->failed = 1;
                }
            }
            __syncwarp();
        } else if (warp == 1 && n_tiles > 0) {
            // -------------------------------------------------------- products
            const uint32_t tm = uniform(tmem);
            const uint32_t q16 = (smem_u32(sQ) & 0x3FFFFu) >> 4, r16 = (smem_u32(ring) & 0x3FFFFu) >> 4;
            constexpr uint32_t kDescHiMnSw128 = (1024u >> 4) | (1u << 14) | (static_cast<uint32_t>(tc::kSwizzle128B) << 29);
            constexpr uint32_t kLboField = (static_cast<uint32_t>(kBlockBytes) >> 4) << 16;
            // Barriers are tested before products are issued and the outcome is looked at behind them; the second product of head sizes
            // above 128 has N = 256.
            auto test = [&](uint64_t* bar, uint32_t parity) { return mbar_test_wait(bar, parity); };
            auto unit_full = [&](int u) { return &ctl->full[u % L::kUnits]; };
            auto unit_parity = [&](int u) -> uint32_t { return (u / L::kUnits) & 1; };
            // scores of one unit of K (past head_dim both operands are zero), row tile x, into buffer x
            auto scores = [&](int x, int u, int h) {
                const uint32_t qa = q16 + ((L::kOwn ? x * L::kBlocks * kBlockBytes : h * L::kUnitBytes) >> 4), ka = r16 + (u % L::kUnits * L::kUnitBytes >> 4);
#pragma unroll
                for (int kk = 0; kk < L::kUnitBlocks * 4; ++kk) {
                    const uint32_t off = static_cast<uint32_t>((kk >> 2) * kBlockBytes + (kk & 3) * 32) >> 4;
                    mma_ss(tm + x * kTile, tc::desc_from_words(qa + off, tc::kDescHiKmajorSw128), tc::desc_from_words(ka + off, tc::kDescHiKmajorSw128),
                           P.idesc_s, (h | kk) > 0 ? 1u : 0u);
                }
            };
            // the product of half of a tile's keys, weights in buffer x; a tile's units lie one behind the other
            auto values = [&](int x, int u, int part, uint32_t more) {
                const uint32_t va = r16 + (u % L::kUnits * L::kUnitBytes >> 4), d = tm + L::kColO + (L::kOwn ? x * DP : 0);
#pragma unroll
                for (int kk = part * 4; kk < part * 4 + 4; ++kk) {
                    mma_ts(d, tm + L::kColP + x * L::kStepP + kk * 8, tc::desc_from_words((va + (kk * 2048 >> 4)) | kLboField, kDescHiMnSw128), P.idesc_o,
                           kk > 0 ? 1u : more);
                }
            };
            bool ok = wait_warp(&ctl->q_full, 0);
            if constexpr (L::kOwn) {
                const int t0 = uniform(tiles[0]), t1 = uniform(tiles[1]), n = max(t0, t1);
                ok = ok && wait_warp(unit_full(0), 0);
                if (tc::elect_one()) {
                    if (ok && t0 > 0) {
                        scores(0, 0, 0);
                        tc::commit(&ctl->s_ready[0]);
                    }
                    if (R == 2 && ok && t1 > 0) {
                        scores(R - 1, 0, 0);
                        tc::commit(&ctl->s_ready[R - 1]);
                    }
                    if (ok) tc::commit(&ctl->empty[0]);
                    bool p0 = false, vf = false;
                    for (int j = 0; j < n && ok; ++j) {
                        const int v = 2 * j + 1, k = 2 * j + 2;
#pragma unroll
                        for (int x = 0; x < R; ++x) {
                            const int t = x == 0 ? t0 : t1;
                            const bool last_use = x == R - 1 || t1 == 0;
                            if (j >= t || !ok) continue;
                            const bool next = j + 1 < t;
                            auto next_scores = [&](bool early) {
                                ok = early || mbar_wait_bounded(unit_full(k), unit_parity(k), kWait);
                                if (!ok) return;
                                scores(x, k, 0);
                                tc::commit(&ctl->s_ready[x]);
                                if (last_use) tc::commit(&ctl->empty[k % L::kUnits]);
                            };
                            if (L::kAhead && next) {
                                ok = mbar_wait_bounded(&ctl->s_read[x], j & 1, kWait);
                                tc::fence_after_thread_sync();
                                if (ok) next_scores(false);
                                if (!ok) continue;
                            }
                            ok = (p0 || mbar_wait_bounded(&ctl->p_ready[x][0], j & 1, kWait)) &&
                                 (vf || mbar_wait_bounded(unit_full(v), unit_parity(v), kWait));
                            if (!ok) continue;
                            tc::fence_after_thread_sync();
                            const bool p1 = test(&ctl->p_ready[x][1], j & 1);
                            values(x, v, 0, j > 0 ? 1u : 0u);
                            ok = p1 || mbar_wait_bounded(&ctl->p_ready[x][1], j & 1, kWait);
                            if (!ok) continue;
                            tc::fence_after_thread_sync();
                            const bool kf = !L::kAhead && next && test(unit_full(k), unit_parity(k));
                            // of the event that comes next: the other row tile's where it has one
                            const bool other = R == 2 && (x == 0 ? j < t1 : j + 1 < t0);
                            values(x, v, 1, 1);
                            if (last_use) tc::commit(&ctl->empty[v % L::kUnits]);
                            if (L::kAhead || !next) tc::commit(&ctl->o_done[x]);
                            p0 = test(&ctl->p_ready[other ? x ^ 1 : x][0], (x == 0 && other ? j : j + 1) & 1);
                            vf = x == 0 && other ? true : test(unit_full(v + 2), unit_parity(v + 2));
                            if (!L::kAhead && next) next_scores(kf);
                        }
                    }
                    if (!ok) {
                        record_error(kErrPackedBarrierTimeout);
                        ctl->failed = 1;
                    }
                }
                __syncwarp();
            } else {
                const int n = uniform(n_tiles);
                if (tc::elect_one()) {
                    auto issue_scores = [&](int e, bool early) {
                        const int u = k_unit(e);
#pragma unroll
                        for (int h = 0; h < L::kHalves; ++h) {
                            ok = ok && (early || mbar_wait_bounded(unit_full(u + h), unit_parity(u + h), kWait));
                            if (!ok) return;
                            early = test(unit_full(u + 1), unit_parity(u + 1));
                            scores(e & 1, u + h, h);
                            tc::commit(&ctl->empty[(u + h) % L::kUnits]);
                        }
                        tc::commit(&ctl->s_ready[e & 1]);
                    };
                    issue_scores(0, false);
                    if (n > 1) issue_scores(1, false);
                    bool p0 = false;
                    for (int e = 0; e < n && ok; ++e) {
                        const int v = L::kHalves * (e == n - 1 ? 2 * e + 1 : 2 * e + 2), x = e & 1;
                        const uint32_t phase = (e >> 1) & 1;
                        const bool v0 = test(unit_full(v), unit_parity(v)), v1 = test(unit_full(v + 1), unit_parity(v + 1));
                        ok = (p0 || mbar_wait_bounded(&ctl->p_ready[x][0], phase, kWait)) && (v0 || mbar_wait_bounded(unit_full(v), unit_parity(v), kWait)) &&
                             (v1 || mbar_wait_bounded(unit_full(v + 1), unit_parity(v + 1), kWait));
                        if (!ok) break;
                        tc::fence_after_thread_sync();
                        const bool p1 = test(&ctl->p_ready[x][1], phase);
                        values(x, v, 0, e > 0 ? 1u : 0u);
                        ok = p1 || mbar_wait_bounded(&ctl->p_ready[x][1], phase, kWait);
                        if (!ok) break;
                        tc::fence_after_thread_sync();
                        const bool next = e + 2 < n, kf = next && test(unit_full(k_unit(e + 2)), unit_parity(k_unit(e + 2)));
                        values(x, v, 1, 1);
                        tc::commit(&ctl->empty[v % L::kUnits]);
                        tc::commit(&ctl->empty[(v + 1) % L::kUnits]);
                        tc::commit(&ctl->o_done[x]);
                        p0 = test(&ctl->p_ready[x ^ 1][0], ((e + 1) >> 1) & 1);
                        if (next) issue_scores(e + 2, kf);
                    }
                    if (!ok) {
                        record_error(kErrPackedBarrierTimeout);
                        ctl->failed = 1;
                    }
                }
                __syncwarp();
            }
        } else if (warp >= 2) {
            // -------------------------------------------------------- V of tiles with masked pairs
            // Rows behind the sequence's end to zero, infinities and NaN out of the product.  x * 0 summed up is NaN if there is one.
            for (int j = kWindow && left_begin < left_end ? left_begin : first_masked; j < n_tiles; ++j) {
                if (kWindow && !looked_over(j)) continue;
                const int u0 = v_unit(j);
                bool ok = wait_warp(&ctl->v_landed[place(j)], 0);
                for (int r = (warp - 2) * 32 + lane; r < kTile && ok; r += 64) {
                    const bool there = real(j * kTile + r) < nk;
                    bool bad = false;
                    for (int h = 0; h < L::kHalves; ++h) {
                        for (int b = 0; b < L::kUnitBlocks; ++b) {
                            uint4* at = reinterpret_cast<uint4*>(ring + (u0 + h) % L::kUnits * L::kUnitBytes + b * kBlockBytes + r * 128);
                            uint4 v[8];
                            uint32_t sum[4] = {0, 0, 0, 0};          // four chains: the check is in the way of short sequences
#pragma unroll
                            for (int c = 0; c < 8; ++c) v[c] = at[c ^ (r & 7)];
#pragma unroll
                            for (int c = 0; c < 8; ++c) {
                                sum[0] = Half16<T>::add_zeros(v[c].x, sum[0]);
                                sum[1] = Half16<T>::add_zeros(v[c].y, sum[1]);
                                sum[2] = Half16<T>::add_zeros(v[c].z, sum[2]);
                                sum[3] = Half16<T>::add_zeros(v[c].w, sum[3]);
                            }
                            if (!there) {
#pragma unroll
                                for (int c = 0; c < 8; ++c) at[c] = make_uint4(0, 0, 0, 0);
                            } else if (((sum[0] | sum[1] | sum[2] | sum[3]) & 0x7fff7fffu) != 0) {
                                bad = true;
                                uint16_t* x = reinterpret_cast<uint16_t*>(at);
                                constexpr uint16_t kExp = std::is_same<T, __nv_bfloat16>::value ? 0x7f80 : 0x7c00;
                                for (int i = 0; i < 64; ++i) {
                                    if ((x[i] & kExp) == kExp) x[i] = 0;
                                }
                            }
                        }
                    }
                    const uint32_t word = __ballot_sync(0xffffffffu, bad);
                    if (lane == 0 && word != 0) {
                        ctl->bad[place(j)][r >> 5] = word;
                        ctl->bad_any = 1;
                    }
                }
                fence_proxy_async_smem();
                if (!meet_and(ok)) {     // both warps leave; the units stay empty, and the products' wait runs out too
                    if (lane == 0) {
                        record_error(kErrPackedBarrierTimeout);
                        ctl->failed = 1;
                    }
                    break;
                }
                if (warp == 2 && lane < L::kHalves) mbar_arrive(&ctl->full[(u0 + lane) % L::kUnits]);
            }
        }
    } else {
        // ------------------------------------------------------------ softmax: group x, thread = row of a tile
        more_registers<L::kManyRegs>();
        const int x = (warp >> 2) - 1;
        const int quarter = warp & 3, row = quarter * 32 + lane;
        const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
        const uint32_t s_at = lanes + x * kTile, p_at = lanes + L::kColP + x * L::kStepP, o_at = lanes + L::kColO + (L::kOwn ? x * DP : 0);
        const int my_tile = L::kOwn ? x : 0;
        const int token = token0 + my_tile * tokens_tile + (row >> P.pack_shift);
        const int limit = token < nq ? row_limit(P, nq, nk, token) - gap : 0;
        const int lowest = row_limit(P, nq, nk, token0 + my_tile * tokens_tile) - gap;       // of the tile's rows that exist
        // of the tile's rows that exist: behind the last key that the window hides from one
        const int behind = kWindow ? row_limit(P, nq, nk, min(token0 + (my_tile + 1) * tokens_tile, nq) - 1) - gap - P.window : 0;
        float ref = -INFINITY, l = 0.0f;
        float l_ref = -INFINITY;         // the reference that l is relative to (one row tile: the groups share ref)
        bool ok = true;
        for (int e = x; e < events; e += 2) {
            if (!active(e)) break;
            const int j = key_tile(e);
            if (!wait_warp(&ctl->s_ready[x], (e >> 1) & 1)) { ok = false; break; }
            tc::fence_after_thread_sync();
            const int key0 = j * kTile;
            const bool masked = key0 + kTile > lowest || (kWindow && key0 < behind && key0 + kTile > P.sinks);
            const int lim = limit - key0;
            uint32_t s[kTile];
            float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < kTile; c += 32) tc::tmem_ld_32x32b_x32(s_at + c, *reinterpret_cast<uint32_t(*)[32]>(s + c));
#pragma unroll
            for (int c = 0; c < kTile; c += 32) tmem_ld_wait_for(s + c);
            if (L::kAhead) {
                tc::fence_before_thread_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctl->s_read[x]);
            }
            if (masked) {
#pragma unroll
                for (int c = 0; c < kTile; c += 32) {    // a bit per column that is seen
                    uint32_t sees = lim >= c + 32 ? 0xffffffffu : (lim > c ? (1u << (lim - c)) - 1 : 0u);
                    if (kWindow) {                       // but not [sinks, limit - window)
                        const int from = min(max(P.sinks - key0 - c, 0), 32), to = min(max(lim - P.window - c, 0), 32);
                        const uint32_t below_to = to == 32 ? 0xffffffffu : (1u << to) - 1, below_from = from == 32 ? 0xffffffffu : (1u << from) - 1;
                        sees &= ~(below_to & ~below_from);
                    }
#pragma unroll
                    for (int i = 0; i < 32; ++i) s[c + i] = (sees >> i) & 1 ? s[c + i] : 0xff800000u;
                }
            }
#pragma unroll
            for (int i = 0; i < kTile; i += 2) top[(i >> 1) & 3] = max3(top[(i >> 1) & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
            const float high = max3(fmaxf(top[0], top[1]), top[2], top[3]) * P.scale2;
            if (!L::kOwn && e > 0) {     // the reference after the event before, from the other group
                if (!wait_warp(&ctl->ref_ready[x ^ 1][quarter], ((e - 1) >> 1) & 1)) { ok = false; break; }
                ref = ctl->ref[row];
            }
            const bool raise = high > ref + kRaise || (ref == -INFINITY && high > ref);
            const float now = raise ? high : ref;
            if (!L::kOwn) {
                ctl->ref[row] = now;
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctl->ref_ready[x][quarter]);
            }
            if (L::kAhead && e >= 2) {       // the last product into this O, which reads what P is written over
                if (!wait_warp(&ctl->o_done[x], ((e >> 1) - 1) & 1)) { ok = false; break; }
                tc::fence_after_thread_sync();
            }
            if (__any_sync(0xffffffffu, raise) && e >= (L::kOwn ? 2 : 1)) {
                // the last product into this O: where P lies in S's columns it was issued before these scores, and is complete
                if (!L::kOwn && !wait_warp(&ctl->o_done[x ^ 1], ((e - 1) >> 1) & 1)) { ok = false; break; }
                tc::fence_after_thread_sync();
                const float f = raise ? ex2(ref - now) : 1.0f;
                for (int c = 0; c < DP; c += 32) {
                    uint32_t o[32];
                    tc::tmem_ld_32x32b_x32(o_at + c, o);
                    tc::tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                    tmem_st_x32(o_at + c, o);
                }
                tmem_st_done();
            }
            ref = now;
            const float base = ref == -INFINITY ? 0.0f : ref;
            if (l_ref != ref) {
                l *= ex2(l_ref - base);
                l_ref = ref;
            }
            // P = 2^(scale2 S - m), its row sum (before rounding), rounded pairs into the columns S was in
            const uint64_t scale = pair(P.scale2, P.scale2), minus = pair(Half16<T>::kLift - base, Half16<T>::kLift - base);
            uint64_t sum[2] = {pair(0.0f, 0.0f), pair(0.0f, 0.0f)};
            if (__builtin_expect(__reduce_max_sync(0xffffffffu, __float_as_uint(fabsf(base))) > __float_as_uint(kFar), 0)) {
                // scores rounded as their reference was; the other rows' stay what they are.  (In local memory, a few at a time: in place the other
                // branch kept fewer registers, and the ragged prompts took 27.3 us.)
                float y[kTile];
                const float up = Half16<T>::kLift - base;
#pragma unroll
                for (int i = 0; i < kTile; ++i) {
                    const float z = __uint_as_float(s[i]);
                    y[i] = fabsf(base) > kFar ? __fadd_rn(__fmul_rn(z, P.scale2), up) : fmaf(z, P.scale2, up);
                }
#pragma unroll 1
                for (int c = 0; c < kTile / 2; c += 8) {
                    uint32_t p[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float a = ex2(y[2 * (c + i)]), b = ex2(y[2 * (c + i) + 1]);
                        sum[i & 1] = add2(sum[i & 1], pair(a, b));
                        p[i] = Half16<T>::pack(a, b);
                    }
                    tmem_st_x8(p_at + c, p);
                    tmem_st_done();
                    if (c % 32 != 24) continue;
                    tc::fence_before_thread_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&ctl->p_ready[x][c / 32]);
                }
            } else {
#pragma unroll
                for (int c = 0; c < kTile / 2; c += 32) {
                    uint32_t p[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        float a, b;
                        unpair(fma2(pair(__uint_as_float(s[2 * (c + i)]), __uint_as_float(s[2 * (c + i) + 1])), scale, minus), a, b);
                        a = ex2(a);
                        b = ex2(b);
                        sum[i & 1] = add2(sum[i & 1], pair(a, b));
                        p[i] = Half16<T>::pack(a, b);
                    }
                    tmem_st_x32(p_at + c, p);
                    tmem_st_done();
                    tc::fence_before_thread_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&ctl->p_ready[x][c / 32]);
                }
            }
            float a, b;
            unpair(add2(sum[0], sum[1]), a, b);
            l += a + b;
        }
        // ------------------------------------------------------------ O / l -> the rows
        if (!L::kOwn) {
            ctl->part_l[x][row] = l;
            ctl->part_m[x][row] = l_ref;
            asm volatile("bar.sync 1, 256;" ::: "memory");
            const float m = fmaxf(ctl->part_m[0][row], ctl->part_m[1][row]), base = m == -INFINITY ? 0.0f : m;
            l = ctl->part_l[0][row] * ex2(ctl->part_m[0][row] - base) + ctl->part_l[1][row] * ex2(ctl->part_m[1][row] - base);
        }
        const int mine = L::kOwn ? tiles[x] : tiles[0];
        if (ok && mine > 0) {
            if (!wait_warp(&ctl->o_done[L::kOwn ? x : (mine - 1) & 1], L::kAhead ? (mine - 1) & 1 : (L::kOwn ? 0 : ((mine - 1) >> 1) & 1))) ok = false;
            tc::fence_after_thread_sync();
        }
        // rows that see no key while the CTA's other row tile does: their queries may still be on the way to where the output is staged
        if (ok && mine == 0 && n_tiles > 0) ok = wait_warp(&ctl->q_full, 0);
        if (!ok && lane == 0) {
            record_error(kErrPackedBarrierTimeout);
            ctl->failed = 1;
        }
        if (ok) {
            const float inv = mine > 0 ? 1.0f / l : 0.0f;
            // through shared memory where Q was (its products are done), each warp its own rows, so that whole rows leave together
            constexpr int kCols = L::kOwn ? DP : DP / 2, kChunks = kCols / 8, kRowsIter = 32 / kChunks, kSwap = 7;
            const int c_lo = L::kOwn ? 0 : x * kCols;
            uint8_t* stage = sQ + (x * 4 + quarter) * 32 * kCols * 2;
            const bool any_bad = mine > 0 && ctl->bad_any != 0;
#pragma unroll 1
            for (int c = 0; c < kCols; c += 32) {
                uint32_t o[32];
                if (mine > 0) {
                    tc::tmem_ld_32x32b_x32(o_at + c_lo + c, o);
                    tc::tmem_ld_wait();
                }
                if (any_bad && token < nq) {             // what was taken out of V, for the rows that see it
                    for (int i = 0; i < (kWindow ? 2 : 1) * kBadTiles * kTile; ++i) {
                        const int key = tile_at(i / kTile) * kTile + i % kTile;
                        if (!((ctl->bad[i >> 7][(i >> 5) & 3] >> (i & 31)) & 1) || key >= limit) continue;
                        if (kWindow && key >= P.sinks && key < limit - P.window) continue;
                        const uint16_t* from = P.v_rows + static_cast<long long>(k0 + real(key)) * P.v_stride[0] +
                                               head_group / P.groups_per_kv * P.v_stride[1];
#pragma unroll
                        for (int n = 0; n < 32; ++n) {
                            if (c_lo + c + n >= P.head_dim) continue;
                            const uint32_t w = from[c_lo + c + n];
                            const float v = Half16<T>::unpack(w).x;
                            if (!(fabsf(v) < INFINITY)) o[n] = __float_as_uint(__uint_as_float(o[n]) + v);
                        }
                    }
                }
#pragma unroll
                for (int n = 0; n < 32; n += 8) {
                    uint32_t w[4] = {0, 0, 0, 0};
                    if (limit > 0) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            w[i] = Half16<T>::pack(__uint_as_float(o[n + 2 * i]) * inv, __uint_as_float(o[n + 2 * i + 1]) * inv);
                        }
                    }
                    *reinterpret_cast<uint4*>(stage + lane * (kCols * 2) + ((((c + n) >> 3) ^ (lane & kSwap)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            __syncwarp();
            // kRowsIter rows at a time: they are heads of one token, or whole tokens, so a lane's offset stays and the step's is uniform
            const int chunk = lane % kChunks, lane_row = lane / kChunks, first_row = quarter * 32, mask = P.pack - 1;
            uint16_t* to = P.out + static_cast<long long>(q0 + token0 + my_tile * tokens_tile + ((first_row + lane_row) >> P.pack_shift)) * P.o_stride[0] +
                           ((head_group << P.pack_shift) + ((first_row + lane_row) & mask)) * P.o_stride[1] + c_lo + chunk * 8;
            const int rows_left = ((nq - token0 - my_tile * tokens_tile) << P.pack_shift) - first_row;       // of this warp that exist
            const uint8_t* from = stage + lane_row * (kCols * 2);
            const bool column = c_lo + chunk * 8 < P.head_dim;
#pragma unroll 4
            for (int r0 = 0; r0 < 32; r0 += kRowsIter) {
                const int r = r0 + lane_row;
                const uint4 v = *reinterpret_cast<const uint4*>(from + r0 * (kCols * 2) + ((chunk ^ (r & kSwap)) << 4));
                if (r < rows_left && column) {
                    const int row0 = first_row + r0, token_step = (row0 >> P.pack_shift) - (first_row >> P.pack_shift), head_step = (row0 & mask) - (first_row & mask);
                    *reinterpret_cast<uint4*>(to + token_step * P.o_stride[0] + head_step * P.o_stride[1]) = v;
                }
            }
        }
        tc::fence_before_thread_sync();
    }
    __syncthreads();
    if (ctl->failed) {                   // copies may still be on their way into this CTA's shared memory
        const long long start = clock64();
        while (clock64() - start < 2000000) {}
        __syncthreads();
    }
    tc::fence_after_thread_sync();
    if (warp == 2) tc::tmem_dealloc(tmem, L::kTmemCols);
}

template <typename T, int DP, int R, bool kWindow>
int launch_packed(const PackedParams& P, unsigned blocks, cudaStream_t stream) {
    constexpr int smem = packed_smem<DP, R>();
    static_assert(Layout<DP, R>::kCtas * (smem + 1024) <= 228 * 1024, "shared memory of an SM");
    static std::atomic<uint64_t> configured{0};
    int dev = 0;
    cudaGetDevice(&dev);
    const uint64_t bit = 1ull << (dev & 63);
    if (!(configured.load(std::memory_order_relaxed) & bit)) {
        if (cudaFuncSetAttribute(packed_attention_kernel<T, DP, R, kWindow>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) {
            return TPB200_ERR_CUDA;
        }
        configured.fetch_or(bit, std::memory_order_relaxed);
    }
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = paged_config(blocks, Layout<DP, R>::kThreads, smem, &attr, stream);
    return cudaLaunchKernelEx(&cfg, packed_attention_kernel<T, DP, R, kWindow>, P) == cudaSuccess ? TPB200_OK : TPB200_ERR_CUDA;
}

// [tokens][heads][head_dim] with element strides, boxes of 64 columns x `heads` x `rows` tokens
bool rows_map(CUtensorMap* map, const void* base, int head_dim, int heads, long long head_stride, int tokens, long long token_stride,
              int box_heads, int box_tokens) {
    const uint64_t dims[3] = {static_cast<uint64_t>(head_dim), static_cast<uint64_t>(heads), static_cast<uint64_t>(tokens)};
    const uint64_t strides[2] = {static_cast<uint64_t>(heads > 1 ? head_stride : head_dim) * 2,
                                 static_cast<uint64_t>(tokens > 1 ? token_stride : static_cast<long long>(head_dim) * heads) * 2};
    const uint32_t box[3] = {64, static_cast<uint32_t>(box_heads), static_cast<uint32_t>(box_tokens)};
    return make_tensor_map_bf16_nd_sw128(map, base, 3, dims, strides, box);
}

}  // namespace

int device_error_packed_attention(int clear) { return read_device_error(clear); }

}  // namespace tpb

namespace tpb {
namespace {

// window 0: all keys up to a query's own
int attend(const tpb200_packed_attention_args* a, int window, int sinks, tpb200_stream_t stream) {
    TPB_REQUIRE(a != nullptr, TPB200_ERR_NULL);
    TPB_REQUIRE((a->flags & ~TPB200_FLAG_PDL) == 0, TPB200_ERR_ENUM);
    TPB_REQUIRE(a->dtype == TPB200_BF16 || a->dtype == TPB200_F16, TPB200_ERR_ENUM);
    TPB_REQUIRE(a->seqs >= 0 && a->q_tokens >= 0 && a->k_tokens >= 0, TPB200_ERR_SHAPE);
    TPB_REQUIRE(a->q_tokens <= kMaxTokens && a->k_tokens <= kMaxTokens, TPB200_ERR_SHAPE);
    TPB_REQUIRE(a->q_heads >= 1 && a->kv_heads >= 1 && a->q_heads % a->kv_heads == 0, TPB200_ERR_SHAPE);
    TPB_REQUIRE(a->head_dim >= 8 && a->head_dim <= 256 && a->head_dim % 8 == 0, TPB200_ERR_SHAPE);
    if (a->seqs == 0 || a->q_tokens == 0) return TPB200_OK;
    TPB_REQUIRE(a->q && a->out && a->cu && (a->k_tokens == 0 || (a->k && a->v)), TPB200_ERR_NULL);
    TPB_REQUIRE(tpb_aligned16(a->q) && tpb_aligned16(a->k) && tpb_aligned16(a->v) && tpb_aligned16(a->out), TPB200_ERR_ALIGN);
    PackedParams P = {};
    TPB_REQUIRE(std::isfinite(a->scale), TPB200_ERR_SHAPE);
    for (int i = 0; i < 2; ++i) {
        const int qn = i == 0 ? a->q_tokens : a->q_heads, kn = i == 0 ? a->k_tokens : a->kv_heads;
        for (const long long st : {a->q_stride[i], a->o_stride[i]}) TPB_REQUIRE(paged_stride(st, qn, a->head_dim) == TPB200_OK, paged_stride(st, qn, a->head_dim));
        for (const long long st : {a->k_stride[i], a->v_stride[i]}) TPB_REQUIRE(paged_stride(st, kn, a->head_dim) == TPB200_OK, paged_stride(st, kn, a->head_dim));
        P.o_stride[i] = qn > 1 ? a->o_stride[i] : 0;
        P.v_stride[i] = kn > 1 ? a->v_stride[i] : 0;
    }
    const int group = a->q_heads / a->kv_heads;
    int pack = 1;
    while (group % (2 * pack) == 0 && pack < 16) pack *= 2;
    for (int p = pack; p > 1; p /= 2) ++P.pack_shift;
    P.pack = pack;
    P.head_groups = a->q_heads / pack;
    P.groups_per_kv = group / pack;
    P.seqs = a->seqs;
    P.q_tokens = a->q_tokens;
    P.k_tokens = a->k_tokens;
    P.head_dim = a->head_dim;
    P.cu = a->cu;
    P.cu_keys = a->cu_keys != nullptr ? a->cu_keys : a->cu;
    P.out = static_cast<uint16_t*>(a->out);
    P.v_rows = static_cast<const uint16_t*>(a->v);
    P.causal = a->causal != 0;
    const bool hides = window > 0 && window < a->k_tokens;       // else no query has a key that it does not see
    P.window = window;
    P.sinks = std::min(sinks, a->k_tokens);
    // the sign of the scale goes into the product (operand A negated), its size into the exponent; none at all would lose the mask
    P.scale2 = fmaxf(fabsf(a->scale) * 1.4426950408889634f, 1.1754944e-38f);
    TPB_REQUIRE(std::isfinite(P.scale2), TPB200_ERR_SHAPE);
    // CTAs read keys and values while others write rows of the output
    const RowSet q_rows(a->q, a->q_stride, a->q_tokens, a->q_heads, a->head_dim), o_rows(a->out, a->o_stride, a->q_tokens, a->q_heads, a->head_dim);
    TPB_REQUIRE(output_fits(o_rows, q_rows), TPB200_ERR_SHAPE);
    TPB_REQUIRE(!rows_meet(o_rows, RowSet(a->k, a->k_stride, a->k_tokens, a->kv_heads, a->head_dim)) &&
                !rows_meet(o_rows, RowSet(a->v, a->v_stride, a->k_tokens, a->kv_heads, a->head_dim)), TPB200_ERR_SHAPE);
    const int DP = a->head_dim <= 64 ? 64 : (a->head_dim <= 128 ? 128 : 256);
    const bool bf = a->dtype == TPB200_BF16;
    // instruction descriptor: fp32 sums, A and B bf16 (1) or fp16 (0), [13] negate A, [16] B MN-major, N >> 3 at 17, M >> 4 at 24
    const uint32_t types = (1u << 4) | (bf ? (1u << 7) | (1u << 10) : 0u) | ((128u >> 4) << 24);
    P.idesc_s = types | (a->scale < 0.0f ? 1u << 13 : 0u) | ((128u >> 3) << 17);
    P.idesc_o = types | (1u << 16) | (static_cast<uint32_t>(DP >> 3) << 17);
    const int rows_tokens = kTile / pack;
    if (!rows_map(&P.q, a->q, a->head_dim, a->q_heads, a->q_stride[1], a->q_tokens, a->q_stride[0], pack, rows_tokens)) return TPB200_ERR_SHAPE;
    if (a->k_tokens > 0) {
        const int keys_box = hides ? kHalf : kTile;
        if (!rows_map(&P.k, a->k, a->head_dim, a->kv_heads, a->k_stride[1], a->k_tokens, a->k_stride[0], 1, keys_box) ||
            !rows_map(&P.v, a->v, a->head_dim, a->kv_heads, a->v_stride[1], a->k_tokens, a->v_stride[0], 1, keys_box)) {
            return TPB200_ERR_SHAPE;
        }
    }
    // Up to head size 128, two row tiles per CTA where sequences are long (each unit of K and V serves both), else one, and two CTAs on an
    // SM: half the rows to fill up, and one's loads and output beside the other's products.  The border is where the two meet on average:
    // 24 sequences of 100 / 8 of 1536, 16 heads of 64: 13.5 us with one, 18.1 with two / 91.6, 92.6; 16 heads of 128: 21.0, 25.2 / 129, 118.
    // Batches of sequences alike; not measured where lengths differ much or queries are few beside the keys.  With a window its keys count, and the border for
    // heads of 128 is 1000: windows of 200 / 400 / 800 / 1500, 4000 tokens, 32 on 8 heads, 95 / 106 / 138 / 194 us with one, 97 / 121 / 149 / 187 with two.
    // That holds for windows shorter than the prompts.  Longer ones, which hide nothing, take that border too: 24 prompts of 200 / 400 / 600 / 1000 tokens, 32
    // on 8 heads of 128, 52 / 101 / 160 / 327 us with a window of 4096, 51 / 100 / 157 / 305 without one; heads of 64 and 256 1 to 5 % more.
    const long long keys = hides ? std::min<long long>(a->k_tokens, (static_cast<long long>(window) + P.sinks) * a->seqs) : a->k_tokens;
    const bool two = DP <= 128 && keys > (DP == 64 || hides ? 1000ll : 200ll) * a->seqs;
    // no more tiles than whole ones and a ragged one per sequence
    const long long tiles = static_cast<long long>(a->q_tokens) / (rows_tokens * (two ? 2 : 1)) + std::min(a->seqs, a->q_tokens);
    const long long blocks = tiles * P.head_groups;
    TPB_REQUIRE(blocks <= 0x7fffffff, TPB200_ERR_SHAPE);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const unsigned n = static_cast<unsigned>(blocks);
    auto launch = [&](auto type, auto windowed) {
        using T = decltype(type);
        constexpr bool W = decltype(windowed)::value;
        if (DP == 64) return two ? launch_packed<T, 64, 2, W>(P, n, s) : launch_packed<T, 64, 1, W>(P, n, s);
        if (DP == 128) return two ? launch_packed<T, 128, 2, W>(P, n, s) : launch_packed<T, 128, 1, W>(P, n, s);
        return launch_packed<T, 256, 1, W>(P, n, s);
    };
    if (hides) return bf ? launch(__nv_bfloat16(), std::true_type()) : launch(__half(), std::true_type());
    return bf ? launch(__nv_bfloat16(), std::false_type()) : launch(__half(), std::false_type());
}

}  // namespace
}  // namespace tpb

extern "C" int tpb200_packed_attention(const tpb200_packed_attention_args* a, tpb200_stream_t stream) { return tpb::attend(a, 0, 0, stream); }

extern "C" int tpb200_packed_attention_window(const tpb200_packed_attention_args* a, int window, int sinks, tpb200_stream_t stream) {
    TPB_REQUIRE(a != nullptr, TPB200_ERR_NULL);
    TPB_REQUIRE(window >= 1 && sinks >= 0 && a->causal, TPB200_ERR_SHAPE);
    return tpb::attend(a, window, sinks, stream);
}
