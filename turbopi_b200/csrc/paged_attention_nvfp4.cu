// Attention of one new token per sequence on a cache of pages held in 4 bits (E2M1 values with an E4M3 scale for every 16), over all keys or over
// a window and the first few: softmax(scale q K^T) V with K = k_scale s c, V = v_scale s c.
//
// As on 16 bits the keys of all items are one line, cut into pieces of equal cost for the warps of a full machine (paged_decode.cuh), and S^T = K Q^T, O^T = V^T P^T run on
// mma.sync with the keys, and the columns of V, on its 16-row side.  But there are 3.6 times fewer bytes for the same products, so that not the
// stream but the issue of the dequantisation bounds it: one conversion and one product with the scale for two values of either, besides 32 products for 16
// keys of 256.  c s is exact in fp16, so nothing is lost there.  What keeps the rest small:
//   * a slot holds keys and their values (64, 32, 32 keys for head sizes up to 64, 128, 256), so that scores never leave the registers of a pass;
//   * a lane's codes are whole groups of 32 values (first product) or DP / 8 neighbouring columns (second): wide loads, one scale conversion per group, since
//     neither product minds the order of its inner or outer dimension;
//   * page ids are looked up for up to 32 tiles at once, a lane each; a lane's addresses in a slot are constants.
//
// Inside a piece (two lengths of one long sequence compared): heads of 256 470 warp instructions for 16 keys, 5.8 TB/s = 0.89 of the measured copy rate; of 128 574 for
// 32, 5.3; of 64 667 for 64, 4.8.  Around it: 2.3 us until a warp knows its piece, 2 until its first slot is there, warps of an SM that end up to a third
// apart, 4-5 us for the second kernel.  Calls in a CUDA graph: 96 sequences of 1 to 8192, 32 on 8 of 128, bf16 (111 MB) 35.3 us = 3.1 TB/s; 5 of 60 to 131 k, 8 on 1 of 256,
// fp16 (124 MB) 34.2 = 3.6; 64 of up to 12,000 under a window of 2048, 16 on 16 of 64 (116 MB) 38.6 = 3.0; one of 762 keys 10.5.  (On 16 bits the first would
// have 394 MB to read.)
#include "paged_decode.cuh"

namespace tpb {
namespace {

// A slot's keys, and its values, in shared memory: rows of DP / 2 bytes of codes, in 128-byte lines whose 16-byte chunks are exchanged so that the
// eight lanes of a phase meet all banks, whether they read two rows (keys) or a column of chunks (values).  Behind the codes of both lie the scales
// of the tiles of keys, then of values: DP bytes a tile, rows of 2 groups.
template <int DP>
constexpr int kKeysOf = Shape<Nvfp4, DP, 1>::kKeys;
template <int DP>
constexpr int kCodesOf = kKeysOf<DP> * DP / 2;           // bytes of a slot's keys, and of its values
template <int DP>
constexpr int kScalesOf = kKeysOf<DP> * DP / 16;
template <int DP>
__device__ __forceinline__ uint32_t code_at(int row, int chunk) {
    constexpr int kPerLine = 256 / DP;                   // rows of a line: 1, 2, 4
    const int line = row / kPerLine, c = row % kPerLine * (DP / 32) + chunk;
    const int turn = DP == 256 ? ((row >> 1) & 3) * 2 ^ (row & 1) * 4 : (DP == 128 ? (line & 3) * 2 : (line & 1) * 2);
    return line * 128 + ((c ^ turn) << 4);
}
// The order of a row's values in the products with the queries is free.  A lane (of four) takes whole groups of 32 values, for DP = 64 a block of 16;
// step kk of 16 takes four of each lane's.
template <int DP>
__device__ __forceinline__ int query_column(int kk, int t) {
    return DP == 64 ? t * 16 + kk * 4 : (t + (kk >> 3) * 4) * 32 + (kk & 7) * 4;
}
__device__ __forceinline__ __half2 e4m3_pair(uint32_t two) {
    __half2_raw r;
    asm("{\n .reg .b32 t;\n cvt.rn.f16x2.e4m3x2 t, %2;\n mov.b32 {%0, %1}, t;\n}\n" : "=h"(r.x), "=h"(r.y) : "h"(static_cast<uint16_t>(two)));
    return r;
}
__device__ __forceinline__ uint32_t bits_of(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }

template <int kBytes>
__device__ __forceinline__ void lds(uint32_t (&w)[kBytes / 4 > 0 ? kBytes / 4 : 1], uint32_t at) {
    if constexpr (kBytes == 16) asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
    else if constexpr (kBytes == 8) asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at) : "memory");
    else if constexpr (kBytes == 4) asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(at) : "memory");
    else if constexpr (kBytes == 2) {
        uint16_t x;
        asm volatile("ld.shared.b16 %0, [%1];" : "=h"(x) : "r"(at) : "memory");
        w[0] = x;
    } else asm volatile("ld.shared.u8 %0, [%1];" : "=r"(w[0]) : "r"(at) : "memory");
}

// Where a lane's codes and scales stand in a slot.  kFull: head_dim fills its 32 * groups and DP; else scales past a row's own are masked (the codes there
// are zeros, but 0 times a NaN would not be).
template <int DP, bool kFull>
struct Lane {
    static constexpr int kCodes = kCodesOf<DP>, kScales = kScalesOf<DP>;
    uint32_t k, v[2], ks, vs;            // keys lane / 4 of 8; values of keys 2 t and 2 t + 1; their scales
    uint32_t k_mask[2], v_mask;
    int row;                             // bytes of a row of scales
    __device__ __forceinline__ Lane(int lane, int groups) {
        const int g = lane >> 2, t = lane & 3;
        row = kFull ? DP / 16 : 2 * groups;
        k = code_at<DP>(g, DP == 64 ? t >> 1 : t) + (DP == 64 ? (t & 1) * 8 : 0);
        ks = 2 * kCodes + g * row + (DP == 64 ? t : 2 * t);
        const int block = DP == 256 ? 2 * g : (DP == 128 ? g : g >> 1);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            v[i] = kCodes + (DP == 256 ? code_at<DP>(2 * t + i, g) : (DP == 128 ? code_at<DP>(2 * t + i, g >> 1) + (g & 1) * 8 : code_at<DP>(2 * t + i, g >> 2) + (g & 3) * 4));
            k_mask[i] = kFull || (DP == 64 ? t < row : 2 * (t + 4 * i) < row) ? 0xffffu : 0u;
        }
        vs = 2 * kCodes + kScales + 2 * t * row + block;
        v_mask = kFull || block < row ? 0xffffu : 0u;
    }
};

// S^T = K Q^T of a slot: sc[16-key block][tile of heads].  Per 32 values of a row: 16 conversions and 16 products with the scale, exact in fp16.
template <int DP, int NT, int kBlocks, bool kFull>
__device__ __forceinline__ void scores4(float (&sc)[kBlocks][NT][4], uint32_t slot, const Lane<DP, kFull>& of, const uint32_t (&qf)[DP / 16][NT][2]) {
    constexpr int kRuns = DP == 256 ? 2 : 1;             // of 32 values, or of 16 (DP = 64), that a lane has of a row
    constexpr int kWords = DP == 64 ? 2 : 4;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) sc[b][n][j] = 0.0f;
    }
    const uint32_t k_at = slot + of.k, s_at = slot + of.ks;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
        for (int run = 0; run < kRuns; ++run) {
            uint32_t w[2][kWords];
            __half2 scale[2][2];                         // [row][block of 16]: the scale twice
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                // chunk t + 4 of a row of eight stands where chunk t would with bit 2 of its place turned
                lds<4 * kWords>(w[r], (run == 0 ? k_at : k_at ^ 64u) + b * 8 * DP + r * 4 * DP);
                uint32_t two[1];
                lds<DP == 64 ? 1 : 2>(two, s_at + b * DP + r * 8 * of.row + run * 8);
                if (!kFull) two[0] &= of.k_mask[run];
                const __half2 f = e4m3_pair(two[0]);
                scale[r][0] = __low2half2(f);
                scale[r][1] = DP == 64 ? scale[r][0] : __high2half2(f);
            }
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                __half2 x[2][4];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    decode_e2m1x8(w[r][i], x[r]);
#pragma unroll
                    for (int c = 0; c < 4; ++c) x[r][c] = __hmul2(x[r][c], scale[r][i / 2]);
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t a[4] = {bits_of(x[0][2 * j]), bits_of(x[1][2 * j]), bits_of(x[0][2 * j + 1]), bits_of(x[1][2 * j + 1])};
                    const int kk = run * 8 + i * 2 + j;
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma16816<__half>(sc[b][n], a, qf[kk][n][0], qf[kk][n][1]);
                }
            }
        }
    }
}

// O^T += V^T P^T of a slot.  The product wants neighbouring keys in a register: the halves of two keys' bytes are exchanged before they are
// converted, four instructions for 16 values, so that a conversion gives the same column of both, and a product applies both scales.  A lane has
// DP / 8 neighbouring columns of four keys out of 16.
template <int DP, int NT, int kBlocks, bool kFull>
__device__ __forceinline__ void values4(float (&o)[DP / 16][NT][4], uint32_t slot, const Lane<DP, kFull>& of, const uint32_t (&p)[kBlocks][NT][2]) {
    constexpr int kWords = DP / 64;                      // of 8 columns
    const uint32_t v_at[2] = {slot + of.v[0], slot + of.v[1]}, s_at = slot + of.vs;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
        uint32_t w[4][kWords], s[4][1];                  // keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            lds<4 * kWords>(w[k], v_at[k & 1] + b * 8 * DP + (k >> 1) * 4 * DP);
            lds<DP == 256 ? 2 : 1>(s[k], s_at + b * DP + ((k >> 1) * 8 + (k & 1)) * of.row);
        }
        __half2 scale[2][DP == 256 ? 2 : 1];             // of a pair of keys, per block of 16 columns
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            uint32_t low = __byte_perm(s[2 * k][0], s[2 * k + 1][0], 0x0040);
            if (!kFull) low &= of.v_mask;
            scale[k][0] = e4m3_pair(low);
            if constexpr (DP == 256) {
                uint32_t high = __byte_perm(s[2 * k][0], s[2 * k + 1][0], 0x0051);
                if (!kFull) high &= of.v_mask;
                scale[k][1] = e4m3_pair(high);
            }
        }
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            __half2 x[2][2][4];                          // [pair of keys][even, odd columns]
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint32_t a = w[2 * k][i], c = w[2 * k + 1][i];
                decode_e2m1x8((a & 0x0f0f0f0fu) | ((c << 4) & 0xf0f0f0f0u), x[k][0]);
                decode_e2m1x8(((a >> 4) & 0x0f0f0f0fu) | (c & 0xf0f0f0f0u), x[k][1]);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int n = 0; n < 4; ++n) x[k][j][n] = __hmul2(x[k][j][n], scale[k][DP == 256 ? i / 2 : 0]);
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const uint32_t a[4] = {bits_of(x[0][0][c]), bits_of(x[0][1][c]), bits_of(x[1][0][c]), bits_of(x[1][1][c])};
#pragma unroll
                for (int n = 0; n < NT; ++n) mma16816<__half>(o[i * 4 + c][n], a, p[b][n][0], p[b][n][1]);
            }
        }
    }
}

// One pass over a warp's piece of the line: per slot (32 or 64 keys, their tiles and those of their values) the scores, the running reference and
// sum of a softmax, and the product with the values.  Two slots are on their way while a third is worked on.  Page ids are looked up for up
// to 32 tiles at a time, a lane each, and asked for that long before they are needed.
template <typename T, int DP, int NT, bool kFull>
__device__ __forceinline__ void attend_tiles(const DecodeParams& P) {
    using Src = Nvfp4;
    using S = Shape<Src, DP, NT>;
    constexpr int kSlots = S::kSlots, kWarps = S::kWarps, kCodes = kCodesOf<DP>, kScales = kScalesOf<DP>;
    constexpr int kKeys = S::kKeys, kBlocks = kKeys / 16, kAhead = 32 / kBlocks;       // slots of a look-up
    static_assert(S::kSlotBytes == 2 * (kCodes + kScales) && (kBlocks == 2 || kBlocks == 4) && kSlots <= 8, "");
    extern __shared__ __align__(128) uint8_t smem[];
    auto* ctl = reinterpret_cast<Control<S>*>(smem + kWarps * kSlots * S::kSlotBytes);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int D = P.cache.head_dim, groups = kFull ? DP / 32 : (D + 31) / 32;
    Piece<Src, S, true> piece;
    if (!piece.find(P, ctl->lengths, warp, lane)) return;        // (the whole CTA)
    // Nobody waits for another here but for speed: a CTA's warps begin together.  96 ragged sequences 40.5 -> 36.3 us, 100 of about 400 26.3 -> 23.0;
    // why it helps where pieces are found at different times was not found out.
    __syncthreads();
    auto& work = piece.work;
    const auto& line = piece.line;
    const int slots = piece.slots, cta = blockIdx.x, worker = cta * kWarps + warp;
    const bool merged = piece.merged;

    // ------------------------------------------------ loads
    uint8_t* ring = smem + warp * kSlots * S::kSlotBytes;
    auto next = work;                    // the first slot that has not been looked up
    int unknown = slots;                 // slots from there on
    int page_id = -1;                    // of this lane's tile of the look-up that begins at `next`
    int known = 0, at = 0;               // slots of the look-up the loads take their tiles from, and which one is next
    long long tile_at = 0;               // this lane's tile of it: byte offset
    uint32_t here = 0;                   // tiles of it that are there and have a key that is seen; the others are not read
    uint32_t gone = 0;                   // tiles of it with a key that is seen, and without a page in the pool
    uint32_t absent = 0;                 // the same of the slots in the ring, four bits each
    auto ahead = [&]() { return min(unknown, min(kAhead, (next.n - next.ci + next.step - 1) / next.step)); };
    // the first key of this lane's tile, and whether one of its keys is seen
    auto own_tile = [&](int& key) {
        auto place = next;
        place.ci += lane / kBlocks * next.step;
        if (lane / kBlocks >= ahead()) return false;
        key = place.first_key(P) + lane % kBlocks * 16;
        return key < next.len && (key < P.sinks || static_cast<int>(min(key + 16u, static_cast<unsigned>(next.len))) > next.len - P.window);
    };
    auto ask_ids = [&]() {
        int key = 0;
        page_id = own_tile(key) ? P.cache.table[next.s * P.cache.table_stride + key / P.cache.page_size] : -1;
    };
    // the queries of an item into the first-level cache, a line a lane: they are read when its first slot is worked on, two slots later
    auto ask_queries = [&](const decltype(piece.work)& place) {
        constexpr int kLines = DP / 64;
        const int kvh = place.h / P.tiles, row0 = (place.h - kvh * P.tiles) * S::kRows;
        for (int i = lane; i < S::kRows * kLines; i += 32) {
            const int r = row0 + i / kLines, c = i % kLines * 64;
            if (r < P.group && c < D) {
                asm volatile("prefetch.global.L1 [%0];" ::"l"(P.q + place.s * P.q_stride[0] + (kvh * P.group + r) * P.q_stride[1] + c));
            }
        }
    };
    auto look_up = [&]() {               // the tiles from `next` on; page ids of those behind them are asked for
        int key = 0;
        const bool in = own_tile(key), there = in && static_cast<unsigned>(page_id) < static_cast<unsigned>(P.cache.num_pages);
        tile_at = 0;
        if (there) {
            tile_at = page_id * P.cache.page_stride + key % P.cache.page_size / 16 * P.cache.row_stride + next.h / P.tiles * P.cache.head_stride;
        }
        here = __ballot_sync(0xffffffffu, there);
        gone = __ballot_sync(0xffffffffu, in && !there);
        if (gone != 0) record_error(kErrPagedIndex);
        if (next.ci == 0) ask_queries(next);
        known = ahead();
        at = 0;
        unknown -= known;
        if (unknown > 0) {
            next.ci += (known - 1) * next.step;
            next.next(P, ctl->lengths);
            ask_ids();
        }
    };
    const int lane_row = lane / S::kLanesRow, lane_col = lane % S::kLanesRow;
    const int from_lane = lane_row * 16 * groups + lane_col * 16, step = S::kRowsIter * 16 * groups;
    const uint32_t to_lane = code_at<DP>(lane_row, lane_col);
    constexpr int kScaleLanes = kScales / 16, kScaleCopies = kScaleLanes / 16;         // copies of 16 bytes for the scales of the keys
    const int scale_tile = (lane & 15) / (DP / 16), scale_chunk = (lane & 15) % (DP / 16);
    static_assert(kScaleLanes % 16 == 0 && (DP / 16) <= 16, "");
    const uint8_t* k_pages = static_cast<const uint8_t*>(P.cache.k_pages);
    const uint8_t* v_pages = static_cast<const uint8_t*>(P.cache.v_pages);
    auto load_slot = [&](int slot) {
        if (at == known) look_up();
        const uint32_t to = smem_u32(ring) + slot * S::kSlotBytes;
        constexpr int kIters = kCodes / 512, kTileIters = kIters / kBlocks;
        static_assert(S::kRowsIter * kTileIters == 16, "");
        const uint32_t there = here >> (at * kBlocks);
        const uint8_t *k = k_pages, *v = v_pages;
        int bytes = 0;
#pragma unroll
        for (int i = 0; i < kIters; ++i) {
            if (i % kTileIters == 0) {
                const long long off = __shfl_sync(0xffffffffu, tile_at, at * kBlocks + i / kTileIters);
                bytes = (there >> (i / kTileIters)) & 1 && (kFull || lane_col < groups) ? 16 : 0;
                k = k_pages + off + (kFull || bytes > 0 ? from_lane : 0);
                v = v_pages + off + (kFull || bytes > 0 ? from_lane : 0);
            }
            // rows further on by kRowsIter stand in the same place of a later line: code_at repeats every eight rows
            const uint32_t row_at = S::kRowsIter % 8 == 0 ? to_lane + i * 512 : code_at<DP>(i * S::kRowsIter + lane_row, lane_col);
            const int on = i % kTileIters * (kFull || bytes > 0 ? step : 0);
            cp_async16(to + row_at, k + on, bytes);
            cp_async16(to + kCodes + row_at, v + on, bytes);
        }
#pragma unroll
        for (int i = 0; i < kScaleCopies; ++i) {         // lanes 0 to 15: of keys
            const int tile = i * (256 / DP) + scale_tile;
            const long long off = __shfl_sync(0xffffffffu, tile_at, at * kBlocks + tile);
            const bool in = (there >> tile) & 1 && (kFull || scale_chunk < 2 * groups);
            cp_async16(to + 2 * kCodes + (lane >> 4) * kScales + i * 256 + (lane & 15) * 16,
                       (lane < 16 ? k_pages : v_pages) + off + (kFull || in ? 256 * groups + scale_chunk * 16 : 0), in ? 16 : 0);
        }
        absent = (absent & ~(15u << (4 * slot))) | ((gone >> (at * kBlocks)) & ((1u << kBlocks) - 1)) << (4 * slot);
        ++at;
    };

    // ------------------------------------------------ queries
    uint32_t qf[DP / 16][NT][2];         // as the B operand, zero past the group and past head_dim
    float scale2[NT][2];                 // of the lane's two query heads of a tile
    float o[DP / 16][NT][4];             // O^T: columns of head_dim by query heads
    float m[NT][2], l[NT][2];            // reference and sum of the lane's two query heads of a tile; l over the lane's keys only
    auto clear = [&]() {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            m[t][0] = m[t][1] = -INFINITY;
            l[t][0] = l[t][1] = 0.0f;
#pragma unroll
            for (int i = 0; i < DP / 16; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[i][t][j] = 0.0f;
        }
    };
    auto start = [&]() {                 // an item's (or its piece's) beginning
        clear();
        const int kvh = work.h / P.tiles, row0 = (work.h - kvh * P.tiles) * S::kRows;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int r = row0 + t * 8 + (lane >> 2);
            const uint16_t* row = P.q + work.s * P.q_stride[0] + (kvh * P.group + r) * P.q_stride[1];
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk) {
                const int c = query_column<DP>(kk, lane & 3);
                const uint2 x = r < P.group && c < D ? __ldg(reinterpret_cast<const uint2*>(row + c)) : make_uint2(0, 0);
                qf[kk][t][0] = x.x;
                qf[kk][t][1] = x.y;
            }
            if (P.scale2 < 0.0f) {       // the sign goes into the queries: scores are compared before they are scaled
#pragma unroll
                for (int kk = 0; kk < DP / 16; ++kk) {
                    qf[kk][t][0] ^= 0x80008000u;
                    qf[kk][t][1] ^= 0x80008000u;
                }
            }
            constexpr float kLeast = 1.1754944e-38f;     // no scale at all would lose the mask
            const float size = fabsf(P.scale2);
            scale2[t][0] = scale2[t][1] = fmaxf(size, kLeast);
            if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                // fp16 queries are taken as they are; bf16 ones are divided by the power of two of their head's largest, which moves into the scale (a
                // query 2^-15 of the largest and below is rounded to a multiple of 2^-24 of it)
                uint32_t top = 0;
#pragma unroll
                for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
                    for (int j = 0; j < 2; ++j) top = max(top, max(qf[kk][t][j] & 0x7fffu, (qf[kk][t][j] >> 16) & 0x7fffu));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const int e = min(max(static_cast<int>(top >> 7), 1), 253);          // exponent field; 2^(127 - e) and its inverse are normal
                const float down = __uint_as_float((254u - e) << 23);
#pragma unroll
                for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float2 x = Half16<T>::unpack(qf[kk][t][j]);
                        qf[kk][t][j] = Half16<__half>::pack(x.x * down, x.y * down);
                    }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t power = static_cast<uint32_t>(__shfl_sync(0xffffffffu, e, ((lane & 3) * 2 + j) * 4)) << 23;
                    // a product past fp32 would make NaN of scores of 0; with the largest number in its place scores that are not 0 are still 2^90 and
                    // more apart, as they would be
                    scale2[t][j] = fminf(fmaxf(size * __uint_as_float(power), kLeast), FLT_MAX);
                }
            }
        }
    };

    const Lane<DP, kFull> of(lane, groups);
    int parts = 0;                       // partial results this warp has left
    bool far = false;                    // a reference whose rounding error is no small part of one
    const int first_ci = work.ci;
    bool from_start = first_ci == 0;
    if (slots > 0) ask_ids();
#pragma unroll
    for (int i = 0; i < kSlots - 1; ++i) {
        if (i < slots) load_slot(i);
        cp_async_commit();
    }
    if (slots > 0) start();
    else clear();
    int slot = 0;
#pragma unroll 1
    for (int i = 0; i < slots; ++i) {
        cp_async_wait<kSlots - 2>();
        __syncwarp();
        if (i + kSlots - 1 < slots) load_slot(slot == 0 ? kSlots - 1 : slot - 1);
        cp_async_commit();
        uint8_t* tiles = ring + slot * S::kSlotBytes;
        const uint32_t off = (absent >> (4 * slot)) & 15u;
        const int key0 = work.first_key(P), valid = work.len - key0;               // keys of the slot, at least one
        const int hidden = P.sinks - key0, shown = valid - P.window;               // [hidden, shown) are not seen
        const bool edge = valid < kKeys || (shown > 0 && hidden < kKeys && hidden < shown);
        float sc[kBlocks][NT][4];
        scores4<DP, NT>(sc, smem_u32(tiles), of, qf);
        // ---- a query head's scores lie in the lanes of equal lane % 4.  The reference is raised only when a score passes it by 8 (weights
        // stay below 2^8), so the maximum crosses the lanes hardly ever.  A slot with a key that is seen has a finite reference, whatever the
        // score: one of -infinity at the end means that there was no key.
        float lowest = kLowest;
        if (edge || off != 0) {
            bool any = false;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int key = b * 16 + (lane >> 2) + r * 8;
                    const bool seen = key < valid && !(key >= hidden && key < shown) && ((off >> b) & 1) == 0;
                    any = any || seen;
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        if (!seen) sc[b][n][2 * r] = sc[b][n][2 * r + 1] = -INFINITY;
                    }
                }
            if (!__any_sync(0xffffffffu, any)) lowest = -INFINITY;
            // a scale that is NaN would pass a weight of 0: none for values that are not seen
            for (int key = lane; key < kKeys; key += 32) {
                if (key < valid && !(key >= hidden && key < shown)) continue;
                uint16_t* of = reinterpret_cast<uint16_t*>(tiles + 2 * kCodes + kScales + key / 16 * DP) + key % 16 * groups;
                for (int c = 0; c < groups; ++c) of[c] = 0;
            }
            __syncwarp();
        }
        float top[NT][2];
        bool raise = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            top[n][0] = top[n][1] = -INFINITY;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
                for (int j = 0; j < 4; ++j) top[n][j & 1] = fmaxf(top[n][j & 1], sc[b][n][j]);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) top[n][j] = fmaxf(top[n][j] * scale2[n][j], lowest);
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
                    for (int d = 0; d < DP / 16; ++d) {
                        o[d][n][j] *= shrink;
                        o[d][n][j + 2] *= shrink;
                    }
                    l[n][j] *= shrink;
                    m[n][j] = now;
                }
            }
            far = false;
#pragma unroll
            for (int n = 0; n < NT; ++n) far = far || fabsf(m[n][0]) > kFar || fabsf(m[n][1]) > kFar;
            far = __any_sync(0xffffffffu, far);
        }
        // ---- weights, rounded to fp16 for the second product (their sum is that of the unrounded ones), transposed into its B operand
        uint32_t p[kBlocks][NT][2];
        auto exponents = [&](auto of_score) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float up[2] = {Half16<__half>::kLift - (m[n][0] == -INFINITY ? 0.0f : m[n][0]), Half16<__half>::kLift - (m[n][1] == -INFINITY ? 0.0f : m[n][1])};
#pragma unroll
                for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                    for (int j = 0; j < 4; ++j) sc[b][n][j] = of_score(sc[b][n][j], scale2[n][j & 1], up[j & 1], m[n][j & 1]);
            }
        };
        if (__builtin_expect(far, 0)) {  // scores rounded as their reference was; the other heads' stay what they are
            exponents([](float x, float f, float up, float ref) { return fabsf(ref) > kFar ? __fadd_rn(__fmul_rn(x, f), up) : fmaf(x, f, up); });
        } else {
            exponents([](float x, float f, float up, float) { return fmaf(x, f, up); });
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                float w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = ex2(sc[b][n][j]);
                l[n][0] += w[0] + w[2];
                l[n][1] += w[1] + w[3];
                p[b][n][0] = transpose8x8(Half16<__half>::pack(w[0], w[1]));
                p[b][n][1] = transpose8x8(Half16<__half>::pack(w[2], w[3]));
            }
        }
        values4<DP, NT>(o, smem_u32(tiles), of, p);
        slot = slot == kSlots - 1 ? 0 : slot + 1;
        const bool item_done = work.ci + work.step >= work.n, last = i == slots - 1;
        if (merged || (!item_done && !last)) {
            work.ci += work.step;
            continue;
        }
        // the slot just used is free until the next load
        __syncwarp();
        if (!store_item<Src, T, S, DP, NT>(P, work, line, reinterpret_cast<float*>(tiles), cta, worker, lane, parts, from_start, item_done, o, m, l)) ++parts;
        if (!last) {
            work.next(P, ctl->lengths);
            from_start = true;
            start();
        }
    }
    cp_async_wait<0>();
    if (!merged) return;
    merge_cta<Src, T, S, DP, NT>(P, work, line, smem, ctl->ml, cta, warp, lane, first_ci == 0, piece.whole_item, o, m, l);
}

template <typename T, int DP, int NT, bool kFull>
__global__ void __launch_bounds__(Shape<Nvfp4, DP, NT>::kThreads, Shape<Nvfp4, DP, NT>::kCtas) paged_attention_nvfp4_kernel(const __grid_constant__ DecodeParams P) {
    pdl_wait_prior_grids();
    pdl_launch_dependents();
    attend_tiles<T, DP, NT, kFull>(P);
}
template <typename T, int kLanes, int kLoads>
__global__ void __launch_bounds__(kJoinThreads) paged_attention_nvfp4_join_kernel(const __grid_constant__ DecodeParams P) {
    pdl_wait_prior_grids();
    pdl_launch_dependents();
    join_parts<Nvfp4, T, kLanes, kLoads>(P);
}

// query heads that go through together: eight, or sixteen where a group has more and their sums leave registers for the rest (head sizes up to 128);
// larger groups read the cache again, mostly out of L2.  38 MB of sequences of 8192, one key head, groups of 8 / 16: heads of 64 17 / 22 us, of 128 17 / 25, of 256
// 18.5 / 25.  Two tiles of heads of 128 have 56 to 168 bytes of spills at the 168 registers that three CTAs an SM leave; with two CTAs they were not timed.
int decode_rows4(int group, int head_dim) { return group <= 8 || head_dim > 128 ? 8 : 16; }

template <typename T, int DP, int NT>
int launch_tiles(const DecodeParams& P, int ctas, cudaStream_t stream) {
    return P.cache.head_dim == DP ? launch_decode<Nvfp4, DP, NT, paged_attention_nvfp4_kernel<T, DP, NT, true>>(P, ctas, stream)
                                  : launch_decode<Nvfp4, DP, NT, paged_attention_nvfp4_kernel<T, DP, NT, false>>(P, ctas, stream);
}
template <typename T>
int launch_tiles(const DecodeParams& P, int ctas, cudaStream_t stream) {
    const int D = P.cache.head_dim;
    if (D > 128) return launch_tiles<T, 256, 1>(P, ctas, stream);
    if (D > 64) return P.rows > 8 ? launch_tiles<T, 128, 2>(P, ctas, stream) : launch_tiles<T, 128, 1>(P, ctas, stream);
    return P.rows > 8 ? launch_tiles<T, 64, 2>(P, ctas, stream) : launch_tiles<T, 64, 1>(P, ctas, stream);
}
template <typename T>
int join_tiles(const DecodeParams& P, int ctas, cudaStream_t stream) {
    constexpr Kernel most = paged_attention_nvfp4_join_kernel<T, 32, 8>, many = paged_attention_nvfp4_join_kernel<T, 8, 8>, few = paged_attention_nvfp4_join_kernel<T, 2, 4>;
    if (!configure<most>(0, true) || !configure<many>(0, true) || !configure<few>(0, true)) return TPB200_ERR_CUDA;
    return launch_join(P, most, many, few, ctas, stream);
}
// CTAs of an SM: the same for one tile of query heads and for two
int ctas_per_sm4(int head_dim) { return head_dim > 128 ? Shape<Nvfp4, 256, 1>::kCtas : Shape<Nvfp4, 128, 1>::kCtas; }
static_assert(Shape<Nvfp4, 64, 1>::kCtas == Shape<Nvfp4, 128, 1>::kCtas, "");

}  // namespace

int device_error_paged_attention_nvfp4(int clear) { return read_device_error(clear); }

}  // namespace tpb

extern "C" size_t tpb200_paged_attention_nvfp4_workspace_size(int q_heads, int kv_heads, int head_dim) {
    using namespace tpb;
    if (q_heads < 1 || kv_heads < 1 || q_heads % kv_heads != 0 || head_dim < 8 || head_dim > 256) return 0;
    const int group = q_heads / kv_heads, rows = std::min(group, decode_rows4(group, head_dim));
    const int ctas = decode_ctas(ctas_per_sm4(head_dim));
    return ctas < 1 ? 0 : decode_scratch(static_cast<size_t>(ctas) * kCtaWarps, rows, head_dim).bytes;
}

extern "C" int tpb200_paged_attention_nvfp4(const tpb200_paged_attention_nvfp4_args* a, tpb200_stream_t stream) {
    using namespace tpb;
    TPB_REQUIRE(a != nullptr, TPB200_ERR_NULL);
    DecodeParams P = {};
    const int st = paged_view_nvfp4(a->cache, &P.cache);
    if (st != TPB200_OK) return st;
    TPB_REQUIRE(a->dtype == TPB200_BF16 || a->dtype == TPB200_F16, TPB200_ERR_ENUM);
    TPB_REQUIRE(a->window >= 0 && a->sinks >= 0 && (a->window > 0 || a->sinks == 0), TPB200_ERR_SHAPE);
    const DecodeCall call = {a->q, a->out, a->q_stride, a->o_stride, a->q_heads, a->scale, a->workspace, a->workspace_bytes, a->flags, a->window, a->sinks,
                             nvfp4_pool_bytes(P.cache)};
    const int D = P.cache.head_dim, group = a->q_heads / P.cache.kv_heads, rows = decode_rows4(group, D);
    const int ctas = decode_ctas(ctas_per_sm4(D));
    const int ready = prepare_decode(call, rows, D <= 64 ? kKeysOf<64> : (D <= 128 ? kKeysOf<128> : kKeysOf<256>), Nvfp4::kItemUnits, ctas, &P);
    if (ready != TPB200_OK || P.cache.seqs == 0) return ready;
    P.scale2 *= a->cache.k_scale;
    TPB_REQUIRE(std::isfinite(P.scale2), TPB200_ERR_SHAPE);
    P.out_scale = a->cache.v_scale;
    const bool bf = a->dtype == TPB200_BF16;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const int done = bf ? launch_tiles<__nv_bfloat16>(P, ctas, s) : launch_tiles<__half>(P, ctas, s);
    if (done != TPB200_OK) return done;
    return bf ? join_tiles<__nv_bfloat16>(P, ctas, s) : join_tiles<__half>(P, ctas, s);
}
