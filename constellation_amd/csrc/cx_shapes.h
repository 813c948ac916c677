// cx_shapes.h — which kernels a call takes and the scratch it needs, from its
// sizes alone.  Plain C++, so that the rules can be checked on the host over
// whole ranges of sizes.
//
// A context's scratch only grows, and growing frees the old buffer, which a
// captured graph may still use.  So what a call asks for covers every call of
// the same entry point and shape with fewer tokens, whatever kernels these take:
// a program that has run its largest call allocates no more, under capture too.
// Parts that belong together share one allocation: a context's first call pays
// for each.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

namespace cx {

// Geometry of the fast grouped kernels.
constexpr int kKB = 128;        // k-block: one scale per 128 columns
constexpr int kTileRows = 16;   // MFMA 16x16x32: 16 weight rows per wave
constexpr int kTileTok = 16;    // 16 token (pair) columns per MFMA tile

constexpr int kDecSplitMaxTokens = 8;  // tokens whose shared gate/up runs as k-parts (8 selection waves)

// The ABI states no alignment of x, and a view's rows may start anywhere.  Direct
// global->LDS loads and bounded buffer loads, 16 bytes a lane, are only given rows
// (and weights) that start on 16 bytes; all others go through plain loads, which
// take any address.
inline bool dma_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Activation rows of one work item that fit the LDS budget next to the
// reduction tile (<= 16 KB); 0 when staging is not worth it or not possible.
inline int lds_rows(int max_lds, int hidden, int max_pairs_per_item, bool x_dma) {
    if (!x_dma || hidden % 512 != 0) return 0;  // rows are copied in 1 KB wave chunks
    const int budget = std::min(max_lds, 65536) - 16384;
    const int rows = budget / (hidden * 2 + 16);
    return (max_pairs_per_item <= rows && max_pairs_per_item <= 4) ? max_pairs_per_item : 0;
}

// ---------------------------------------------------------------------------
// One expert over 1..4 tokens (split-K down launch).
constexpr int kDownKsRows = 4;    // tokens
constexpr int kDownKsGroups = 2;  // 16-row groups per workgroup

inline bool expert_small_shape(int hidden, int inter) {
    const int nkg = hidden / kKB, nkd = inter / kKB;
    return hidden % (kDownKsGroups * kTileRows) == 0 && (nkg == 56 || nkg == 8 || nkg == 4) && (nkd == 16 || nkd == 4);
}

// One expert over 5..64 tokens (single mode, cx_few.h): gate/up writes h in the
// order the down launch reads it, few_scratch_bytes of it.  The limits, one
// expert of 7168 x 2048, us a call: 1..4 tokens stay on the k-part launches,
// whose rows keep their bits whatever the batch (2 tokens 12.4 against 13.3, 4
// tokens 14.7 against 13.4); 5 tokens 23.7 / 13.5; 64 tokens 31.4 against 41.1
// with the ping-pong GEMM, 65 tokens 45.4 / 41.3.
constexpr int kFewMinTokens = 5, kFewMaxTokens = 64;
constexpr size_t kFewHBlk = 8192;  // h bytes of a 16-token tile and 128 columns: 2 planes x 4 steps x 1 KB
constexpr int kFewGuWaves = 8;     // waves of a gate/up workgroup

// LDS of a gate/up workgroup: a block of x, later a partial tile, per wave and tile.
constexpr int few_gu_lds(int tiles) { return kFewGuWaves * tiles * 4096; }

inline int few_tiles(int n_tokens) { return (n_tokens + kTileTok - 1) / kTileTok; }

// The most tokens whose LDS a workgroup of this device can have (32 with 64 KB).
inline int few_max_tokens(int max_lds) { return std::min(kFewMaxTokens, max_lds / few_gu_lds(1) * kTileTok); }

inline size_t few_scratch_bytes(int n_tokens, int inter) {
    return (size_t)few_tiles(n_tokens) * (inter / kKB) * kFewHBlk;
}

inline bool few_ok(int hidden, int inter, int n_tokens, int max_lds) {
    const int nkg = hidden / kKB, nkd = inter / kKB;
    return hidden % kKB == 0 && inter % kKB == 0 && (nkg == 56 || nkg == 8 || nkg == 4) && (nkd == 16 || nkd == 4) &&
           n_tokens >= kFewMinTokens && n_tokens <= few_max_tokens(max_lds);
}

// The ping-pong GEMM (cx_pp.h).
constexpr int kPpRowsGu = 128;  // inter rows (of gate and of up) per gate/up workgroup
constexpr int kPpRowsDn = 256;  // hidden rows per down workgroup
constexpr int kPpMinBlocks = 4;  // 128-column blocks of a row: the ring's last blocks are peeled off
constexpr int kPpLds = 160 * 1024;  // one workgroup per CU

inline bool pp_ok(int hidden, int inter, int max_lds) {
    return inter % kPpRowsGu == 0 && hidden % kPpRowsDn == 0 && hidden / kKB >= kPpMinBlocks &&
           inter / kKB >= kPpMinBlocks && max_lds >= kPpLds;
}

// Shapes with 64-pair grouped kernels of their own (cx_grouped.h).
inline bool grp_shape(int hidden, int inter) {
    const int nkg = hidden / kKB, nkd = inter / kKB;
    return hidden % kKB == 0 && inter % kKB == 0 && (nkg == 56 || nkg == 8 || nkg == 4) && (nkd == 16 || nkd == 4);
}

// A grouped call of at least this many pairs per resident expert, on average,
// takes 128-pair items through the ping-pong GEMM: there the matrix cores bound
// the work as much as HBM does, and 64-pair items stream an expert's weights once
// for each.  us a layer with 64 and with 128-pair items at 20 / 32 / 48 / 64 / 80 /
// 128 pairs per expert, 7168 x 2048 with the shared expert:
//   256 experts  2226 2524 3037 3917 4909 6704   2153 2354 2630 3154 3559 5357
//   64 experts   614 666 783 982 1243 1660       624 713 778 864 937 1406
//   64, none shared  535 598 708 904 1132 1514   523 569 622 741 816 1276
// The shared expert's items, all full, run last: where the others last for few
// rounds of the CUs, 128 pairs at the end cost more than fewer reads of the weights
// save, up to 63 pairs (8 experts, which fit one round, gain from 20: 121 / 105; 4
// gain up to 48, 121 / 117, and from 80, but lose between, 125 / 142 at 64).
// Rows of few blocks gain later, a ring's fill and drain being a larger part of an
// item, and the later the fewer the experts, as the halved count of items leaves CUs
// idle: 7168 x 512 (hidden x inter), 256 experts 683 765 908 1171 1488 2070 and 732
// 807 936 1048 1181 1728; 64 / 80 / 96 pairs of 1024 x 512, 64 experts 76 91 109 and
// 86 91 96, 16 experts 44 45 44 and 51 47 51.
constexpr int kBigPairs = 128;
inline int big_min_pairs(int hidden, int inter, int n_resident, bool shared, int n_cu) {
    if (!grp_shape(hidden, inter)) return 20;
    const int wgs = (n_resident + (shared ? 1 : 0)) * (inter / kPpRowsGu);  // gate/up, an item each
    if (hidden / kKB == 56 && inter / kKB == 16) return !shared || wgs <= n_cu || wgs >= 8 * n_cu ? 20 : 64;
    return n_resident >= 256 ? 64 : n_resident >= 32 ? 80 : kBigPairs;
}

// Kernels of one expert on the fast paths.  Above 16 tokens the 64-token items of
// the grouped kernels leave most CUs idle (16 gate/up workgroups at 17..64
// tokens): 66 / 108 us at 32 / 300 tokens against 42 / 59 with the ping-pong GEMM.
// x_dma, gu_dma, down_dma: x, the gate and up and the down weights are dma_aligned.
enum ExpertPath { kPathGeneric, kPathSmall, kPathTiles, kPathFew };

struct ExpertRoute {
    ExpertPath path;
    bool pp_gate_up, pp_down;  // kPathTiles: this launch by the ping-pong GEMM
    int np_lds;                // rows of x staged in LDS
};

inline ExpertRoute expert_route(int n_tokens, int hidden, int inter, int max_lds, bool x_dma, bool gu_dma, bool down_dma) {
    ExpertRoute r{kPathTiles, false, false, n_tokens <= kTileTok ? lds_rows(max_lds, hidden, n_tokens, x_dma) : 0};
    if (x_dma && few_ok(hidden, inter, n_tokens, max_lds)) {
        r.path = kPathFew;
    } else if (n_tokens <= kDownKsRows && expert_small_shape(hidden, inter)) {
        r.path = kPathSmall;
    } else if (n_tokens > kTileTok && pp_ok(hidden, inter, max_lds)) {
        r.pp_gate_up = x_dma && gu_dma;
        r.pp_down = down_dma;
    }
    return r;
}

// Scratch of a call on one expert: h in fp32 (generic kernels), in fragment order
// (few-token path), as fp32 k-part sums of gate and up (1..4 tokens), or as two
// bf16 planes, the lo plane at h_lo_offset.
constexpr size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }
constexpr size_t gu_part_bytes(int n_tokens, int inter) { return sizeof(float) * 2 * 2 * (size_t)n_tokens * inter; }
constexpr size_t h_lo_offset(int n_tokens, int inter) { return align256((size_t)n_tokens * inter * 2); }

inline size_t expert_call_bytes(ExpertPath path, int n_tokens, int inter) {
    switch (path) {
        case kPathGeneric: return (size_t)n_tokens * inter * 4;
        case kPathSmall: return gu_part_bytes(n_tokens, inter);
        case kPathFew: return few_scratch_bytes(n_tokens, inter);
        default: return h_lo_offset(n_tokens, inter) + (size_t)n_tokens * inter * 2;
    }
}

// The same of a context, for the paths of all calls with up to n_tokens tokens.
// Above kFewMaxTokens tokens the lo plane has a buffer of its own (a first call of
// 300 tokens took 78 us with two allocations of 1.2 MB and 89 to 114 with one of 2.4).
struct ExpertScratch {
    size_t bytes, lo_bytes;
};

inline ExpertScratch expert_scratch(int n_tokens, int hidden, int inter, int max_lds) {
    const bool small = expert_small_shape(hidden, inter);
    const int few = std::min(n_tokens, few_max_tokens(max_lds)), both = std::min(n_tokens, kFewMaxTokens);
    const size_t plane = n_tokens > both ? (size_t)n_tokens * inter * 2 : 0;
    return {std::max({small ? expert_call_bytes(kPathSmall, std::min(n_tokens, kDownKsRows), inter) : 0,
                      few_ok(hidden, inter, few, max_lds) ? expert_call_bytes(kPathFew, few, inter) : 0,
                      small && n_tokens <= kDownKsRows ? 0 : expert_call_bytes(kPathTiles, both, inter), plane}),
            plane};
}

// ---------------------------------------------------------------------------
// Router logits of many tokens in 16 x 32 tiles (k_route_logits_mfma): widths.
constexpr int kLgWaves = 8;    // K split
constexpr int kLgRing = 4;     // chunks in flight per wave

inline bool route_mfma_ok(int hidden) { return hidden % (kLgWaves * 32 * kLgRing) == 0; }

// Router logits of 4 to 256 tokens (k_route_logits_split): K slices, 0: another
// kernel.  Its 16 x 16 tiles win while one round of 256 CUs holds them: us a call
// with them and with the 16 x 32 tiles, 256 experts 256 / 300 tokens 30.6 / 42.1 and
// 46.9 / 42.2; 384 experts 160 / 176 / 256 tokens 137 / 150, 155 / 150 and 153 / 147;
// 512 experts 128 / 129 / 256 tokens 34.0 / 43.8, 47.2 / 43.8 and 48.9 / 44.2.  The
// selection reads every slice of its experts, so that above 384 experts a workgroup
// per expert row is still the faster at 4 tokens (512 experts 18.6 against 20.8).
// (Widths that only they and the kernel of a workgroup per expert row take keep
// them up to 256 tokens.)
constexpr int kLsMinTokens = 4, kLsMaxTokens = 256;
constexpr int kLsMaxTiles = 256;
constexpr int kLsWaves = 4;
constexpr int kLsMaxSlices = 8;

inline int route_slices(int n_tokens, int hidden, int n_experts) {
    if (n_tokens < kLsMinTokens + (n_experts > 384) || n_tokens > kLsMaxTokens || hidden % (kLsWaves * 32) != 0) return 0;
    const int tiles = (n_experts + kTileRows - 1) / kTileRows * ((n_tokens + kTileTok - 1) / kTileTok);
    if (tiles > kLsMaxTiles && route_mfma_ok(hidden)) return 0;
    int s = n_tokens <= 32 ? 8 : n_tokens <= 64 ? 4 : n_tokens <= 128 ? 2 : 1;
    while (hidden % (kLsWaves * 32 * s) != 0) s /= 2;
    return s;
}

// Scratch of a router call, offsets in bytes: logits [T, E] in fp64; their slices
// (slices x tokens is at most 256: 8 x 32, 4 x 64, 2 x 128); and for a layer with a
// decode pipeline (`decode`) its one-token scores s, c [E] and, with a shared
// expert, the k-part gate/up sums of up to kDecSplitMaxTokens tokens (dec_inter: its
// inter, else 0).  Up to 16 tokens of such a layer need no slices.
constexpr int kLsPartTokens = 256;

struct RouteScratch {
    size_t part, scores, gu_part, bytes;
};

inline RouteScratch route_scratch(int n_tokens, int hidden, int n_experts, bool decode, int dec_inter) {
    const bool part = n_tokens >= kLsMinTokens && hidden % (kLsWaves * 32) == 0 && !(decode && n_tokens <= kTileTok);
    RouteScratch z;
    z.part = align256(sizeof(double) * (size_t)n_tokens * n_experts);
    z.scores = z.part + align256(part ? sizeof(double) * kLsPartTokens * (size_t)n_experts : 0);
    z.gu_part = z.scores + align256(decode ? sizeof(double) * 2 * (size_t)n_experts : 0);
    z.bytes = z.gu_part + (decode ? gu_part_bytes(std::min(n_tokens, kDecSplitMaxTokens), dec_inter) : 0);
    return z;
}

// ---------------------------------------------------------------------------
// The plan of a grouped call (PlanPtrs).
constexpr int kPlanHdrInts = 8;
constexpr size_t kItemRecBytes = 88, kSlotRecBytes = 24;

struct PlanSizes {
    int max_slots, max_pairs, max_items, item_cap, maxt;
};

inline PlanSizes plan_sizes(int n_tokens, int top_k, int n_experts, int has_shared) {
    PlanSizes z;
    z.maxt = n_tokens <= kTileTok ? 1 : 4;
    z.item_cap = kTileTok * z.maxt;
    z.max_slots = std::min(n_tokens * top_k, n_experts) + has_shared;
    z.max_pairs = n_tokens * top_k + n_tokens * has_shared;
    z.max_items = z.max_slots + (z.max_pairs + z.item_cap - 1) / z.item_cap;
    return z;
}

// dense: a decode plan, which also fills pair_row.
inline size_t plan_bytes(const PlanSizes& z, int n_tokens, int top_k, bool dense) {
    const size_t ints = kPlanHdrInts + 3 * (size_t)z.max_slots + 3 * (size_t)z.max_items +
                        2 * (size_t)z.max_pairs + (size_t)n_tokens * (top_k + 1) +
                        (dense ? (size_t)z.max_pairs : 0);
    return kItemRecBytes * (size_t)z.max_items + kSlotRecBytes * (size_t)z.max_slots + ints * 4;
}

// Bytes of the plan buffer: the plan with the smallest items (16 pairs) and
// pair_row, so that neither the item size nor the pipeline makes it shrink.
inline size_t plan_buffer_bytes(int n_tokens, int top_k, int n_experts, int has_shared) {
    PlanSizes z = plan_sizes(n_tokens, top_k, n_experts, has_shared);
    z.max_items = z.max_slots + (z.max_pairs + kTileTok - 1) / kTileTok;
    return plan_bytes(z, n_tokens, top_k, true);
}

// ---------------------------------------------------------------------------
// Rows around the experts and 4-bit products.
constexpr int kSortMaxExperts = 1024;  // the counts of a workgroup's waves fit its LDS
constexpr int kQ4MaxSide = 1 << 24;    // rows and columns of a 4-bit matrix
constexpr int kNormMaxHidden = 65536;  // a row in the registers of 1024 threads, 64 values each

constexpr int kRowThreads = 256;       // workgroup of the gather and combine kernels

// Columns of a row that is summed: those that the last threads look at, past its end, still fit an int.
constexpr int kMaxRowWidth = INT32_MAX - 8 * kRowThreads;

// A launch's threads are counted in 32 bits.
inline bool rows_grid_ok(int64_t workgroups, int threads) { return workgroups * threads < ((int64_t)1 << 32); }

// Routes of a token that one workgroup of the combine's gradient takes: one each while workgroups are few, up to eight
// together, on one read of dout, once there are many.  Where that turns depends on the pairs and on
// the width of the accesses, little on the rows' bytes (us, one each and together; bf16 rows of 7168, 8 a token: 384
// tokens 22.4 and 26.7, 512: 28.8 and 29.1, 640: 36.0 and 32.8; 16 a token: 256 tokens 26.1 and 29.2, 384: 36.3 and
// 35.5; of 1024, 8 a token: 320 tokens 8.2 and 8.4, 512: 11.8 and 9.1; fp32 of 7168, 6 a token: 320 tokens 26.6 and
// 27.1, 640: 49.0 and 42.2; rows at odd addresses, fp32 of 2001, 6 a token: 256 tokens 9.4 and 9.7, 320: 13.1 and 11.2;
// bf16 of 2001, 16 a token: 96 tokens 9.0 and 10.3, 128: 11.3 and 10.7).
inline int combine_grad_routes(int64_t pairs, bool vec) { return pairs < (vec ? 3500 : 1800) ? 1 : 8; }

// Rows of x per work item: up to 4 for the decode kernel, which stages them in LDS; up to 16
// for the kernel of few rows, which reads them from L2; up to 128 for the GEMM (64 where
// it keeps a second set of sums).
constexpr int kQ4GemmRows = 128;
constexpr int kQ4DecWaves = 8, kQ4DecPieces = 2;  // waves and, of a staged row, 8-value pieces a thread
constexpr int kQ4DecCols = kQ4DecPieces * 64 * kQ4DecWaves * 8;
constexpr int kQ4LdsPad = 64;  // bytes behind a staged row, so that four rows lie in different banks
inline size_t q4_dec_lds(int cols, int rows) { return (size_t)rows * ((size_t)((cols + 127) / 128) * (256 + 4) + kQ4LdsPad); }
inline int q4_dec_rows(int cols) {
    int rows = cols <= kQ4DecCols ? 4 : 0;
    while (rows > 0 && q4_dec_lds(cols, rows) > 63 * 1024) --rows;
    return rows;
}
// LDS of the down projections and sum of one token's routes: up to 512 columns in two planes, 16 sums and a
// weight per route, a wave each.
constexpr int kQ4SumHeld = 4;  // 8-value pieces of a row per lane
constexpr int q4_sum_pitch(int cols) { return 2 * ((cols > 384 ? 4 : (cols + 127) / 128) * 256 + kQ4LdsPad); }
inline size_t q4_sum_lds(int cols, int routes) { return (size_t)routes * (q4_sum_pitch(cols) + 68); }
// A layer on one token's routes, without a plan.
inline bool q4_routes_ok(int n_tokens, int top_k, int hidden, int inter, int shared) {
    return n_tokens == 1 && hidden <= kQ4DecCols && inter <= kQ4SumHeld * 512 && top_k + shared <= 16 &&
           q4_sum_lds(inter, top_k + shared) <= 63 * 1024;
}
// The kernel of a product by its items' rows (us, bf16).
// Few rows while items of 16 rows, at most one short one per matrix, take fewer than 2^30 multiply-adds: few
// launches decide there, and beyond it the reads of x from L2 (one matrix of 4096 x 7168, 32 and 48 rows: 20.1
// and 28.6, GEMM 24.0 and 27.5; 7168 x 2048, 64 rows: 18.6 and 22.0; 1000 x 2048, 128: 10.1 and 25.2; 16 matrices of
// 1024 x 2048, 96 and 256 rows: 19 and 28, GEMM 22 and 22; 64 of 1024 x 1024, 96 rows: 22 and 17), half of that
// for many rows in e4m3, which the GEMM takes as they are (512 x 512, 1024 and 2048 rows: 11.6 and 21.7, GEMM
// 16.0 and 17.4; in bf16 10.5 and 19.7, 24.8 and 26.7); and for up to
// 16 rows of one matrix of any size (18432 x 7168, 16 rows: 32.8, GEMM at 17 31.1).  Its reads of x need whole
// pieces of 8 columns: otherwise it is left to short rows (4096 x 7161, 5 to 16 rows: 26 to 42, GEMM 22).
// The decode kernel while matrices of a stack have one row on average (64 of 4096 x 7168, 64 rows: 122, GEMM 162;
// 96 rows 173 and 177) and for rows without whole pieces as far as it goes; the GEMM for the rest.
constexpr double kQ4FewWork = 1 << 30;
inline int q4_item_rows(int64_t n_rows, int n_mats, int rows, int cols, bool two_sums) {
    const int dec = q4_dec_rows(cols);
    if (dec > 0 && n_rows <= (n_mats > 1 ? n_mats : cols % 8 != 0 ? dec : 0)) return dec;
    const int64_t items = n_mats == 1 ? (n_rows + kTileTok - 1) / kTileTok : std::min<int64_t>(n_mats, n_rows) + n_rows / kTileTok;
    const bool small = (n_mats == 1 && items <= 1) || (double)items * kTileTok * rows * cols < (two_sums && n_rows > 128 ? kQ4FewWork / 2 : kQ4FewWork);
    return small && (cols % 8 == 0 || cols <= 1024) ? kTileTok : two_sums ? kQ4GemmRows / 2 : kQ4GemmRows;
}
// Of a layer of up to `cols` columns, whose second product reads the first one's fp32 rows of `inter` columns, two
// planes of each: the decode kernel or the GEMM.
inline int q4_layer_dec_rows(int cols, int inter) {
    int dec = q4_dec_rows(cols);
    while (dec > 0 && q4_dec_lds(inter, 2 * dec) > 63 * 1024) --dec;
    return dec;
}
inline int q4_layer_rows(int64_t n_rows, int n_mats, int cols, int inter = 0) {
    const int dec = q4_layer_dec_rows(cols, inter);
    return dec > 0 && n_rows <= std::max(n_mats, dec) ? dec : kQ4GemmRows;
}

// Ranges of the columns that the GEMM deals to workgroups of their own, whose partial sums a
// second launch adds: as many as cost least by this estimate, in us.  A workgroup (256
// weight rows, an item of nt 16-row tiles) takes 0.6 + 0.17 nt a column tile on a CU of its own
// (measured: 0.94, 1.2 and 1.96 with 2, 4 and 8), 1 + nt / 10 times that beside a second one; the
// partial sums are written and read at 4.5 MB a us, and the launch is 3.
constexpr int kQ4GemmBlock = 16;  // row tiles of a workgroup
inline int64_t q4_gemm_items(int64_t n_rows, int n_mats, int item_rows) {
    return std::max<int64_t>(n_mats > 1 ? std::min<int64_t>(n_mats, n_rows) : 1, (n_rows + item_rows - 1) / item_rows);
}
inline int q4_gemm_splits(int row_tiles, int col_tiles, int64_t n_rows, int n_mats, int item_rows) {
    if (n_rows <= 0) return 1;
    const int64_t items = q4_gemm_items(n_rows, n_mats, item_rows);
    const double nt = std::min<double>(item_rows / 16, std::max(2.0, (double)((n_rows + 16 * items - 1) / (16 * items))));
    const int64_t wgs = items * ((row_tiles + kQ4GemmBlock - 1) / kQ4GemmBlock);
    int best = 1;
    double least = 0;
    for (int s = 1; s <= 16 && (s == 1 || col_tiles / s >= 2); s *= 2) {
        const double rounds = (double)((wgs * s + 511) / 512), beside = wgs * s > 256 ? 1 + nt / 10 : 1;
        const double cost = rounds * ((col_tiles + s - 1) / s) * (0.6 + 0.17 * nt) * beside +
                            (s > 1 ? 3 + 2.0 * s * (double)n_rows * row_tiles * 64 / 4.5e6 : 0);
        if (s == 1 || cost < least) least = cost, best = s;
    }
    return best;
}

// The most rows of partial sums (ranges times rows) that a call of up to n_rows rows has: with more rows
// come fewer ranges, so that a smaller call may need more.  The estimate's items and nt stay the same over an interval
// of rows; within it only the partial sums' own cost grows with the rows, in proportion to the ranges, so
// that the ranges are the most at its first row.  Items beyond one per matrix are at least half full, 32 rows, whose
// partial sums cost 0.0018 us a row tile and more; what ranges can save is less than a round of workgroups, 3.6 us a
// column tile, so that there are none from 2000 row tiles of items per column tile on.
inline int64_t q4_gemm_part_rows(int row_tiles, int col_tiles, int64_t n_rows, int n_mats, int item_rows) {
    int64_t most = 0;
    for (int64_t n = 1, end; n <= n_rows; n = end + 1) {
        const int64_t items = q4_gemm_items(n, n_mats, item_rows), nt = std::max<int64_t>(2, (n + 16 * items - 1) / (16 * items));
        if (items > n_mats && items * row_tiles >= 2000 * (int64_t)col_tiles) break;
        end = n < n_mats ? n : std::min({n_rows, items * item_rows, items * 16 * nt});
        const int s = q4_gemm_splits(row_tiles, col_tiles, n, n_mats, item_rows);
        if (s > 1) most = std::max(most, s * end);
    }
    return most;
}

// Rows of each of the n items that `rows` rows are cut to (the last has what is left): equal
// ones of whole 16-row tiles, so that the last is not a short one.  n is the least that holds
// them, so no item is empty: (n - 1) shares are at most (n - 1) * item_rows, fewer than the rows.
constexpr int q4_item_share(int n, int rows) {
    return n == 0 ? 0 : n == 1 || rows < 16 * n ? (rows + n - 1) / n : (rows + 16 * n - 1) / (16 * n) * 16;
}

// Items of up to item_rows rows over n_mats matrices, entry 0 (the head) included: at
// most one short item per matrix that has rows, and one of rows without a matrix.
inline int64_t q4_max_items(int64_t n_rows, int n_mats, int item_rows) {
    return 2 + (n_rows < n_mats ? n_rows : n_mats) + n_rows / item_rows;
}
// The same for every call of up to n_rows rows, whatever kernel it takes: none has shorter items than the
// decode kernel (16 rows where that does not go).
inline int64_t q4_most_items(int64_t n_rows, int n_mats, int dec_rows) {
    return q4_max_items(n_rows, n_mats, dec_rows > 0 ? dec_rows : kTileTok);
}

}  // namespace cx
