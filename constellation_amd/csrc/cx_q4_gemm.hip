// cx_q4_gemm.hip — launches of the GEMM with 4-bit weights.
#include "cx_q4_gemm.h"

namespace cx {

namespace {
int splits_of(const cx_q4_desc& w, int64_t n_rows, int n_mats, int item_rows) {
    return item_rows > kTileTok ? q4_gemm_splits(q4_row_tiles(w), q4_col_tiles(w), n_rows, n_mats, item_rows) : 1;
}
}  // namespace

size_t q4_part_bytes(const cx_q4_desc& w, int64_t n_rows, int n_mats, int item_rows) {
    const int s = splits_of(w, n_rows, n_mats, item_rows);
    return s > 1 ? (size_t)s * n_rows * q4_row_tiles(w) * 64 : 0;
}

size_t q4_most_part_bytes(const cx_q4_desc& w, int64_t n_rows, int n_mats, int item_rows) {
    if (item_rows <= kTileTok) return 0;
    return (size_t)q4_gemm_part_rows(q4_row_tiles(w), q4_col_tiles(w), n_rows, n_mats, item_rows) * q4_row_tiles(w) * 64;
}

hipError_t launch_q4_gemm(const Q4Launch& L, hipStream_t s) {
    Q4GemmArgs a{};
    a.w = L.w;
    a.shared = L.shared;
    a.x = static_cast<const uint16_t*>(L.x);
    a.x_row_scale = L.x_type == kQ4E4m3 ? nullptr : L.x_scale;  // set where the rows were scaled
    a.x_scale = L.x_scale;
    a.item_rows = L.item_rows;
    a.RT = q4_row_tiles(L.w);
    a.KT = q4_col_tiles(L.w);
    a.padded = a.KT * (L.x_type == kQ4F32 ? 256 : 128);
    a.n_x = L.n_x;
    a.n_rows = L.n_rows;
    a.top_k = L.top_k;
    a.order = L.order;
    a.items = L.items;
    a.y = L.y;
    a.y_type = L.y_type;
    constexpr int kRtw = kQ4GemmBlock / kQ4GemmWaves;
    a.part = L.part;
    a.splits = splits_of(L.w, L.n_rows, L.n_mats, L.item_rows);
    a.RB = (a.RT + kQ4GemmWaves * kRtw - 1) / (kQ4GemmWaves * kRtw);
    const int64_t items = L.items != nullptr ? L.max_items : (L.n_rows + L.item_rows - 1) / L.item_rows;
    auto of = [&](auto ng) {
        return L.x_type == kQ4E4m3 ? k_q4_gemm<ng, kRtw, true, false> : L.x_type == kQ4F32 ? k_q4_gemm<ng, kRtw, false, true> : k_q4_gemm<ng, kRtw, false, false>;
    };
    auto k = L.w.group == 128  ? of(std::integral_constant<int, 1>{})
             : L.w.group == 64 ? of(std::integral_constant<int, 2>{})
                               : of(std::integral_constant<int, 4>{});
    cx_launch(k, dim3((unsigned)(items * a.RB * a.splits)), dim3(64 * kQ4GemmWaves), 0, s, a);
    if (a.splits > 1) {
        const int width = L.w.gated ? L.w.rows / 2 : L.w.rows, units = (width + 3) / 4;
        cx_launch(k_q4_sum, dim3((unsigned)(((int64_t)L.n_rows * units + 255) / 256)), dim3(256), 0, s, static_cast<const float*>(L.part),
                  a.splits, L.n_rows, a.RT * 16, L.w.gated, width, L.y, L.y_type, units);
    }
    return hipGetLastError();
}

}  // namespace cx
