// cx_q4_gemm.hip — launches of the GEMM with 4-bit weights.
#include "cx_q4_gemm.h"

namespace cx {

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
    a.padded = a.KT * 128;
    a.n_x = L.n_x;
    a.n_rows = L.n_rows;
    a.top_k = L.top_k;
    a.order = L.order;
    a.items = L.items;
    a.y = L.y;
    a.y_type = L.y_type;
    constexpr int kRtw = 4;
    a.RB = (a.RT + kQ4GemmWaves * kRtw - 1) / (kQ4GemmWaves * kRtw);
    const int64_t items = L.items != nullptr ? L.max_items : (L.n_rows + L.item_rows - 1) / L.item_rows;
    const bool xs = L.x_type == kQ4E4m3;
    auto k = L.w.group == 128  ? (xs ? k_q4_gemm<1, kRtw, true> : k_q4_gemm<1, kRtw, false>)
             : L.w.group == 64 ? (xs ? k_q4_gemm<2, kRtw, true> : k_q4_gemm<2, kRtw, false>)
                               : (xs ? k_q4_gemm<4, kRtw, true> : k_q4_gemm<4, kRtw, false>);
    cx_launch(k, dim3((unsigned)(items * a.RB)), dim3(64 * kQ4GemmWaves), 0, s, a);
    return hipGetLastError();
}

}  // namespace cx
