// cx_q4_dec.hip — launches of the decode kernel with 4-bit weights.
#include <algorithm>

#include "cx_q4_dec.h"

namespace cx {

namespace {

template <int XT, int NG>
hipError_t dec_launch(const Q4DecArgs& A, int64_t items, hipStream_t s) {
    const size_t lds = std::max<size_t>(q4_dec_lds(A.L.w.cols, A.lds_rows * (XT == kQ4F32 ? 2 : 1)), kQ4DecWaves * 1024);
    // A ring of 8: one token through 8 experts takes 42 us with 4 to 8 places, 45 with 14 and 52 with 20 (registers
    // that waves then lack); 4 in the sum's kernel: 41.3 us, 42.2 with 8, 43.3 with 16.
    cx_launch(k_q4_dec<XT, NG, 8>, dim3((unsigned)(items * A.row_blocks)), dim3(64 * kQ4DecWaves), (uint32_t)lds, s, A);
    return hipGetLastError();
}

template <int XT>
hipError_t dec_groups(const Q4DecArgs& A, int64_t items, hipStream_t s) {
    return A.L.w.group == 128 ? dec_launch<XT, 1>(A, items, s) : A.L.w.group == 64 ? dec_launch<XT, 2>(A, items, s) : dec_launch<XT, 4>(A, items, s);
}

}  // namespace

hipError_t launch_q4_dec(const Q4Launch& L, const Q4Routes* routes, int splits, int64_t items, hipStream_t s) {
    Q4DecArgs A{};
    A.L = L;
    if (routes) A.routes = *routes;
    A.RT = q4_row_tiles(L.w);
    A.KT = q4_col_tiles(L.w);
    A.splits = splits;
    A.row_blocks = (A.RT + kQ4DecWaves / splits - 1) / (kQ4DecWaves / splits);
    A.lds_rows = routes ? 1 : std::min(L.item_rows, L.n_rows);
    switch (L.x_type) {
        case kQ4Bf16: return dec_groups<kQ4Bf16>(A, items, s);
        case kQ4Fp16: return dec_groups<kQ4Fp16>(A, items, s);
        case kQ4F32: return dec_groups<kQ4F32>(A, items, s);
        default: return dec_groups<kQ4E4m3>(A, items, s);
    }
}

hipError_t launch_q4_dec_sum(const Q4DecSumArgs& A, int n_tokens, hipStream_t s) {
    const int ke = A.routes.top_k + A.routes.shared;
    auto k = A.w.group == 128 ? k_q4_dec_sum<1> : A.w.group == 64 ? k_q4_dec_sum<2> : k_q4_dec_sum<4>;
    cx_launch(k, dim3((unsigned)(n_tokens * A.RT)), dim3(64 * ke), (uint32_t)q4_sum_lds(A.w.cols, ke), s, A);
    return hipGetLastError();
}

}  // namespace cx
