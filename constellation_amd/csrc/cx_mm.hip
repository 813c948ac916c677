// cx_mm.hip — products with 16-bit weights as the program holds them: plain and gated.
#include "cx_mm_few.h"

namespace cx {
namespace {

using Big = MmShape<2, 4, 8, 4, 2>;
using Small = MmShape<2, 2, 4, 4, 2>;

template <class T, class S, bool GATED, bool DMA>
hipError_t run(MmLaunch& L, hipStream_t s) {
    const int out = GATED ? S::BM / 2 : S::BM, width = GATED ? L.rows / 2 : L.rows;
    L.m_tiles = (width + out - 1) / out;
    cx_launch(k_mm<T, S, GATED, DMA>, dim3(mm_grid(L, S::BN)), dim3(S::kThreads), 0, s, L);
    return hipGetLastError();
}

template <class T, bool GATED>
hipError_t pick(MmLaunch& L, hipStream_t s) {
    const bool dma = L.cols % (16 / T::kEl) == 0 && mm_at16(L.x) && mm_at16(L.w);
    const MmFew f = mm_few_form(L.n_rows, L.n_mats, L.rows, L.cols, T::kEl);
    if (f.rows > 0) return mm_few<T, GATED>(L, f, dma, s);
    if (!dma) return run<T, Small, GATED, false>(L, s);
    return mm_big(L.n_rows, L.offsets ? L.n_mats : 1, L.rows) ? run<T, Big, GATED, true>(L, s) : run<T, Small, GATED, true>(L, s);
}

}  // namespace

hipError_t launch_mm(MmLaunch L, hipStream_t s) {
    if (L.type == CX_DTYPE_BF16) return L.gated ? pick<MmBf16, true>(L, s) : pick<MmBf16, false>(L, s);
    if (L.type == CX_DTYPE_FP16) return L.gated ? pick<MmF16, true>(L, s) : pick<MmF16, false>(L, s);
    return launch_mm_i8(L, s);
}

}  // namespace cx
