// cx_mm_grad.hip — gradients of the products with 16-bit weights, and of the gate between them.
#include "cx_mm.h"

namespace cx {
namespace {

template <class T, class S>
hipError_t dx(MmLaunch& L, hipStream_t s) {
    cx_launch(k_mm_dx<T, S>, dim3(mm_grid(L, L.cols)), dim3(S::kThreads), 0, s, L);
    return hipGetLastError();
}

template <class T>
hipError_t dx_pick(MmLaunch& L, hipStream_t s) {
    const hipError_t e = L.form.kind == 2 ? dx<T, MmBig>(L, s) : dx<T, MmSmall>(L, s);
    return e != hipSuccess || L.splits == 1 ? e : launch_mm_sum(L, L.cols, false, s);
}

template <class T>
hipError_t dw_pick(MmLaunch& L, hipStream_t s) {
    static_assert(MmSmall::BM == 128 && MmSmall::BN == 128 && MmBig::BM == 256 && MmBig::BN == 256 && MmMid::BM == 256 && MmMid::BN == 128, "mm_dw_grid");
    const int kind = mm_dw_kind(L.n_rows, L.n_mats, L.rows, L.cols), m = kind == 1 ? MmSmall::BM : MmBig::BM;
    const dim3 grid((unsigned)mm_dw_grid(kind, L.n_mats, L.rows, L.cols));
    L.m_tiles = (L.cols + m - 1) / m;
    if (kind == 1)
        cx_launch(k_mm_dw<T, MmSmall>, grid, dim3(MmSmall::kThreads), 0, s, L);
    else if (kind == 2)
        cx_launch(k_mm_dw<T, MmBig>, grid, dim3(MmBig::kThreads), 0, s, L);
    else
        cx_launch(k_mm_dw_short<T, MmMid>, grid, dim3(MmMid::kThreads), 0, s, L);
    return hipGetLastError();
}

// h = silu(g) u has dg = dh u sig(g) (1 + g (1 - sig(g))) and du = dh silu(g); each rounded once.  One value
// of dh, g and u a lane, 8 where rows allow 16-byte accesses.  HBM bounds it: 16384 rows of 2048 (335 MB) in 77 us.  Within
// the products that read it, each would form it again for every tile (56 of 128 columns).
template <bool BF, int N>
__global__ __launch_bounds__(256) void k_gate_grad(const uint16_t* dh, const uint16_t* pre, int64_t n_rows, int inter, uint16_t* dpre, int pitch) {
    const int per = (inter + N - 1) / N;
    const int64_t total = n_rows * per;
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < total; at += (int64_t)gridDim.x * 256) {
        const int64_t p = at / per;
        const int c = (int)(at - p * per) * N;
        typedef uint16_t V __attribute__((ext_vector_type(N == 1 ? 2 : N)));
        auto value = [](uint16_t h) { return BF ? __uint_as_float((uint32_t)h << 16) : (float)__builtin_bit_cast(_Float16, h); };
        auto round = [](float f) { return (uint16_t)(BF ? bf16_rne(f) : f16_rne(f)); };
        V d = {}, g = {}, u = {}, a, b;
        const int64_t o = p * 2 * inter + c, to = p * pitch + c;
        if constexpr (N == 1) {
            d[0] = dh[p * inter + c], g[0] = pre[o], u[0] = pre[o + inter];
        } else {
            d = *reinterpret_cast<const V*>(dh + p * inter + c);
            g = *reinterpret_cast<const V*>(pre + o);
            u = *reinterpret_cast<const V*>(pre + o + inter);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float x = value(g[i]), t = value(d[i]), sig = 1.0f / (1.0f + expf(-x));
            a[i] = round(t * value(u[i]) * sig * (1.0f + x * (1.0f - sig)));
            b[i] = round(t * x * sig);
        }
        if constexpr (N == 1) {
            dpre[to] = a[0], dpre[to + inter] = b[0];
        } else {
            *reinterpret_cast<V*>(dpre + to) = a;
            *reinterpret_cast<V*>(dpre + to + inter) = b;
        }
        if (c == 0)
            for (int i = 2 * inter; i < pitch; ++i) dpre[p * pitch + i] = 0;
    }
}

}  // namespace

hipError_t launch_mm_dx(MmLaunch L, hipStream_t s) { return L.type == CX_DTYPE_BF16 ? dx_pick<MmBf16>(L, s) : dx_pick<MmF16>(L, s); }
hipError_t launch_mm_dw(MmLaunch L, hipStream_t s) { return L.type == CX_DTYPE_BF16 ? dw_pick<MmBf16>(L, s) : dw_pick<MmF16>(L, s); }

hipError_t launch_gate_grad(const void* dh, const void* pre, int type, int64_t n_rows, int inter, void* dpre, int pitch, hipStream_t s) {
    const bool vec = inter % 8 == 0 && mm_at16(dh) && mm_at16(pre) && mm_at16(dpre);
    const int64_t wgs = (n_rows * ((inter + (vec ? 7 : 0)) / (vec ? 8 : 1)) + 255) / 256;
    auto k = type == CX_DTYPE_BF16 ? (vec ? k_gate_grad<true, 8> : k_gate_grad<true, 1>) : (vec ? k_gate_grad<false, 8> : k_gate_grad<false, 1>);
    cx_launch(k, dim3((unsigned)std::min<int64_t>(wgs, 8192)), dim3(256), 0, s, static_cast<const uint16_t*>(dh), static_cast<const uint16_t*>(pre),
              n_rows, inter, static_cast<uint16_t*>(dpre), pitch);
    return hipGetLastError();
}

}  // namespace cx
