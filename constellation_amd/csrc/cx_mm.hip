// cx_mm.hip — products with 16-bit weights as the program holds them: plain and gated; and the sums of partial
// products.
#include "cx_mm_few.h"

namespace cx {
namespace {

template <class T, class S, bool GATED>
hipError_t run(MmLaunch& L, hipStream_t s) {
    cx_launch(k_mm<T, S, GATED>, dim3(mm_grid(L, L.rows)), dim3(S::kThreads), 0, s, L);
    return hipGetLastError();
}

template <class T, bool GATED>
hipError_t pick(MmLaunch& L, hipStream_t s) {
    if (L.form.kind == 0) return mm_few<T, GATED>(L, L.cols % 8 == 0, s);
    const hipError_t e = L.form.kind == 2 ? run<T, MmBig, GATED>(L, s) : run<T, MmSmall, GATED>(L, s);
    return e != hipSuccess || L.splits == 1 ? e : launch_mm_sum(L, L.rows, GATED, s);
}

// The matrix that row p belongs to: the one before the first whose offset lies behind it; n_mats: none.
__device__ __forceinline__ int mm_mat_of(const int32_t* offsets, int n_mats, int n_rows, int p) {
    if (offsets == nullptr) return 0;
    int first = n_mats + 1;
    for (int e = 1 + (threadIdx.x & 63); e <= n_mats; e += 64)
        if (mm_cut(offsets[e], n_rows) > p) first = min(first, e);
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) first = min(first, __shfl_xor(first, m));
    return first > n_mats ? n_mats : first - 1;
}

// The ranges' sums of a row, added in order, and what follows the sums.  A row and 1024 of its outputs a workgroup.  The
// partial sums come from L2, where they were just written: 4 ranges of 256 rows by 4096 (17 MB) take 7 us of 32.
template <bool I8>
__global__ __launch_bounds__(256) void k_mm_sum(MmLaunch L, int out, int gated, int chunks) {
    const int p = blockIdx.x / chunks, c = (blockIdx.x - p * chunks) * 1024 + threadIdx.x * 4, width = gated ? out / 2 : out;
    const int mat = mm_mat_of(L.offsets, L.n_mats, L.n_rows, p), left = width - c;
    if (left <= 0) return;
    const int xr = mat == L.n_mats && L.offsets != nullptr ? -1 : L.dy != nullptr ? p : mm_row_of_x(L, p);
    float v[2][4] = {};
    if (xr >= 0) {
        for (int h = 0; h <= gated; ++h) {
            const float* src = L.part + (size_t)p * out + (h ? width : 0) + c;
            const size_t range = (size_t)L.n_rows * out;
            const bool vec = width % 4 == 0;
            int n[4] = {};
            for (int s = 0; s < L.splits; ++s) {
                float d[4];
                if (vec) {
                    const f32x4 q = *reinterpret_cast<const f32x4*>(src + s * range);
#pragma unroll
                    for (int i = 0; i < 4; ++i) d[i] = q[i];
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) d[i] = i < left ? src[s * range + i] : 0.0f;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (I8)
                        n[i] += __float_as_int(d[i]);
                    else
                        v[h][i] += d[i];
                }
            }
            if constexpr (I8) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (i < left) v[h][i] = (float)n[i] * L.x_scale[xr] * L.w_scale[(size_t)mat * out + (h ? width : 0) + c + i];
            }
        }
    }
    auto put = [&](void* y, int type, int64_t at, const float (&f)[4]) {
        if (type == CX_DTYPE_F32) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < left) static_cast<float*>(y)[at + i] = f[i];
        } else if (width % 4 == 0 && (reinterpret_cast<uintptr_t>(y) & 7) == 0) {
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(y) + at) = uint2{cast_out(f[0], type) | (cast_out(f[1], type) << 16), cast_out(f[2], type) | (cast_out(f[3], type) << 16)};
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < left) static_cast<uint16_t*>(y)[at + i] = (uint16_t)cast_out(f[i], type);
        }
    };
    if (gated) {
        if (L.pre != nullptr) {
            put(L.pre, L.type, (int64_t)p * out + c, v[0]);
            put(L.pre, L.type, (int64_t)p * out + width + c, v[1]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) v[0][i] = mm_silu(v[0][i]) * v[1][i];
    }
    put(L.y, L.y_type, (int64_t)p * width + c, v[0]);
}

// Rows to rows of whole pieces, a piece of 16 bytes a lane.  HBM bounds it: 16 matrices of 714 x 2001 (46 MB) in 16.5 us.
// Read by the products themselves, through registers instead of straight to LDS, such rows cost more: 3001 rows by
// 4096 x 2001 93 us where copies and product take 68, its gradients 177 and 141 (67 and 58).
template <int EL>
__global__ __launch_bounds__(256) void k_mm_pad(MmPad p) {
    const int per = p.pitch / (16 / EL);
    const int64_t total = p.rows * per;
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < total; at += (int64_t)gridDim.x * 256) {
        const int64_t row = total <= 0xFFFFFFFFll ? (uint32_t)at / (uint32_t)per : at / per;
        if (p.offsets != nullptr) {
            const int64_t mat = row / p.mat_rows;
            // cut offsets give it no rows either; the first offset is taken for 0
            if (p.offsets[mat + 1] <= 0 || (mat > 0 && p.offsets[mat + 1] <= p.offsets[mat])) continue;
        }
        const int c = (int)(at - row * per) * (16 / EL);
        static_cast<u32x4*>(p.dst)[at] = mm_piece<EL, false>(static_cast<const char*>(p.src) + (row * p.cols + c) * EL, p.cols - c);
    }
}

}  // namespace

hipError_t launch_mm_pad(const MmPad& p, hipStream_t s) {
    const int64_t wgs = (p.rows * (p.pitch / (16 / p.el)) + 255) / 256;
    cx_launch(p.el == 1 ? k_mm_pad<1> : k_mm_pad<2>, dim3((unsigned)std::min<int64_t>(wgs, 16384)), dim3(256), 0, s, p);
    return hipGetLastError();
}

hipError_t launch_mm_sum(const MmLaunch& L, int out, bool gated, hipStream_t s) {
    const int chunks = mm_sum_chunks(gated ? out / 2 : out);
    cx_launch(L.type == kMmI8 ? k_mm_sum<true> : k_mm_sum<false>, dim3((unsigned)((int64_t)L.n_rows * chunks)), dim3(256), 0, s, L, out, (int)gated, chunks);
    return hipGetLastError();
}

hipError_t launch_mm(MmLaunch L, hipStream_t s) {
    const int el = L.type == kMmI8 ? 1 : 2;
    L.x_pitch = L.w_pitch = L.cols;
    if (L.pad_w != nullptr) {
        const int pitch = mm_pitch(L.cols, el);
        hipError_t e = launch_mm_pad(MmPad{L.x, L.pad_x, el, L.cols, pitch, L.n_x, nullptr, 1}, s);
        if (e == hipSuccess) e = launch_mm_pad(MmPad{L.w, L.pad_w, el, L.cols, pitch, (int64_t)L.n_mats * L.rows, L.offsets, L.rows}, s);
        if (e != hipSuccess) return e;
        L.x = L.pad_x;
        L.w = L.pad_w;
        L.x_pitch = L.w_pitch = pitch;
    }
    if (L.type == CX_DTYPE_BF16) return L.gated ? pick<MmBf16, true>(L, s) : pick<MmBf16, false>(L, s);
    if (L.type == CX_DTYPE_FP16) return L.gated ? pick<MmF16, true>(L, s) : pick<MmF16, false>(L, s);
    return launch_mm_i8(L, s);
}

}  // namespace cx
