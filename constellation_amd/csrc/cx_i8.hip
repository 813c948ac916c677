// cx_i8.hip — rows to 8-bit integers with a scale each, and products of such rows with
// 8-bit weights: y[p, n] = xs[p] ws[n] sum over k of x[p, k] w[n, k], the sum exact in 32 bits.
#include "cx_mm_few.h"

namespace cx {
namespace {

template <class S, bool GATED>
hipError_t run(MmLaunch& L, hipStream_t s) {
    cx_launch(k_mm<MmI8, S, GATED>, dim3(mm_grid(L, L.rows)), dim3(S::kThreads), 0, s, L);
    return hipGetLastError();
}

template <bool GATED>
hipError_t pick(MmLaunch& L, hipStream_t s) {
    if (L.form.kind == 0) return mm_few<MmI8, GATED>(L, L.cols % 16 == 0, s);
    const hipError_t e = L.form.kind == 2 ? run<MmBig, GATED>(L, s) : run<MmSmall, GATED>(L, s);
    return e != hipSuccess || L.splits == 1 ? e : launch_mm_sum(L, L.rows, GATED, s);
}

constexpr int kI8Threads = 256, kI8Held = 4;  // pieces of 8 values of a row that a thread holds

__device__ __forceinline__ void i8_piece(const void* x, int type, size_t at, int left, bool vec, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    if (left <= 0) return;
    if (type == CX_DTYPE_F32) {
        const float* p = static_cast<const float*>(x) + at;
        if (vec) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = a[i], v[i + 4] = b[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < left) v[i] = p[i];
        }
        return;
    }
    const uint16_t* p = static_cast<const uint16_t*>(x) + at;
    uint32_t h[8] = {};
    if (vec) {
        const u32x4 d = ld16(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = i & 1 ? d[i >> 1] >> 16 : d[i >> 1] & 0xFFFFu;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < left) h[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        v[i] = type == CX_DTYPE_BF16 ? __uint_as_float(h[i] << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)h[i]);
}

// A row's largest size, then codes from correctly rounded quotients.  W waves have a row, 4 / W rows a workgroup, and hold
// it in registers between the two (up to 2048 W columns), so that it is read once.  1024 rows of 7168 in 9.4 us of a series
// (12.4 traced after a pause), where a copy of the same bytes takes 4.5: a row's load, its maximum and its codes wait for each other.
template <int W>
__global__ __launch_bounds__(kI8Threads) void k_quantize_i8(const void* x, int type, int n_rows, int cols, int8_t* q, float* scale) {
    __shared__ uint32_t part[kI8Threads / 64];
    constexpr int kThreads = 64 * W, kSpan = kI8Held * kThreads * 8;
    const int tid = threadIdx.x % kThreads, at_row = blockIdx.x * (kI8Threads / kThreads) + threadIdx.x / kThreads;
    if (at_row >= n_rows) return;  // W 4: none
    const size_t row = (size_t)at_row * cols;
    const bool vec = cols % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0, wide = cols % 8 == 0 && (reinterpret_cast<uintptr_t>(q) & 7) == 0;
    float v[kI8Held][8];
    uint32_t most = 0;  // as bits: of sizes the larger one has the larger bits, and a NaN is the largest
    auto take = [&](const float (&f)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(f[i]) & 0x7FFFFFFFu);
    };
#pragma unroll
    for (int i = 0; i < kI8Held; ++i) {
        const int c = (i * kThreads + tid) * 8;
        i8_piece(x, type, row + c, cols - c, vec, v[i]);
        take(v[i]);
    }
    for (int c = kSpan + tid * 8; c < cols; c += kThreads * 8) {
        float f[8];
        i8_piece(x, type, row + c, cols - c, vec, f);
        take(f);
    }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, m));
    if constexpr (W > 1) {
        if ((tid & 63) == 0) part[tid >> 6] = most;
        __syncthreads();
        most = max(max(part[0], part[1]), max(part[2], part[3]));
    }
    const float s = most > 0x7F800000u ? __uint_as_float(most) : fmaxf(__uint_as_float(most) / 127.0f, 1e-12f);
    if (tid == 0) scale[at_row] = s;
    auto put = [&](int c, const float (&f)[8]) {
        uint32_t d[2] = {};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float r = rintf(f[i] / s);
            d[i >> 2] |= ((uint32_t)(r == r ? (int)fminf(fmaxf(r, -127.0f), 127.0f) : 0) & 0xFFu) << (8 * (i & 3));
        }
        if (wide) {
            *reinterpret_cast<uint2*>(q + row + c) = uint2{d[0], d[1]};
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < cols) q[row + c + i] = (int8_t)(d[i >> 2] >> (8 * (i & 3)));
        }
    };
#pragma unroll
    for (int i = 0; i < kI8Held; ++i) {
        const int c = (i * kThreads + tid) * 8;
        if (c < cols) put(c, v[i]);
    }
    for (int c = kSpan + tid * 8; c < cols; c += kThreads * 8) {
        float f[8];
        i8_piece(x, type, row + c, cols - c, vec, f);
        put(c, f);
    }
}

}  // namespace

hipError_t launch_mm_i8(MmLaunch L, hipStream_t s) { return L.gated ? pick<true>(L, s) : pick<false>(L, s); }

hipError_t launch_quantize_i8(const void* x, int x_type, int n_rows, int cols, int8_t* q, float* scale, hipStream_t s) {
    // a wave each and four, us: rows of 512: 256 3.4 and 3.5, 1024 3.6 and 4.7, 4096 5.1 and 10.6; of 1024: 512 3.9 and 3.8, 1500 4.4 and
    // 5.7, 2048 4.5 and 7.0; of 2048: one 4.0 and 2.5, 512 4.9 and 3.8, 1024 5.1 and 5.3, 2048 6.2 and 7.6, 16384 30 and 46
    const int rows = cols <= 512 || (cols <= 2048 && n_rows >= 2048) ? 4 : 1;  // of a workgroup
    const int most = rows << 23;                                               // of a launch, whose threads are counted in 32 bits
    const size_t row = (size_t)cols * (x_type == CX_DTYPE_F32 ? 4 : 2);
    for (int64_t r = 0; r < n_rows; r += most) {
        const int n = (int)std::min<int64_t>(most, n_rows - r);
        cx_launch(rows == 4 ? k_quantize_i8<1> : k_quantize_i8<4>, dim3((unsigned)((n + (int64_t)rows - 1) / rows)), dim3(kI8Threads), 0, s,
                  static_cast<const char*>(x) + r * row, x_type, n, cols, q + r * cols, scale + r);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace cx
