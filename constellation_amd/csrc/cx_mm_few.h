// cx_mm_few.h — the forward products for few rows of x per matrix: the weights stream once from
// memory to the matrix cores, without LDS.
#pragma once

#include "cx_mm.h"

namespace cx {

// 16 bytes of a row, `have` elements of which exist.  VEC: all or none of them, at an address that 16 divides.
template <int EL, bool VEC>
__device__ __forceinline__ u32x4 mm_piece(const char* q, int have) {
    if constexpr (VEC) {
        return ld16(have > 0 ? q : reinterpret_cast<const char*>(mm_zeros));
    } else {
        constexpr int kWhole = 16 / EL;
        u32x4 v = {};
        if (have >= kWhole) return ((const __attribute__((address_space(1))) MmPacked*)q)->v;
#pragma unroll
        for (int e = 0; e < kWhole - 1; ++e) {
            if (e >= have) continue;
            if constexpr (EL == 1)
                v[e / 4] |= (uint32_t)reinterpret_cast<const uint8_t*>(q)[e] << (8 * (e & 3));
            else
                v[e / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(q)[e] << (16 * (e & 1));
        }
        return v;
    }
}

// Up to 16 rows fit one MFMA's columns, so that the weights are read once and nothing is shared that LDS would serve.  Memory
// bounds it: 1 row by 4096 x 7168 gated 14.8 us on weights from HBM (4.0 TB/s) and 12.4 after itself, when the last-level cache
// holds the 59 MB (4.7 TB/s); 69 through LDS; 16 rows 20, where x costs L2 as many bytes as the weights cost HBM; 232 rows over
// 64 matrices, which no cache holds, 197 to 238 by the deal (about 4.7 TB/s); 8-bit 8.4.  Rows at odd
// addresses (7161 columns) 24: lanes' pieces straddle lines; with more of them in flight it was 26.
//
// A workgroup's 8 waves are `splits` ranges of the columns times 8 / splits groups of RW tiles of 16 weight
// rows (gated: 8 gate rows and the same 8 up rows, so that both factors of an output meet in two lanes of
// a wave); the ranges' sums are added in order.  A wave has U steps of 128 bytes of its rows in flight ahead of the
// U that it multiplies, of weights and of up to 16 rows of x, which come from L2.
template <class T, int RW, bool GATED, bool VEC>
__global__ __launch_bounds__(64 * kMmFewWaves, 2) void k_mm_few(MmLaunch L, int splits, int row_blocks) {
    typedef typename T::Acc Acc;
    constexpr int EL = T::kEl, kStep = 128 / EL, U = !VEC ? 1 : RW == 1 ? 4 : 2;
    __shared__ __attribute__((aligned(16))) uint32_t red[kMmFewWaves][RW][256];
    const int idx = blockIdx.x / row_blocks, block = blockIdx.x - idx * row_blocks;
    const int wave = wave_id(), lane = threadIdx.x & 63, t = lane & 15, q = lane >> 4;
    if (L.offsets != nullptr && blockIdx.x == 0 && wave == kMmFewWaves - 1) mm_check(L.offsets, L.n_mats, L.n_rows, L.err_flag);
    const MmItem it = mm_item(L.offsets, L.n_mats, L.n_rows, 16, idx);
    if (it.rows <= 0) return;
    const int groups = kMmFewWaves / splits, rg = wave / splits, ks = wave - rg * splits;
    constexpr int kCols = GATED ? 8 : 16;  // outputs of a tile
    const int width = GATED ? L.rows / 2 : L.rows, tile0 = (block * groups + rg) * RW, tiles = (width + kCols - 1) / kCols;
    if (it.mat < 0) {
        const int m0 = block * groups * RW * kCols, cols = groups * RW * kCols;
        mm_clear(L.y, L.y_type, it.begin, it.rows, width, m0, cols, 64 * kMmFewWaves);
        if (GATED && L.pre != nullptr)
            for (int h = 0; h < 2; ++h)
                for (int r = 0; r < it.rows; ++r) mm_clear(L.pre, T::kType, 2 * (int64_t)(it.begin + r) + h, 1, width, m0, cols, 64 * kMmFewWaves);
        return;
    }
    auto source = [&](int r) {  // row of x of row r of the item, < 0: none
        const int p = it.begin + min(r, it.rows - 1);
        if (L.order == nullptr) return p;
        const int pair = L.order[p], xr = pair / L.top_k;
        return pair < 0 || xr >= L.n_x ? -1 : xr;
    };
    const size_t pitch = (size_t)L.cols * EL;
    const char *wp[RW];
#pragma unroll
    for (int m = 0; m < RW; ++m) {
        const int r = (tile0 + m) * kCols + t % kCols, n = min(r, width - 1) + (GATED && t >= 8 ? width : 0);  // rows past the matrix: its last one again
        wp[m] = static_cast<const char*>(L.w) + ((size_t)it.mat * L.rows + n) * pitch + q * 16;
    }
    const char* xp = static_cast<const char*>(L.x) + (size_t)max(source(t), 0) * pitch + q * 16;
    const int steps = (L.cols + kStep - 1) / kStep, per = (steps + splits - 1) / splits, k0 = ks * per, k1 = tile0 >= tiles ? 0 : min(steps, k0 + per);
    u32x4 a[2][U][RW][2], x[2][U][2];
    Acc acc[RW] = {};
    auto fetch = [&](int k, auto to) {  // past the range: its last step again, not multiplied
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int kk = min(k + u, k1 - 1);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int have = L.cols - kk * kStep - (4 * j + q) * (16 / EL);
                const size_t at = (size_t)kk * 128 + j * 64;
#pragma unroll
                for (int m = 0; m < RW; ++m) a[to][u][m][j] = mm_piece<EL, VEC>(wp[m] + at, have);
                x[to][u][j] = mm_piece<EL, VEC>(xp + at, have);
            }
        }
    };
    auto multiply = [&](int k, auto from) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (k + u >= k1) break;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int m = 0; m < RW; ++m) acc[m] = T::mma(a[from][u][m][j], x[from][u][j], acc[m]);
        }
    };
    constexpr std::integral_constant<int, 0> even{};
    constexpr std::integral_constant<int, 1> odd{};
    if (k0 < k1) fetch(k0, even);
    for (int k = k0; k < k1; k += 2 * U) {
        if (k + U < k1) fetch(k + U, odd);
        multiply(k, even);
        if (k + U >= k1) break;
        if (k + 2 * U < k1) fetch(k + 2 * U, even);
        multiply(k + U, odd);
    }
#pragma unroll
    for (int m = 0; m < RW; ++m) *reinterpret_cast<u32x4*>(&red[wave][m][t * 16 + q * 4]) = __builtin_bit_cast(u32x4, acc[m]);
    __syncthreads();
    // outputs: 16 lanes have a tile's 16 sums of one row of x
    auto put = [](void* y, int type, int64_t at, float f) {
        if (type == CX_DTYPE_F32)
            static_cast<float*>(y)[at] = f;
        else
            static_cast<uint16_t*>(y)[at] = (uint16_t)cast_out(f, type);
    };
    for (int i = threadIdx.x; i < groups * RW * 256; i += 64 * kMmFewWaves) {
        // neighbours: the sums of a tile, the tiles of the group, the rows of x
        const int r = i & 15, m = i / 16 % RW, g = i / (16 * RW) % groups, row = i / (16 * RW * groups);
        if (row >= it.rows) break;
        const int xr = source(row), c = ((block * groups + g) * RW + m) * kCols + r % kCols, n = min(c, width - 1) + (GATED && r >= 8 ? width : 0);
        float v;
        if constexpr (EL == 1) {
            int s = 0;
            for (int k = 0; k < splits; ++k) s += (int)red[g * splits + k][m][row * 16 + r];
            v = (float)s * (xr < 0 ? 0.0f : L.x_scale[xr]) * L.w_scale[(size_t)it.mat * L.rows + n];
        } else {
            v = 0.0f;
            for (int k = 0; k < splits; ++k) v += __uint_as_float(red[g * splits + k][m][row * 16 + r]);
        }
        if (xr < 0) v = 0.0f;
        const int64_t p = it.begin + row;
        if constexpr (GATED) {
            const float up = __shfl_down(v, 8);
            if (c < width && L.pre != nullptr) put(L.pre, T::kType, p * L.rows + n, v);
            if (c < width && r < 8) put(L.y, L.y_type, p * width + c, mm_silu(v) * up);
        } else if (c < width) {
            put(L.y, L.y_type, p * width + c, v);
        }
    }
}

template <class T, int RW, bool GATED>
hipError_t mm_few_run(MmLaunch& L, bool vec, hipStream_t s) {
    const int splits = L.form.splits, blocks = (int)mm_few_blocks(L.form, L.rows);
    const int64_t items = mm_items(L.n_rows, L.n_mats, L.offsets != nullptr, 16);
    cx_launch(vec ? k_mm_few<T, RW, GATED, true> : k_mm_few<T, RW, GATED, false>, dim3((unsigned)(items * blocks)), dim3(64 * kMmFewWaves), 0, s, L,
              splits, blocks);
    return hipGetLastError();
}

template <class T, bool GATED>
hipError_t mm_few(MmLaunch& L, bool vec, hipStream_t s) {
    return L.form.tiles == 1 ? mm_few_run<T, 1, GATED>(L, vec, s) : mm_few_run<T, 2, GATED>(L, vec, s);
}

}  // namespace cx
