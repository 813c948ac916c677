// cx_q4.h — kernels of the products with 4-bit weights.
//
// Layout of a packed matrix: tiles of 16 rows x 128 columns, 1 KB each, the tiles of
// 16 rows one after another.  Lane l of a wave holds the codes that an MFMA 16x16x32
// takes from it in one 16-byte piece: row l % 16; dword j the columns 32 j + 8 (l / 16)
// .. + 7, so that MFMA j covers the columns 32 j .. 32 j + 31, within one group of any
// size, and a wave's load of a tile is one contiguous 1 KB.  The tile's scales are
// fp16 [16 rows][128 / group], divided by a power of two per row that lies behind
// them all as fp32 [n_mats][row tiles][16].
// A `gated` matrix has 8 rows of its first half and the same 8 of its second half in
// a tile, so that both factors of an output meet in one accumulator tile.
#pragma once

#include "cx_device.h"

namespace cx {

constexpr int kQ4Tile = 1024;     // bytes of a tile's codes
constexpr int kQ4FewWaves = 8;

__host__ __device__ inline int q4_row_tiles(const cx_q4_desc& w) { return w.gated ? (w.rows / 2 + 7) / 8 : (w.rows + 15) / 16; }
__host__ __device__ inline int q4_col_tiles(const cx_q4_desc& w) { return (w.cols + 127) / 128; }

__host__ __device__ inline const float* q4_row_scales(const cx_q4_desc& w) {
    return reinterpret_cast<const float*>(w.scales + (size_t)w.n_mats * q4_row_tiles(w) * q4_col_tiles(w) * (128 / w.group) * 16);
}

// Eight codes -> eight bf16 / fp16, exact.
__device__ __forceinline__ bf16x8 q4_bf16(uint32_t w) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 1);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 3);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ f16x8 q4_f16(uint32_t w) {
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 1);
    const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 3);
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// x's columns col .. col + 7 of one row as MFMA operand bits; columns past the
// row's end are zeros (the codes there are, too, but a NaN times zero is not).
template <int XT>
__device__ __forceinline__ u32x4 q4_x8(const void* row, int col, int cols, bool vec) {
    if constexpr (XT == kQ4E4m3) {
        const uint8_t* p = static_cast<const uint8_t*>(row) + col;
        uint32_t a = 0, b = 0;
        if (vec) {
            if (col < cols) {
                const uint2 v = *reinterpret_cast<const uint2*>(p);
                a = v.x, b = v.y;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (col + i < cols) (i < 4 ? a : b) |= (uint32_t)p[i] << (8 * (i & 3));
        }
        return __builtin_bit_cast(u32x4, cvt8_bf16(a, b));
    } else {
        const uint16_t* p = static_cast<const uint16_t*>(row) + col;
        u32x4 v = {};
        if (vec) {
            if (col < cols) v = ld16(p);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (col + i < cols) v[i >> 1] |= (uint32_t)p[i] << (16 * (i & 1));
        }
        return v;
    }
}

__device__ __forceinline__ float q4_scale(const uint32_t* sc, int i) {
    return static_cast<float>(__builtin_bit_cast(f16x2, sc[i >> 1])[i & 1]);
}

__device__ __forceinline__ void q4_store(const Q4Launch& L, size_t at, float v) {
    if (L.y_type == CX_DTYPE_F32) {
        static_cast<float*>(L.y)[at] = v;
    } else if (L.y_type == kQ4Planes) {
        const uint32_t hi = bf16_rne(v);
        static_cast<uint16_t*>(L.y)[at] = (uint16_t)hi;
        static_cast<uint16_t*>(L.y_lo)[at] = (uint16_t)bf16_rne(v - __uint_as_float(hi << 16));
    } else {
        static_cast<uint16_t*>(L.y)[at] = (uint16_t)cast_out(v, L.y_type);
    }
}

// Up to 16 rows of x against 16 rows of weights per workgroup, the columns dealt to
// its waves tile by tile and the partial tiles summed in wave order.
template <int XT, int NG>
__global__ __launch_bounds__(64 * kQ4FewWaves) void k_q4_few(Q4Launch L, int RT, int KT) {
    __shared__ float red[kQ4FewWaves][256];
    const int idx = blockIdx.x / RT, rt = blockIdx.x - idx * RT;
    const int wave = wave_id(), lane = threadIdx.x & 63, t = lane & 15, q = lane >> 4;
    int expert = 0, begin = idx * kTileTok, np = min(kTileTok, L.n_rows - begin);
    if (L.items != nullptr) {
        if (idx >= L.items[0].expert) return;
        expert = L.items[1 + idx].expert;
        begin = L.items[1 + idx].begin;
        np = L.items[1 + idx].rows;
    }
    const bool other = expert == L.w.n_mats;
    const cx_q4_desc& w = other ? L.shared : L.w;
    const size_t tile0 = ((size_t)(other ? 0 : max(expert, 0)) * RT + rt) * KT;
    const int p = begin + t, cols = L.w.cols;
    int xr = t < np && expert >= 0 ? p : -1;
    if (xr >= 0 && L.order != nullptr) {
        const int pair = L.order[p];
        xr = pair < 0 ? -1 : pair / L.top_k;
    }
    const bool live = xr >= 0 && xr < L.n_x;
    xr = live ? xr : 0;
    constexpr int kEl = XT == kQ4E4m3 ? 1 : 2;
    const char* x = static_cast<const char*>(L.x) + (size_t)xr * cols * kEl;
    const char* xl = XT == kQ4Planes ? static_cast<const char*>(L.x_lo) + (size_t)xr * cols * 2 : nullptr;
    const bool vec = cols % 8 == 0 && (reinterpret_cast<uintptr_t>(L.x) & (8 * kEl - 1)) == 0;
    f32x4 acc = {};
    for (int kt = wave; kt < KT && expert >= 0; kt += kQ4FewWaves) {
        const u32x4 a = ld16(w.codes + (tile0 + kt) * kQ4Tile + lane * 16);
        const uint32_t* sc = reinterpret_cast<const uint32_t*>(w.scales + (tile0 + kt) * 16 * NG) + q * 2 * NG;
        const float xs = XT == kQ4E4m3 && live ? L.x_scale[(size_t)xr * KT + kt] : 1.0f;
        f32x4 part = {};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int col = kt * 128 + 32 * j + 8 * q;
            const u32x4 b = live ? q4_x8<XT>(x, col, cols, vec) : u32x4{};
            if constexpr (XT == kQ4Fp16) {
                part = Mma<true>::mma(q4_f16(a[j]), Mma<true>::bits(b), part);
            } else {
                part = Mma<false>::mma(q4_bf16(a[j]), Mma<false>::bits(b), part);
                if constexpr (XT == kQ4Planes)
                    part = Mma<false>::mma(q4_bf16(a[j]), Mma<false>::bits(live ? q4_x8<XT>(xl, col, cols, vec) : u32x4{}), part);
            }
            if ((j + 1) % (4 / NG) == 0) {
                const int g = j / (4 / NG);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[i] += q4_scale(sc, i * NG + g) * (XT == kQ4E4m3 ? xs * part[i] : part[i]);
                part = f32x4{};
            }
        }
    }
    *reinterpret_cast<f32x4*>(&red[wave][t * 16 + q * 4]) = acc;
    __syncthreads();
    if (threadIdx.x >= 256) return;
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < kQ4FewWaves; ++i) v += red[i][threadIdx.x];
    const int tt = threadIdx.x >> 4, r = threadIdx.x & 15;
    v *= q4_row_scales(w)[tile0 / KT * 16 + (threadIdx.x & 15)];
    if (L.w.gated) {
        const float up = __shfl_down(v, 8);
        v = v / (1.0f + __expf(-v)) * up;
    }
    const int n = L.w.gated ? rt * 8 + r : rt * 16 + r, width = L.w.gated ? L.w.rows / 2 : L.w.rows;
    if (tt < np && n < width && (!L.w.gated || r < 8)) q4_store(L, (size_t)(begin + tt) * width + n, v);
}

}  // namespace cx
