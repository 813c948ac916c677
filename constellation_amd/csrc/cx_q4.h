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

#include <type_traits>

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

// Two fp32 values as two fp16 planes: in x each rounded to 11 bits, in y what that leaves of it,
// rounded to 11 bits again: together within 2^-23 of the value, or 2^-25 where the rest
// is below fp16's normal numbers.  Of an infinity or a NaN nothing is left.
__device__ __forceinline__ uint2 q4_planes(float a, float b) {
    const uint32_t ha = f16_rne(a), hb = f16_rne(b);
    auto rest = [](float v, uint32_t h) {
        const float r = v - static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(h)));
        return f16_rne(__builtin_fabsf(v) < __builtin_inff() ? r : 0.0f);
    };
    return uint2{ha | (hb << 16), rest(a, ha) | (rest(b, hb) << 16)};
}

// x's columns col .. col + 7 of one row as MFMA operand bits, element by element; columns past
// the row's end are zeros (the codes there are, too, but a NaN times zero is not).
template <int XT>
__device__ __forceinline__ u32x4 q4_x8(const char* row, int col, int cols) {
    if constexpr (XT == kQ4E4m3) {
        const uint8_t* p = reinterpret_cast<const uint8_t*>(row) + col;
        uint32_t a = 0, b = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i < cols) (i < 4 ? a : b) |= (uint32_t)p[i] << (8 * (i & 3));
        return u32x4{a, b, 0, 0};
    } else {
        const uint16_t* p = reinterpret_cast<const uint16_t*>(row) + col;
        u32x4 v = {};
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i < cols) v[i >> 1] |= (uint32_t)p[i] << (16 * (i & 1));
        return v;
    }
}

__device__ __forceinline__ float q4_scale(const uint32_t* sc, int i) {
    return static_cast<float>(__builtin_bit_cast(f16x2, sc[i >> 1])[i & 1]);
}

__device__ __forceinline__ void q4_store(const Q4Launch& L, size_t at, float v) {
    if (L.y_type == CX_DTYPE_F32) {
        static_cast<float*>(L.y)[at] = v;
    } else {
        static_cast<uint16_t*>(L.y)[at] = (uint16_t)cast_out(v, L.y_type);
    }
}

// Up to 16 rows of x against RW row tiles of weights per wave: the kernel streams a matrix's
// weights once per item.  With one row the latency of its loads bounds it, of weights and of x from L2 (18432 x
// 7168: 70 MB in 22.8 us, 3.1 of the 5 TB/s that the decode kernel reaches on more matrices; 4096 x
// 7168 in 7.2, of which a launch's ramp and the reduction are half), with 16 the reads of x, as many
// bytes as four times the weights' codes over RW, from L2 (32 and 11.7 us).  Products are of the bf16
// (fp16) x as it is with the codes, exact; the scales come to the fp32 sums of their group.
//  A workgroup's 8 waves are `splits` ranges of the columns times
// 8 / splits groups of row tiles; the partial sums of a group's ranges are added in order.
// Each wave keeps U column tiles of codes in flight ahead of those that it multiplies;
// the rows of x come from L2, for RW row tiles at once.
// VEC: rows of x as 16-byte (e4m3: 8-byte) bounded buffer loads, whose absent rows and
// columns read as zeros without a branch.
template <int XT, int NG, int RW, bool VEC>
__global__ __launch_bounds__(64 * kQ4FewWaves, 2) void k_q4_few(Q4Launch L, int RT, int KT, int splits, int row_blocks) {
    constexpr int kEl = XT == kQ4E4m3 ? 1 : 2;
    constexpr int U = !VEC ? 1 : RW == 1 ? 4 : 2;
    __shared__ float red[kQ4FewWaves][RW][256];
    const int idx = blockIdx.x / row_blocks, block = blockIdx.x - idx * row_blocks;
    const int wave = wave_id(), lane = threadIdx.x & 63, t = lane & 15, q = lane >> 4;
    const int groups = kQ4FewWaves / splits;
    int expert = 0, begin = idx * L.item_rows, np = min(L.item_rows, L.n_rows - begin);
    if (L.items != nullptr) {
        if (idx >= L.items[0].expert) return;
        const Q4Item it = ld_uniform(L.items + 1 + idx);
        expert = it.expert;
        begin = it.begin;
        np = it.rows;
    }
    const bool other = expert == L.w.n_mats;
    const cx_q4_desc& w = other ? L.shared : L.w;
    const size_t mat = other ? 0 : (size_t)max(expert, 0);
    const int cols = L.w.cols, rg = wave / splits, ks = wave - rg * splits;
    const int rt0 = (block * groups + rg) * RW;
    auto source = [&](int r) {  // row of x of row r of the item, -1: none
        int xr = r < np && expert >= 0 ? begin + r : -1;
        if (xr >= 0 && L.order != nullptr) {
            const int pair = L.order[xr];
            xr = pair < 0 ? -1 : pair / L.top_k;
        }
        return xr < L.n_x ? xr : -1;
    };
    const uint8_t* wp[RW];
    const uint16_t* sp[RW];
#pragma unroll
    for (int m = 0; m < RW; ++m) {
        const size_t tile = (mat * RT + min(rt0 + m, RT - 1)) * (size_t)KT;
        wp[m] = w.codes + tile * kQ4Tile;
        sp[m] = w.scales + tile * 16 * NG;
    }
    const int per = (KT + splits - 1) / splits, k0 = ks * per, k1 = expert < 0 || rt0 >= RT ? 0 : min(KT, k0 + per);
    u32x4 a[2][U][RW];
    uint32_t s[2][U][RW][2 * NG];
    auto fetch = [&](int kt0, auto to) {  // past the range: the last tile again, whose products are not added
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int kt = min(kt0 + u, k1 - 1);
#pragma unroll
            for (int m = 0; m < RW; ++m) {
                a[to][u][m] = ld16(wp[m] + (size_t)kt * kQ4Tile + (uint32_t)lane * 16);
                const uint32_t* sc = reinterpret_cast<const uint32_t*>(sp[m] + (size_t)kt * 16 * NG) + (uint32_t)q * 2 * NG;
#pragma unroll
                for (int i = 0; i < 2 * NG; ++i) s[to][u][m][i] = sc[i];
            }
        }
    };
    if (k0 < k1) fetch(k0, std::integral_constant<int, 0>{});
    const int xr = source(t);  // the lane's row
    const bool live = xr >= 0;
    const size_t row = (size_t)(live ? xr : 0) * cols * kEl;
    const char* x = static_cast<const char*>(L.x) + row;
    const uint32_t size = VEC ? (uint32_t)((size_t)L.n_x * cols * kEl) : 0;
    const __amdgpu_buffer_rsrc_t rx = make_rsrc(L.x, size);
    f32x4 acc[RW] = {};
    auto multiply = [&](int kt0, auto from) {
        u32x4 b[U][4];
        float xs[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int col = (kt0 + u) * 128 + 32 * j + 8 * q;
                const bool is = live && kt0 + u < k1 && col < cols;
                if constexpr (VEC) {
                    const uint32_t at = is ? (uint32_t)row + (uint32_t)col * kEl : kOob;
                    if constexpr (XT == kQ4E4m3) {
                        typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
                        const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rx, at, 0, 0));
                        b[u][j] = u32x4{v[0], v[1], 0, 0};
                    } else {
                        b[u][j] = bld16(rx, at);
                    }
                } else {
                    b[u][j] = is ? q4_x8<XT>(x, col, cols) : u32x4{};
                }
            }
            xs[u] = 1.0f;
            if constexpr (XT == kQ4E4m3) xs[u] = live ? L.x_scale[(size_t)xr * KT + min(kt0 + u, KT - 1)] : 1.0f;
        }
        if (kt0 + U < k1) fetch(kt0 + U, std::integral_constant<int, 1 - from>{});
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (kt0 + u >= k1) break;
            f32x4 part[RW] = {};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                u32x4 b0 = b[u][j];
                if constexpr (XT == kQ4E4m3) b0 = __builtin_bit_cast(u32x4, cvt8_bf16(b0[0], b0[1]));
#pragma unroll
                for (int m = 0; m < RW; ++m) {
                    if constexpr (XT == kQ4Fp16) {
                        part[m] = Mma<true>::mma(q4_f16(a[from][u][m][j]), Mma<true>::bits(b0), part[m]);
                    } else {
                        part[m] = Mma<false>::mma(q4_bf16(a[from][u][m][j]), Mma<false>::bits(b0), part[m]);
                    }
                    if ((j + 1) % (4 / NG) == 0) {
                        const int g = j / (4 / NG);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            acc[m][i] += q4_scale(s[from][u][m], i * NG + g) * (XT == kQ4E4m3 ? xs[u] * part[m][i] : part[m][i]);
                        part[m] = f32x4{};
                    }
                }
            }
        }
    };
    for (int kt = k0; kt < k1; kt += 2 * U) {
        multiply(kt, std::integral_constant<int, 0>{});
        if (kt + U < k1) multiply(kt + U, std::integral_constant<int, 1>{});
    }
#pragma unroll
    for (int m = 0; m < RW; ++m) *reinterpret_cast<f32x4*>(&red[wave][m][t * 16 + q * 4]) = acc[m];
    __syncthreads();
    // a row group's tiles by the threads of its waves, 256 outputs at a time
    const int width = L.w.gated ? L.w.rows / 2 : L.w.rows;
    for (int i = threadIdx.x; i < groups * RW * 256; i += 64 * kQ4FewWaves) {
        const int g = i / (RW * 256), m = i / 256 % RW, rt = (block * groups + g) * RW + m, tt = (i & 255) >> 4, r = i & 15;
        float v = 0.0f;
        for (int k = 0; k < splits; ++k) v += red[g * splits + k][m][i & 255];
        v *= q4_row_scales(w)[(mat * RT + min(rt, RT - 1)) * 16 + r];
        if (L.w.gated) {
            const float up = __shfl_down(v, 8);
            v = v / (1.0f + expf(-v)) * up;
        }
        const int n = L.w.gated ? rt * 8 + r : rt * 16 + r;
        if (tt < np && rt < RT && n < width && (!L.w.gated || r < 8)) q4_store(L, (size_t)(begin + tt) * width + n, v);
    }
}

}  // namespace cx
