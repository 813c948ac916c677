// cx_q4_gemm.h — products with 4-bit weights for many rows of x per matrix: a GEMM
// whose weights go from memory to the matrix cores through registers alone.
#pragma once

#include "cx_q4.h"

namespace cx {

// The rows of x as a workgroup reads them: fp16, whole 128-column tiles, aligned.
struct Q4GemmArgs {
    cx_q4_desc w, shared;
    const uint16_t* x;        // [n_x, padded]
    const float* x_row_scale; // nullable [n_x]
    int padded;               // columns of a row of x: KT * 128
    int n_x, n_rows, top_k;
    const int32_t* order;
    const Q4Item* items;
    void* y;
    int y_type;
    int RT, KT, RB;           // row tiles, column tiles, row blocks
};

constexpr int kQ4GemmWaves = 4;

// Workgroup: 4 waves of RTW row tiles each against an item of up to 16 NT rows of x.
// Each wave converts its own rows' codes, times their scales, to fp16 (exactly, see
// k_q4_row_scales) for the MFMAs of all the item's rows; the rows of x go through a
// double buffer in LDS, fetched a column tile ahead through registers.
template <int NG, int RTW, int NT>
__device__ __forceinline__ void q4_gemm_tile(const Q4GemmArgs& L, unsigned char* lds, const cx_q4_desc& w, size_t mat, int rb,
                                             int begin, int rows) {
    constexpr int kBuf = NT * 4096;  // 16 NT rows x 256 bytes
    const int wave = wave_id(), lane = threadIdx.x & 63, t = lane & 15, q = lane >> 4;
    const int KT = L.KT;
    // x: thread i % 16 of a row's 16 threads takes 16-byte piece i % 16
    const int tr = threadIdx.x >> 4, piece = threadIdx.x & 15;
    uint32_t xoff[NT];  // in 16-byte pieces; rows that do not exist read row 0 and are never stored
    uint32_t zero = 0;  // rows of the order without a pair
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const int r = i * 16 + tr, p = begin + (r < rows ? r : 0);
        int xr = p;
        if (L.order != nullptr) {
            const int pair = L.order[p];
            xr = pair < 0 ? -1 : pair / L.top_k;
        }
        if (xr < 0 || xr >= L.n_x) {
            xr = 0;
            zero |= 1u << i;
        }
        xoff[i] = (uint32_t)xr * (uint32_t)(L.padded / 8) + piece;
    }
    const u32x4* xg = reinterpret_cast<const u32x4*>(L.x);
    const uint8_t* wp[RTW];
    const uint16_t* sp[RTW];
#pragma unroll
    for (int m = 0; m < RTW; ++m) {
        const int rt = min((rb * kQ4GemmWaves + wave) * RTW + m, L.RT - 1);
        const size_t tile = (mat * L.RT + rt) * (size_t)KT;
        wp[m] = w.codes + tile * kQ4Tile + lane * 16;
        sp[m] = w.scales + tile * 16 * NG + t * NG;
    }
    typedef uint16_t Sc __attribute__((ext_vector_type(NG == 1 ? 2 : NG)));
    f32x4 acc[NT][RTW] = {};
    u32x4 a_next[RTW], x_next[NT];
    Sc s_next[RTW];
    auto fetch = [&](int kt) {
#pragma unroll
        for (int m = 0; m < RTW; ++m) {
            a_next[m] = ld16(wp[m] + (size_t)kt * kQ4Tile);
            if constexpr (NG == 1)
                s_next[m][0] = sp[m][kt * 16];
            else
                s_next[m] = *reinterpret_cast<const Sc*>(sp[m] + kt * 16 * NG);
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) x_next[i] = ld16(xg + (size_t)xoff[i] + kt * 16);
    };
    auto publish = [&](int buf) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
            *reinterpret_cast<u32x4*>(lds + buf * kBuf + (i * 16 + tr) * 256 + (piece ^ tr) * 16) =
                zero >> i & 1 ? u32x4{} : x_next[i];
    };
    fetch(0);
    publish(0);
    __syncthreads();
    for (int kt = 0; kt < KT; ++kt) {
        u32x4 a[RTW];
        Sc s[RTW];
#pragma unroll
        for (int m = 0; m < RTW; ++m) a[m] = a_next[m], s[m] = s_next[m];
        if (kt + 1 < KT) fetch(kt + 1);
        const unsigned char* in = lds + (kt & 1) * kBuf + t * 256;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f16x8 fa[RTW];
#pragma unroll
            for (int m = 0; m < RTW; ++m) {
                const _Float16 sc = __builtin_bit_cast(_Float16, (uint16_t)s[m][j * NG / 4]);
                const f16x8 c = q4_f16(a[m][j]);
                fa[m] = c * f16x8{sc, sc, sc, sc, sc, sc, sc, sc};
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const u32x4 b = *reinterpret_cast<const u32x4*>(in + n * 4096 + (((j * 4 + q) ^ t) * 16));
#pragma unroll
                for (int m = 0; m < RTW; ++m) acc[n][m] = Mma<true>::mma(fa[m], Mma<true>::bits(b), acc[n][m]);
            }
        }
        if (kt + 1 < KT) publish((kt + 1) & 1);
        __syncthreads();
    }
    const int width = w.gated ? w.rows / 2 : w.rows;
    const float* rs = q4_row_scales(w) + mat * L.RT * 16;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int r = n * 16 + t, p = begin + r;
        float xs = 1.0f;
        if (L.x_row_scale != nullptr && r < rows) {
            const int xr = L.order != nullptr ? max(L.order[p], 0) / L.top_k : p;
            xs = xr < L.n_x ? L.x_row_scale[xr] : 1.0f;
        }
#pragma unroll
        for (int m = 0; m < RTW; ++m) {
            const int rt = (rb * kQ4GemmWaves + wave) * RTW + m;
            f32x4 v = acc[n][m];
            if (rt < L.RT) v *= *reinterpret_cast<const f32x4*>(rs + rt * 16 + 4 * q);
            v *= f32x4{xs, xs, xs, xs};
            int c = rt * 16 + 4 * q;
            bool mine = rt < L.RT && r < rows;
            if (w.gated) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float up = __shfl_xor(v[i], 32);
                    v[i] = v[i] / (1.0f + __expf(-v[i])) * up;
                }
                c = rt * 8 + 4 * q;
                mine = mine && q < 2;
            }
            const size_t at = (size_t)p * width + c;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (!mine || c + i >= width) continue;
                if (L.y_type == CX_DTYPE_F32)
                    static_cast<float*>(L.y)[at + i] = v[i];
                else
                    static_cast<uint16_t*>(L.y)[at + i] = (uint16_t)cast_out(v[i], L.y_type);
            }
        }
    }
}

template <int NG, int RTW>
__global__ __launch_bounds__(64 * kQ4GemmWaves, 2) void k_q4_gemm(Q4GemmArgs L) {
    __shared__ __attribute__((aligned(16))) unsigned char lds[2 * 8 * 4096];
    const int idx = blockIdx.x / L.RB, rb = blockIdx.x - idx * L.RB;
    int expert = 0, begin = idx * kQ4GemmRows, rows = min(kQ4GemmRows, L.n_rows - begin);
    if (L.items != nullptr) {
        if (idx >= L.items[0].expert) return;
        const Q4Item it = ld_uniform(L.items + 1 + idx);
        expert = it.expert;
        begin = it.begin;
        rows = it.rows;
    }
    if (expert < 0) {  // rows behind the last matrix's
        const int width = L.w.gated ? L.w.rows / 2 : L.w.rows, per = kQ4GemmWaves * RTW * (L.w.gated ? 8 : 16);
        const int size = L.y_type == CX_DTYPE_F32 ? 2 : 1;  // in 16-bit units
        for (int r = 0; r < rows; ++r)
            for (int c = threadIdx.x; c < per * size; c += 64 * kQ4GemmWaves)
                if (rb * per * size + c < width * size) static_cast<uint16_t*>(L.y)[((size_t)(begin + r) * width) * size + rb * per * size + c] = 0;
        return;
    }
    const bool other = expert == L.w.n_mats;
    const cx_q4_desc& w = other ? L.shared : L.w;
    const size_t mat = other ? 0 : (size_t)expert;
    if (rows > 96)
        q4_gemm_tile<NG, RTW, 8>(L, lds, w, mat, rb, begin, rows);
    else if (rows > 64)
        q4_gemm_tile<NG, RTW, 6>(L, lds, w, mat, rb, begin, rows);
    else if (rows > 32)
        q4_gemm_tile<NG, RTW, 4>(L, lds, w, mat, rb, begin, rows);
    else
        q4_gemm_tile<NG, RTW, 2>(L, lds, w, mat, rb, begin, rows);
}

}  // namespace cx
