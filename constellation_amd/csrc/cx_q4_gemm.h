// cx_q4_gemm.h — products with 4-bit weights for many rows of x per matrix: a GEMM
// whose weights go from memory to the matrix cores through registers alone.
#pragma once

#include <type_traits>

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
// k_q4_row_scales) for the MFMAs of all the item's rows; the rows of x go straight from
// memory to one of two LDS buffers, a column tile ahead.  The buffers are two objects:
// the compiler then knows that reads of one need not wait for loads into the other.
constexpr int kQ4GemmBuf = kQ4GemmRows * 256;

// s_waitcnt vmcnt(0) lgkmcnt(0), then a barrier: the loads into the other buffer have
// arrived, and no wave still reads this one.
__device__ __forceinline__ void q4_gemm_turn() {
    __builtin_amdgcn_s_waitcnt(0x70);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

template <int NG, int RTW, int NT>
__device__ __forceinline__ void q4_gemm_tile(const Q4GemmArgs& L, unsigned char* lds0, unsigned char* lds1, const cx_q4_desc& w,
                                             size_t mat, int rb, int begin, int rows) {
    const int wave = wave_id(), lane = threadIdx.x & 63, t = lane & 15, q = lane >> 4;
    const int KT = L.KT;
    // x: load i brings rows 16 i + 4 wave .. + 3 of the item, each lane 16 bytes; slot s of
    // row r gets the row's piece s ^ (r % 16), so that the 16 rows of a fragment lie in
    // 16 different places of the banks.
    const int tr = threadIdx.x >> 4, piece = (threadIdx.x & 15) ^ tr;
    uint32_t xoff[NT];  // in 16-byte pieces; rows that do not exist read another and are never stored
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const int r = i * 16 + tr;
        int xr = begin + (r < rows ? r : 0);
        if (L.order != nullptr) xr = max(L.order[xr], 0) / L.top_k;
        xoff[i] = (uint32_t)(xr < L.n_x ? xr : 0) * (uint32_t)(L.padded / 8) + piece;
    }
    const uint8_t* wp[RTW];
    const uint16_t* sp[RTW];
#pragma unroll
    for (int m = 0; m < RTW; ++m) {
        const int rt = min((rb * kQ4GemmWaves + wave) * RTW + m, L.RT - 1);
        const size_t tile = (mat * L.RT + rt) * (size_t)KT;
        wp[m] = w.codes + tile * kQ4Tile + lane * 16;
        sp[m] = w.scales + tile * 16 * NG + t * NG;
    }
    struct Sc {  // the lane's row's scales of a tile
        uint32_t d[(NG + 1) / 2];
    };
    f32x4 acc[NT][RTW] = {};
    u32x4 a[2][RTW];
    Sc s[2][RTW];
    auto fetch = [&](int kt, auto to, unsigned char* buf) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(L.x + ((size_t)xoff[i] + kt * 16) * 8),
                                             (__attribute__((address_space(3))) void*)(buf + i * 4096 + wave * 1024), 16, 0, 0);
#pragma unroll
        for (int m = 0; m < RTW; ++m) {
            a[to][m] = ld16(wp[m] + (size_t)kt * kQ4Tile);
            if constexpr (NG == 1)
                s[to][m].d[0] = sp[m][kt * 16];
            else
                s[to][m] = *reinterpret_cast<const Sc*>(sp[m] + kt * 16 * NG);
        }
    };
    auto multiply = [&](auto from, const unsigned char* buf) {
        // Steps of RTW MFMAs on one fragment of x, in this order: the fragment after the
        // next is read and the next columns' weights are converted while they run.
        const unsigned char* in = buf + t * 256;
        constexpr int kSteps = 4 * NT;
        f16x8 fa[2][RTW];
        u32x4 b[3];
        auto convert = [&](int j, int m) {
            const int g = j * NG / 4;
            const _Float16 sc = __builtin_bit_cast(f16x2, s[from][m].d[g / 2])[g % 2];
            fa[j & 1][m] = q4_f16(a[from][m][j]) * f16x8{sc, sc, sc, sc, sc, sc, sc, sc};
        };
        auto read = [&](int i) { b[i % 3] = *reinterpret_cast<const u32x4*>(in + i % NT * 4096 + (((i / NT * 4 + q) ^ t) * 16)); };
        read(0);
        read(1);
#pragma unroll
        for (int m = 0; m < RTW; ++m) convert(0, m);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int j = i / NT, n = i % NT;
            __builtin_amdgcn_sched_barrier(0);
            if (i + 2 < kSteps) read(i + 2);
            if (j < 3)
#pragma unroll
                for (int m = n * RTW / NT; m < (n + 1) * RTW / NT; ++m) convert(j + 1, m);
#pragma unroll
            for (int m = 0; m < RTW; ++m) acc[n][m] = Mma<true>::mma(fa[j & 1][m], Mma<true>::bits(b[i % 3]), acc[n][m]);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    constexpr std::integral_constant<int, 0> even{};
    constexpr std::integral_constant<int, 1> odd{};
    fetch(0, even, lds0);
    q4_gemm_turn();
    for (int kt = 0; kt < KT; kt += 2) {
        if (kt + 1 < KT) fetch(kt + 1, odd, lds1);
        multiply(even, lds0);
        q4_gemm_turn();
        if (kt + 1 >= KT) break;
        if (kt + 2 < KT) fetch(kt + 2, even, lds0);
        multiply(odd, lds1);
        q4_gemm_turn();
    }
    const int width = w.gated ? w.rows / 2 : w.rows;
    const float* rs = q4_row_scales(w) + mat * L.RT * 16;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int r = n * 16 + t, p = begin + r;
        float xs = 1.0f;
        bool none = false;  // a row of the order without a pair: zeros
        if (r < rows && (L.order != nullptr || L.x_row_scale != nullptr)) {
            const int pair = L.order != nullptr ? L.order[p] : p * L.top_k, xr = pair / L.top_k;
            none = pair < 0 || xr >= L.n_x;
            if (!none && L.x_row_scale != nullptr) xs = L.x_row_scale[xr];
        }
#pragma unroll
        for (int m = 0; m < RTW; ++m) {
            const int rt = (rb * kQ4GemmWaves + wave) * RTW + m;
            f32x4 v = acc[n][m];
            if (rt < L.RT) v *= *reinterpret_cast<const f32x4*>(rs + rt * 16 + 4 * q);
            v = none ? f32x4{} : v * f32x4{xs, xs, xs, xs};
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
    __shared__ __attribute__((aligned(16))) unsigned char lds0[kQ4GemmBuf], lds1[kQ4GemmBuf];
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
        q4_gemm_tile<NG, RTW, 8>(L, lds0, lds1, w, mat, rb, begin, rows);
    else if (rows > 64)
        q4_gemm_tile<NG, RTW, 6>(L, lds0, lds1, w, mat, rb, begin, rows);
    else if (rows > 32)
        q4_gemm_tile<NG, RTW, 4>(L, lds0, lds1, w, mat, rb, begin, rows);
    else
        q4_gemm_tile<NG, RTW, 2>(L, lds0, lds1, w, mat, rb, begin, rows);
}

}  // namespace cx
