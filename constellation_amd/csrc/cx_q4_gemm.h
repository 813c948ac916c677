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
    const float* x_scale;     // XS: [n_x, KT]
    int padded;               // columns of a row of x: KT * 128, twice that with two planes
    int n_x, n_rows, top_k;
    const int32_t* order;
    const Q4Item* items;
    void* y;
    int y_type;
    float* part;              // [splits, n_rows, RT * 16]
    int item_rows, splits;
    int RT, KT, RB;           // row tiles, column tiles, row blocks
};

constexpr int kQ4GemmWaves = 4;

// Workgroup: 4 waves of RTW row tiles each against an item of up to 16 NT rows of x.
// Each wave converts its own rows' codes, times their scales, to fp16 (exactly, see
// k_q4_row_scales) for the MFMAs of all the item's rows; the rows of x go straight from
// memory to one of two LDS buffers, a column tile ahead.  The buffers are two objects:
// the compiler then knows that reads of one need not wait for loads into the other.
//
// What bounds it: issue.  Beside an MFMA of 16 cycles a wave converts codes (a pack of two codes and
// a product with the scale for every two weights), reads a fragment of x and waits its turn; with
// 8 tiles of rows to a conversion and two workgroups a CU the matrix cores are busy 71 % of the time
// (4096 rows by 4096 x 7168: 192 us, 1.25 PFLOP/s; a library's bf16 product reaches 1.43 on
// this card).  Fewer rows per item amortise a conversion less: 1024 tokens over 64 experts, gate/up 472
// us and 63 %; the down product, whose h is two planes on one conversion, 439 us and 67 %.  Steps that led here,
// at that size (both products and what is around them): x through registers 1476 us, straight to LDS with
// fragments two steps ahead 1000, outputs turned in LDS 935, equal items and wide conversions 819, long
// items first 789; h in two planes 955 (11 bits of h were too few for fp16 and fp32 outputs).
constexpr int kQ4GemmBuf = kQ4GemmRows * 256;

// s_waitcnt vmcnt(0) lgkmcnt(0), then a barrier: the loads into the other buffer have
// arrived, and no wave still reads this one.
__device__ __forceinline__ void q4_gemm_turn() {
    __builtin_amdgcn_s_waitcnt(0x70);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// The accumulators, times the rows' powers of two, to y.  A wave turns 16 rows of x at a
// time in its own part of the LDS, so that it stores whole lines of y (as they lie in
// the accumulators, a lane has 4 neighbours of one row: 8 bytes in 16 bits).
template <int RTW, int NT>
__device__ __forceinline__ void q4_gemm_store(const Q4GemmArgs& L, const f32x4 (&acc)[NT][RTW], unsigned char* lds, const cx_q4_desc& w,
                                              size_t mat, int rb, int ks, int begin, int rows) {
    constexpr int kPitch = RTW * 16 + 4;  // floats; 16 rows' pieces then lie in different banks
    static_assert(16 * kPitch * 4 * kQ4GemmWaves <= kQ4GemmBuf, "turned tiles");
    const int wave = wave_id(), lane = threadIdx.x & 63, t = lane & 15, q = lane >> 4;
    float* turn = reinterpret_cast<float*>(lds) + wave * 16 * kPitch;
    const int rt0 = (rb * kQ4GemmWaves + wave) * RTW;
    const bool parts = L.splits > 1, gated = w.gated && !parts;  // partial sums: tiles as they are
    const int width = parts ? L.RT * 16 : gated ? w.rows / 2 : w.rows;
    const int c0 = rt0 * (gated ? 8 : 16), cols = RTW * (gated ? 8 : 16);  // of this wave
    void* out = parts ? L.part + (size_t)ks * L.n_rows * width : L.y;
    const bool wide = parts || L.y_type == CX_DTYPE_F32;
    const bool vec = width % (wide ? 4 : 8) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
    const int per = wide ? 4 : 8, lanes = cols / per;  // columns of a lane's store, lanes of a row
    f32x4 rs[RTW];
#pragma unroll
    for (int m = 0; m < RTW; ++m)
        rs[m] = *reinterpret_cast<const f32x4*>(q4_row_scales(w) + (mat * L.RT + min(rt0 + m, L.RT - 1)) * 16 + 4 * q);
    // rows n * 16 + t: whether they exist in x (rows of the order without a pair are zeros) and their power of two
    float xs[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int r = n * 16 + t, p = begin + r;
        xs[n] = 1.0f;
        if (r < rows && (L.order != nullptr || L.x_row_scale != nullptr)) {
            const int pair = L.order != nullptr ? L.order[p] : p, xr = L.order != nullptr ? pair / L.top_k : p;  // top_k: of an order only
            if (pair < 0 || xr >= L.n_x)
                xs[n] = 0.0f;
            else if (L.x_row_scale != nullptr)
                xs[n] = L.x_row_scale[xr];
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        if (n * 16 >= rows) continue;
#pragma unroll
        for (int m = 0; m < RTW; ++m) {
            f32x4 v = acc[n][m] * rs[m];
            v = xs[n] == 0.0f ? f32x4{} : v * f32x4{xs[n], xs[n], xs[n], xs[n]};
            int c = m * 16 + 4 * q;
            if (gated) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float up = __shfl_xor(v[i], 32);
                    v[i] = v[i] / (1.0f + expf(-v[i])) * up;
                }
                c = m * 8 + 4 * (q & 1);
            }
            if (!gated || q < 2) *reinterpret_cast<f32x4*>(turn + t * kPitch + c) = v;
        }
        __builtin_amdgcn_wave_barrier();
        for (int i = lane; i < 16 * lanes; i += 64) {
            const int r = i / lanes, c = (i - r * lanes) * per, left = width - c0 - c;
            if (n * 16 + r >= rows || left <= 0) continue;
            const float* src = turn + r * kPitch + c;
            const size_t at = (size_t)(begin + n * 16 + r) * width + c0 + c;
            if (wide) {
                const f32x4 v = *reinterpret_cast<const f32x4*>(src);
                float* y = static_cast<float*>(out) + at;
                if (vec) {
                    *reinterpret_cast<f32x4*>(y) = v;
                } else {
                    for (int k = 0; k < min(left, 4); ++k) y[k] = src[k];
                }
            } else {
                uint16_t* y = static_cast<uint16_t*>(out) + at;
                if (vec) {
                    const f32x4 a = *reinterpret_cast<const f32x4*>(src), b = *reinterpret_cast<const f32x4*>(src + 4);
                    *reinterpret_cast<u32x4*>(y) = u32x4{cast_out(a[0], L.y_type) | (cast_out(a[1], L.y_type) << 16), cast_out(a[2], L.y_type) | (cast_out(a[3], L.y_type) << 16),
                                                         cast_out(b[0], L.y_type) | (cast_out(b[1], L.y_type) << 16), cast_out(b[2], L.y_type) | (cast_out(b[3], L.y_type) << 16)};
                } else {
                    for (int k = 0; k < min(left, 8); ++k) y[k] = (uint16_t)cast_out(src[k], L.y_type);
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// XS (e4m3 rows of x, as fp16): each column tile's sums are scaled by the row's x_scale in
// fp32 before they are added up, with items of up to 64 rows for the second set of sums.
// The matrix cores' own 8-bit products would be twice as fast, but drop what lies 2^13
// below the largest product of an instruction, and sums here are kept to fp32.  The second set of
// sums costs a multiply-add per MFMA and 4 values, and half the rows per conversion: 3001
// rows by 7168 x 2048 in 101 to 116 us, 0.8 to 0.87 PFLOP/s (128 rows and one workgroup a CU: 8 % slower).
//
// PL (fp32 rows of x, the h of a layer, as two fp16 planes; row p of x is row p of y): a buffer holds 64
// columns, 8 pieces of a row's first plane and the 8 of its second, so that a buffer and a turn have
// as many MFMAs as without planes and a conversion serves both planes of all rows.  Items of up to 64 rows, whose
// weights bound them, have a whole column tile of both planes in a buffer instead, and half the turns (16 and 128
// tokens over 64 experts 342 and 357 us, in halves 349 and 375).
template <int NG, int RTW, int NT, bool XS, bool PL>
__device__ __forceinline__ void q4_gemm_tile(const Q4GemmArgs& L, unsigned char* lds0, unsigned char* lds1, const cx_q4_desc& w,
                                             size_t mat, int rb, int ks, int begin, int rows) {
    const int wave = wave_id(), lane = threadIdx.x & 63, t = lane & 15, q = lane >> 4;
    const int KT = L.KT;
    // x: load i brings rows 16 i + 4 wave .. + 3 of the item, each lane 16 bytes; slot s of
    // row r gets the row's piece s ^ (r % 16), so that the 16 rows of a fragment lie in
    // 16 different places of the banks.
    const int tr = threadIdx.x >> 4, piece = (threadIdx.x & 15) ^ tr;
    constexpr bool kHalf = PL && NT > 4;         // a fetch is half a column tile
    constexpr int kPieces = PL && !kHalf ? 2 : 1;  // 256-byte pieces of a row in a fetch
    const uint32_t pitch = (uint32_t)L.padded * 2;
    uint32_t xoff[NT];  // in bytes; rows that do not exist read another and are never stored
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const int r = i * 16 + tr;
        int xr = (PL ? 0 : begin) + (r < rows ? r : 0);
        if (!PL && L.order != nullptr) xr = max(L.order[xr], 0) / L.top_k;
        xoff[i] = (uint32_t)(PL || xr < L.n_x ? xr : 0) * pitch + piece * 16;
    }
    const int rt0 = min((rb * kQ4GemmWaves + wave) * RTW, L.RT - 1), rts = min(RTW, L.RT - rt0);  // row tiles past the matrix: its last one again
    const size_t tile0 = (mat * L.RT + rt0) * (size_t)KT;
    const uint8_t* wp = w.codes + tile0 * kQ4Tile;
    const uint16_t* sp = w.scales + tile0 * 16 * NG;
    // kBounded: loads of a lane's 32-bit place and a scalar one, with planes of the item's own rows, where the compiler
    // spills otherwise: with planes (down products of 1024 tokens over 64 experts 439 us, 599 with plain loads) and with
    // the four scales of groups of 32 (1024 rows by 4096 x 7168: 74.6 us, 84.9). The others are faster with plain loads
    // (4096 rows by 4096 x 7168, groups of 64 and 128: 192 and 193 us, 199 bounded; e4m3, 3001 rows by 7168 x 2048: 108.4, 110.8).
    constexpr bool kBounded = PL || (NG == 4 && !XS);
    const __amdgpu_buffer_rsrc_t rx = make_rsrc(reinterpret_cast<const char*>(L.x) + (PL ? (size_t)begin * pitch : 0), (PL ? (uint32_t)rows : (uint32_t)L.n_x) * pitch);
    const __amdgpu_buffer_rsrc_t rw = make_rsrc(wp, (uint32_t)(rts * KT) * kQ4Tile), rs = make_rsrc(sp, (uint32_t)(rts * KT) * 32 * NG);
    // of a fetch: the lane's codes, and its row's scales
    typedef uint32_t Codes __attribute__((ext_vector_type(kHalf ? 2 : 4)));
    struct Sc {
        uint32_t d[kHalf ? 1 : (NG + 1) / 2];
    };
    f32x4 acc[NT][RTW] = {}, sum[XS ? NT : 1][RTW] = {};
    Codes a[2][RTW];
    Sc s[2][RTW];
    uint32_t xso = 0;  // XS: wave 0 brings the rows' scales, a lane each, behind their 64 rows
    if constexpr (XS) {
        static_assert(NT <= 4, "64 rows");
        int xr = begin + (lane < rows ? lane : 0);
        if (L.order != nullptr) xr = max(L.order[xr], 0) / L.top_k;
        xso = (uint32_t)(xr < L.n_x ? xr : 0) * (uint32_t)KT;
    }
    auto fetch = [&](int part, auto to, unsigned char* buf) {  // part: column tile (kHalf: its half `to`)
#pragma unroll
        for (int i = 0; i < NT * kPieces; ++i) {
            const auto at = (__attribute__((address_space(3))) void*)(buf + i * 4096 + wave * 1024);
            if constexpr (kBounded)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, at, 16, xoff[i % NT], (part * kPieces + i / NT) * 256, 0, 0);
            else
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(reinterpret_cast<const char*>(L.x) + (size_t)part * 256 + xoff[i]), at, 16, 0, 0);
        }
#pragma unroll
        for (int m = 0; m < RTW; ++m) {
            const int tile = min(m, rts - 1) * KT + (kHalf ? part >> 1 : part);
            if constexpr (!kBounded) {
                a[to][m] = ld16(wp + (size_t)tile * kQ4Tile + (uint32_t)lane * 16);
                if constexpr (NG == 1)
                    s[to][m].d[0] = (sp + (size_t)tile * 16)[(uint32_t)t];
                else
                    s[to][m] = *reinterpret_cast<const Sc*>(sp + (size_t)tile * 16 * NG + (uint32_t)t * NG);
                continue;
            }
            if constexpr (kHalf)
                a[to][m] = __builtin_bit_cast(Codes, __builtin_amdgcn_raw_buffer_load_b64(rw, lane * 16 + to * 8, tile * kQ4Tile, 0));
            else
                a[to][m] = __builtin_bit_cast(Codes, __builtin_amdgcn_raw_buffer_load_b128(rw, lane * 16, tile * kQ4Tile, 0));
            if constexpr (NG == 1)
                s[to][m].d[0] = __builtin_amdgcn_raw_buffer_load_b16(rs, t * 2, tile * 32, 0);
            else if constexpr (NG == 2 || kHalf)  // the tile's two scales, or its half's two of four
                s[to][m].d[0] = __builtin_amdgcn_raw_buffer_load_b32(rs, t * 2 * NG + (NG == 4 ? to * 4 : 0), tile * 32 * NG, 0);
            else
                s[to][m] = __builtin_bit_cast(Sc, __builtin_amdgcn_raw_buffer_load_b64(rs, t * 8, tile * 128, 0));
        }
        if constexpr (XS)
            if (wave == 0)
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(L.x_scale + part + xso),
                                                 (__attribute__((address_space(3))) void*)(buf + 16384), 4, 0, 0);
    };
    auto scaled_add = [&](const unsigned char* buf, int n) {
        if constexpr (XS) {
            const float x = *reinterpret_cast<const float*>(buf + 16384 + (n * 16 + t) * 4);
#pragma unroll
            for (int m = 0; m < RTW; ++m) {
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[n][m][i] = __builtin_fmaf(x, acc[n][m][i], sum[n][m][i]);
                asm volatile("" : "+v"(sum[n][m]));
            }
        }
    };
    auto multiply = [&](auto from, const unsigned char* buf) {
        // Steps of RTW MFMAs on one fragment of x, in this order: the fragment after the
        // next is read and the next columns' weights are converted while they run.
        const unsigned char* in = buf + t * 256;
        constexpr int kSteps = 4 * NT * kPieces, kOf = PL ? 2 * NT : NT;  // steps that share a conversion: those of all rows, with planes of both
        f16x8 fa[2][RTW];
        u32x4 b[3];
        auto convert = [&](int j, int m) {  // of the fetch's columns 32 j .. + 31
            const int g = (kHalf ? from * 2 + j : j) * NG / 4 - (kHalf && NG == 4 ? from * 2 : 0);
            const _Float16 sc = __builtin_bit_cast(f16x2, s[from][m].d[g / 2])[g % 2];
            fa[j & 1][m] = q4_f16(a[from][m][j]) * f16x8{sc, sc, sc, sc, sc, sc, sc, sc};
        };
        auto read = [&](int i) {
            const int j = i / kOf, plane = i % kOf / NT, piece = PL ? plane * 2 + j % 2 : j;
            b[i % 3] = *reinterpret_cast<const u32x4*>(in + ((PL ? j / 2 * NT : 0) + i % NT) * 4096 + (((piece * 4 + q) ^ t) * 16));
        };
        read(0);
        read(1);
#pragma unroll
        for (int m = 0; m < RTW; ++m) convert(0, m);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int j = i / kOf, at = i % kOf, n = i % NT;
            __builtin_amdgcn_sched_barrier(0);
            if (i + 2 < kSteps) read(i + 2);
            if (j + 1 < kSteps / kOf && at >= kOf - NT)  // late: registers
#pragma unroll
                for (int m = n * RTW / NT; m < (n + 1) * RTW / NT; ++m) convert(j + 1, m);
#pragma unroll
            for (int m = 0; m < RTW; ++m)
                acc[n][m] = Mma<true>::mma(fa[j & 1][m], Mma<true>::bits(b[i % 3]), XS && j == 0 ? f32x4{} : acc[n][m]);
            if (XS && j == 3 && n > 0) scaled_add(buf, n - 1);  // while this step's products are on their way
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (XS) {
            scaled_add(buf, NT - 1);
        } else {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int m = 0; m < RTW; ++m) asm volatile("" : "+v"(acc[n][m]));  // keeps the sums where they are: no copies of them at the loop's end
        }
    };
    constexpr std::integral_constant<int, 0> even{};
    constexpr std::integral_constant<int, 1> odd{};
    constexpr int kParts = kHalf ? 2 : 1;  // of a column tile
    const int per = (KT + L.splits - 1) / L.splits, k0 = ks * per * kParts, k1 = min(KT * kParts, k0 + per * kParts);
    if (k0 < k1) fetch(k0, even, lds0);
    q4_gemm_turn();
    for (int k = k0; k < k1; k += 2) {
        if (kHalf || k + 1 < k1) fetch(k + 1, odd, lds1);
        multiply(even, lds0);
        q4_gemm_turn();
        if (!kHalf && k + 1 >= k1) break;
        if (k + 2 < k1) fetch(k + 2, even, lds0);
        multiply(odd, lds1);
        q4_gemm_turn();
    }
    if constexpr (XS)
        q4_gemm_store<RTW, NT>(L, sum, lds0, w, mat, rb, ks, begin, rows);
    else
        q4_gemm_store<RTW, NT>(L, acc, lds0, w, mat, rb, ks, begin, rows);
}

template <int NG, int RTW, bool XS, bool PL>
__global__ __launch_bounds__(64 * kQ4GemmWaves, 2) void k_q4_gemm(Q4GemmArgs L) {
    __shared__ __attribute__((aligned(16))) unsigned char lds0[kQ4GemmBuf], lds1[kQ4GemmBuf];
    const int per = L.RB * L.splits, idx = blockIdx.x / per, unit = blockIdx.x - idx * per, ks = unit / L.RB, rb = unit - ks * L.RB;
    int expert = 0, begin = idx * L.item_rows, rows = min(L.item_rows, L.n_rows - begin);
    if (L.items != nullptr) {
        if (idx >= L.items[0].expert) return;
        const Q4Item it = ld_uniform(L.items + 1 + idx);
        expert = it.expert;
        begin = it.begin;
        rows = it.rows;
    }
    if (expert < 0) {  // rows behind the last matrix's
        const bool parts = L.splits > 1, wide = parts || L.y_type == CX_DTYPE_F32;
        const int width = parts ? L.RT * 16 : L.w.gated ? L.w.rows / 2 : L.w.rows;
        const int n = kQ4GemmWaves * RTW * (L.w.gated && !parts ? 8 : 16), left = width - rb * n;
        char* out = parts ? reinterpret_cast<char*>(L.part + (size_t)ks * L.n_rows * width) : static_cast<char*>(L.y);
        const size_t el = wide ? 4 : 2;
        for (int r = 0; r < rows; ++r)
            for (int c = threadIdx.x * 2; c < min(n, left) * (int)el; c += 128 * kQ4GemmWaves)
                *reinterpret_cast<uint16_t*>(out + ((size_t)(begin + r) * width + rb * n) * el + c) = 0;
        return;
    }
    const bool other = expert == L.w.n_mats;
    const cx_q4_desc& w = other ? L.shared : L.w;
    const size_t mat = other ? 0 : (size_t)expert;
    auto tile = [&](auto nt) {
        q4_gemm_tile<NG, RTW, nt, XS, PL>(L, lds0, lds1, w, mat, rb, ks, begin, rows);
    };
    if constexpr (!XS) {
        if (rows > 112) return tile(std::integral_constant<int, 8>{});
        if (rows > 96) return tile(std::integral_constant<int, 7>{});
        if (rows > 80) return tile(std::integral_constant<int, 6>{});
        if (rows > 64) return tile(std::integral_constant<int, 5>{});
    }
    if (rows > 48)
        tile(std::integral_constant<int, 4>{});
    else if (rows > 32)
        tile(std::integral_constant<int, 3>{});
    else
        tile(std::integral_constant<int, 2>{});
}

// The partial sums of the ranges, added in order, and what follows the sums.
__global__ __launch_bounds__(256) void k_q4_sum(const float* part, int splits, int n_rows, int pitch, int gated, int width, void* y,
                                                int y_type, int units) {
    const size_t at = (size_t)blockIdx.x * 256 + threadIdx.x;
    const size_t p = at / units;
    const int n = (int)(at - p * units) * 4;
    if (p >= (size_t)n_rows) return;
    const float* src = part + p * pitch + (gated ? n / 8 * 16 + n % 8 : n);
    f32x4 a = {}, b = {};
    for (int s = 0; s < splits; ++s) {
        a += *reinterpret_cast<const f32x4*>(src + (size_t)s * n_rows * pitch);
        if (gated) b += *reinterpret_cast<const f32x4*>(src + (size_t)s * n_rows * pitch + 8);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float v = gated ? a[i] / (1.0f + expf(-a[i])) * b[i] : a[i];
        if (n + i >= width) continue;
        if (y_type == CX_DTYPE_F32)
            static_cast<float*>(y)[p * width + n + i] = v;
        else
            static_cast<uint16_t*>(y)[p * width + n + i] = (uint16_t)cast_out(v, y_type);
    }
}

}  // namespace cx
