// cx_q4_dec.h — products with 4-bit weights for up to four rows of x per item: decode.
#pragma once

#include "cx_q4.h"

namespace cx {

struct Q4DecArgs {
    Q4Launch L;
    Q4Routes routes;
    int RT, KT;
    int splits;      // ranges of the columns per row tile
    int row_blocks;  // workgroups per item
    int lds_rows;    // rows of x staged, at most 4
};

// A wave's ring of column tiles of one row tile: codes, and the scales of the lane's row.  The
// loads are bounded, so that tiles past the range read as zeros and cost nothing.
template <int NG, int U>
struct Q4Ring {
    u32x4 a[U];
    uint32_t s[U][(NG + 1) / 2];

    __device__ __forceinline__ void fetch(__amdgpu_buffer_rsrc_t codes, __amdgpu_buffer_rsrc_t scales, int kt, int u, int lane) {
        a[u] = bld16(codes, (uint32_t)kt * kQ4Tile + (uint32_t)lane * 16);
        const uint32_t at = (uint32_t)kt * 32 * NG + (uint32_t)(lane & 15) * 2 * NG;
        if constexpr (NG == 1) {
            s[u][0] = __builtin_amdgcn_raw_buffer_load_b16(scales, at, 0, 0);
        } else if constexpr (NG == 2) {
            s[u][0] = __builtin_amdgcn_raw_buffer_load_b32(scales, at, 0, 0);
        } else {
            typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
            const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(scales, at, 0, 0));
            s[u][0] = v[0], s[u][1] = v[1];
        }
    }
    // The lane's eight weights of MFMA j of the tile in place u.
    __device__ __forceinline__ f16x8 weights(int u, int j) const {
        const int g = j * NG / 4;
        const _Float16 sc = __builtin_bit_cast(f16x2, s[u][g / 2])[g % 2];
        return q4_f16(a[u][j]) * f16x8{sc, sc, sc, sc, sc, sc, sc, sc};
    }
};

// A wave takes one row tile and one range of the column tiles; the partial sums of the ranges
// are added in order.  HBM bounds it as long as enough bytes are in flight: a wave's ring holds U
// tiles of codes (1 KB each) and refills a place as soon as it has multiplied it.  Gate and up
// of 8 experts of 7168 x 2048 for one token, 121 MB: 24 us, 5 TB/s; 64 rows over 40 of 64 matrices of 4096 x 7168,
// 605 MB: 122 us.  (x from L2, as the kernel of few rows has it: 161 us.)
//
// x is staged once per workgroup as fp16 in LDS: fp16 and e4m3 values as they are, others
// times the power of two that brings the row's largest value to 2^14 .. 2^15 (bf16 is then
// exact down to 2^-31 of it).  fp32, the h of an expert, is staged as two planes (q4_planes), whose
// products are two of the MFMA's 16 columns, so that the second one costs LDS and no time.  The codes
// times their scales are exact in fp16 (k_q4_row_scales), so the MFMAs sum exact products.
template <int XT, int NG, int U>
__global__ __launch_bounds__(64 * kQ4DecWaves) void k_q4_dec(Q4DecArgs A) {
    constexpr bool kScaled = XT == kQ4E4m3;  // a scale per row and column tile
    constexpr int kPlanes = XT == kQ4F32 ? 2 : 1;
    const Q4Launch& L = A.L;
    __shared__ float row_up[4];
    __shared__ uint32_t tops[4][kQ4DecWaves];
    extern __shared__ __attribute__((aligned(16))) unsigned char staged[];
    const int RT = A.RT, KT = A.KT, idx = blockIdx.x / A.row_blocks, block = blockIdx.x - idx * A.row_blocks;
    const int wave = wave_id(), lane = threadIdx.x & 63, t = lane & 15, q = lane >> 4, tid = threadIdx.x;
    const int groups = kQ4DecWaves / A.splits, rg = wave / A.splits, ks = wave - rg * A.splits;
    int expert = 0, begin = idx * L.item_rows, np = min(L.item_rows, L.n_rows - begin);
    if (L.items != nullptr) {
        if (idx >= L.items[0].expert) return;
        const Q4Item it = ld_uniform(L.items + 1 + idx);
        expert = it.expert;
        begin = it.begin;
        np = it.rows;
    }
    int x_row = -1;  // with routes: the token
    if (A.routes.ids != nullptr || A.routes.shared) {
        const int ke = A.routes.top_k + A.routes.shared;
        x_row = idx / ke;
        expert = A.routes.expert(x_row, idx - x_row * ke, L.w.n_mats);
        if (block == 0 && wave == 0) {
            const int k = idx - x_row * ke, err = A.routes.fault(x_row, k, L.w.n_mats, A.routes.before(x_row, k, lane));
            if (err && lane == 0) atomicOr(A.routes.err_flag, err);
        }
        if (expert < 0) return;  // its row is not read
    }
    const bool other = expert == L.w.n_mats;
    const cx_q4_desc& w = other ? L.shared : L.w;
    const size_t mat = other ? 0 : (size_t)max(expert, 0);
    const int cols = L.w.cols, pitch = KT * 256 + kQ4LdsPad, rt = block * groups + rg;
    float* xs_lds = reinterpret_cast<float*>(staged + A.lds_rows * pitch);  // kScaled (one plane): [lds_rows][KT]

    const size_t tile0 = (mat * RT + min(rt, RT - 1)) * (size_t)KT;
    const int per = (KT + A.splits - 1) / A.splits, k0 = ks * per, k1 = expert < 0 || rt >= RT ? k0 : min(KT, k0 + per);
    const __amdgpu_buffer_rsrc_t rw = make_rsrc(w.codes + tile0 * kQ4Tile, (uint32_t)max(k1, 0) * kQ4Tile);
    const __amdgpu_buffer_rsrc_t rs = make_rsrc(w.scales + tile0 * 16 * NG, (uint32_t)max(k1, 0) * 32 * NG);
    Q4Ring<NG, U> ring;

    // ---- x: loads first, so that waiting for them does not wait for the weights
    constexpr int kWords = XT == kQ4F32 ? 8 : XT == kQ4E4m3 ? 2 : 4;  // of a piece of 8 values
    const bool vec = cols % 8 == 0 && (reinterpret_cast<uintptr_t>(L.x) & (XT == kQ4E4m3 ? 7 : 15)) == 0;
    for (int r = 0; r < A.lds_rows; ++r) {
        int xr = r < np && expert >= 0 ? begin + r : -1;
        if (xr >= 0 && L.order != nullptr) {
            const int pair = L.order[xr];
            xr = pair < 0 ? -1 : pair / L.top_k;
        }
        if (x_row >= 0) xr = x_row;
        if (xr >= L.n_x) xr = -1;
        const size_t row = (size_t)max(xr, 0) * cols;
        uint32_t v[kQ4DecPieces][kWords];
#pragma unroll
        for (int i = 0; i < kQ4DecPieces; ++i) {
            const int c = (i * 64 * kQ4DecWaves + tid) * 8;
#pragma unroll
            for (int k = 0; k < kWords; ++k) v[i][k] = 0;
            if (xr < 0 || c >= cols) continue;
            const char* src = static_cast<const char*>(L.x) + (row + c) * (kWords / 2);
            if (vec) {
                if constexpr (kWords == 2) {
                    const uint2 d = *reinterpret_cast<const uint2*>(src);
                    v[i][0] = d.x, v[i][1] = d.y;
                } else {
#pragma unroll
                    for (int k = 0; k < kWords; k += 4) {
                        const u32x4 d = ld16(src + 4 * k);
#pragma unroll
                        for (int n = 0; n < 4; ++n) v[i][k + n] = d[n];
                    }
                }
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    if (c + k >= cols) continue;
                    if constexpr (kWords == 8)
                        v[i][k] = reinterpret_cast<const uint32_t*>(src)[k];
                    else if constexpr (kWords == 4)
                        v[i][k / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(src)[k] << (16 * (k & 1));
                    else
                        v[i][k / 4] |= (uint32_t)reinterpret_cast<const uint8_t*>(src)[k] << (8 * (k & 3));
                }
            }
        }
        if (r == 0) {
#pragma unroll
            for (int u = 0; u < U; ++u) ring.fetch(rw, rs, k0 + u, u, lane);
        }
        auto bits = [&](int i, int k) -> uint32_t {  // value k of piece i as fp32
            if constexpr (XT == kQ4F32)
                return v[i][k];
            else
                return k & 1 ? v[i][k / 2] & 0xFFFF0000u : v[i][k / 2] << 16;
        };
        float up = 1.0f;
        if constexpr (XT == kQ4Bf16 || XT == kQ4F32) {
            uint32_t most = 0;
#pragma unroll
            for (int i = 0; i < kQ4DecPieces; ++i)
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const uint32_t b = bits(i, k) & 0x7FFFFFFFu;
                    if (b < 0x7F800000u) most = max(most, b);  // infinities and NaN stay themselves
                }
#pragma unroll
            for (int m = 32; m >= 1; m >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, m));
            if (lane == 0) tops[r][wave] = most;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kQ4DecWaves; ++i) most = max(most, tops[r][i]);
            const int e = most == 0 ? 127 : min(max((int)(most >> 23) - 14, 1), 253);
            up = __uint_as_float((uint32_t)(254 - e) << 23);
            if (tid == 0) row_up[r] = __uint_as_float((uint32_t)e << 23);
        } else if (tid == 0) {
            row_up[r] = 1.0f;
        }
#pragma unroll
        for (int i = 0; i < kQ4DecPieces; ++i) {
            const int p = i * 64 * kQ4DecWaves + tid;
            if (p >= KT * 16) continue;
            u32x4 o;
            if constexpr (XT == kQ4F32) {
                u32x4 lo;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint2 two = q4_planes(__uint_as_float(v[i][2 * k]) * up, __uint_as_float(v[i][2 * k + 1]) * up);
                    o[k] = two.x, lo[k] = two.y;
                }
                *reinterpret_cast<u32x4*>(staged + (r * 2 + 1) * pitch + p * 16) = lo;
            } else if constexpr (XT == kQ4Fp16) {
                o = u32x4{v[i][0], v[i][1], v[i][2], v[i][3]};
            } else if constexpr (XT == kQ4E4m3) {
                o = __builtin_bit_cast(u32x4, cvt8_f16(v[i][0], v[i][1]));
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    o[k] = f16_rne(__uint_as_float(bits(i, 2 * k)) * up) | (f16_rne(__uint_as_float(bits(i, 2 * k + 1)) * up) << 16);
            }
            *reinterpret_cast<u32x4*>(staged + r * kPlanes * pitch + p * 16) = o;
        }
        if constexpr (kScaled)
            for (int k = tid; k < KT; k += 64 * kQ4DecWaves) xs_lds[r * KT + k] = xr >= 0 ? L.x_scale[(size_t)xr * KT + k] : 0.0f;
    }
    __syncthreads();

    // ---- the products; lanes of rows that are not there read another row, whose sums are dropped
    const int lr = kPlanes == 2 ? min(t & 3, A.lds_rows - 1) : min(t, A.lds_rows - 1);
    const unsigned char* in = staged + (kPlanes == 2 ? lr * 2 + (t >> 2 & 1) : lr) * pitch + q * 16;  // columns 4 .. 7: the second plane
    f32x4 acc[2] = {};
    auto multiply = [&](int kt, int u) {
        u32x4 b[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) b[j] = *reinterpret_cast<const u32x4*>(in + kt * 256 + j * 64);
        f32x4 part[2] = {};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f32x4& sum = kScaled ? part[j & 1] : acc[j & 1];
            sum = Mma<true>::mma(ring.weights(u, j), Mma<true>::bits(b[j]), sum);
        }
        if constexpr (kScaled) {
            const float x = xs_lds[lr * KT + kt];
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[0][i] += x * (part[0][i] + part[1][i]);
        }
    };
    for (int kt = k0; kt < k1; kt += U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (kt + u >= k1) break;
            __builtin_amdgcn_sched_barrier(0);
            multiply(kt + u, u);
            ring.fetch(rw, rs, kt + U + u, u, lane);
        }
    }
    acc[0] += acc[1];
    __syncthreads();  // x has been read: the sums take its place
    float(*red)[256] = reinterpret_cast<float(*)[256]>(staged);
    *reinterpret_cast<f32x4*>(&red[wave][t * 16 + q * 4]) = acc[0];
    __syncthreads();
    const int width = L.w.gated ? L.w.rows / 2 : L.w.rows;
    for (int i = tid; i < groups * 64; i += 64 * kQ4DecWaves) {  // 4 rows x 16 of each row tile
        const int g = i >> 6, o = block * groups + g, tt = (i & 63) >> 4, r = i & 15;
        float v = 0.0f;
        for (int k = 0; k < A.splits; ++k) {
            v += red[g * A.splits + k][i & 63];
            if constexpr (kPlanes == 2) v += red[g * A.splits + k][64 + (i & 63)];
        }
        v *= q4_row_scales(w)[(mat * RT + min(o, RT - 1)) * 16 + r] * row_up[min(tt, A.lds_rows - 1)];
        if (L.w.gated) {
            const float other_half = __shfl_down(v, 8);
            v = v / (1.0f + expf(-v)) * other_half;
        }
        const int n = L.w.gated ? o * 8 + r : o * 16 + r;
        if (tt < np && o < RT && n < width && (!L.w.gated || r < 8)) q4_store(L, (size_t)(begin + tt) * width + n, v);
    }
}

// The down projections of a token's routes and their weighted sum, for a few tokens: a wave per
// route, all on the same row tile, whose results are summed in route order (the shared
// expert last) and rounded once.  Each wave stages its own row of h in two planes as k_q4_dec does,
// 512 columns at a time, so the only barrier is the one before the sum.  Even columns of the MFMA
// take the first plane, odd ones the second.  HBM: 8 routes of 7168 x 2048, 61 MB in 13.8 us, 4.4 TB/s
// (13.0 with h rounded to the first plane).
template <int NG>
__global__ __launch_bounds__(1024) void k_q4_dec_sum(Q4DecSumArgs A) {
    constexpr int U = 4;  // column tiles in flight: those of 512 columns
    extern __shared__ __attribute__((aligned(16))) unsigned char staged[];
    const int RT = A.RT, KT = A.KT, tok = blockIdx.x / RT, rt = blockIdx.x - tok * RT;
    const int wave = wave_id(), lane = threadIdx.x & 63, t = lane & 15, q = lane >> 4;
    const int ke = A.routes.top_k + A.routes.shared, cols = A.w.cols, pitch = q4_sum_pitch(cols), k = wave;
    float* red = reinterpret_cast<float*>(staged + ke * pitch);  // [ke][16]
    float* weight = red + ke * 16;
    unsigned char* mine = staged + wave * pitch;
    const int lo_at = min(KT, 4) * 256 + kQ4LdsPad;  // of the second plane
    // in the order of their waits: h's row and the token's other ids, then the weights
    const __amdgpu_buffer_rsrc_t rh = make_rsrc(A.h + ((size_t)tok * ke + k) * cols, (uint32_t)cols * 4);
    u32x4 held[kQ4SumHeld][2];
    if (cols % 8 == 0) {
#pragma unroll
        for (int i = 0; i < kQ4SumHeld; ++i)
#pragma unroll
            for (int d = 0; d < 2; ++d) held[i][d] = bld16(rh, (uint32_t)(i * 64 + lane) * 32 + 16 * d);
    } else {
#pragma unroll
        for (int i = 0; i < kQ4SumHeld; ++i)
#pragma unroll
            for (int d = 0; d < 8; ++d) held[i][d >> 2][d & 3] = __builtin_amdgcn_raw_buffer_load_b32(rh, (uint32_t)(i * 64 + lane) * 32 + 4 * d, 0, 0);
    }
    const int before = A.routes.before(tok, k, lane), expert = A.routes.expert(tok, k, A.w.n_mats);
    const bool other = expert == A.w.n_mats;
    const cx_q4_desc& w = other ? A.shared : A.w;
    const size_t tile0 = ((size_t)(other ? 0 : max(expert, 0)) * RT + rt) * (size_t)KT;
    const uint32_t tiles = expert < 0 ? 0 : (uint32_t)KT;  // none: zeros
    const __amdgpu_buffer_rsrc_t rw = make_rsrc(w.codes + tile0 * kQ4Tile, tiles * kQ4Tile);
    const __amdgpu_buffer_rsrc_t rs = make_rsrc(w.scales + tile0 * 16 * NG, tiles * 32 * NG);
    Q4Ring<NG, U> ring;
#pragma unroll
    for (int u = 0; u < U; ++u) ring.fetch(rw, rs, u, u, lane);
    __builtin_amdgcn_sched_barrier(0);
    // a route that is left out: no weight, whatever its row holds (the gate/up launch has reported it)
    const bool used = expert >= 0 && A.routes.fault(tok, k, A.w.n_mats, before) == 0;
    if (lane == 0) weight[k] = !used ? 0.0f : k < A.routes.top_k ? A.routes.weights[(size_t)tok * A.routes.top_k + k] : 1.0f;
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < kQ4SumHeld; ++i)
#pragma unroll
        for (int d = 0; d < 8; ++d) {
            const uint32_t b = held[i][d >> 2][d & 3] & 0x7FFFFFFFu;
            if (b < 0x7F800000u) most = max(most, b);
        }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, m));
    const int e = most == 0 ? 127 : min(max((int)(most >> 23) - 14, 1), 253);
    const float up = __uint_as_float((uint32_t)(254 - e) << 23), down = __uint_as_float((uint32_t)e << 23);
    f32x4 acc[2] = {};
#pragma unroll
    for (int i = 0; i < kQ4SumHeld; ++i) {  // 512 columns: a piece of 8 a lane
        const int k0 = i * 4;
        if (k0 >= KT) break;
        const int c = lane * 16, part = min(KT - k0, 4) * 256;
        if (c < part) {
            u32x4 hi, lo;
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const uint2 two = q4_planes(__uint_as_float(held[i][d >> 1][2 * (d & 1)]) * up, __uint_as_float(held[i][d >> 1][2 * (d & 1) + 1]) * up);
                hi[d] = two.x, lo[d] = two.y;
            }
            *reinterpret_cast<u32x4*>(mine + c) = hi;
            *reinterpret_cast<u32x4*>(mine + lo_at + c) = lo;
        }
        __builtin_amdgcn_wave_barrier();
        const unsigned char* in = mine + (t & 1) * lo_at + q * 16;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (k0 + u >= KT) break;
            __builtin_amdgcn_sched_barrier(0);
            u32x4 b[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = *reinterpret_cast<const u32x4*>(in + u * 256 + j * 64);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j & 1] = Mma<true>::mma(ring.weights(u, j), Mma<true>::bits(b[j]), acc[j & 1]);
            ring.fetch(rw, rs, k0 + 4 + u, u, lane);
        }
        __builtin_amdgcn_wave_barrier();
    }
    f32x4 both = acc[0] + acc[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) both[i] += __shfl_xor(both[i], 1);
    if (t == 0) {
        const f32x4 scale = *reinterpret_cast<const f32x4*>(q4_row_scales(w) + tile0 / KT * 16 + 4 * q);
#pragma unroll
        for (int i = 0; i < 4; ++i) red[k * 16 + 4 * q + i] = used ? both[i] * scale[i] * down : 0.0f;
    }
    __syncthreads();
    const int n = rt * 16 + threadIdx.x;
    if (threadIdx.x >= 16 || n >= A.w.rows) return;
    float v = 0.0f;
    for (int r = 0; r < ke; ++r) v += weight[r] * red[r * 16 + threadIdx.x];
    const size_t at = (size_t)tok * A.w.rows + n;
    static_cast<uint16_t*>(A.y)[at] = (uint16_t)cast_out(v, A.out_dtype);
    if (A.y_f32 != nullptr) A.y_f32[at] = v;
}

}  // namespace cx
