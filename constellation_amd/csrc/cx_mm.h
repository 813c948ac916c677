// cx_mm.h — tiles of products with weights as the program holds them, row-major in 16 bits
// or 8-bit integers, and of the 16-bit products' gradients:
//   forward   y[p, n] = sum over k of x[p, k] w[n, k]
//   at x      dx[p, k] = sum over n of dy[p, n] w[n, k]
//   at w      dw[n, k] = sum over p of dy[p, n] x[p, k]
// A stack of matrices takes the rows of its offsets; a workgroup finds its own run of
// rows in them, so that no plan is launched before it.
#pragma once

#include <type_traits>

#include "cx_device.h"

namespace cx {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// v_mfma 32x32 of 16 bytes a lane and operand: lane l holds row (column) l % 32, contraction bytes 16 (l / 32)
// .. + 15 of 32; a result's element i is row 8 (i / 4) + 4 (l / 32) + i % 4, column l % 32.
struct MmBf16 {
    static constexpr int kType = CX_DTYPE_BF16, kEl = 2;
    typedef f32x16 Acc;
    static __device__ __forceinline__ Acc mma(u32x4 a, u32x4 b, Acc c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
struct MmF16 {
    static constexpr int kType = CX_DTYPE_FP16, kEl = 2;
    typedef f32x16 Acc;
    static __device__ __forceinline__ Acc mma(u32x4 a, u32x4 b, Acc c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};
struct MmI8 {
    static constexpr int kType = kMmI8, kEl = 1;
    typedef i32x16 Acc;
    static __device__ __forceinline__ Acc mma(u32x4 a, u32x4 b, Acc c) {
        return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
    }
};

// ---------------------------------------------------------------------------
// Runs of rows.  Offsets that go back or leave the rows are cut to what is there: matrix
// e has the rows from the largest of the offsets up to e's to the largest up to e + 1's.
struct MmItem {
    int mat, begin, rows;  // mat < 0: rows behind the last matrix's; rows 0: no such item
};

__device__ __forceinline__ int mm_cut(int v, int n_rows) { return min(max(v, 0), n_rows); }

// One wave reports offsets that are out of order.
__device__ __forceinline__ void mm_check(const int32_t* offsets, int n_mats, int n_rows, int* err_flag) {
    bool bad = false;
    for (int e = threadIdx.x & 63; e < n_mats; e += 64) {
        const int a = offsets[e], b = offsets[e + 1];
        bad = bad || a > b || a < 0 || b > n_rows || (e == 0 && a != 0);
    }
    if (__ballot(bad) != 0 && (threadIdx.x & 63) == 0) atomicOr(err_flag, kErrBadRow);
}

__device__ __forceinline__ int wave_scan_max(int v, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(v, d);
        v = lane >= d ? max(v, o) : v;
    }
    return v;
}
__device__ __forceinline__ int wave_scan_add(int v, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(v, d);
        v += lane >= d ? o : 0;
    }
    return v;
}

// Run idx of up to item_rows rows, of whole tiles of TILE (uniform in a wave; each wave finds it by itself).
template <int TILE>
__device__ __forceinline__ MmItem mm_item(const int32_t* offsets, int n_mats, int n_rows, int item_rows, int idx) {
    if (offsets == nullptr) {
        const int begin = idx * item_rows;
        return MmItem{0, begin, begin < n_rows ? min(item_rows, n_rows - begin) : 0};
    }
    const int lane = threadIdx.x & 63;
    int held = 0, before = 0;  // rows and runs of the matrices so far
    for (int e0 = 0; e0 < n_mats; e0 += 64) {
        const int e = e0 + lane;
        const int top = wave_scan_max(max(held, e < n_mats ? mm_cut(offsets[e + 1], n_rows) : 0), lane);
        const int up = __shfl_up(top, 1), begin = lane == 0 ? held : up, rows = top - begin;
        const int n = (rows + item_rows - 1) / item_rows, end = before + wave_scan_add(n, lane);
        const uint64_t past = __ballot(end > idx);
        if (past != 0) {
            const int l = __builtin_ctzll(past);
            const int r = __shfl(rows, l), m = __shfl(n, l), first = __shfl(end, l) - m, i = idx - first;
            const int share = mm_share(m, r, TILE);  // equal runs
            return MmItem{e0 + l, __builtin_amdgcn_readfirstlane(__shfl(begin, l) + i * share), __builtin_amdgcn_readfirstlane(min(share, r - i * share))};
        }
        held = __shfl(top, 63);
        before = __shfl(end, 63);
    }
    const int begin = held + (idx - before) * item_rows;
    return MmItem{-1, begin, begin < n_rows && begin >= held ? min(item_rows, n_rows - begin) : 0};
}

// The rows of one matrix.
__device__ __forceinline__ MmItem mm_rows_of(const int32_t* offsets, int n_rows, int mat) {
    if (offsets == nullptr) return MmItem{0, 0, n_rows};
    int lo = 0;
    for (int e = 1 + (threadIdx.x & 63); e <= mat; e += 64) lo = max(lo, mm_cut(offsets[e], n_rows));
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) lo = max(lo, __shfl_xor(lo, m));
    const int hi = max(lo, mm_cut(offsets[mat + 1], n_rows));
    return MmItem{mat, __builtin_amdgcn_readfirstlane(lo), __builtin_amdgcn_readfirstlane(hi - lo)};
}

// ---------------------------------------------------------------------------
// A workgroup's tile: WM x WN waves of TM x TN results of 32 x 32.  m is the direction in which the
// output is contiguous, n its rows.
template <int WM_, int WN_, int TM_, int TN_>
struct MmShape {
    static constexpr int WM = WM_, WN = WN_, TM = TM_, TN = TN_;
    static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves;
    static constexpr int BM = WM * TM * 32, BN = WN * TN * 32;
    static constexpr int kStage = (BM + BN) * 128;  // bytes of LDS of a step of the contraction
};

static __device__ __attribute__((aligned(16))) const uint32_t mm_zeros[4] = {};

// 16 bytes at any alignment.
struct __attribute__((packed)) MmPacked {
    u32x4 v;
};

// The pieces of 16 bytes that a thread brings to LDS for one operand of a step, R rows (columns) wide.
//  TR false: rows that are contiguous in the contraction, 128 bytes of each.  Row r's piece c lies
//    in place c ^ (r % 8) ^ (r / 8 % 2), so that the 16 rows which a wave reads at a time lie in different banks.
//  TR true: 64 rows of the contraction, R 16-bit columns of each.  32-byte chunk c of row j lies in place
//    c ^ 2 (j % 4), for the transposing reads of four rows at a time.
// Places are 32 bits from a uniform base, which moves with the steps.
template <int R, int THREADS, int EL, bool TR>
struct MmSrc {
    static constexpr int P = R * 8 / THREADS;
    static constexpr int kStepRows = THREADS * 8 / R;  // TR: rows between a thread's pieces
    static constexpr int kStep = 128 / EL;             // elements of the contraction in a step
    const char* base;
    uint32_t off[TR ? 1 : P];
    uint32_t gap;  // TR: bytes between a thread's pieces
    size_t move;   // bytes between steps
    int first;     // place in the step's contraction of the thread's pieces' first element (TR: of its first piece)
    int left;      // TR: elements from the piece's first to the row's end

    // offset(r): bytes from base to row r
    template <class F>
    __device__ __forceinline__ void rows(const void* base_, F offset) {
        static_assert(!TR, "");
        const int t = threadIdx.x, c = (t & 7) ^ ((t >> 3) & 7) ^ ((t >> 6) & 1);
        base = static_cast<const char*>(base_);
        move = 128;
        first = c * (16 / EL);
#pragma unroll
        for (int i = 0; i < P; ++i) off[i] = offset(i * (THREADS / 8) + (t >> 3)) + c * 16;
    }
    // columns col0 .. of a matrix `width` wide; those past it read others, and their results are not stored
    __device__ __forceinline__ void cols(const void* base_, int col0, int width) {
        static_assert(TR, "");
        const int t = threadIdx.x, piece = t % (R / 8);
        first = t / (R / 8);
        const int col = col0 + (((piece >> 1) ^ (2 * (first & 3))) * 2 + (piece & 1)) * 8;
        base = static_cast<const char*>(base_);
        left = width - col;
        off[0] = (uint32_t)first * (uint32_t)width * 2 + (left > 0 ? col * 2 : 0);
        gap = (uint32_t)kStepRows * (uint32_t)width * 2;
        move = (size_t)width * 128;
    }
    __device__ __forceinline__ const char* piece(int i, int k) const {
        return base + (size_t)k * move + (TR ? off[0] + (uint32_t)i * gap : off[TR ? 0 : i]);
    }
    // Straight to LDS: whole pieces that start on 16 bytes.  What lies past the contraction's n elements is zeros.
    __device__ __forceinline__ void fetch(unsigned char* lds, int k, int n) const {
        auto bring = [&](int i, const char* q) {
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)q,
                                             (__attribute__((address_space(3))) void*)(lds + i * THREADS * 16 + wave_id() * 1024), 16, 0, 0);
        };
        if ((k + 1) * kStep <= n) {
#pragma unroll
            for (int i = 0; i < P; ++i) bring(i, piece(i, k));
        } else {
#pragma unroll
            for (int i = 0; i < P; ++i)
                bring(i, k * kStep + first + (TR ? i * kStepRows : 0) < n ? piece(i, k) : reinterpret_cast<const char*>(mm_zeros));
        }
    }
    // Through registers: rows of any width at any address.
    __device__ __forceinline__ void load(u32x4 (&v)[P], int k, int n) const {
        constexpr int kWhole = 16 / EL;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int have = TR ? (k * kStep + first + i * kStepRows < n ? left : 0) : n - k * kStep - first;
            const char* q = piece(i, k);
            v[i] = u32x4{};
            if (have >= kWhole) {
                v[i] = ((const __attribute__((address_space(1))) MmPacked*)q)->v;
            } else if (have > 0) {
#pragma unroll
                for (int e = 0; e < kWhole - 1; ++e) {
                    if (e >= have) continue;
                    if constexpr (EL == 1)
                        v[i][e / 4] |= (uint32_t)reinterpret_cast<const uint8_t*>(q)[e] << (8 * (e & 3));
                    else
                        v[i][e / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(q)[e] << (16 * (e & 1));
                }
            }
        }
    }
    __device__ __forceinline__ void put(unsigned char* lds, const u32x4 (&v)[P]) const {
#pragma unroll
        for (int i = 0; i < P; ++i) *reinterpret_cast<u32x4*>(lds + (i * THREADS + threadIdx.x) * 16) = v[i];
    }
};

// A wave's fragments of an operand, T of 32 rows (columns) from row r0 of the tile on.
template <int R, int T, bool TR>
struct MmFrag {
    uint32_t at[TR ? T : 4];
    __device__ __forceinline__ MmFrag(int r0) {
        const int l = threadIdx.x & 63;
        if constexpr (TR) {
            const int g = l >> 4, i = l & 15;
#pragma unroll
            for (int t = 0; t < T; ++t)
                at[t] = (8 * (g >> 1) + (i >> 2)) * R * 2 + (((r0 / 16 + 2 * t + (g & 1)) ^ (2 * (i >> 2))) * 32) + (i & 3) * 8;
        } else {
            const int key = (l & 7) ^ ((l >> 3) & 1);
#pragma unroll
            for (int s = 0; s < 4; ++s) at[s] = (r0 + (l & 31)) * 128 + (((2 * s + (l >> 5)) ^ key) * 16);
        }
    }
    __device__ __forceinline__ void read(u32x4 (&f)[T], const unsigned char* lds, int s) const {
#pragma unroll
        for (int t = 0; t < T; ++t) {
            if constexpr (TR) {
                union {
                    s16x4 h[2];
                    u32x4 v;
                } u;
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    u.h[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds + at[t] + (16 * s + 4 * h) * R * 2));
                f[t] = u.v;
            } else {
                f[t] = *reinterpret_cast<const u32x4*>(lds + at[s] + t * 4096);
            }
        }
    }
};

// s_waitcnt vmcnt(0) lgkmcnt(0), then a barrier: what was fetched is there, and no wave still reads what was
// read before.
__device__ __forceinline__ void mm_turn() {
    __builtin_amdgcn_s_waitcnt(0x70);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// acc[m][n] += A B over `steps` steps of 128 bytes (64 rows) of a contraction of n elements.  Steps go through two
// buffers of LDS, which are two objects: the compiler then knows that reads of one need not wait for loads into the
// other.  A step is four MFMA depths; the fragments of a depth are read while the depth before multiplies,
// and a step's last depth multiplies while the next step's first fragments are read, behind the barrier.
template <class T, class S, bool AT, bool BT, bool DMA>
__device__ __forceinline__ void mm_core(const MmSrc<S::BM, S::kThreads, T::kEl, AT>& a, const MmSrc<S::BN, S::kThreads, T::kEl, BT>& b,
                                        int n, int k0, int k1, unsigned char* lds0, unsigned char* lds1, typename T::Acc (&acc)[S::TM][S::TN]) {
    constexpr int kB = S::BM * 128;
    const int wave = wave_id();
    const MmFrag<S::BM, S::TM, AT> fa(wave % S::WM * S::TM * 32);
    const MmFrag<S::BN, S::TN, BT> fb(wave / S::WM * S::TN * 32);
#pragma unroll
    for (int m = 0; m < S::TM; ++m)
#pragma unroll
        for (int t = 0; t < S::TN; ++t) acc[m][t] = typename T::Acc{};
    if (k0 >= k1) return;
    u32x4 va[MmSrc<S::BM, S::kThreads, T::kEl, AT>::P], vb[MmSrc<S::BN, S::kThreads, T::kEl, BT>::P];  // DMA: not used
    auto fetch = [&](int k, unsigned char* buf) {
        if constexpr (DMA) {
            a.fetch(buf, k, n);
            b.fetch(buf + kB, k, n);
        } else {
            a.load(va, k, n);
            b.load(vb, k, n);
        }
    };
    auto put = [&](unsigned char* buf) {
        if constexpr (!DMA) {
            a.put(buf, va);
            b.put(buf + kB, vb);
        }
    };
    u32x4 xa[2][S::TM], xb[2][S::TN];
    auto read = [&](int s, const unsigned char* buf) {
        fa.read(xa[s & 1], buf, s);
        fb.read(xb[s & 1], buf + kB, s);
    };
    auto multiply = [&](int s) {
#pragma unroll
        for (int m = 0; m < S::TM; ++m)
#pragma unroll
            for (int t = 0; t < S::TN; ++t) acc[m][t] = T::mma(xa[s & 1][m], xb[s & 1][t], acc[m][t]);
#if defined(__HIP_DEVICE_COMPILE__)  // keeps the sums where they are: no copies of them at the loop's end
        if (s == 3)
#pragma unroll
            for (int m = 0; m < S::TM; ++m)
#pragma unroll
                for (int t = 0; t < S::TN; ++t) asm volatile("" : "+v"(acc[m][t]));
#endif
    };
    auto step = [&](int k, unsigned char* buf, unsigned char* other) {
        if (!DMA && k + 1 < k1) fetch(k + 1, other);
#pragma unroll
        for (int s = 0; s < 3; ++s) {
            __builtin_amdgcn_sched_barrier(0);
            read(s + 1, buf);
            multiply(s);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (!DMA && k + 1 < k1) put(other);
        mm_turn();
        if (DMA && k + 2 < k1) fetch(k + 2, buf);
        if (k + 1 < k1) read(0, other);
        multiply(3);
    };
    fetch(k0, lds0);
    put(lds0);
    mm_turn();
    if (DMA && k0 + 1 < k1) fetch(k0 + 1, lds1);
    read(0, lds0);
    int k = k0;
    for (; k + 1 < k1; k += 2) {
        step(k, lds0, lds1);
        step(k + 1, lds1, lds0);
    }
    if (k < k1) step(k, lds0, lds1);
}

// 32 rows of W * 32 outputs, from a wave's results through its own part of LDS, so that it stores whole lines.
// v: results whose m is consecutive; row(n) is where in `out` row n starts (elements), < 0: not stored.
template <int W, class F>
__device__ __forceinline__ void mm_put(const f32x16 (&v)[W], float* turn, void* out, int type, bool vec, int m0, int width, F row) {
    constexpr int kChunks = W * 8;  // of four floats
    const int l = threadIdx.x & 63, n = l & 31;
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int c = w * 8 + 2 * g + (l >> 5);
            *reinterpret_cast<f32x4*>(turn + n * W * 32 + (c ^ (n & (kChunks - 1))) * 4) = f32x4{v[w][4 * g], v[w][4 * g + 1], v[w][4 * g + 2], v[w][4 * g + 3]};
        }
    __builtin_amdgcn_wave_barrier();
    const int per = type == CX_DTYPE_F32 ? 4 : 8, lanes = W * 32 / per;  // columns of a lane's store, lanes of a row
    for (int i = l; i < 32 * lanes; i += 64) {
        const int r = i / lanes, c = (i - r * lanes) * per, left = width - m0 - c;
        const int64_t at = row(r);
        if (at < 0 || left <= 0) continue;
        const float* src = turn + r * W * 32;
        const f32x4 a = *reinterpret_cast<const f32x4*>(src + ((c / 4) ^ (r & (kChunks - 1))) * 4);
        if (type == CX_DTYPE_F32) {
            float* y = static_cast<float*>(out) + at + m0 + c;
            if (vec) {
                *reinterpret_cast<f32x4*>(y) = a;
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (k < left) y[k] = a[k];
            }
        } else {
            const f32x4 b = *reinterpret_cast<const f32x4*>(src + ((c / 4 + 1) ^ (r & (kChunks - 1))) * 4);
            uint32_t h[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) h[k] = cast_out(a[k], type), h[4 + k] = cast_out(b[k], type);
            uint16_t* y = static_cast<uint16_t*>(out) + at + m0 + c;
            if (vec) {
                *reinterpret_cast<u32x4*>(y) = u32x4{h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16), h[6] | (h[7] << 16)};
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (k < left) y[k] = (uint16_t)h[k];
            }
        }
    }
    __builtin_amdgcn_wave_barrier();
}

// Zeros in rows n of out[.., m0 .. m0 + cols - 1].
__device__ __forceinline__ void mm_clear(void* out, int type, int64_t first, int rows, int width, int m0, int cols, int threads) {
    const int n = min(cols, width - m0);
    for (int r = 0; r < rows; ++r)
        for (int c = threadIdx.x; c < n; c += threads) {
            const int64_t at = (first + r) * width + m0 + c;
            if (type == CX_DTYPE_F32)
                static_cast<float*>(out)[at] = 0.0f;
            else
                static_cast<uint16_t*>(out)[at] = 0;
        }
}

__device__ __forceinline__ float mm_silu(float g) { return g / (1.0f + expf(-g)); }

__device__ __forceinline__ bool mm_vec(const void* p, int width, int type) {
    return width % (type == CX_DTYPE_F32 ? 4 : 8) == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0;
}

// ---------------------------------------------------------------------------
// Forward.  m: weight rows; a gated tile has TM / 2 results of gate rows and the same rows of the up
// half per wave, so that both factors of an output meet in one lane.
template <class T, class S, bool GATED, bool DMA>
__global__ __launch_bounds__(S::kThreads, 2) void k_mm(MmLaunch L) {
    __shared__ __attribute__((aligned(16))) unsigned char lds0[S::kStage], lds1[S::kStage];
    static_assert(S::kWaves * 8192 <= S::kStage, "turned results");
    constexpr int kOut = GATED ? S::BM / 2 : S::BM;  // columns of y
    const MmTile tile = mm_tile(blockIdx.x, L.m_tiles, L.by_item);
    if (L.offsets != nullptr && blockIdx.x == 0 && wave_id() == 0) mm_check(L.offsets, L.n_mats, L.n_rows, L.err_flag);
    if (tile.m >= L.m_tiles) return;
    const MmItem it = mm_item<32>(L.offsets, L.n_mats, L.n_rows, S::BN, tile.item);
    if (it.rows <= 0) return;
    const int width = GATED ? L.rows / 2 : L.rows, m0 = tile.m * kOut;
    if (it.mat < 0) {
        mm_clear(L.y, L.y_type, it.begin, it.rows, width, m0, kOut, S::kThreads);
        if (GATED && L.pre != nullptr)
            for (int h = 0; h < 2; ++h)
                for (int r = 0; r < it.rows; ++r) mm_clear(L.pre, T::kType, 2 * (int64_t)(it.begin + r) + h, 1, width, m0, kOut, S::kThreads);
        return;
    }
    MmSrc<S::BM, S::kThreads, T::kEl, false> a;
    MmSrc<S::BN, S::kThreads, T::kEl, false> b;
    const size_t pitch = (size_t)L.cols * T::kEl;
    // weight rows from the tile's first on; those past the matrix are its last one again, and not stored
    constexpr int half = S::TM / 2;  // gated: results of gate rows
    a.rows(static_cast<const char*>(L.w) + ((size_t)it.mat * L.rows + m0) * pitch, [&](int r) {
        const int n = GATED ? min(m0 + (r / (S::TM * 32) * half + r / 32 % half) * 32 + r % 32, width - 1) + (r / 32 % S::TM < half ? 0 : width)
                            : min(m0 + r, width - 1);
        return (uint32_t)(n - m0) * (uint32_t)pitch;
    });
    // the row of x of row r of the item, < 0: none, and row 0 is read in its place
    auto source = [&](int r) {
        const int p = it.begin + min(r, it.rows - 1);
        if (L.order == nullptr) return p;
        const int pair = L.order[p], xr = pair / L.top_k;
        return pair < 0 || xr >= L.n_x ? -1 : xr;
    };
    const int x0 = L.order == nullptr ? it.begin : 0;
    b.rows(static_cast<const char*>(L.x) + (size_t)x0 * pitch, [&](int r) { return (uint32_t)(max(source(r), x0) - x0) * (uint32_t)pitch; });
    typename T::Acc acc[S::TM][S::TN];
    mm_core<T, S, false, false, DMA>(a, b, L.cols, 0, (L.cols + 128 / T::kEl - 1) / (128 / T::kEl), lds0, lds1, acc);
    // results to y
    const int wave = wave_id(), l = threadIdx.x & 63, wm = wave % S::WM, n0 = wave / S::WM * S::TN * 32;
    float* turn = reinterpret_cast<float*>(lds0 + wave * 8192);
    f32x16 v[S::TM];
#pragma unroll
    for (int t = 0; t < S::TN; ++t) {
        const int nt = n0 + t * 32;
        if (nt >= it.rows) break;
        const int xr = source(nt + (l & 31));
        const float xs = T::kEl == 1 ? (xr < 0 ? 0.0f : L.x_scale[xr]) : 1.0f;
#pragma unroll
        for (int m = 0; m < S::TM; ++m) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float f = (float)acc[m][t][i];
                if constexpr (T::kEl == 1) {
                    const int c = 8 * (i >> 2) + 4 * (l >> 5) + (i & 3);
                    const int n = GATED ? min(m0 + (wm * half + m % half) * 32 + c, width - 1) + (m < half ? 0 : width)
                                        : min(m0 + (wm * S::TM + m) * 32 + c, width - 1);
                    f = f * xs * L.w_scale[(size_t)it.mat * L.rows + n];
                }
                v[m][i] = xr < 0 ? 0.0f : f;
            }
        }
        auto row = [&](int64_t w, int64_t off) {
            return [=](int r) { return nt + r < it.rows ? (int64_t)(it.begin + nt + r) * w + off : (int64_t)-1; };
        };
        if constexpr (GATED) {
            f32x16 g[half], u[half], h[half];
#pragma unroll
            for (int m = 0; m < half; ++m) {
                g[m] = v[m];
                u[m] = v[half + m];
#pragma unroll
                for (int i = 0; i < 16; ++i) h[m][i] = mm_silu(g[m][i]) * u[m][i];
            }
            const int mw = m0 + wm * half * 32;
            if (L.pre != nullptr) {
                const bool vec = mm_vec(L.pre, width, T::kType);
                mm_put<half>(g, turn, L.pre, T::kType, vec, mw, width, row(2 * (int64_t)width, 0));
                mm_put<half>(u, turn, L.pre, T::kType, vec, mw, width, row(2 * (int64_t)width, width));
            }
            mm_put<half>(h, turn, L.y, L.y_type, mm_vec(L.y, width, L.y_type), mw, width, row(width, 0));
        } else {
            const bool vec = mm_vec(L.y, width, L.y_type);
#pragma unroll
            for (int m = 0; m < S::TM; m += 2) {
                f32x16 o[2] = {v[m], v[m + 1]};
                mm_put<2>(o, turn, L.y, L.y_type, vec, m0 + (wm * S::TM + m) * 32, width, row(width, 0));
            }
        }
    }
}

// The gradient at x.  m: columns of the weights, read across their rows; n: rows of dy.
template <class T, class S, bool DMA>
__global__ __launch_bounds__(S::kThreads, 2) void k_mm_dx(MmLaunch L) {
    __shared__ __attribute__((aligned(16))) unsigned char lds0[S::kStage], lds1[S::kStage];
    const MmTile tile = mm_tile(blockIdx.x, L.m_tiles, L.by_item);
    if (L.offsets != nullptr && blockIdx.x == 0 && wave_id() == 0) mm_check(L.offsets, L.n_mats, L.n_rows, L.err_flag);
    if (tile.m >= L.m_tiles) return;
    const MmItem it = mm_item<32>(L.offsets, L.n_mats, L.n_rows, S::BN, tile.item);
    if (it.rows <= 0) return;
    const int width = L.cols, m0 = tile.m * S::BM;
    if (it.mat < 0) return mm_clear(L.y, L.y_type, it.begin, it.rows, width, m0, S::BM, S::kThreads);
    MmSrc<S::BM, S::kThreads, 2, true> a;
    MmSrc<S::BN, S::kThreads, 2, false> b;
    a.cols(static_cast<const char*>(L.w) + (size_t)it.mat * L.rows * L.cols * 2, m0, width);
    b.rows(static_cast<const char*>(L.dy) + (size_t)it.begin * L.rows * 2, [&](int r) { return (uint32_t)min(r, it.rows - 1) * (uint32_t)L.rows * 2; });
    f32x16 acc[S::TM][S::TN];
    mm_core<T, S, true, false, DMA>(a, b, L.rows, 0, (L.rows + 63) / 64, lds0, lds1, acc);
    const int wave = wave_id(), n0 = wave / S::WM * S::TN * 32;
    float* turn = reinterpret_cast<float*>(lds0 + wave * 8192);
    const bool vec = mm_vec(L.y, width, L.y_type);
#pragma unroll
    for (int t = 0; t < S::TN; ++t) {
        const int nt = n0 + t * 32;
        if (nt >= it.rows) break;
#pragma unroll
        for (int m = 0; m < S::TM; m += 2) {
            f32x16 o[2] = {acc[m][t], acc[m + 1][t]};
            mm_put<2>(o, turn, L.y, L.y_type, vec, m0 + (wave % S::WM * S::TM + m) * 32, width,
                      [&](int r) { return nt + r < it.rows ? (int64_t)(it.begin + nt + r) * width : (int64_t)-1; });
        }
    }
}

// The gradient at the weights of each matrix.  m: their columns; n: their rows.
template <class T, class S, bool DMA>
__global__ __launch_bounds__(S::kThreads, 2) void k_mm_dw(MmLaunch L) {
    __shared__ __attribute__((aligned(16))) unsigned char lds0[S::kStage], lds1[S::kStage];
    if (L.offsets != nullptr && blockIdx.x == 0 && wave_id() == 0) mm_check(L.offsets, L.n_mats, L.n_rows, L.err_flag);
    const int n_tiles = (L.rows + S::BN - 1) / S::BN, per = n_tiles * L.m_tiles, mat = blockIdx.x / per, i = blockIdx.x - mat * per;
    const int n0 = i / L.m_tiles * S::BN, m0 = (i - i / L.m_tiles * L.m_tiles) * S::BM;
    const MmItem it = mm_rows_of(L.offsets, L.n_rows, mat);
    MmSrc<S::BM, S::kThreads, 2, true> a;
    MmSrc<S::BN, S::kThreads, 2, true> b;
    a.cols(static_cast<const char*>(L.x) + (size_t)it.begin * L.cols * 2, m0, L.cols);
    b.cols(static_cast<const char*>(L.dy) + (size_t)it.begin * L.rows * 2, n0, L.rows);
    f32x16 acc[S::TM][S::TN];
    mm_core<T, S, true, true, DMA>(a, b, it.rows, 0, (it.rows + 63) / 64, lds0, lds1, acc);
    const int wave = wave_id(), nw = n0 + wave / S::WM * S::TN * 32;
    float* turn = reinterpret_cast<float*>(lds0 + wave * 8192);
    const bool vec = mm_vec(L.y, L.cols, L.y_type);
#pragma unroll
    for (int t = 0; t < S::TN; ++t)
#pragma unroll
        for (int m = 0; m < S::TM; m += 2) {
            f32x16 o[2] = {acc[m][t], acc[m + 1][t]};
            mm_put<2>(o, turn, L.y, L.y_type, vec, m0 + (wave % S::WM * S::TM + m) * 32, L.cols, [&](int r) {
                const int n = nw + t * 32 + r;
                return n < L.rows ? ((int64_t)mat * L.rows + n) * L.cols : (int64_t)-1;
            });
        }
}

}  // namespace cx
