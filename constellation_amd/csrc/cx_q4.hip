// cx_q4.hip — products with 4-bit weights (e2m1 codes, a bf16 scale per row and
// 32, 64 or 128 columns): y[t, n] = sum over groups g of s[n, g] * sum over k in g of
// c[n, k] * x[t, k], for one matrix or a stack of them, the rows of x dealt to the
// stack's matrices by work items.
#include "cx_q4.h"

namespace cx {
namespace {

// Source row of row r of row tile rt; -1: padding.
__device__ __forceinline__ int q4_src_row(const cx_q4_desc& w, int rt, int r) {
    if (!w.gated) return rt * 16 + r < w.rows ? rt * 16 + r : -1;
    const int half = w.rows / 2, n = rt * 8 + (r & 7);
    return n < half ? (r < 8 ? n : half + n) : -1;
}

__global__ __launch_bounds__(256) void k_q4_pack(cx_q4_desc w, const uint8_t* codes, const uint16_t* scales,
                                                 const float* row_scale, uint32_t* dst, uint16_t* dst_scale,
                                                 int64_t tiles) {
    const int RT = q4_row_tiles(w), KT = q4_col_tiles(w), lane = threadIdx.x & 63;
    const int groups = (w.cols + w.group - 1) / w.group, NG = 128 / w.group;
    const int stride = (w.cols + 1) / 2, r = lane & 15, q = lane >> 4;
    for (int64_t tile = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); tile < tiles; tile += (int64_t)gridDim.x * 4) {
        const int kt = (int)(tile % KT), rt = (int)(tile / KT % RT);
        const int64_t mat = tile / KT / RT;
        const int n = q4_src_row(w, rt, r);
        const uint8_t* src = codes + (mat * w.rows + n) * (int64_t)stride;
        uint32_t d[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            d[j] = 0;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const int col = kt * 128 + 32 * j + 8 * q + 2 * b;
                if (n < 0 || col >= w.cols) continue;
                uint32_t v = src[col / 2];
                if (col + 1 >= w.cols) v &= 0xFu;
                d[j] |= v << (8 * b);
            }
        }
        *reinterpret_cast<u32x4*>(dst + tile * 256 + lane * 4) = u32x4{d[0], d[1], d[2], d[3]};
        if (lane < 16 * NG) {  // [16 rows][group]
            const int g = lane % NG, r2 = lane / NG, n2 = q4_src_row(w, rt, r2), at = kt * NG + g;
            const float up = n2 >= 0 ? 1.0f / row_scale[(mat * RT + rt) * 16 + r2] : 1.0f;
            const float s = n2 >= 0 && at < groups ? __uint_as_float((uint32_t)scales[(mat * w.rows + n2) * (int64_t)groups + at] << 16) : 0.0f;
            dst_scale[tile * 16 * NG + lane] = (uint16_t)f16_rne(s * up);
        }
    }
}

// Per row the power of two that brings its largest scale to 2^11 .. 2^12: below it, a
// code times a scale (2 and 8 significant bits) is exact in fp16 over 27 binades of
// scales, and smaller ones are off by less than 2^-36 of the row's largest weight.
// The powers run from 2^-126 to 2^116, whose reciprocals are normal numbers, too.
__global__ __launch_bounds__(256) void k_q4_row_scales(cx_q4_desc w, const uint16_t* scales, float* row_scale, int64_t rows) {
    const int RT = q4_row_tiles(w), lane = threadIdx.x & 63, groups = (w.cols + w.group - 1) / w.group;
    for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < rows; i += (int64_t)gridDim.x * 4) {
        const int r = (int)(i & 15), rt = (int)(i / 16 % RT), n = q4_src_row(w, rt, r);
        const uint16_t* src = scales + (i / 16 / RT * w.rows + n) * (int64_t)groups;
        uint32_t most = 0;
        for (int g = lane; n >= 0 && g < groups; g += 64) {
            const uint32_t v = src[g] & 0x7FFFu;
            if (v < 0x7F80u) most = max(most, v);  // infinities and NaN stay themselves
        }
#pragma unroll
        for (int m = 32; m >= 1; m >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, m));
        const int e = min(max((int)(most >> 7) - 11, 1), 243);
        if (lane == 0) row_scale[i] = most == 0 ? 1.0f : __uint_as_float((uint32_t)e << 23);
    }
}

// Rows of x as fp16 times a power of two per row, in rows of whole 128-column tiles,
// zeros behind the row.  The row's largest value comes to 2^14 .. 2^15, so bf16
// values (8 significant bits) are exact down to 2^-31 of it and the others off by less than
// 2^-39 of it: nothing next to the sums' own 2^-24.  fp32 values come in two planes (q4_planes), 64 columns
// of the first, then the same of the second.
//
// A row is read once, kRowPieces pieces of 8 values a thread in registers (wider rows are read
// again for what lies behind), 16 bytes at a time where it starts on them.  1024 bf16 rows of 7168 take 9
// us, 8192 fp32 rows of 2048 26 (134 MB, 5.1 TB/s), 3001 e4m3 rows of 2048 7.
constexpr int kRowPieces = 4;

template <int DT>
__device__ __forceinline__ void q4_row_piece(const void* x, size_t row, int c, int cols, bool vec, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    if (c >= cols) return;
    if constexpr (DT == CX_DTYPE_F32) {
        const float* p = static_cast<const float*>(x) + row + c;
        if (vec) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < cols) v[i] = p[i];
        }
    } else if constexpr (DT == CX_DTYPE_E4M3) {
        const uint8_t* p = static_cast<const uint8_t*>(x) + row + c;
        uint32_t a = 0, b = 0;
        if (vec) {
            const uint2 d = *reinterpret_cast<const uint2*>(p);
            a = d.x, b = d.y;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < cols) (i < 4 ? a : b) |= (uint32_t)p[i] << (8 * (i & 3));
        }
        const f16x8 f = cvt8_f16(a, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)f[i];
    } else {
        const uint16_t* p = static_cast<const uint16_t*>(x) + row + c;
        uint32_t h[8] = {};
        if (vec) {
            const u32x4 d = ld16(p);
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = i & 1 ? d[i >> 1] >> 16 : d[i >> 1] & 0xFFFFu;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < cols) h[i] = p[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = DT == CX_DTYPE_BF16 ? __uint_as_float(h[i] << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)h[i]);
    }
}

// e4m3 rows (exact in fp16) and fp16 rows are copied as they are, with a scale of 1.
template <int DT>
__global__ __launch_bounds__(256) void k_q4_rows(const void* x, int cols, int padded, uint16_t* dst, float* scale) {
    __shared__ uint32_t part[4];
    const int tid = threadIdx.x;
    const size_t row = (size_t)blockIdx.x * cols, out = (size_t)blockIdx.x * padded * (DT == CX_DTYPE_F32 ? 2 : 1);
    constexpr int kEl = DT == CX_DTYPE_F32 ? 4 : DT == CX_DTYPE_E4M3 ? 1 : 2, kSpan = kRowPieces * 256 * 8;
    const bool vec = cols % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & (kEl == 1 ? 7 : 15)) == 0;
    float v[kRowPieces][8];
#pragma unroll
    for (int i = 0; i < kRowPieces; ++i) q4_row_piece<DT>(x, row, (i * 256 + tid) * 8, cols, vec, v[i]);
    float up = 1.0f;
    if constexpr (DT == CX_DTYPE_BF16 || DT == CX_DTYPE_F32) {
        uint32_t most = 0;
        auto take = [&](const float (&f)[8]) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t b = __float_as_uint(f[i]) & 0x7FFFFFFFu;
                if (b < 0x7F800000u) most = max(most, b);
            }
        };
#pragma unroll
        for (int i = 0; i < kRowPieces; ++i) take(v[i]);
        for (int c = kSpan + tid * 8; c < cols; c += 2048) {
            float f[8];
            q4_row_piece<DT>(x, row, c, cols, vec, f);
            take(f);
        }
#pragma unroll
        for (int m = 32; m >= 1; m >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, m));
        if ((tid & 63) == 0) part[tid >> 6] = most;
        __syncthreads();
        most = max(max(part[0], part[1]), max(part[2], part[3]));
        const int e = most == 0 ? 127 : min(max((int)(most >> 23) - 14, 1), 253);
        up = __uint_as_float((uint32_t)(254 - e) << 23);
        if (tid == 0) scale[blockIdx.x] = __uint_as_float((uint32_t)e << 23);
    } else if (tid == 0) {
        scale[blockIdx.x] = 1.0f;
    }
    auto put = [&](int c, const float (&f)[8]) {
        u32x4 o;
        if constexpr (DT == CX_DTYPE_F32) {
            u32x4 lo;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint2 p = q4_planes(f[2 * i] * up, f[2 * i + 1] * up);
                o[i] = p.x, lo[i] = p.y;
            }
            uint16_t* to = dst + out + c / 64 * 128 + c % 64;
            *reinterpret_cast<u32x4*>(to) = o;
            *reinterpret_cast<u32x4*>(to + 64) = lo;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = f16_rne(f[2 * i] * up) | (f16_rne(f[2 * i + 1] * up) << 16);
            *reinterpret_cast<u32x4*>(dst + out + c) = o;
        }
    };
#pragma unroll
    for (int i = 0; i < kRowPieces; ++i)
        if ((i * 256 + tid) * 8 < padded) put((i * 256 + tid) * 8, v[i]);
    for (int c = kSpan + tid * 8; c < padded; c += 2048) {
        float f[8];
        q4_row_piece<DT>(x, row, c, cols, vec, f);
        put(c, f);
    }
}

// The runs of rows that `offsets` give each matrix, cut to item_rows.  Offsets that
// go back or past the rows are cut to what is there, so that no item leaves it.
__global__ __launch_bounds__(1024) void k_q4_items(const int32_t* offsets, int n_mats, int n_rows, int item_rows,
                                                   Q4Item* items, int* err_flag) {
    __shared__ int top[1024], totals[2 * Q4LongFirst::kClasses];
    const int e = threadIdx.x;
    if (e < 2 * Q4LongFirst::kClasses) totals[e] = 0;
    const int raw0 = offsets[min(e, n_mats)], raw1 = offsets[min(e + 1, n_mats)];
    if (e < n_mats && (raw0 > raw1 || raw0 < 0 || raw1 > n_rows || (e == 0 && raw0 != 0))) atomicOr(err_flag, kErrBadRow);
    top[e] = min(max(raw1, 0), n_rows);
    __syncthreads();
    for (int d = 1; d < 1024; d <<= 1) {  // running maximum
        const int v = e >= d ? max(top[e], top[e - d]) : top[e];
        __syncthreads();
        top[e] = v;
        __syncthreads();
    }
    const int begin = e == 0 ? 0 : top[e - 1], rows = e < n_mats ? top[e] - begin : 0;
    const Q4LongFirst list{totals};
    const int n = list.items(rows, item_rows);
    list.count(n, rows);
    __syncthreads();
    q4_put_items(items + 1 + list.place(n, rows), n, e, begin, rows, 0, 1);
    const int all = list.all();
    const int held = top[1023], rest = (n_rows - held + item_rows - 1) / item_rows;
    q4_put_items(items + 1 + all, rest, -1, held, n_rows - held, e, 1024);  // rows behind the last matrix's: zeros
    if (e == 0) items[0] = Q4Item{all + rest, held, 0, 0};
}

}  // namespace

size_t q4_code_bytes(const cx_q4_desc& w) { return (size_t)w.n_mats * q4_row_tiles(w) * q4_col_tiles(w) * kQ4Tile; }
size_t q4_scale_bytes(const cx_q4_desc& w) {
    return (size_t)w.n_mats * q4_row_tiles(w) * ((size_t)q4_col_tiles(w) * (128 / w.group) * 32 + 64);
}

hipError_t launch_q4_pack(const cx_q4_desc& w, const uint8_t* codes, const uint16_t* scales, hipStream_t s) {
    const int64_t rows = (int64_t)w.n_mats * q4_row_tiles(w) * 16, tiles = rows / 16 * q4_col_tiles(w);
    float* row_scale = const_cast<float*>(q4_row_scales(w));
    auto wgs = [](int64_t units) { return dim3((unsigned)std::min<int64_t>((units + 3) / 4, 16384)); };
    cx_launch(k_q4_row_scales, wgs(rows), dim3(256), 0, s, w, scales, row_scale, rows);
    cx_launch(k_q4_pack, wgs(tiles), dim3(256), 0, s, w, codes, scales, row_scale,
              reinterpret_cast<uint32_t*>(const_cast<uint8_t*>(w.codes)), const_cast<uint16_t*>(w.scales), tiles);
    return hipGetLastError();
}

hipError_t launch_q4_items(const int32_t* offsets, int n_mats, int n_rows, int item_rows, Q4Item* items, int* err_flag,
                           hipStream_t s) {
    cx_launch(k_q4_items, dim3(1), dim3(1024), 0, s, offsets, n_mats, n_rows, item_rows, items, err_flag);
    return hipGetLastError();
}

namespace {

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

// Ranges of the columns per row tile: up to `all` waves in the launch (16 a CU are 4096), of at least 2
// column tiles each.  The kernel of few rows, whose waves wait for x now and then, takes twice as many
// (18432 x 7168, 1 and 16 rows: 22.8 and 32 us, with 4096 waves 26.8 and 39.8); the decode kernel does not gain.
int column_splits(int64_t waves, int KT, int most, int64_t all) {
    int n = 1;
    while (n < most && waves * n * 2 <= all && KT / n >= 4) n *= 2;
    return n;
}

// The matrices that have rows, at most.
int64_t busy_mats(const Q4Launch& L) { return L.items != nullptr ? std::min(L.n_rows, L.w.n_mats) : (L.n_rows + L.item_rows - 1) / L.item_rows; }
int64_t item_bound(const Q4Launch& L) { return L.items != nullptr ? L.max_items : (L.n_rows + L.item_rows - 1) / L.item_rows; }

template <int XT, int NG>
hipError_t few_launch(const Q4Launch& L, hipStream_t s) {
    const int RT = q4_row_tiles(L.w), KT = q4_col_tiles(L.w), el = L.x_type == kQ4E4m3 ? 1 : 2;
    const int64_t busy = busy_mats(L);
    const bool vec = L.w.cols % 8 == 0 && (reinterpret_cast<uintptr_t>(L.x) & (8 * el - 1)) == 0 && (int64_t)L.n_x * L.w.cols * el < (int64_t)kOob;
    // two row tiles a wave, on one read of x, where that leaves enough waves (7168 x 2048, 1 row: 5.5 and 8.2 us;
    // 4096 x 7168: 8.0 and 7.2, 512 x 512: 5.1 and 4.4)
    const int rw = RT > 256 ? 2 : 1, splits = column_splits(busy * ((RT + rw - 1) / rw), KT, kQ4FewWaves, 8192);
    const int per = kQ4FewWaves / splits * rw, row_blocks = (RT + per - 1) / per;
    auto k = vec ? (rw == 2 ? k_q4_few<XT, NG, 2, true> : k_q4_few<XT, NG, 1, true>) : (rw == 2 ? k_q4_few<XT, NG, 2, false> : k_q4_few<XT, NG, 1, false>);
    cx_launch(k, dim3((unsigned)(item_bound(L) * row_blocks)), dim3(64 * kQ4FewWaves), 0, s, L, RT, KT, splits, row_blocks);
    return hipGetLastError();
}

template <int XT>
hipError_t few_groups(const Q4Launch& L, hipStream_t s) {
    return L.w.group == 128 ? few_launch<XT, 1>(L, s) : L.w.group == 64 ? few_launch<XT, 2>(L, s) : few_launch<XT, 4>(L, s);
}

}  // namespace

bool q4_grid_ok(const Q4Launch& L) {
    const int RT = q4_row_tiles(L.w);
    if (!rows_grid_ok(item_bound(L) * (RT + 16), 1024)) return false;
    return L.item_rows <= kTileTok || (rows_grid_ok(L.n_x, 256) && rows_grid_ok((int64_t)L.n_rows * RT * 4 / 256 + 1, 256) &&
                                       // the GEMM's places in x, in bytes; of two planes within an item
                                       (L.x_type == kQ4F32 ? (int64_t)L.item_rows * 2 : (int64_t)L.n_x) * q4_col_tiles(L.w) * 256 < ((int64_t)1 << 32));
}

size_t q4_x_scratch(const cx_q4_desc& w, int n_x, int planes) { return up256((size_t)n_x * q4_col_tiles(w) * 256 * planes) + up256((size_t)n_x * 4); }

hipError_t launch_q4_routes(const Q4Launch& L, const Q4Launch& D, const Q4Routes& routes, int n_tokens, void* y, int out_dtype,
                            float* y_f32, hipStream_t s) {
    const int ke = routes.top_k + routes.shared;
    const int64_t pairs = (int64_t)n_tokens * ke;
    const hipError_t e = launch_q4_dec(L, &routes, column_splits(pairs * q4_row_tiles(L.w), q4_col_tiles(L.w), kQ4DecWaves, 4096), pairs, s);
    if (e != hipSuccess) return e;
    return launch_q4_dec_sum(Q4DecSumArgs{D.w, D.shared, routes, static_cast<const float*>(D.x), y, y_f32, out_dtype,
                                          q4_row_tiles(D.w), q4_col_tiles(D.w)}, n_tokens, s);
}

hipError_t launch_q4(const Q4Launch& L, hipStream_t s) {
    if (L.item_rows < kTileTok) return launch_q4_dec(L, nullptr, column_splits(busy_mats(L) * q4_row_tiles(L.w), q4_col_tiles(L.w), kQ4DecWaves, 4096), item_bound(L), s);
    if (L.item_rows > kTileTok) {
        const int padded = q4_col_tiles(L.w) * 128;
        Q4Launch G = L;
        if (L.x_type != kQ4Fp16 || padded != L.w.cols || !dma_aligned(L.x)) {
            uint16_t* x = static_cast<uint16_t*>(L.x_scratch);
            float* scale = reinterpret_cast<float*>(static_cast<char*>(L.x_scratch) + up256((size_t)L.n_x * padded * (L.x_type == kQ4F32 ? 4 : 2)));
            auto k = L.x_type == kQ4Bf16   ? k_q4_rows<CX_DTYPE_BF16>
                     : L.x_type == kQ4Fp16 ? k_q4_rows<CX_DTYPE_FP16>
                     : L.x_type == kQ4F32  ? k_q4_rows<CX_DTYPE_F32>
                                           : k_q4_rows<CX_DTYPE_E4M3>;
            if (L.n_x > 0) cx_launch(k, dim3((unsigned)L.n_x), dim3(256), 0, s, L.x, L.w.cols, padded, x, scale);
            G.x = x;
            if (L.x_type != kQ4E4m3) G.x_scale = scale;
        }
        return launch_q4_gemm(G, s);
    }
    switch (L.x_type) {
        case kQ4Bf16: return few_groups<kQ4Bf16>(L, s);
        case kQ4Fp16: return few_groups<kQ4Fp16>(L, s);
        default: return few_groups<kQ4E4m3>(L, s);
    }
}

}  // namespace cx
