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
                                                 uint32_t* dst, uint16_t* dst_scale, int64_t tiles) {
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
        if (lane < 16 * NG) {  // [quarter][group][4 rows]
            const int i = lane & 3, g = (lane >> 2) % NG, n2 = q4_src_row(w, rt, (lane >> 2) / NG * 4 + i);
            const int at = kt * NG + g;
            dst_scale[tile * 16 * NG + lane] = n2 >= 0 && at < groups ? scales[(mat * w.rows + n2) * (int64_t)groups + at] : 0;
        }
    }
}

// The runs of rows that `offsets` give each matrix, cut to item_rows.  Offsets that
// go back or past the rows are cut to what is there, so that no item leaves it.
__global__ __launch_bounds__(1024) void k_q4_items(const int32_t* offsets, int n_mats, int n_rows, int item_rows,
                                                   Q4Item* items, int* err_flag) {
    __shared__ int top[1024], cnt[1024];
    const int e = threadIdx.x;
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
    const int n = (rows + item_rows - 1) / item_rows;
    cnt[e] = n;
    __syncthreads();
    for (int d = 1; d < 1024; d <<= 1) {
        const int v = e >= d ? cnt[e] + cnt[e - d] : cnt[e];
        __syncthreads();
        cnt[e] = v;
        __syncthreads();
    }
    Q4Item* at = items + 1 + cnt[e] - n;
    for (int i = 0; i < n; ++i) at[i] = Q4Item{e, begin + i * item_rows, min(item_rows, rows - i * item_rows), 0};
    const int held = top[1023], all = cnt[1023], rest = (n_rows - held + item_rows - 1) / item_rows;
    for (int i = e; i < rest; i += 1024)  // rows behind the last matrix's: zeros
        items[1 + all + i] = Q4Item{-1, held + i * item_rows, min(item_rows, n_rows - held - i * item_rows), 0};
    if (e == 0) items[0] = Q4Item{all + rest, held, 0, 0};
}

}  // namespace

size_t q4_code_bytes(const cx_q4_desc& w) { return (size_t)w.n_mats * q4_row_tiles(w) * q4_col_tiles(w) * kQ4Tile; }
size_t q4_scale_bytes(const cx_q4_desc& w) {
    return (size_t)w.n_mats * q4_row_tiles(w) * q4_col_tiles(w) * (128 / w.group) * 32;
}

hipError_t launch_q4_pack(const cx_q4_desc& w, const uint8_t* codes, const uint16_t* scales, hipStream_t s) {
    const int64_t tiles = (int64_t)w.n_mats * q4_row_tiles(w) * q4_col_tiles(w);
    const unsigned wgs = (unsigned)std::min<int64_t>((tiles + 3) / 4, 16384);
    cx_launch(k_q4_pack, dim3(wgs), dim3(256), 0, s, w, codes, scales, reinterpret_cast<uint32_t*>(const_cast<uint8_t*>(w.codes)),
              const_cast<uint16_t*>(w.scales), tiles);
    return hipGetLastError();
}

hipError_t launch_q4_items(const int32_t* offsets, int n_mats, int n_rows, int item_rows, Q4Item* items, int* err_flag,
                           hipStream_t s) {
    cx_launch(k_q4_items, dim3(1), dim3(1024), 0, s, offsets, n_mats, n_rows, item_rows, items, err_flag);
    return hipGetLastError();
}

int q4_item_rows(const cx_q4_desc& w, int n_rows, int n_mats) {
    (void)w, (void)n_rows, (void)n_mats;
    return kTileTok;
}

namespace {
int64_t few_workgroups(const Q4Launch& L) {
    return (L.items != nullptr ? L.max_items : (L.n_rows + kTileTok - 1) / kTileTok) * q4_row_tiles(L.w);
}

template <int XT>
hipError_t few_groups(const Q4Launch& L, hipStream_t s) {
    const int RT = q4_row_tiles(L.w);
    auto k = L.w.group == 128 ? k_q4_few<XT, 1> : L.w.group == 64 ? k_q4_few<XT, 2> : k_q4_few<XT, 4>;
    cx_launch(k, dim3((unsigned)few_workgroups(L)), dim3(64 * kQ4FewWaves), 0, s, L, RT, q4_col_tiles(L.w));
    return hipGetLastError();
}
}  // namespace

bool q4_grid_ok(const Q4Launch& L) { return rows_grid_ok(few_workgroups(L), 64 * kQ4FewWaves); }

hipError_t launch_q4(const Q4Launch& L, hipStream_t s) {
    switch (L.x_type) {
        case kQ4Bf16: return few_groups<kQ4Bf16>(L, s);
        case kQ4Fp16: return few_groups<kQ4Fp16>(L, s);
        case kQ4E4m3: return few_groups<kQ4E4m3>(L, s);
        default: return few_groups<kQ4Planes>(L, s);
    }
}

}  // namespace cx
