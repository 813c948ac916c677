// cx_rows.hip — the rows around the experts: RMS norm with the residual's
// addition and an e4m3 output, token-expert pairs sorted by expert, and rows
// gathered into that order and summed back, with the sum's gradient.
#include <algorithm>

#include "cx_device.h"

namespace cx {
namespace {

// Eight consecutive values of a row as fp32.  VEC: the row and the address allow
// 16-byte accesses and `left` is 8 or more; otherwise `left` of them exist.
template <int DT, bool VEC>
__device__ __forceinline__ void load8(const void* base, size_t at, int left, float (&v)[8]) {
    if constexpr (DT == CX_DTYPE_F32) {
        const float* p = static_cast<const float*>(base) + at;
        if constexpr (VEC) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = i < left ? p[i] : 0.0f;
        }
    } else {
        const uint16_t* p = static_cast<const uint16_t*>(base) + at;
        uint32_t h[8];
        if constexpr (VEC) {
            const u32x4 a = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) h[2 * i] = a[i] & 0xFFFFu, h[2 * i + 1] = a[i] >> 16;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = i < left ? p[i] : 0u;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (DT == CX_DTYPE_BF16)
                v[i] = __uint_as_float(h[i] << 16);
            else
                v[i] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(h[i])));
        }
    }
}

template <bool VEC>
__device__ __forceinline__ void load8(const void* base, int dtype, size_t at, int left, float (&v)[8]) {
    if (dtype == CX_DTYPE_BF16)
        load8<CX_DTYPE_BF16, VEC>(base, at, left, v);
    else if (dtype == CX_DTYPE_FP16)
        load8<CX_DTYPE_FP16, VEC>(base, at, left, v);
    else
        load8<CX_DTYPE_F32, VEC>(base, at, left, v);
}

template <int DT, bool VEC>
__device__ __forceinline__ void store8(void* base, size_t at, int left, const float (&v)[8]) {
    if constexpr (DT == CX_DTYPE_F32) {
        float* p = static_cast<float*>(base) + at;
        if constexpr (VEC) {
            *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
            *reinterpret_cast<f32x4*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < left) p[i] = v[i];
        }
    } else {
        uint16_t* p = static_cast<uint16_t*>(base) + at;
        uint32_t h[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = cast_out(v[i], DT);
        if constexpr (VEC) {
            *reinterpret_cast<u32x4*>(p) = u32x4{h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16), h[6] | (h[7] << 16)};
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < left) p[i] = static_cast<uint16_t>(h[i]);
        }
    }
}

template <bool VEC>
__device__ __forceinline__ void store8(void* base, int dtype, size_t at, int left, const float (&v)[8]) {
    if (dtype == CX_DTYPE_BF16)
        store8<CX_DTYPE_BF16, VEC>(base, at, left, v);
    else if (dtype == CX_DTYPE_FP16)
        store8<CX_DTYPE_FP16, VEC>(base, at, left, v);
    else
        store8<CX_DTYPE_F32, VEC>(base, at, left, v);
}

template <int DT>
__device__ __forceinline__ float rounded(float f) {
    if constexpr (DT == CX_DTYPE_BF16)
        return __uint_as_float(bf16_rne(f) << 16);
    else if constexpr (DT == CX_DTYPE_FP16)
        return static_cast<float>(static_cast<_Float16>(f));
    else
        return f;
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m);
    return v;
}

// Largest value of the lane's row of 16 lanes.
__device__ __forceinline__ uint32_t row16_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xF, 0xF, true));  // row_ror 1, 2, 4, 8
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xF, 0xF, true));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xF, 0xF, true));
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xF, 0xF, true));
}

// ---------------------------------------------------------------------------
// s = rnd(x + residual);  y = s / sqrt(mean(s^2) + eps) * weight;
// per 128 columns: c = max(max|y| / 448, 1e-12), q = e4m3(y / c).
//
// A row stays in registers between its sum of squares and its outputs, so each
// input is read once and each output written once: HBM bounds it.  A thread holds
// VPT pieces of 8 columns; the 16 pieces of a scale block are 16 neighbouring lanes,
// whose maximum is four DPP steps.  |y| is compared as bits, which orders a NaN
// above all numbers: its block's scale is NaN too.
template <int DT, bool VEC, int VPT>
__global__ __launch_bounds__(1024) void k_rms_norm(NormArgs a) {
    __shared__ float part[16];
    const int H = a.hidden, tid = threadIdx.x;
    const size_t row = (size_t)blockIdx.x * (size_t)H;
    float s[VPT][8];
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int c = (i * (int)blockDim.x + tid) * 8, left = H - c;
#pragma unroll
        for (int j = 0; j < 8; ++j) s[i][j] = 0.0f;
        if (left <= 0) continue;
        load8<DT, VEC>(a.x, row + c, left, s[i]);
        if (a.residual != nullptr) {
            float r[8];
            load8<DT, VEC>(a.residual, row + c, left, r);
#pragma unroll
            for (int j = 0; j < 8; ++j) s[i][j] = rounded<DT>(s[i][j] + r[j]);
        }
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int c = (i * (int)blockDim.x + tid) * 8, left = H - c;
        if (a.sum != nullptr && left > 0) store8<DT, VEC>(a.sum, row + c, left, s[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) ss += s[i][j] * s[i][j];
    }
    ss = wave_sum(ss);
    if ((tid & 63) == 0) part[tid >> 6] = ss;
    __syncthreads();
    ss = 0.0f;
    for (int w = 0; w < (int)blockDim.x >> 6; ++w) ss += part[w];
    const float inv = 1.0f / sqrtf(ss / (float)H + a.eps);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int v = i * (int)blockDim.x + tid, c = v * 8, left = H - c;
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = 1.0f;
        if (left > 0 && a.weight != nullptr) load8<VEC>(a.weight, a.w_dtype, c, left, w);
        uint32_t most = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            s[i][j] = s[i][j] * inv * w[j];
            if (j < left) most = max(most, __float_as_uint(s[i][j]) & 0x7FFFFFFFu);
        }
        if (a.y != nullptr && left > 0) store8<VEC>(a.y, a.y_dtype, row + c, left, s[i]);
        if (a.q == nullptr) continue;
        float scale = __uint_as_float(row16_max(most)) / 448.0f;
        scale = scale < 1e-12f ? 1e-12f : scale;
        if (left <= 0) continue;
        if ((v & 15) == 0) a.q_scale[(size_t)blockIdx.x * (size_t)((H + 127) >> 7) + (v >> 4)] = scale;
        const float up = 1.0f / scale;
        uint32_t b[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            int d = __builtin_amdgcn_cvt_pk_fp8_f32(s[i][4 * j] * up, s[i][4 * j + 1] * up, 0, false);
            b[j] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(s[i][4 * j + 2] * up, s[i][4 * j + 3] * up, d, true);
        }
        uint8_t* q = a.q + row + c;
        if constexpr (VEC) {
            *reinterpret_cast<uint2*>(q) = uint2{b[0], b[1]};
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j < left) q[j] = (uint8_t)(b[j >> 2] >> (8 * (j & 3)));
        }
    }
}

template <int DT, bool VEC>
hipError_t norm_vpt(const NormArgs& a, hipStream_t s) {
    const int nvec = (a.hidden + 7) / 8;
    const int vpt = nvec <= 1024 ? 1 : nvec <= 2048 ? 2 : nvec <= 4096 ? 4 : 8;
    const int threads = ((nvec + vpt - 1) / vpt + 63) / 64 * 64;
    auto k = vpt == 1 ? k_rms_norm<DT, VEC, 1> : vpt == 2 ? k_rms_norm<DT, VEC, 2> : vpt == 4 ? k_rms_norm<DT, VEC, 4> : k_rms_norm<DT, VEC, 8>;
    cx_launch(k, dim3((unsigned)a.n_tokens), dim3((unsigned)threads), 0, s, a);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Pairs sorted by expert: a stable counting sort.  Pair i = t * K' + k, K' = top_k,
// or top_k + 1 where a shared expert takes every token as its last route; key =
// the expert, the shared one after all others, pairs without an expert last.
//
// Up to 64 workgroups each place a share of consecutive pairs.  Each counts the
// keys of all pairs and of those before its share, so none waits for another; within
// its share, 512 pairs at a time, a pair's rank is its rank in the wave (the lanes
// of the same key, one ballot per bit of the key) after the counts of the waves and
// pairs before.  Counts are integers: the order of the atomics changes nothing.
constexpr int kSortThreads = 512, kSortWaves = kSortThreads / 64;
constexpr int kSortKeys = kSortMaxExperts + 2;  // experts, the shared one, none

// First index of each key from its count, in place; entry n gets the total.
__device__ __forceinline__ void scan_counts(int* v, int n, int* wave_tot) {
    constexpr int kPer = (kSortKeys + kSortThreads) / kSortThreads;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    int own[kPer], sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        own[i] = tid * kPer + i < n ? v[tid * kPer + i] : 0;
        sum += own[i];
    }
    int inc = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(inc, d);
        if (lane >= d) inc += o;
    }
    if (lane == 63) wave_tot[w] = inc;
    __syncthreads();
    int base = inc - sum;
    for (int i = 0; i < w; ++i) base += wave_tot[i];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        if (tid * kPer + i <= n) v[tid * kPer + i] = base;
        base += own[i];
    }
    __syncthreads();
}

__global__ __launch_bounds__(kSortThreads) void k_sort_tokens(SortArgs a) {
    __shared__ int first[kSortKeys + 1], next[kSortKeys + 1], items[kSortKeys + 1];
    __shared__ int hist[kSortWaves][kSortKeys];
    __shared__ int wave_tot[kSortWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int K = a.top_k, E = a.n_experts, KE = K + a.shared, NK = E + a.shared, P = a.n_tokens * KE;
    const int bits = 32 - __builtin_clz(NK);
    const int chunks = (P + kSortThreads - 1) / kSortThreads;
    const int per = (chunks + (int)gridDim.x - 1) / (int)gridDim.x * kSortThreads;
    const int begin = min(P, (int)blockIdx.x * per), end = min(P, begin + per);
    int err = 0;
    auto key = [&](int i) {
        const int t = i / KE, k = i - t * KE;
        if (k == K) return E;  // the shared expert
        const int32_t* row = a.ids + (size_t)t * K;
        const int e = row[k];
        if (e < 0) return NK;
        int bad = e >= E ? kErrBadExpertId : 0;
        if (a.weights != nullptr) {
            for (int j = 0; j < k; ++j)
                if (row[j] == e) bad |= kErrDuplicateRoute;
            if (!route_weight_ok(a.weights[(size_t)t * K + k])) bad |= kErrBadWeight;
        }
        err |= bad;
        return bad ? NK : e;
    };
    for (int e = tid; e <= NK + 1; e += kSortThreads) first[e] = next[e] = 0;
    __syncthreads();
    for (int i = tid; i < P; i += kSortThreads) {
        const int e = key(i);
        atomicAdd(&first[e], 1);
        if (i < begin) atomicAdd(&next[e], 1);
    }
    __syncthreads();
    if (blockIdx.x == 0 && a.items != nullptr) {
        for (int e = tid; e < NK; e += kSortThreads) items[e] = (first[e] + a.item_rows - 1) / a.item_rows;
        __syncthreads();
        scan_counts(items, NK, wave_tot);
    }
    scan_counts(first, NK + 1, wave_tot);
    if (blockIdx.x == 0) {
        if (a.offsets != nullptr)
            for (int e = tid; e <= E; e += kSortThreads) a.offsets[e] = first[e];
        if (a.items != nullptr) {
            for (int e = tid; e < NK; e += kSortThreads)
                for (int i = items[e], p = first[e]; p < first[e + 1]; ++i, p += a.item_rows)
                    a.items[1 + i] = Q4Item{e, p, min(a.item_rows, first[e + 1] - p), 0};
            if (tid == 0) a.items[0] = Q4Item{items[NK], first[NK], 0, 0};
        }
        if (err && a.err_flag != nullptr) atomicOr(a.err_flag, err);
    }
    for (int e = tid; e <= NK; e += kSortThreads) next[e] += first[e];
    for (int c = begin; c < end; c += kSortThreads) {
        for (int e = tid; e < kSortWaves * kSortKeys; e += kSortThreads) (&hist[0][0])[e] = 0;
        __syncthreads();
        const int i = c + tid;
        const bool live = i < end;
        const int e = live ? key(i) : NK;
        uint64_t same = __ballot(live);
        for (int b = 0; b < bits; ++b) {
            const uint64_t set = __ballot((e >> b) & 1);
            same &= ((e >> b) & 1) ? set : ~set;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1));
        if (live && rank == 0) hist[wave][e] = __popcll(same);
        __syncthreads();
        for (int b = tid; b <= NK; b += kSortThreads) {
            int at = next[b];
            for (int w = 0; w < kSortWaves; ++w) {
                const int n = hist[w][b];
                hist[w][b] = at;
                at += n;
            }
            next[b] = at;
        }
        __syncthreads();
        if (live) {
            const int row = hist[wave][e] + rank;
            const bool held = e < NK;
            a.place[i] = held ? row : ~row;
            a.order[row] = held ? i : ~i;
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------
// Rows into sorted order: one read of a token's row, a write per route.  A piece
// of W bytes of one token per thread; the token's places are wave-uniform loads.
// Copies bytes, so it takes rows of any type.
template <class V>
__global__ __launch_bounds__(kRowThreads) void k_gather_rows(const V* x, V* xs, const int32_t* place, int top_k, int n_rows,
                                                     int pieces, int chunks, int* err_flag) {
    const int t = blockIdx.x / chunks, c = (blockIdx.x - t * chunks) * kRowThreads + threadIdx.x;
    if (c >= pieces) return;
    const V v = x[(size_t)t * pieces + c];
    for (int k = 0; k < top_k; ++k) {
        const int p = place[(size_t)t * top_k + k], row = p < 0 ? ~p : p;
        if (row >= n_rows) {
            atomicOr(err_flag, kErrBadRow);
            continue;
        }
        xs[(size_t)row * pieces + c] = p < 0 ? V{} : v;
    }
}

// The widest access that rows and addresses allow.
int gather_width(const GatherArgs& g) {
    const uintptr_t any = reinterpret_cast<uintptr_t>(g.x) | reinterpret_cast<uintptr_t>(g.xs) | g.row_bytes | 16;
    return (int)(any & (~any + 1));
}

template <class V>
hipError_t gather_as(const GatherArgs& g, hipStream_t s) {
    const int pieces = (int)(g.row_bytes / sizeof(V)), chunks = (pieces + kRowThreads - 1) / kRowThreads;
    cx_launch(k_gather_rows<V>, dim3((unsigned)(g.n_tokens * chunks)), dim3(kRowThreads), 0, s, static_cast<const V*>(g.x),
              static_cast<V*>(g.xs), g.place, g.top_k, g.n_tokens * g.top_k, pieces, chunks, g.err_flag);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// out[t] = sum over k, in this order and in fp32, of w[t, k] * ys[place[t, k]], then
// + add[t], rounded once.  Eight columns of one token per thread; the loads of eight
// routes are in flight together.
template <int DT, bool VEC>
__global__ __launch_bounds__(kRowThreads) void k_combine_rows(CombineArgs a, int chunks) {
    const int t = blockIdx.x / chunks, c = ((blockIdx.x - t * chunks) * kRowThreads + threadIdx.x) * 8;
    const int H = a.hidden, K = a.top_k, left = H - c;
    if (left <= 0) return;
    float acc[8] = {};
    for (int k0 = 0; k0 < K; k0 += 8) {
        float v[8][8], w[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const size_t i = (size_t)t * K + k0 + k;
            int p = k0 + k < K ? a.place[i] : -1;
            if (p >= a.n_rows) {
                atomicOr(a.err_flag, kErrBadRow);
                p = -1;
            }
            w[k] = p < 0 ? 0.0f : a.weights != nullptr && k0 + k < a.weights_step ? a.weights[(size_t)t * a.weights_step + k0 + k] : 1.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[k][j] = 0.0f;
            if (p >= 0) load8<DT, VEC>(a.ys, (size_t)p * H + c, left, v[k]);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] += w[k] * v[k][j];
    }
    if (a.add != nullptr) {
        float v[8];
        load8<VEC>(a.add, a.out_dtype, (size_t)t * H + c, left, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] += v[j];
    }
    store8<VEC>(a.out, a.out_dtype, (size_t)t * H + c, left, acc);
    if (a.out_f32 != nullptr) store8<CX_DTYPE_F32, VEC>(a.out_f32, (size_t)t * H + c, left, acc);
}

// Its gradient: dys[place[t, k]] = w[t, k] * dout[t] and dw[t, k] = <dout[t],
// ys[place[t, k]]>; rows of pairs without an expert get zeros.  A workgroup takes
// up to eight routes of one token, so dout is read once for them and each row of ys
// and dys is touched once; the sums over columns are per thread in fp32, then over
// the lanes and waves in a fixed order.
template <int DT, bool VEC>
__global__ __launch_bounds__(kRowThreads) void k_combine_grad(CombineGradArgs a, int routes, int splits) {
    __shared__ float part[4][8];
    const int t = blockIdx.x / splits, k0 = (blockIdx.x - t * splits) * routes;
    const int H = a.hidden, n = min(routes, a.top_k - k0), tid = threadIdx.x;
    const size_t first = (size_t)t * a.top_k + k0;
    int row[8];
    float w[8], dot[8] = {};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const int p = k < n ? a.place[first + k] : 0;
        row[k] = p < 0 ? ~p : p;
        w[k] = k < n && p >= 0 ? (a.weights != nullptr ? a.weights[first + k] : 1.0f) : 0.0f;
        if (k >= n) row[k] = -1;
        if (row[k] >= a.n_rows) {
            atomicOr(a.err_flag, kErrBadRow);
            row[k] = -1;
        }
        if (k < n && p < 0 && row[k] >= 0) row[k] |= INT32_MIN;  // zeros, no product
    }
    for (int c = tid * 8; c < H; c += kRowThreads * 8) {
        const int left = H - c;
        float d[8], v[8][8];
        load8<VEC>(a.dout, a.dout_dtype, (size_t)t * H + c, left, d);
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (row[k] >= 0) load8<DT, VEC>(a.ys, (size_t)row[k] * H + c, left, v[k]);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (row[k] == -1) continue;
            float o[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (row[k] >= 0) dot[k] += d[j] * v[k][j];
                o[j] = row[k] >= 0 ? w[k] * d[j] : 0.0f;
            }
            store8<DT, VEC>(a.dys, (size_t)(row[k] & INT32_MAX) * H + c, left, o);
        }
    }
    if (a.dw == nullptr) return;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float v = wave_sum(dot[k]);
        if ((tid & 63) == 0) part[tid >> 6][k] = v;
    }
    __syncthreads();
    if (tid < n) a.dw[first + tid] = part[0][tid] + part[1][tid] + part[2][tid] + part[3][tid];
}

bool at16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }  // also true of NULL

}  // namespace

hipError_t launch_rms_norm(const NormArgs& a, hipStream_t s) {
    const bool vec = a.hidden % 8 == 0 && at16(a.x) && at16(a.residual) && at16(a.sum) && at16(a.y) && at16(a.weight) &&
                     (reinterpret_cast<uintptr_t>(a.q) & 7) == 0;
    if (a.x_dtype == CX_DTYPE_BF16) return vec ? norm_vpt<CX_DTYPE_BF16, true>(a, s) : norm_vpt<CX_DTYPE_BF16, false>(a, s);
    if (a.x_dtype == CX_DTYPE_FP16) return vec ? norm_vpt<CX_DTYPE_FP16, true>(a, s) : norm_vpt<CX_DTYPE_FP16, false>(a, s);
    return vec ? norm_vpt<CX_DTYPE_F32, true>(a, s) : norm_vpt<CX_DTYPE_F32, false>(a, s);
}

hipError_t launch_sort_tokens(const SortArgs& a, hipStream_t s) {
    const int64_t pairs = (int64_t)a.n_tokens * (a.top_k + a.shared);
    const int64_t wgs = std::max<int64_t>(1, std::min<int64_t>(64, (pairs + kSortThreads - 1) / kSortThreads));
    cx_launch(k_sort_tokens, dim3((unsigned)wgs), dim3(kSortThreads), 0, s, a);
    return hipGetLastError();
}

int64_t gather_workgroups(const GatherArgs& g) {
    const int64_t pieces = (int64_t)g.row_bytes / gather_width(g);
    return g.n_tokens * ((pieces + kRowThreads - 1) / kRowThreads);
}

hipError_t launch_gather_rows(const GatherArgs& g, hipStream_t s) {
    switch (gather_width(g)) {
        case 16: return gather_as<uint4>(g, s);
        case 8: return gather_as<uint2>(g, s);
        case 4: return gather_as<uint32_t>(g, s);
        case 2: return gather_as<uint16_t>(g, s);
        default: return gather_as<uint8_t>(g, s);
    }
}

int64_t combine_workgroups(const CombineArgs& a) { return (int64_t)a.n_tokens * ((a.hidden + 8 * kRowThreads - 1) / (8 * kRowThreads)); }

hipError_t launch_combine_rows(const CombineArgs& a, hipStream_t s) {
    const bool vec = a.hidden % 8 == 0 && at16(a.ys) && at16(a.add) && at16(a.out) && at16(a.out_f32);
    const int chunks = (a.hidden + 8 * kRowThreads - 1) / (8 * kRowThreads);
    auto k = a.ys_dtype == CX_DTYPE_BF16   ? (vec ? k_combine_rows<CX_DTYPE_BF16, true> : k_combine_rows<CX_DTYPE_BF16, false>)
             : a.ys_dtype == CX_DTYPE_FP16 ? (vec ? k_combine_rows<CX_DTYPE_FP16, true> : k_combine_rows<CX_DTYPE_FP16, false>)
                                           : (vec ? k_combine_rows<CX_DTYPE_F32, true> : k_combine_rows<CX_DTYPE_F32, false>);
    cx_launch(k, dim3((unsigned)(a.n_tokens * chunks)), dim3(kRowThreads), 0, s, a, chunks);
    return hipGetLastError();
}

hipError_t launch_combine_grad(const CombineGradArgs& a, hipStream_t s) {
    const bool vec = a.hidden % 8 == 0 && at16(a.ys) && at16(a.dys) && at16(a.dout);
    const int routes = a.n_tokens < 1024 ? 1 : 8, splits = (a.top_k + routes - 1) / routes;
    auto k = a.ys_dtype == CX_DTYPE_BF16   ? (vec ? k_combine_grad<CX_DTYPE_BF16, true> : k_combine_grad<CX_DTYPE_BF16, false>)
             : a.ys_dtype == CX_DTYPE_FP16 ? (vec ? k_combine_grad<CX_DTYPE_FP16, true> : k_combine_grad<CX_DTYPE_FP16, false>)
                                           : (vec ? k_combine_grad<CX_DTYPE_F32, true> : k_combine_grad<CX_DTYPE_F32, false>);
    cx_launch(k, dim3((unsigned)(a.n_tokens * splits)), dim3(kRowThreads), 0, s, a, routes, splits);
    return hipGetLastError();
}

}  // namespace cx
