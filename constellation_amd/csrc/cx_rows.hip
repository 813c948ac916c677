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

// Two values rounded to a 16-bit type (nearest even), the first in the lower half.
template <int DT>
__device__ __forceinline__ uint32_t round2(float a, float b) {
    if constexpr (DT == CX_DTYPE_BF16)
        return __builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(a), static_cast<__bf16>(b)});  // one v_cvt_pk_bf16_f32
    else
        return __builtin_bit_cast(uint32_t, f16x2{static_cast<_Float16>(a), static_cast<_Float16>(b)});
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
        const u32x4 h = {round2<DT>(v[0], v[1]), round2<DT>(v[2], v[3]), round2<DT>(v[4], v[5]), round2<DT>(v[6], v[7])};
        if constexpr (VEC) {
            *reinterpret_cast<u32x4*>(p) = h;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < left) p[i] = static_cast<uint16_t>(h[i >> 1] >> (16 * (i & 1)));
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
// input is read once and each output written once: HBM bounds it (4096 rows of 7168 bf16 with
// residual, sum and e4m3: 206 MB in 42 us, 4.9 TB/s; 357 of 1411 fp16: 7 us).  One row is latency: 5.3 us
// for a load, a barrier, a load of the weight and the stores.  A thread holds VPT pieces of 8 columns; the 16 pieces of a scale block are 16 neighbouring lanes,
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
            for (int j = 0; j < 8; ++j) s[i][j] += r[j];
            if constexpr (DT != CX_DTYPE_F32) {
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const uint32_t h = round2<DT>(s[i][j], s[i][j + 1]);
                    s[i][j] = DT == CX_DTYPE_BF16 ? __uint_as_float(h << 16) : (float)__builtin_bit_cast(f16x2, h)[0];
                    s[i][j + 1] = DT == CX_DTYPE_BF16 ? __uint_as_float(h & 0xFFFF0000u) : (float)__builtin_bit_cast(f16x2, h)[1];
                }
            }
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
        // n: y before the row's factor, exact for 16-bit rows and weights
        float n[8];
        uint32_t most = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            n[j] = s[i][j] * w[j];
            most = max(most, __float_as_uint(n[j]) & 0x7FFFFFFFu);  // columns past the row are zeros
        }
        if (a.y != nullptr && left > 0) {
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = s[i][j] * inv * w[j];
            store8<VEC>(a.y, a.y_dtype, row + c, left, y);
        }
        if (a.q == nullptr) continue;
        const float top = __uint_as_float(row16_max(most));
        float scale = top * inv / 448.0f;
        const bool plain = scale >= 1e-12f && top > 1e-30f && top < 1e30f;  // neither zeros nor infinities nor NaN
        if (!plain) {  // a whole block's lanes: from y itself
            most = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                n[j] = s[i][j] * inv * w[j];
                most = max(most, __float_as_uint(n[j]) & 0x7FFFFFFFu);
            }
            scale = __uint_as_float(row16_max(most)) / 448.0f;
            scale = scale < 1e-12f ? 1e-12f : scale;
        }
        if (left <= 0) continue;
        if ((v & 15) == 0) a.q_scale[(size_t)blockIdx.x * (size_t)((H + 127) >> 7) + (v >> 4)] = scale;
        // y / scale = 448 n / top: the row's factor, and with it its rounding, falls out.  The division is
        // refined to a correctly rounded one, since a code flips where the quotient crosses a border.
        const float by = plain ? top : scale, inv_by = 1.0f / by, gain = plain ? 448.0f : 1.0f;
        auto quotient = [&](int j) {
            const float num = n[j] * gain, r = num * inv_by, better = __builtin_fmaf(__builtin_fmaf(-r, by, num), inv_by, r);
            return plain ? better : r;
        };
        uint32_t b[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            int d = __builtin_amdgcn_cvt_pk_fp8_f32(quotient(4 * j), quotient(4 * j + 1), 0, false);
            b[j] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(quotient(4 * j + 2), quotient(4 * j + 3), d, true);
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
// Pairs sorted by expert: a stable counting sort of the ids, i = t * top_k + k; ids that
// name no expert have the last key.  Where a shared expert takes every token as one more
// route, its rows follow those of all experts, in token order.
//
// Up to 64 workgroups each place a share of consecutive ids.  Each counts the keys of
// all ids, those before its share apart, so none waits for another; within its share, 512
// ids at a time, an id's rank is its rank in the wave (the lanes of the same key, one
// ballot per bit of the key) after the counts of the waves and ids before.  Counts are
// integers: the order of the atomics changes nothing.  Reading the ids, from L2, bounds it, so
// eight loads a thread are in flight: 32,768 ids over 256 experts in 13 us (40 with one load at
// a time); 232 ids in one workgroup 3.5.
constexpr int kSortThreads = 512, kSortWaves = kSortThreads / 64, kSortLoads = 8;
constexpr int kSortKeys = kSortMaxExperts + 2;  // experts, the shared one, none

// First index of each key from its count, in place; entry n gets the total.
template <int PER>
__device__ __forceinline__ void scan_counts(int* v, int n, int* wave_tot) {
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    int own[PER], sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        own[i] = tid * PER + i < n ? v[tid * PER + i] : 0;
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
#pragma unroll
    for (int i = 0; i < kSortWaves; ++i)
        if (i < w) base += wave_tot[i];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (tid * PER + i <= n) v[tid * PER + i] = base;
        base += own[i];
    }
    __syncthreads();
}

// SMALL: up to 512 ids and 510 keys: one workgroup, whose ranks give the counts.
template <bool SMALL>
__global__ __launch_bounds__(kSortThreads) void k_sort_tokens(SortArgs a) {
    constexpr int kKeys = SMALL ? kSortThreads : kSortKeys, kPer = SMALL ? 1 : (kSortKeys + kSortThreads) / kSortThreads;
    __shared__ int first[kKeys + 1], next[kKeys + 1], totals[2 * Q4LongFirst::kClasses];
    __shared__ int hist[kSortWaves][kKeys];
    __shared__ int wave_tot[kSortWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int K = a.top_k, KE = K + a.shared, NK = a.n_experts, N = a.n_tokens * K;  // key NK: none
    const int bits = 32 - __builtin_clz(NK);
    const int chunks = (N + kSortThreads - 1) / kSortThreads;
    const int per = (chunks + (int)gridDim.x - 1) / (int)gridDim.x * kSortThreads;
    const int begin = min(N, (int)blockIdx.x * per), end = min(N, begin + per);
    auto key = [&](int id) { return id >= 0 && id < NK ? id : NK; };
    int err = 0;
    auto place = [&](int i, int e, int row) {
        const int t = i / K, k = i - t * K;
        bool held = e < NK;
        if (held && a.weights != nullptr) {
            // a repeated expert or a bad weight: the row stays, no token takes it
            int bad = route_weight_ok(a.weights[i]) ? 0 : kErrBadWeight;
            for (int j = 1; j <= k; ++j)
                if (a.ids[i - j] == e) bad |= kErrDuplicateRoute;
            err |= bad;
            held = bad == 0;
        }
        const int pair = t * KE + k;
        a.place[pair] = held ? row : ~row;
        a.order[row] = e < NK ? pair : ~pair;
    };
    auto rank_in_wave = [&](int e, bool live, int& count) {
        uint64_t same = __ballot(live);
        for (int b = 0; b < bits; ++b) {
            const uint64_t set = __ballot((e >> b) & 1);
            same &= ((e >> b) & 1) ? set : ~set;
        }
        count = __popcll(same);
        return __popcll(same & ((1ull << lane) - 1));
    };
    const int own = SMALL && tid < N ? a.ids[tid] : 0;
    for (int e = tid; e <= NK + 1; e += kSortThreads) first[e] = next[e] = 0;
    if (tid < 2 * Q4LongFirst::kClasses) totals[tid] = 0;
    if constexpr (SMALL) {
        for (int w = 0; w < kSortWaves; ++w)
            if (tid <= NK) hist[w][tid] = 0;
    }
    __syncthreads();
    int own_rank = 0;
    if constexpr (SMALL) {
        int n;
        own_rank = rank_in_wave(key(own), tid < N, n);
        if (tid < N && own_rank == 0) hist[wave][key(own)] = n;
        if (tid < N && own >= NK) err |= kErrBadExpertId;
        __syncthreads();
        if (tid <= NK) {
            int at = 0;
#pragma unroll
            for (int w = 0; w < kSortWaves; ++w) {
                const int c = hist[w][tid];
                hist[w][tid] = at;
                at += c;
            }
            first[tid] = at;
        }
    } else {
        for (int i0 = 0; i0 < N; i0 += kSortLoads * kSortThreads) {
            int id[kSortLoads];
#pragma unroll
            for (int u = 0; u < kSortLoads; ++u) id[u] = a.ids[min(i0 + u * kSortThreads + tid, N - 1)];
#pragma unroll
            for (int u = 0; u < kSortLoads; ++u) {
                const int i = i0 + u * kSortThreads + tid;
                if (i >= N) continue;
                if (id[u] >= NK) err |= kErrBadExpertId;
                atomicAdd(i < begin ? &next[key(id[u])] : &first[key(id[u])], 1);
            }
        }
        __syncthreads();
        for (int e = tid; e <= NK; e += kSortThreads) first[e] += next[e];
    }
    __syncthreads();
    scan_counts<kPer>(first, NK + 1, wave_tot);
    const int shared_row = first[NK];  // the shared expert's rows, then those without an expert
    const int none = a.shared ? a.n_tokens : 0;
    if (blockIdx.x == 0) {
        if (a.offsets != nullptr)
            for (int e = tid; e <= NK; e += kSortThreads) a.offsets[e] = first[e];
        if (a.items != nullptr) {
            const int more = (none + a.item_rows - 1) / a.item_rows;  // of the shared expert, whose items are the longest
            q4_put_items(a.items + 1, more, NK, shared_row, none, tid, kSortThreads);
            const Q4LongFirst list{totals};
            for (int e = tid; e < NK; e += kSortThreads) {
                const int rows = first[e + 1] - first[e];
                list.count(list.items(rows, a.item_rows), rows);
            }
            __syncthreads();
            for (int e = tid; e < NK; e += kSortThreads) {
                const int rows = first[e + 1] - first[e], n = list.items(rows, a.item_rows);
                q4_put_items(a.items + 1 + more + list.place(n, rows), n, e, first[e], rows, 0, 1);
            }
            const int all = more + list.all();
            if (tid == 0) a.items[0] = Q4Item{all, shared_row + none, 0, 0};
        }
    }
    if (a.shared)
        for (int t = blockIdx.x * kSortThreads + tid; t < a.n_tokens; t += gridDim.x * kSortThreads) {
            a.place[t * KE + K] = shared_row + t;
            a.order[shared_row + t] = t * KE + K;
        }
    auto row_of = [&](int e, int at) { return e < NK ? at : at + none; };
    if constexpr (SMALL) {
        if (tid < N) {
            const int e = key(own);
            place(tid, e, row_of(e, first[e] + hist[wave][e] + own_rank));
        }
    } else {
        for (int e = tid; e <= NK; e += kSortThreads) next[e] += first[e];
        for (int c = begin; c < end; c += kSortThreads) {
            const int i = c + tid;
            const bool live = i < end;
            const int e = live ? key(a.ids[i]) : NK;
            for (int b = tid; b <= NK; b += kSortThreads)
#pragma unroll
                for (int w = 0; w < kSortWaves; ++w) hist[w][b] = 0;
            int n;
            const int rank = rank_in_wave(e, live, n);
            __syncthreads();
            if (live && rank == 0) hist[wave][e] = n;
            __syncthreads();
            for (int b = tid; b <= NK; b += kSortThreads) {
                int at = next[b];
#pragma unroll
                for (int w = 0; w < kSortWaves; ++w) {
                    const int h = hist[w][b];
                    hist[w][b] = at;
                    at += h;
                }
                next[b] = at;
            }
            __syncthreads();
            if (live) place(i, e, row_of(e, hist[wave][e] + rank));
            __syncthreads();
        }
    }
    if (err && a.err_flag != nullptr) atomicOr(a.err_flag, err);
}

// ---------------------------------------------------------------------------
// Rows into sorted order: one read of a token's row, a write per route.  A piece
// of W bytes of one token per thread; the token's places are wave-uniform loads.
// Copies bytes, so it takes rows of any type.  HBM bounds it: 4096 rows of 7168 bf16 to 32,768,
// 528 MB in 95 to 111 us, 4.7 to 5.5 TB/s.  (A workgroup per sorted row would read x top_k times.)
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
    const int pieces = (int)(g.row_bytes / sizeof(V)), chunks = (int)(((int64_t)pieces + kRowThreads - 1) / kRowThreads);
    cx_launch(k_gather_rows<V>, dim3((unsigned)(g.n_tokens * chunks)), dim3(kRowThreads), 0, s, static_cast<const V*>(g.x),
              static_cast<V*>(g.xs), g.place, g.top_k, g.n_tokens * g.top_k, pieces, chunks, g.err_flag);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Eight columns of a thread for the sums below: with VEC the eight from 8 * lane on, as
// 16-byte accesses; otherwise every kRowThreads-th, so that neighbouring threads still touch
// neighbouring values of rows that start anywhere.  A load is kept as it arrives, so
// that the loads of several rows are in flight together.
template <int DT, bool VEC>
struct Cols {
    static constexpr int kStep = VEC ? 1 : kRowThreads;
    uint32_t d[VEC ? (DT == CX_DTYPE_F32 ? 8 : 4) : 8];

    // columns at, at + kStep, ...; `left` of the row's columns are left from `at` on (those past them repeat the last)
    __device__ __forceinline__ void load(const void* base, size_t at, int left) {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < (int)(sizeof(d) / 16); ++i) {
                const u32x4 v = ld16(static_cast<const char*>(base) + at * (DT == CX_DTYPE_F32 ? 4 : 2) + 16 * i);
#pragma unroll
                for (int j = 0; j < 4; ++j) d[4 * i + j] = v[j];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const size_t p = at + min(i * kStep, (left - 1) / kStep * kStep);
                if constexpr (DT == CX_DTYPE_F32)
                    d[i] = static_cast<const uint32_t*>(base)[p];
                else
                    d[i] = static_cast<const uint16_t*>(base)[p];
            }
        }
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (DT == CX_DTYPE_F32) return __uint_as_float(d[i]);
        const uint32_t h = !VEC ? d[i] : i & 1 ? d[i >> 1] >> 16 : d[i >> 1] & 0xFFFFu;
        if constexpr (DT == CX_DTYPE_BF16) return __uint_as_float(h << 16);
        return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(h)));
    }
};

// The same with the type known at run time.
template <bool VEC>
__device__ __forceinline__ void load_cols(const void* base, int dtype, size_t at, int left, float (&v)[8]) {
    auto as = [&](auto c) {
        c.load(base, at, left);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c.get(i);
    };
    if (dtype == CX_DTYPE_BF16)
        as(Cols<CX_DTYPE_BF16, VEC>{});
    else if (dtype == CX_DTYPE_FP16)
        as(Cols<CX_DTYPE_FP16, VEC>{});
    else
        as(Cols<CX_DTYPE_F32, VEC>{});
}

template <bool VEC>
__device__ __forceinline__ void store_cols(void* base, int dtype, size_t at, int left, const float (&v)[8]) {
    if constexpr (VEC) {
        store8<true>(base, dtype, at, left, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i * kRowThreads >= left) continue;
            if (dtype == CX_DTYPE_F32)
                static_cast<float*>(base)[at + i * kRowThreads] = v[i];
            else
                static_cast<uint16_t*>(base)[at + i * kRowThreads] = (uint16_t)cast_out(v[i], dtype);
        }
    }
}

// A thread's first column of the c-th 8 * kRowThreads columns of a row.
template <bool VEC>
__device__ __forceinline__ int first_col(int c) {
    return c * 8 * kRowThreads + (VEC ? 8 : 1) * (int)threadIdx.x;
}

// out[t] = sum over k, in this order and in fp32, of w[t, k] * ys[place[t, k]], then
// + add[t], rounded once.  Eight columns of one token per thread; the loads of eight
// routes are in flight together (145 us without, 122 with, where 32,768 bf16 rows of 7168 come to
// 4096 tokens and are added: 588 MB, 4.8 TB/s, HBM).  Widths that 8 does not divide: below.
template <int DT, bool VEC>
__global__ __launch_bounds__(kRowThreads) void k_combine_rows(CombineArgs a, int chunks) {
    const int t = blockIdx.x / chunks, H = a.hidden, K = a.top_k, c = first_col<VEC>(blockIdx.x - t * chunks), left = H - c;
    if (left <= 0) return;
    float acc[8] = {};
    for (int k0 = 0; k0 < K; k0 += 8) {
        Cols<DT, VEC> v[8];
        int p[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            p[k] = k0 + k < K ? a.place[(size_t)t * K + k0 + k] : -1;
            if (p[k] >= a.n_rows) {
                atomicOr(a.err_flag, kErrBadRow);
                p[k] = -1;
            }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)  // of a pair without an expert: row 0, which is there, and left out below
            v[k].load(a.ys, (size_t)max(p[k], 0) * H + c, left);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (p[k] < 0) continue;
            const float w = a.weights != nullptr && k0 + k < a.weights_step ? a.weights[(size_t)t * a.weights_step + k0 + k] : 1.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] += w * v[k].get(j);
        }
    }
    if (a.add != nullptr) {
        float v[8];
        load_cols<VEC>(a.add, a.out_dtype, (size_t)t * H + c, left, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] += v[j];
    }
    store_cols<VEC>(a.out, a.out_dtype, (size_t)t * H + c, left, acc);
    if (a.out_f32 != nullptr) store_cols<VEC>(a.out_f32, CX_DTYPE_F32, (size_t)t * H + c, left, acc);
}

// Its gradient: dys[place[t, k]] = w[t, k] * dout[t] and dw[t, k] = <dout[t],
// ys[place[t, k]]>; rows of pairs without an expert get zeros.  A workgroup takes
// up to eight routes of one token, so dout is read once for them and each row of ys
// and dys is touched once; the sums over columns are per thread in fp32, then over
// the lanes and waves in a fixed order.  HBM bounds it: 2048 tokens of 8 rows of 7168 bf16,
// 499 MB in 126 us, 4.0 TB/s (reads and writes half and half).
template <int DT, bool VEC>
__global__ __launch_bounds__(kRowThreads) void k_combine_grad(CombineGradArgs a, int routes, int splits) {
    constexpr int kNone = -1, kZeros = INT32_MIN;  // no such route; a row of zeros (kZeros | row)
    __shared__ float part[4][8];
    const int t = blockIdx.x / splits, k0 = (blockIdx.x - t * splits) * routes;
    const int H = a.hidden, n = min(routes, a.top_k - k0), tid = threadIdx.x;
    const size_t first = (size_t)t * a.top_k + k0;
    int row[8];
    float w[8], dot[8] = {};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const int p = k < n ? a.place[first + k] : 0, at = p < 0 ? ~p : p;
        w[k] = k < n && a.weights != nullptr ? a.weights[first + k] : 1.0f;
        row[k] = k >= n || at >= a.n_rows ? kNone : p < 0 ? at | kZeros : at;
        if (k < n && at >= a.n_rows) atomicOr(a.err_flag, kErrBadRow);
    }
    for (int b = 0, c = first_col<VEC>(0); c < H; c = first_col<VEC>(++b)) {
        const int left = H - c;
        float d[8];
        Cols<DT, VEC> v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < routes) v[k].load(a.ys, (size_t)max(row[k], 0) * H + c, left);
        load_cols<VEC>(a.dout, a.dout_dtype, (size_t)t * H + c, left, d);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (row[k] == kNone) continue;
            float o[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const bool in = VEC || j * kRowThreads < left;
                if (row[k] >= 0 && in) dot[k] += d[j] * v[k].get(j);
                o[j] = row[k] >= 0 ? w[k] * d[j] : 0.0f;
            }
            store_cols<VEC>(a.dys, DT, (size_t)(row[k] & INT32_MAX) * H + c, left, o);
        }
    }
    if (a.dw == nullptr) return;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        if (k >= routes) break;
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
    const int64_t ids = (int64_t)a.n_tokens * a.top_k;
    if (ids <= kSortThreads && a.n_experts + 2 <= kSortThreads) {
        cx_launch(k_sort_tokens<true>, dim3(1), dim3(kSortThreads), 0, s, a);
    } else {
        const int64_t wgs = std::clamp<int64_t>((ids + kSortThreads - 1) / kSortThreads, 1, 64);
        cx_launch(k_sort_tokens<false>, dim3((unsigned)wgs), dim3(kSortThreads), 0, s, a);
    }
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
    const int routes = combine_grad_routes((int64_t)a.n_tokens * a.top_k, vec), splits = (a.top_k + routes - 1) / routes;
    auto k = a.ys_dtype == CX_DTYPE_BF16   ? (vec ? k_combine_grad<CX_DTYPE_BF16, true> : k_combine_grad<CX_DTYPE_BF16, false>)
             : a.ys_dtype == CX_DTYPE_FP16 ? (vec ? k_combine_grad<CX_DTYPE_FP16, true> : k_combine_grad<CX_DTYPE_FP16, false>)
                                           : (vec ? k_combine_grad<CX_DTYPE_F32, true> : k_combine_grad<CX_DTYPE_F32, false>);
    cx_launch(k, dim3((unsigned)(a.n_tokens * splits)), dim3(kRowThreads), 0, s, a, routes, splits);
    return hipGetLastError();
}

}  // namespace cx
