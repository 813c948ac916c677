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

typedef int i32x4 __attribute__((ext_vector_type(4)));

// v_mfma 16x16 of 16 bytes a lane and operand: lane l holds row (column) l % 16, bytes 16 (l / 16) .. + 15 of 64 of the
// contraction; a result's element i is row 4 (l / 16) + i, column l % 16.
struct MmBf16 {
    static constexpr int kType = CX_DTYPE_BF16, kEl = 2;
    typedef f32x4 Acc;
    static __device__ __forceinline__ Acc mma(u32x4 a, u32x4 b, Acc c) { return Mma<false>::mma(Mma<false>::bits(a), Mma<false>::bits(b), c); }
};
struct MmF16 {
    static constexpr int kType = CX_DTYPE_FP16, kEl = 2;
    typedef f32x4 Acc;
    static __device__ __forceinline__ Acc mma(u32x4 a, u32x4 b, Acc c) { return Mma<true>::mma(Mma<true>::bits(a), Mma<true>::bits(b), c); }
};
struct MmI8 {
    static constexpr int kType = kMmI8, kEl = 1;
    typedef i32x4 Acc;
    static __device__ __forceinline__ Acc mma(u32x4 a, u32x4 b, Acc c) {
        return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
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

// Run idx of up to item_rows rows, of whole tiles of 16 (uniform in a wave; each wave finds it by itself).
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
            const int share = mm_share(m, r);  // equal runs
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
// A workgroup's tile: WM x WN waves of TM x TN results of 16 x 16.  m is the direction in which the
// output is contiguous, n its rows.
template <int WM_, int WN_, int TM_, int TN_, int SLOTS>
struct MmShape {
    static constexpr int WM = WM_, WN = WN_, TM = TM_, TN = TN_;
    static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves;
    static constexpr int BM = WM * TM * 16, BN = WN * TN * 16;
    // LDS: a step of the contraction is 128 bytes of each row (column) of an operand; SLOTS steps of n, one more of m
    static constexpr int kSlots = SLOTS, kStepM = BM * 128, kStepN = BN * 128, kEndM = (SLOTS + 1) * kStepM;
    static constexpr int kLds = kEndM + SLOTS * kStepN;
};

static __device__ __attribute__((aligned(16))) const uint32_t mm_zeros[4] = {};

// 16 bytes at any alignment.
struct __attribute__((packed)) MmPacked {
    u32x4 v;
};

// A pointer that is the same in all lanes, in scalar registers.
__device__ __forceinline__ const char* mm_uniform(const void* p) {
    const uint64_t v = (uint64_t)p;
    return (const char*)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)v) | ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(v >> 32)) << 32));
}

// The pieces of 16 bytes that a thread brings to LDS for one operand of a step, R rows (columns) wide.
//  TR false: rows that are contiguous in the contraction, 128 bytes of each: whole lines, as L2 is asked for half of
//    them one by one (64 bytes of each and twice the steps: 4096 rows by 4096 x 7168, loads alone 159 us, 138 with
//    lines).  Row r's piece c lies in place c ^ (r % 8) ^ (r / 8 % 2), so that the 16 rows which a wave reads at a time
//    lie in different banks.
//  TR true: ROWS rows of the contraction, R 16-bit columns of each.  32-byte chunk c of row j lies in place
//    c ^ (2 (j % 4) + j / 8 % 2), for the transposing reads of four rows at a time, by two groups of lanes.
// Places are 32 bits from a uniform base, which moves with the steps.
template <int R, int THREADS, int EL, bool TR, int ROWS = 64>
struct MmSrc {
    static constexpr int P = R * (TR ? ROWS : 64) / 8 / THREADS;
    static constexpr int kStepRows = THREADS * 8 / R;  // TR: rows between a thread's pieces
    static constexpr int kStep = TR ? ROWS : 128 / EL;  // elements of the contraction in a step
    static constexpr int kAlt = TR && kStepRows == 8 ? 2 : 1;  // TR: pieces that lie in different places of their rows
    static_assert(!TR || kStepRows % 8 == 0, "swizzle");
    const char* base;
    uint32_t off[TR ? kAlt : P];
    uint32_t gap;  // TR: bytes between a thread's pieces
    size_t move;   // bytes between steps
    int first;     // place in the step's contraction of the thread's pieces' first element (TR: of its first piece)

    // offset(r): bytes from base to row r
    template <class F>
    __device__ __forceinline__ void rows(const void* base_, F offset) {
        static_assert(!TR, "");
        const int t = threadIdx.x, c = (t & 7) ^ ((t >> 3) & 7) ^ ((t >> 6) & 1);
        base = mm_uniform(base_);
        move = 128;
        first = c * (16 / EL);
#pragma unroll
        for (int i = 0; i < P; ++i) off[i] = offset(i * (THREADS / 8) + (t >> 3)) + c * 16;
    }
    // columns col0 .. of a matrix `width` wide, rows `pitch` apart; those past it read others, and their results are not stored
    __device__ __forceinline__ void cols(const void* base_, int pitch, int col0, int width) {
        static_assert(TR, "");
        const int t = threadIdx.x, piece = t % (R / 8);
        first = t / (R / 8);
        base = mm_uniform(base_);
#pragma unroll
        for (int i = 0; i < kAlt; ++i) {
            const int row = first + i * kStepRows, col = col0 + (((piece >> 1) ^ (2 * (row & 3) + (row >> 3 & 1))) * 2 + (piece & 1)) * 8;
            off[i] = (uint32_t)first * (uint32_t)pitch * 2 + (col < width ? col * 2 : 0);
        }
        gap = (uint32_t)kStepRows * (uint32_t)pitch * 2;
        move = (size_t)pitch * 2 * ROWS;
    }
    __device__ __forceinline__ uint32_t place(int i) const { return TR ? off[i % kAlt] + (uint32_t)i * gap : off[TR ? 0 : i]; }
    // Piece i of the step that starts at `from`.
    __device__ __forceinline__ const char* piece(int i, const char* from) const { return from + place(i); }
    __device__ __forceinline__ const char* step(int k) const { return base + (size_t)k * move; }
    // Straight to LDS, piece i of a step that starts at `from`, to `lds` + the wave's part: whole pieces that start on 16
    // bytes.  It takes `from` from scalar registers and the lane's 32-bit place as it is: with a sum of 64 bits before
    // each load, loads took as much issue as MFMAs.
    __device__ __forceinline__ void fetch(unsigned char* lds, int i, const char* from) const {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(make_rsrc(from, 0xFFFFFFFFu), (__attribute__((address_space(3))) void*)(lds + i * THREADS * 16), 16,
                                                 (int)place(i), 0, 0, 0);
    }
    // The same for any step k: what lies past the contraction's n elements is zeros.
    __device__ __forceinline__ void fetch_to(unsigned char* lds, int i, int k, int n) const {
        const char* q = k * kStep + first + (TR ? i * kStepRows : 0) < n ? piece(i, step(k)) : reinterpret_cast<const char*>(mm_zeros);
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)q, (__attribute__((address_space(3))) void*)(lds + i * THREADS * 16), 16, 0, 0);
    }
};

__device__ __forceinline__ uint32_t mm_lds_addr(const unsigned char* p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) unsigned char*)p;
}

// Fragment reads are written as asm: of plain loads the compiler cannot tell which slot a pending direct load
// writes, and waits for all of them.  Every output is an operand of mm_wait, so it stays live and unread until the
// read has landed; that the compiler neither copies nor spills one before is checked on the built kernels
// (tests/test_matmul_fragments.py).
template <int OFF>
__device__ __forceinline__ void mm_read16(u32x4& v, uint32_t at) {
    static_assert(OFF >= 0 && OFF < 65536, "offset field");
    asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(v) : "v"(at), "i"(OFF));
}
template <int OFF>
__device__ __forceinline__ void mm_read_tr(uint64_t& v, uint32_t at) {
    static_assert(OFF >= 0 && OFF < 65536, "offset field");
    asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(v) : "v"(at), "i"(OFF));
}

// f(integral_constant 0), ..., f(integral_constant N - 1)
template <int N, int I = 0, class F>
__device__ __forceinline__ void mm_each(F f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        mm_each<N, I + 1>(f);
    }
}

// A wave's fragments of an operand, T tiles of 16 rows (columns) from row r0 of the tile on, of 64 bytes (32 rows) of the
// contraction: the halves S of a step.  TR: the four rows' halves of a fragment are reads of their own.
template <int R, bool TR, int T>
struct MmFrag {
    static constexpr int kReads = TR ? 2 : 1, kPlaces = TR ? T : 2;
    union Held {
        u32x4 v;
        uint64_t h[2];
    };
    uint32_t at[kPlaces];
    __device__ __forceinline__ MmFrag(int r0, uint32_t lds) {
        const int l = threadIdx.x & 63, g = l >> 4, i = l & 15;
        if constexpr (TR) {
#pragma unroll
            for (int t = 0; t < T; ++t)
                at[t] = lds + (8 * g + (i >> 2)) * R * 2 + (((r0 / 16 + t) ^ (2 * (i >> 2) + (g & 1))) * 32) + (i & 3) * 8;
        } else {
            const int key = (i & 7) ^ (i >> 3);
#pragma unroll
            for (int s = 0; s < 2; ++s) at[s] = lds + (r0 + i) * 128 + (((4 * s + g) ^ key) * 16);
        }
    }
    template <int S, int I>
    __device__ __forceinline__ void read(Held& f, uint32_t slot) const {
        if constexpr (TR) {
            mm_read_tr<32 * S * R * 2>(f.h[0], at[I] + slot);
            mm_read_tr<(32 * S + 4) * R * 2>(f.h[1], at[I] + slot);
        } else {
            mm_read16<I * 2048>(f.v, at[S] + slot);
        }
    }
};

// All LDS reads and writes of the wave have landed, those into the N fragments of `f` among them.
template <int N, class H>
__device__ __forceinline__ void mm_wait(H (&f)[N]) {
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(f[0].v));
#pragma unroll
    for (int i = 1; i < N; ++i) asm volatile("" : "+v"(f[i].v));
#endif
}

__device__ __forceinline__ void mm_barrier() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// acc[m][n] += A B over steps k0 .. k1 - 1 of 128 bytes (64 rows) of a contraction of n elements.
//
// Steps go through two rings of slots in LDS.  A step is four depths, both halves of the wave's m against all of its n for
// both halves of the contraction; the fragments of a depth are read while the depth before it multiplies.  Before a step's
// last depth the wave waits for the next step's loads and passes the barrier, behind which no wave reads this step any
// more; its last depth then multiplies while the next step's first fragments are read.  Loads into the slots that became
// free go out one by one between MFMAs: of B at once, of A, whose ring is a slot longer, during the next step.  The steady
// loop has no conditions; they cost more than the waits (4096 rows by 4096 x 7168: 220 us, 190 without).
//
// 171 to 176 us there with 256 x 256 results a CU (1.37 to 1.41 PFLOP/s; 8-bit 94, 2.57).  What bounds it is power: rows of
// zeros take a third less time at the same instructions, as the clock falls with what MFMAs switch.
template <class T, class S, bool AT, bool BT>
__device__ __forceinline__ void mm_core(const MmSrc<S::BM, S::kThreads, T::kEl, AT>& a, const MmSrc<S::BN, S::kThreads, T::kEl, BT>& b,
                                        int n, int k0, int k1, unsigned char* lds, typename T::Acc (&acc)[S::TM][S::TN]) {
    typedef MmFrag<S::BM, AT, S::TM> FA;
    typedef MmFrag<S::BN, BT, S::TN> FB;
    constexpr int kLoadsA = S::BM * 8 / S::kThreads, kLoadsB = S::BN * 8 / S::kThreads;
    constexpr int kHalf = S::TM / 2, kMma = kHalf * S::TN;
    const int wave = wave_id();
    const FA fa(wave % S::WM * S::TM * 16, mm_lds_addr(lds));
    const FB fb(wave / S::WM * S::TN * 16, mm_lds_addr(lds) + S::kEndM);
#pragma unroll
    for (int m = 0; m < S::TM; ++m)
#pragma unroll
        for (int t = 0; t < S::TN; ++t) acc[m][t] = typename T::Acc{};
    if (k0 >= k1) return;
    unsigned char *lds_b = lds + S::kEndM, *to_a = lds + wave * 1024, *to_b = lds_b + wave * 1024;
    typename FA::Held xa[2][kHalf];  // of the depth and the next
    typename FB::Held xb[2][S::TN];  // of the half of the contraction and the next
    const char *pa = a.step(k0 + S::kSlots), *pb = b.step(k0 + S::kSlots - 1);  // of the next loads
    // depth D of step k multiplies; the next one's fragments are read from slots `ra` and `rb` beside it, and a share of
    // the loads that slots became free for goes out: B's in depths 3 and 0, A's in 1 and 2, evenly.  STEADY: they are of
    // whole steps.
    auto depth = [&](auto d, auto steady, int k, uint32_t ra, uint32_t rb, int to) {
        constexpr int D = decltype(d)::value, N = (D + 1) & 3;
        constexpr bool B = D == 3 || D == 0;
        constexpr int kAll = B ? kLoadsB : kLoadsA, kFirst = D == 0 || D == 2 ? (kAll + 1) / 2 : 0, kShare = D == 0 || D == 2 ? kAll / 2 : (kAll + 1) / 2;
        constexpr int kReads = kHalf + (N & 1 ? 0 : S::TN);  // the next depth's half of m, and n where its half of the contraction is new
        const int step = D == 0 ? k + S::kSlots - 1 : k + S::kSlots;
        __builtin_amdgcn_s_setprio(1);
        mm_each<kMma>([&](auto i) {
            constexpr int m = i.value / S::TN, t = i.value % S::TN;
            mm_each<kReads>([&](auto r) {  // at the first half of the MFMAs, evenly
                if constexpr (r.value * (kMma / 2) / kReads == i.value) {
                    if constexpr (r.value < kHalf)
                        fa.template read<N / 2, N % 2 * kHalf + r.value>(xa[N % 2][r.value], ra);
                    else
                        fb.template read<N / 2, r.value - kHalf>(xb[N / 2][r.value - kHalf], rb);
                }
            });
            mm_each<kShare>([&](auto r) {
                constexpr int j = kFirst + r.value;
                if constexpr (r.value * kMma / kShare != i.value) return;
                if constexpr (decltype(steady)::value) {
                    if constexpr (B)
                        b.fetch(to_b + to, j, pb);
                    else
                        a.fetch(to_a + to, j, pa);
                } else if (step < k1) {
                    if constexpr (B)
                        b.fetch_to(to_b + to, j, step, n);
                    else
                        a.fetch_to(to_a + to, j, step, n);
                }
            });
            typename T::Acc& sum = acc[D % 2 * kHalf + m][t];
            sum = T::mma(xa[D % 2][m].v, xb[D / 2][t].v, sum);
            __builtin_amdgcn_sched_barrier(0);
        });
        __builtin_amdgcn_s_setprio(0);
        mm_wait(xa[N % 2]);
        if constexpr (N % 2 == 0) mm_wait(xb[N / 2]);
    };
    constexpr std::integral_constant<int, 0> d0{};
    constexpr std::integral_constant<int, 1> d1{};
    constexpr std::integral_constant<int, 2> d2{};
    constexpr std::integral_constant<int, 3> d3{};
    // step k + 1 has landed when only the loads of later steps are in flight
    auto arrived = [&](int k) {
        const int later = k1 - 2 - k;
        if (later >= S::kSlots - 1)
            vm_wait<(S::kSlots - 1) * kLoadsA + (S::kSlots - 2) * kLoadsB>();
        else if (S::kSlots > 3 && later == 2)
            vm_wait<2 * (kLoadsA + kLoadsB)>();
        else if (S::kSlots > 2 && later == 1)
            vm_wait<kLoadsA + kLoadsB>();
        else
            vm_wait<0>();
    };
    static_assert(S::kSlots >= 2 && S::kSlots <= 4, "arrived()");
#pragma unroll
    for (int i = 0; i < S::kSlots; ++i) {
        if (k0 + i >= k1) break;
#pragma unroll
        for (int j = 0; j < kLoadsA; ++j) a.fetch_to(to_a + i * S::kStepM, j, k0 + i, n);
#pragma unroll
        for (int j = 0; j < (i < S::kSlots - 1 ? kLoadsB : (kLoadsB + 1) / 2); ++j) b.fetch_to(to_b + i * S::kStepN, j, k0 + i, n);
    }
    if (k1 - k0 >= S::kSlots)
        vm_wait<(S::kSlots - 1) * kLoadsA + (S::kSlots - 2) * kLoadsB + (kLoadsB + 1) / 2>();
    else
        vm_wait<0>();
    mm_barrier();
    mm_each<kHalf>([&](auto r) { fa.template read<0, r.value>(xa[0][r.value], 0); });
    mm_each<S::TN>([&](auto r) { fb.template read<0, r.value>(xb[0][r.value], 0); });
    mm_wait(xa[0]);
    mm_wait(xb[0]);
    int sa = 0, sb = 0, was_a = S::kEndM - S::kStepM, was_b = (S::kSlots - 1) * S::kStepN;  // slots of the step, and of the one before it
    auto step = [&](auto steady, int k) {
        const int na = sa + S::kStepM == S::kEndM ? 0 : sa + S::kStepM, nb = sb + S::kStepN == S::kSlots * S::kStepN ? 0 : sb + S::kStepN;
        depth(d0, steady, k, sa, sb, was_b);
        pb += b.move;
        depth(d1, steady, k, sa, sb, was_a);
        depth(d2, steady, k, sa, sb, was_a);
        pa += a.move;
        if constexpr (decltype(steady)::value)
            vm_wait<(S::kSlots - 1) * kLoadsA + (S::kSlots - 2) * kLoadsB>();
        else
            arrived(k);
        mm_barrier();
        __builtin_amdgcn_sched_barrier(0);
        depth(d3, steady, k, na, nb, sb);  // past the last step it reads what lies in the rings, not used
#if defined(__HIP_DEVICE_COMPILE__)  // keeps the sums where they are: no copies of them at the loop's end
#pragma unroll
        for (int m = 0; m < S::TM; ++m)
#pragma unroll
            for (int t = 0; t < S::TN; ++t) asm volatile("" : "+v"(acc[m][t]));
#endif
        was_a = sa;
        was_b = sb;
        sa = na;
        sb = nb;
    };
    int k = k0;
    for (const int whole = min(k1, n / MmSrc<S::BM, S::kThreads, T::kEl, AT>::kStep); k + S::kSlots < whole; ++k) step(std::true_type{}, k);
    for (; k < k1; ++k) step(std::false_type{}, k);
    mm_barrier();
}

// The same for the gradient at the weights, whose operands both lie across the contraction: steps of 32 rows, which are whole lines
// all the same, so that three of them for 256 x 128 results leave room for a second workgroup on the CU.  A matrix's share of
// rows is short and its results are many: one workgroup stores while the other multiplies (32 matrices of 4096 x 7168, 512 rows
// each: with one of 256 x 256 results a CU 1226 us, of which 370 were stores that nothing ran beside; so 1120 to 1180, 1284 traced
// after a pause).  Matrix cores are 43 % busy: the 1.88 GB of results go through the L2 that holds the operands, which are
// fetched 4.7 times (1.72 GB for 0.37).
template <class S>
struct MmShort {
    static constexpr int kSlots = 3, kStepM = S::BM * 64, kStepN = S::BN * 64, kStep = kStepM + kStepN, kLds = kSlots * kStep;
    typedef MmSrc<S::BM, S::kThreads, 2, true, 32> A;
    typedef MmSrc<S::BN, S::kThreads, 2, true, 32> B;
};
template <class T, class S>
__device__ __forceinline__ void mm_core_short(const typename MmShort<S>::A& a, const typename MmShort<S>::B& b, int n, unsigned char* lds,
                                              typename T::Acc (&acc)[S::TM][S::TN]) {
    typedef MmShort<S> H;
    typedef MmFrag<S::BM, true, S::TM> FA;
    typedef MmFrag<S::BN, true, S::TN> FB;
    constexpr int kHalf = S::TM / 2, kMma = kHalf * S::TN, kLoads = H::A::P + H::B::P, kLate = kLoads / 2;
    const int wave = wave_id(), k1 = (n + 31) / 32;
    const FA fa(wave % S::WM * S::TM * 16, mm_lds_addr(lds));
    const FB fb(wave / S::WM * S::TN * 16, mm_lds_addr(lds) + H::kStepM);
#pragma unroll
    for (int m = 0; m < S::TM; ++m)
#pragma unroll
        for (int t = 0; t < S::TN; ++t) acc[m][t] = typename T::Acc{};
    if (k1 == 0) return;
    unsigned char* to = lds + wave * 1024;
    // load j of a step: A's first
    auto load = [&](auto steady, int j, int k, const char* pa, const char* pb, int slot) {
        if constexpr (decltype(steady)::value) {
            if (j < H::A::P)
                a.fetch(to + slot, j, pa);
            else
                b.fetch(to + slot + H::kStepM, j - H::A::P, pb);
        } else if (k < k1) {
            if (j < H::A::P)
                a.fetch_to(to + slot, j, k, n);
            else
                b.fetch_to(to + slot + H::kStepM, j - H::A::P, k, n);
        }
    };
#pragma unroll
    for (int i = 0; i < 3; ++i)
#pragma unroll
        for (int j = 0; j < (i < 2 ? kLoads : kLoads - kLate); ++j) load(std::false_type{}, j, i, nullptr, nullptr, i * H::kStep);
    if (k1 >= 3)
        vm_wait<2 * kLoads - kLate>();
    else
        vm_wait<0>();
    mm_barrier();
    typename FA::Held xa[2][kHalf];
    typename FB::Held xb[2][S::TN];
    mm_each<kHalf>([&](auto r) { fa.template read<0, r.value>(xa[0][r.value], 0); });
    mm_each<S::TN>([&](auto r) { fb.template read<0, r.value>(xb[0][r.value], 0); });
    mm_wait(xa[0]);
    mm_wait(xb[0]);
    int slot = 0, was = 2 * H::kStep;
    const char *pa = a.step(2), *pb = b.step(2);  // of the next loads
    // half D of m of step k, whose n is in xb[Q]; beside it the fragments of the next half (from slot `from`) and a share of the loads
    // of step k + 2 or k + 3
    auto half = [&](auto d, auto q, auto steady, int k, uint32_t from, int slot_to) {
        constexpr int D = decltype(d)::value, Q = decltype(q)::value, kReads = kHalf + (D == 1 ? S::TN : 0), kShare = D == 1 ? kLoads - kLate : kLate;
        __builtin_amdgcn_s_setprio(1);
        mm_each<kMma>([&](auto i) {
            constexpr int m = i.value / S::TN, t = i.value % S::TN;
            mm_each<kReads>([&](auto r) {
                if constexpr (r.value * (kMma / 2) / kReads == i.value) {
                    if constexpr (r.value < kHalf)
                        fa.template read<0, (1 - D) * kHalf + r.value>(xa[1 - D][r.value], from);
                    else
                        fb.template read<0, r.value - kHalf>(xb[1 - Q][r.value - kHalf], from);
                }
            });
            mm_each<kShare>([&](auto r) {
                if constexpr (r.value * kMma / kShare == i.value) load(steady, (D == 1 ? 0 : kLoads - kLate) + r.value, k + 2 + D, pa, pb, slot_to);
            });
            typename T::Acc& sum = acc[D * kHalf + m][t];
            sum = T::mma(xa[D][m].v, xb[Q][t].v, sum);
            __builtin_amdgcn_sched_barrier(0);
        });
        __builtin_amdgcn_s_setprio(0);
        mm_wait(xa[1 - D]);
        if constexpr (D == 1) mm_wait(xb[1 - Q]);
    };
    constexpr std::integral_constant<int, 0> d0{};
    constexpr std::integral_constant<int, 1> d1{};
    auto step = [&](auto q, auto steady, int k) {
        const int next = slot == 2 * H::kStep ? 0 : slot + H::kStep;
        half(d0, q, steady, k, slot, was);
        pa += a.move;
        pb += b.move;
        if (decltype(steady)::value || k + 2 < k1)
            vm_wait<kLoads>();
        else
            vm_wait<0>();
        mm_barrier();
        half(d1, q, steady, k, next, slot);  // past the last step it reads what lies in the ring, not used
#if defined(__HIP_DEVICE_COMPILE__)  // keeps the sums where they are: no copies of them at the loop's end
#pragma unroll
        for (int m = 0; m < S::TM; ++m)
#pragma unroll
            for (int t = 0; t < S::TN; ++t) asm volatile("" : "+v"(acc[m][t]));
#endif
        was = slot;
        slot = next;
    };
    int k = 0;
    for (const int whole = n / 32; k + 4 < whole; k += 2) {
        step(d0, std::true_type{}, k);
        step(d1, std::true_type{}, k + 1);
    }
    for (; k + 1 < k1; k += 2) {
        step(d0, std::false_type{}, k);
        step(d1, std::false_type{}, k + 1);
    }
    if (k < k1) step(d0, std::false_type{}, k);
}

// Two values rounded to 16 bits, by the hardware's conversions (nearest even, NaN stay NaN).
__device__ __forceinline__ uint32_t mm_round2(float a, float b, bool bf) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 v = {a, b};
    return bf ? __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2)) : __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}

// 16 rows of W * 16 outputs, from a wave's results through its own part of LDS (W KB), so that it stores whole lines.
// v(w, i): element i of result w, whose m follow each other; row(n) is where in `out` row n starts (elements), < 0: not stored.
template <int W, bool WIDE, class F>
__device__ __forceinline__ void mm_put_rows(const float* turn, void* out, bool bf, bool vec, int m0, int width, F row) {
    constexpr int kChunks = W * 4, kPer = WIDE ? 4 : 8, kLanes = W * 16 / kPer;  // columns of a lane's store, lanes of a row
    const int l = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < 16 * kLanes / 64; ++i) {
        const int r = (i * 64 + l) / kLanes, c = (i * 64 + l) % kLanes * kPer, left = width - m0 - c;
        const int64_t at = row(r);
        if (at < 0 || left <= 0) continue;
        const float* src = turn + r * W * 16;
        const f32x4 a = *reinterpret_cast<const f32x4*>(src + ((c / 4) ^ (r & (kChunks - 1))) * 4);
        u32x4 v;
        if constexpr (WIDE) {
            v = __builtin_bit_cast(u32x4, a);
        } else {
            const f32x4 b = *reinterpret_cast<const f32x4*>(src + ((c / 4 + 1) ^ (r & (kChunks - 1))) * 4);
            v = u32x4{mm_round2(a[0], a[1], bf), mm_round2(a[2], a[3], bf), mm_round2(b[0], b[1], bf), mm_round2(b[2], b[3], bf)};
        }
        char* y = static_cast<char*>(out) + (at + m0 + c) * (WIDE ? 4 : 2);
        if (vec) {
            *reinterpret_cast<u32x4*>(y) = v;
        } else if (left >= kPer) {
            ((__attribute__((address_space(1))) MmPacked*)y)->v = v;
        } else {
#pragma unroll
            for (int k = 0; k < kPer - 1; ++k) {
                if (k >= left) continue;
                if constexpr (WIDE)
                    reinterpret_cast<uint32_t*>(y)[k] = v[k];
                else
                    reinterpret_cast<uint16_t*>(y)[k] = (uint16_t)(v[k / 2] >> (16 * (k & 1)));
            }
        }
    }
}

template <int W, class V, class F>
__device__ __forceinline__ void mm_put(V v, float* turn, void* out, int type, bool vec, int m0, int width, F row) {
    constexpr int kChunks = W * 4;  // of four floats
    const int l = threadIdx.x & 63, n = l & 15;
#pragma unroll
    for (int w = 0; w < W; ++w)
        *reinterpret_cast<f32x4*>(turn + n * W * 16 + ((w * 4 + (l >> 4)) ^ (n & (kChunks - 1))) * 4) = f32x4{v(w, 0), v(w, 1), v(w, 2), v(w, 3)};
    __builtin_amdgcn_wave_barrier();
    if (type == CX_DTYPE_F32)
        mm_put_rows<W, true>(turn, out, false, vec, m0, width, row);
    else
        mm_put_rows<W, false>(turn, out, type == CX_DTYPE_BF16, vec, m0, width, row);
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
// A shape with the fewest tiles in n that hold `rows`: a short item multiplies less.
template <class S, int TN = 1, class F>
__device__ __forceinline__ void mm_fit(int rows, F f) {
    if constexpr (TN < S::TN) {
        if (rows > S::WN * TN * 16) return mm_fit<S, TN + 1>(rows, f);
    }
    f(MmShape<S::WM, S::WN, S::TM, TN, S::kSlots>{});
}

// This workgroup's tile, range of the contraction and run of rows; false: none, or one of rows behind the last matrix,
// which are cleared.
struct MmWork {
    MmItem it;
    int m0, ks;
};
__device__ __forceinline__ bool mm_work(const MmLaunch& L, int tile_cols, int width, int threads, bool halves, MmWork* w) {
    const MmTile tile = mm_tile(blockIdx.x, L.m_tiles * L.splits, L.by_item);
    if (L.offsets != nullptr && blockIdx.x == 0 && wave_id() == 0) mm_check(L.offsets, L.n_mats, L.n_rows, L.err_flag);
    if (tile.m >= L.m_tiles * L.splits) return false;
    w->it = mm_item(L.offsets, L.n_mats, L.n_rows, L.item_rows, tile.item);
    w->ks = tile.m / L.m_tiles;
    w->m0 = (tile.m - w->ks * L.m_tiles) * tile_cols;
    if (w->it.rows <= 0) return false;
    if (w->it.mat >= 0) return true;
    if (L.splits == 1) {  // otherwise with the sums
        mm_clear(L.y, L.y_type, w->it.begin, w->it.rows, width, w->m0, tile_cols, threads);
        if (halves && L.pre != nullptr)
            for (int h = 0; h < 2; ++h)
                for (int r = 0; r < w->it.rows; ++r) mm_clear(L.pre, L.type, 2 * (int64_t)(w->it.begin + r) + h, 1, width, w->m0, tile_cols, threads);
    }
    return false;
}

// The row of x of row p (in the order, if there is one), < 0: none.
__device__ __forceinline__ int mm_row_of_x(const MmLaunch& L, int p) {
    if (L.order == nullptr) return p;
    const int pair = L.order[p], xr = pair / L.top_k;
    return pair < 0 || xr >= L.n_x ? -1 : xr;
}

// Forward: a workgroup reads its weights and rows once each from L2.  32 matrices of 4096 x 7168, gated, 512 rows each on
// average: 967 to 1054 us when dealt unevenly (854 evenly, 1.13 PFLOP/s; one matrix of 4096 rows 1.4), matrix cores 70 % busy.
// Two things bound it: traffic, as each item of up to 256 rows reads its matrix again (4.8 GB fetched where 2.1 are
// unique, about 5 TB/s, a copy's rate), and tiles that an item's last rows do not fill.  m: weight rows; a gated tile has TM / 2 results of gate rows and the same rows of the up
// half per wave, so that both factors of an output meet in one lane.
template <class T, class S, bool GATED>
__device__ __forceinline__ void mm_forward(const MmLaunch& L, const MmWork& work, unsigned char* lds) {
    static_assert(S::kWaves * S::TM * 1024 <= S::kLds, "turned results");
    const MmItem it = work.it;
    const int width = GATED ? L.rows / 2 : L.rows, m0 = work.m0;
    MmSrc<S::BM, S::kThreads, T::kEl, false> a;
    MmSrc<S::BN, S::kThreads, T::kEl, false> b;
    const size_t pitch = (size_t)L.w_pitch * T::kEl, x_pitch = (size_t)L.x_pitch * T::kEl;
    // weight rows from the tile's first on; those past the matrix are its last one again, and not stored
    constexpr int half = S::TM / 2;  // gated: results of gate rows
    a.rows(static_cast<const char*>(L.w) + ((size_t)it.mat * L.rows + m0) * pitch, [&](int r) {
        const int n = GATED ? min(m0 + (r / (S::TM * 16) * half + r / 16 % half) * 16 + r % 16, width - 1) + (r / 16 % S::TM < half ? 0 : width)
                            : min(m0 + r, width - 1);
        return (uint32_t)(n - m0) * (uint32_t)pitch;
    });
    // a row that is not there reads row 0, and its results are zeros
    const int x0 = L.order == nullptr ? it.begin : 0;
    b.rows(static_cast<const char*>(L.x) + (size_t)x0 * x_pitch, [&](int r) {
        return (uint32_t)(max(mm_row_of_x(L, it.begin + min(r, it.rows - 1)), x0) - x0) * (uint32_t)x_pitch;
    });
    typename T::Acc acc[S::TM][S::TN];
    const int steps = (L.cols + 128 / T::kEl - 1) / (128 / T::kEl), per = (steps + L.splits - 1) / L.splits, k0 = work.ks * per;
    mm_core<T, S, false, false>(a, b, L.cols, k0, min(steps, k0 + per), lds, acc);
    // results to y
    const int wave = wave_id(), l = threadIdx.x & 63, wm = wave % S::WM, n0 = wave / S::WM * S::TN * 16;
    float* turn = reinterpret_cast<float*>(lds + wave * S::TM * 1024);
    const int mw = m0 + wm * (GATED ? half : S::TM) * 16;  // of the wave
    auto row = [&](int nt, int64_t w, int64_t off) {
        return [=](int r) { return nt + r < it.rows ? (int64_t)(it.begin + nt + r) * w + off : (int64_t)-1; };
    };
    if (L.splits > 1) {  // sums as they are, of this range of the contraction
        float* part = L.part + (size_t)work.ks * L.n_rows * L.rows;
        const bool vec = mm_vec(part, width, CX_DTYPE_F32);
#pragma unroll
        for (int t = 0; t < S::TN; ++t) {
            const int nt = n0 + t * 16;
            if (nt >= it.rows) break;
            auto bits = [&](int m, int i) {
                const auto e = acc[m][t][i];  // of an element itself __builtin_bit_cast takes its vector's first
                return __builtin_bit_cast(float, e);
            };
            if constexpr (GATED) {
                mm_put<half>(bits, turn, part, CX_DTYPE_F32, vec, mw, width, row(nt, L.rows, 0));
                mm_put<half>([&](int w, int i) { return bits(half + w, i); }, turn, part, CX_DTYPE_F32, vec, mw, width, row(nt, L.rows, width));
            } else {
                mm_put<S::TM>(bits, turn, part, CX_DTYPE_F32, vec, mw, width, row(nt, L.rows, 0));
            }
        }
        return;
    }
    f32x4 ws[T::kEl == 1 ? S::TM : 1];
    if constexpr (T::kEl == 1) {
#pragma unroll
        for (int m = 0; m < S::TM; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = 4 * (l >> 4) + i;
                ws[m][i] = L.w_scale[(size_t)it.mat * L.rows + (GATED ? min(mw + m % half * 16 + c, width - 1) + (m < half ? 0 : width) : min(mw + m * 16 + c, width - 1))];
            }
    }
    const bool vec = mm_vec(L.y, width, L.y_type), pvec = GATED && L.pre != nullptr && mm_vec(L.pre, width, T::kType);
#pragma unroll
    for (int t = 0; t < S::TN; ++t) {
        const int nt = n0 + t * 16;
        if (nt >= it.rows) break;
        const int xr = mm_row_of_x(L, it.begin + min(nt + (l & 15), it.rows - 1));
        const float xs = T::kEl == 1 ? (xr < 0 ? 0.0f : L.x_scale[xr]) : 1.0f;
        auto value = [&](int m, int i) {
            float f = (float)acc[m][t][i];
            if constexpr (T::kEl == 1) f = f * xs * ws[m][i];
            return xr < 0 ? 0.0f : f;
        };
        if constexpr (GATED) {
            if (L.pre != nullptr) {
                mm_put<half>([&](int w, int i) { return value(w, i); }, turn, L.pre, T::kType, pvec, mw, width, row(nt, 2 * (int64_t)width, 0));
                mm_put<half>([&](int w, int i) { return value(half + w, i); }, turn, L.pre, T::kType, pvec, mw, width, row(nt, 2 * (int64_t)width, width));
            }
            mm_put<half>([&](int w, int i) { return mm_silu(value(w, i)) * value(half + w, i); }, turn, L.y, L.y_type, vec, mw, width, row(nt, width, 0));
        } else {
            mm_put<S::TM>(value, turn, L.y, L.y_type, vec, mw, width, row(nt, width, 0));
        }
    }
}

template <class T, class S, bool GATED>
__global__ __launch_bounds__(S::kThreads, 2) void k_mm(MmLaunch L) {
    __shared__ __attribute__((aligned(16))) unsigned char lds[S::kLds];
    MmWork work;
    if (!mm_work(L, GATED ? S::BM / 2 : S::BM, GATED ? L.rows / 2 : L.rows, S::kThreads, GATED, &work)) return;
    mm_fit<S>(work.it.rows, [&](auto s) { mm_forward<T, decltype(s), GATED>(L, work, lds); });
}

// The gradient at x.  m: columns of the weights, read across their rows by transposing reads, so that no transposed copy of
// them is made; n: rows of dy.  16384 rows by 32 x 4096 x 7168: 950 to 975 us, matrix cores 67 % busy
// and 4.9 GB fetched (5 TB/s): every item reads its matrix again, as in the forward product.
template <class T, class S>
__device__ __forceinline__ void mm_dx(const MmLaunch& L, const MmWork& work, unsigned char* lds) {
    const MmItem it = work.it;
    const int width = L.cols, m0 = work.m0;
    MmSrc<S::BM, S::kThreads, 2, true> a;
    MmSrc<S::BN, S::kThreads, 2, false> b;
    a.cols(static_cast<const char*>(L.w) + (size_t)it.mat * L.rows * L.w_pitch * 2, L.w_pitch, m0, width);
    b.rows(static_cast<const char*>(L.dy) + (size_t)it.begin * L.dy_pitch * 2, [&](int r) { return (uint32_t)min(r, it.rows - 1) * (uint32_t)L.dy_pitch * 2; });
    f32x4 acc[S::TM][S::TN];
    const int steps = (L.rows + 63) / 64, per = (steps + L.splits - 1) / L.splits, k0 = work.ks * per;
    mm_core<T, S, true, false>(a, b, L.rows, k0, min(steps, k0 + per), lds, acc);
    const int wave = wave_id(), n0 = wave / S::WM * S::TN * 16;
    float* turn = reinterpret_cast<float*>(lds + wave * S::TM * 1024);
    void* out = L.splits > 1 ? L.part + (size_t)work.ks * L.n_rows * width : L.y;
    const int type = L.splits > 1 ? CX_DTYPE_F32 : L.y_type;
    const bool vec = mm_vec(out, width, type);
#pragma unroll
    for (int t = 0; t < S::TN; ++t) {
        const int nt = n0 + t * 16;
        if (nt >= it.rows) break;
        mm_put<S::TM>([&](int m, int i) { return acc[m][t][i]; }, turn, out, type, vec, m0 + wave % S::WM * S::TM * 16, width,
                      [&](int r) { return nt + r < it.rows ? (int64_t)(it.begin + nt + r) * width : (int64_t)-1; });
    }
}

template <class T, class S>
__global__ __launch_bounds__(S::kThreads, 2) void k_mm_dx(MmLaunch L) {
    __shared__ __attribute__((aligned(16))) unsigned char lds[S::kLds];
    MmWork work;
    if (!mm_work(L, S::BM, L.cols, S::kThreads, false, &work)) return;
    mm_fit<S>(work.it.rows, [&](auto s) { mm_dx<T, decltype(s)>(L, work, lds); });
}

// The gradient at the weights of each matrix, the contraction over its rows of x: both operands lie across it.  A matrix
// without rows gets zeros.  m: the weights' columns; n: their rows.  One of 4096 x 7168 with 4096 rows: 187 us (1.29 PFLOP/s).
template <class T, class S>
__global__ __launch_bounds__(S::kThreads, 2) void k_mm_dw(MmLaunch L) {
    __shared__ __attribute__((aligned(16))) unsigned char lds[S::kLds];
    if (L.offsets != nullptr && blockIdx.x == 0 && wave_id() == 0) mm_check(L.offsets, L.n_mats, L.n_rows, L.err_flag);
    const int n_tiles = (L.rows + S::BN - 1) / S::BN, per = n_tiles * L.m_tiles, mat = blockIdx.x / per, i = blockIdx.x - mat * per;
    const int n0 = i / L.m_tiles * S::BN, m0 = (i - i / L.m_tiles * L.m_tiles) * S::BM;
    const MmItem it = mm_rows_of(L.offsets, L.n_rows, mat);
    MmSrc<S::BM, S::kThreads, 2, true> a;
    MmSrc<S::BN, S::kThreads, 2, true> b;
    a.cols(static_cast<const char*>(L.x) + (size_t)it.begin * L.x_pitch * 2, L.x_pitch, m0, L.cols);
    b.cols(static_cast<const char*>(L.dy) + (size_t)it.begin * L.dy_pitch * 2, L.dy_pitch, n0, L.rows);
    f32x4 acc[S::TM][S::TN];
    mm_core<T, S, true, true>(a, b, it.rows, 0, (it.rows + 63) / 64, lds, acc);
    const int wave = wave_id(), nw = n0 + wave / S::WM * S::TN * 16;
    float* turn = reinterpret_cast<float*>(lds + wave * S::TM * 1024);
    const bool vec = mm_vec(L.y, L.cols, L.y_type);
#pragma unroll
    for (int t = 0; t < S::TN; ++t)
        mm_put<S::TM>([&](int m, int i) { return acc[m][t][i]; }, turn, L.y, L.y_type, vec, m0 + wave % S::WM * S::TM * 16, L.cols, [&](int r) {
            const int n = nw + t * 16 + r;
            return n < L.rows ? ((int64_t)mat * L.rows + n) * L.cols : (int64_t)-1;
        });
}

// The same with short steps, two workgroups a CU.
template <class T, class S>
__global__ __launch_bounds__(S::kThreads, 2) void k_mm_dw_short(MmLaunch L) {
    __shared__ __attribute__((aligned(16))) unsigned char lds[MmShort<S>::kLds];
    static_assert(S::kWaves * S::TM * 1024 <= MmShort<S>::kLds, "turned results");
    if (L.offsets != nullptr && blockIdx.x == 0 && wave_id() == 0) mm_check(L.offsets, L.n_mats, L.n_rows, L.err_flag);
    // tiles of a matrix in blocks of eight in n, down m; XCD b % 8 takes 64 in turn, which share operands in its L2
    const int n_tiles = (L.rows + S::BN - 1) / S::BN, per = n_tiles * L.m_tiles;
    const int64_t total = (int64_t)L.n_mats * per, x = blockIdx.x & 7, i = blockIdx.x >> 3, tile = (i / 64 * 8 + x) * 64 + i % 64;
    if (tile >= total) return;
    const int mat = (int)(tile / per), j = (int)(tile - (int64_t)mat * per), block = j / (8 * L.m_tiles), r = j - block * 8 * L.m_tiles, wide = min(8, n_tiles - block * 8);
    const int m0 = r / wide * S::BM, n0 = (block * 8 + r % wide) * S::BN;
    const MmItem it = mm_rows_of(L.offsets, L.n_rows, mat);
    typename MmShort<S>::A a;
    typename MmShort<S>::B b;
    a.cols(static_cast<const char*>(L.x) + (size_t)it.begin * L.x_pitch * 2, L.x_pitch, m0, L.cols);
    b.cols(static_cast<const char*>(L.dy) + (size_t)it.begin * L.dy_pitch * 2, L.dy_pitch, n0, L.rows);
    f32x4 acc[S::TM][S::TN];
    mm_core_short<T, S>(a, b, it.rows, lds, acc);
    const int wave = wave_id(), nw = n0 + wave / S::WM * S::TN * 16;
    mm_barrier();
    float* turn = reinterpret_cast<float*>(lds + wave * S::TM * 1024);
    const bool vec = mm_vec(L.y, L.cols, L.y_type);
#pragma unroll
    for (int t = 0; t < S::TN; ++t)
        mm_put<S::TM>([&](int m, int i) { return acc[m][t][i]; }, turn, L.y, L.y_type, vec, m0 + wave % S::WM * S::TM * 16, L.cols, [&](int r) {
            const int n = nw + t * 16 + r;
            return n < L.rows ? ((int64_t)mat * L.rows + n) * L.cols : (int64_t)-1;
        });
}

// Tiles of m and of n in waves, by the launch's form: 256 or 128 in m; n as in MmForm.
using MmBig = MmShape<2, 4, 8, 4, 2>;
using MmSmall = MmShape<2, 2, 4, 4, 2>;
using MmMid = MmShape<2, 2, 8, 4, 2>;  // of the gradient at the weights

}  // namespace cx
