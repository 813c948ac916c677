"""Products with 4-bit weights through the GEMM, against their formulas in 64 bits on
the CPU.  Tolerances count roundings, as in test_gpu_q4.py: a sum of n exact products
is off by at most n 2^-24 of the sum of their sizes, and the output's rounding adds
half a step.
"""
from __future__ import annotations

import pytest
import torch

from test_gpu_q4 import BF, F8, HF, SF, TINY, U, dense, make, make_x, near, product_ref, rand, rounded

pytestmark = pytest.mark.gpu

# fp16's largest value is 65504 and its next would be 65536: what lies at or past their middle rounds to an infinity
HF_OVER = 65520.0


def near_out(got, want, e, what):
    """near() for an output rounded to its type, fp16's infinities included."""
    got = got.cpu()
    if got.dtype == HF:
        over, may = want.abs() - e >= HF_OVER, want.abs() + e >= HF_OVER
        inf = torch.isinf(got) & (torch.signbit(got) == torch.signbit(want))
        assert bool(inf[over].all()), what
        got = torch.where(may & inf, want, got.double())
        near(got, want, rounded(want, e, HF), what)
    else:
        near(got, want, rounded(want, e, got.dtype), what)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T,N,K,group", [(18, 40, 1025, 64), (150, 24, 1030, 128)])
def test_top_k_without_an_order(gpu, T, N, K, group, dtype):
    """Without an order row p of y is row p of x, whatever top_k is: a row's power of two belongs to that row."""
    from constellation_amd.engine import Q4Matrix
    codes, scales = make(T, 1, N, K, group)
    w = Q4Matrix.pack(codes.cuda(), scales.cuda(), K, group=group)
    try:
        # rows whose sizes differ by powers of two, so that another row's factor shows
        x = rand(1, T, K, dtype=dtype) * (2.0 ** (torch.arange(T) % 5).to(dtype))[:, None]
        want, e = product_ref(x.double(), dense(codes, scales, K, group)[0], False)
        for top_k in (1, 0, -3, 7, 1 << 30):
            print(f"[q4 gemm] no order, top_k {top_k} {dtype}", flush=True)
            y = gpu.q4_matmul(w, x.cuda(), top_k=top_k)
            torch.cuda.synchronize()
            near(y, want, rounded(want, e, dtype), top_k)
    finally:
        w.free()


# Rows, outputs and columns of one matrix whose products take the GEMM (test_q4_kernel_choice.py): widths that
# 8 does not divide go there with few rows, others with 2^30 multiply-adds.  More than 8192 columns are more
# than the conversion of a row holds in registers.
ONE = [(9, 66, 1025), (17, 130, 1030), (49, 256, 1411), (70, 258, 1100), (129, 320, 1027), (600, 1040, 2048), (530, 1282, 2048),
       (2000, 1024, 1030), (2100, 1026, 1154), (21, 48, 9001), (130, 1024, 9216)]


@pytest.mark.parametrize("dtype", [BF, HF, F8])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("T,N,K", ONE)
def test_one_matrix(gpu, T, N, K, gated, dtype):
    """Each group size and type of output, with and without ranges of the columns."""
    from constellation_amd.engine import Q4Matrix
    for group in (32, 64, 128) if T < 500 else (64 if gated else 32,):
        codes, scales = make(T + N, 1, N, K, group)
        w = Q4Matrix.pack(codes.cuda(), scales.cuda(), K, group=group, gated=gated)
        try:
            x, xs, x64 = make_x(K, T, K, dtype)
            want, e = product_ref(x64, dense(codes, scales, K, group)[0], gated)
            if dtype == F8:
                e = e * 2  # the row's scale is a factor of its own
            for out in (BF, HF, SF) if group != 64 or T >= 500 else (None,):
                print(f"[q4 gemm] {T}x{K} by {N} group {group} gated {gated} {dtype} to {out}", flush=True)
                y = gpu.q4_matmul(w, x.cuda(), x_scale=None if xs is None else xs.cuda(), out_dtype=out)
                torch.cuda.synchronize()
                near_out(y, want, e, (group, out))
        finally:
            w.free()


STACKS = [(70, 3, 50, 1030), (300, 5, 96, 1025), (700, 40, 34, 1100), (2100, 3, 1024, 1030), (2090, 2, 1030, 1027)]


@pytest.mark.parametrize("dtype,group", [(BF, 128), (HF, 64), (F8, 32), (F8, 64), (F8, 128)])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("P,E,N,K", STACKS)
def test_stack(gpu, P, E, N, K, gated, dtype, group):
    """Rows dealt by offsets, as they lie and through an order with entries that are negative or past x;
    rows behind the last matrix are zeros, in memory that held something else."""
    from constellation_amd.engine import Q4Matrix
    codes, scales = make(P + E, E, N, K, group)
    w = Q4Matrix.pack(codes.cuda(), scales.cuda(), K, group=group, gated=gated)
    W = dense(codes, scales, K, group)
    g = torch.Generator().manual_seed(P)
    held = P - max(3, P // 9)
    off = torch.cat((torch.tensor([0]), torch.sort(torch.randint(0, held + 1, (E - 1,), generator=g)).values, torch.tensor([held])))
    top_k = 3
    n_x = -(-P // top_k)
    order = torch.randperm(P, generator=g)
    order[held:] = ~order[held:]
    lost = torch.randperm(held, generator=g)[:max(2, held // 20)]
    order[lost[::2]] = ~order[lost[::2]]
    order[lost[1::2]] = n_x * top_k + order[lost[1::2]]
    try:
        x, xs, x64 = make_x(3, P, K, dtype)
        for ordered, out in ((False, BF), (True, HF), (True, SF)):
            print(f"[q4 gemm] stack {P} over {E} {N}x{K} group {group} {dtype} gated {gated} ordered {ordered}", flush=True)
            n = n_x if ordered else P
            src = torch.where(order < 0, n, order // top_k) if ordered else torch.arange(P)
            rows = torch.cat((x64[:n], torch.zeros(1, K, dtype=torch.float64)))[src.clamp(max=n)]
            want, tol = torch.zeros(P, w.out_cols, dtype=torch.float64), torch.zeros(P, w.out_cols, dtype=torch.float64)
            for e in range(E):
                a, b = int(off[e]), int(off[e + 1])
                if a < b:
                    want[a:b], tol[a:b] = product_ref(rows[a:b], W[e], gated)
            torch.full((P * w.out_cols * 2,), float("nan"), device="cuda")  # goes back to the allocator
            y = gpu.q4_matmul(w, x[:n].cuda(), x_scale=None if xs is None else xs[:n].cuda(), offsets=off.to(torch.int32).cuda(),
                              order=order.to(torch.int32).cuda() if ordered else None, top_k=top_k, out_dtype=out)
            torch.cuda.synchronize()
            near_out(y, want, 2 * tol, (ordered, out))
            if ordered:
                assert not y[lost.cuda()].any()
            assert not y[held:].any()
        gpu.sync()
    finally:
        w.free()


@pytest.mark.parametrize("dtype", [BF, HF, F8])
@pytest.mark.parametrize("K", [1025, 1030])
def test_nan_and_infinite_rows_stay_in_their_rows(gpu, K, dtype):
    from constellation_amd.engine import Q4Matrix
    print(f"[q4 gemm] nan and infinite rows {K} {dtype}", flush=True)
    T, N = 90, 40
    codes, scales = make(T, 1, N, K, 32)
    codes |= 0x11  # no zeros: a NaN or an infinity reaches every output of its row
    w = Q4Matrix.pack(codes.cuda(), scales.cuda(), K, group=32)
    try:
        x, xs, _ = make_x(1, T, K, dtype)
        xs = None if xs is None else xs.cuda()
        clean = gpu.q4_matmul(w, x.cuda(), x_scale=xs, out_dtype=SF)
        x[3, K - 1] = float("nan")
        x[40, 7] = float("inf") if dtype != F8 else float("nan")
        x[89, 0] = float("-inf") if dtype != F8 else float("nan")
        y = gpu.q4_matmul(w, x.cuda(), x_scale=xs, out_dtype=SF)
        torch.cuda.synchronize()
        bad = torch.zeros(T, dtype=torch.bool)
        bad[[3, 40, 89]] = True
        assert torch.equal(y[~bad.cuda()], clean[~bad.cuda()])
        assert not bool(torch.isfinite(y[bad.cuda()]).any())
    finally:
        w.free()


# tokens, routes, experts, hidden, inter, shared: layers of the GEMM, over 8192 columns with any number of tokens
GEMM_LAYERS = [(40, 2, 3, 1040, 330, 1), (1, 2, 2, 40, 8200, 0), (3, 2, 3, 8328, 24, 1), (90, 3, 4, 1000, 2056, 0), (1, 40, 45, 8200, 16, 1)]
# ... and of the decode kernel; `alone`: one token's two launches without a plan, up to 16 routes of up to 2048 columns
DEC_LAYERS = [(1, 15, 20, 256, 136, 1, True), (1, 16, 40, 1000, 64, 0, True), (1, 17, 40, 256, 130, 0, False), (1, 16, 20, 256, 64, 1, False),
              (1, 2, 4, 96, 2049, 0, False), (2, 2, 5, 72, 8192, 0, False), (1, 9, 12, 512, 2048, 0, True), (4, 6, 30, 8190, 24, 1, False)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T,K,E,H,I,shared", GEMM_LAYERS + [c[:6] for c in DEC_LAYERS])
def test_layers(gpu, T, K, E, H, I, shared, dtype):
    """Layers at the limits of their kernels: many routes, wide rows, wide experts."""
    from constellation_amd.engine import Q4Layer, Q4Matrix
    from test_gpu_q4 import layer_ref
    print(f"[q4 gemm] layer {T}x{K} of {E} {H}x{I} shared {shared} {dtype}", flush=True)
    group = 32 if I % 64 else 128
    gu, dn, sg, sd = (make(i + T, n, *s, group) for i, (n, s) in
                      enumerate(((E, (2 * I, H)), (E, (H, I)), (1, (2 * I, H)), (1, (H, I)))))
    mats = [Q4Matrix.pack(c.cuda(), s.cuda(), k, group=group, gated=gt)
            for (c, s), k, gt in ((gu, H, True), (dn, I, False), (sg, H, True), (sd, I, False))]
    try:
        layer = Q4Layer(gpu, mats[0], mats[1], (mats[2], mats[3]) if shared else None)
        x = rand(5, T, H, dtype=dtype)
        g = torch.Generator().manual_seed(6)
        ids = torch.rand(T, E, generator=g).topk(K, dim=1).indices.to(torch.int32)
        ids[torch.rand(T, K, generator=g) < 0.1] = -1
        w = torch.rand(T, K, generator=g)
        y, yf = gpu.moe(layer, x.cuda(), ids.cuda(), w.cuda(), want_f32=True)
        torch.cuda.synchronize()
        gpu.sync()
        D = [dense(c, s, k, group) for (c, s), k in ((gu, H), (dn, I), (sg, H), (sd, I))]
        want, tol = layer_ref(x.double(), ids, w, D[0], D[1], 2.0 ** -22, (D[2], D[3]) if shared else None)
        near(yf, want, tol, "fp32")
        near(y, want, rounded(want, tol, dtype), "rounded")
    finally:
        for m in mats:
            m.free()


@pytest.mark.parametrize("dtype", [BF, HF])
def test_rows_up_to_the_last_place_in_32_bits(gpu, dtype):
    """299,000 rows of 7168, whose places in x end just below 4 GB."""
    from constellation_amd.engine import Q4Matrix
    T, N, K = 299_000, 24, 7168
    print(f"[q4 gemm] {T}x{K} by {N} {dtype}", flush=True)
    codes, scales = make(1, 1, N, K, 128)
    w = Q4Matrix.pack(codes.cuda(), scales.cuda(), K)
    try:
        x = torch.empty(T, K, dtype=dtype, device="cuda")
        x[:] = torch.randn(1000, K, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(dtype).repeat(T // 1000, 1)
        some = torch.cat((torch.arange(2), torch.arange(T // 2 - 3, T // 2 + 3), torch.arange(T - 20, T)))
        x[some.cuda()] = rand(2, some.numel(), K, dtype=dtype).cuda()  # rows that are found nowhere else
        y = gpu.q4_matmul(w, x)
        torch.cuda.synchronize()
        want, e = product_ref(x[some.cuda()].cpu().double(), dense(codes, scales, K, 128)[0], False)
        near(y.cpu()[some], want, rounded(want, e, dtype), dtype)
    finally:
        torch.cuda.synchronize()
        w.free()


@pytest.mark.parametrize("dtype,group", [(BF, 32), (HF, 64), (F8, 128)])
@pytest.mark.parametrize("P,n_x,N,K", [(3, 40, 48, 256), (4, 2, 64, 1030), (16, 5, 48, 512), (70, 9, 50, 264), (33, 200, 40, 1025), (300, 31, 48, 1100)])
def test_order_of_one_matrix(gpu, P, n_x, N, K, dtype, group):
    """Rows of one matrix's product by an order alone: some twice, some never, some that are not there."""
    from constellation_amd.engine import Q4Matrix
    print(f"[q4 gemm] order of one {P} from {n_x} {N}x{K} {dtype}", flush=True)
    codes, scales = make(P, 1, N, K, group)
    w = Q4Matrix.pack(codes.cuda(), scales.cuda(), K, group=group)
    try:
        x, xs, x64 = make_x(3, n_x, K, dtype)
        g = torch.Generator().manual_seed(P)
        for top_k in (1, 5):
            order = torch.randint(0, n_x * top_k, (P,), generator=g)
            order[0], order[-1] = -1 - order[0], n_x * top_k
            src = torch.where(order < 0, n_x, order // top_k).clamp(max=n_x)
            rows = torch.cat((x64, torch.zeros(1, K, dtype=torch.float64)))[src]
            want, e = product_ref(rows, dense(codes, scales, K, group)[0], False)
            y = gpu.q4_matmul(w, x.cuda(), x_scale=None if xs is None else xs.cuda(), order=order.to(torch.int32).cuda(), top_k=top_k, out_dtype=SF)
            torch.cuda.synchronize()
            near(y, want, 2 * e + TINY[SF], top_k)
            assert not y[0].any() and not y[-1].any()
    finally:
        w.free()


def test_scratch_of_the_largest_call_serves_smaller_ones(gpu):
    """One allocation of what the largest call asks for, at its exact size, under calls of every kernel."""
    import ctypes as C
    from constellation_amd._lib import BF16, F32, check, lib
    from constellation_amd.engine import Q4Matrix
    print("[q4 gemm] one scratch", flush=True)
    N, K, most = 7168, 2048, 4096
    codes, scales = make(1, 1, N, K, 128)
    w = Q4Matrix.pack(codes.cuda(), scales.cuda(), K)
    try:
        size = lib().cx_q4_scratch(C.byref(w.desc), BF16, most, most, 0)
        scratch = torch.empty(size, dtype=torch.uint8, device="cuda")
        x = rand(1, most, K, dtype=BF).cuda()
        for T in (most, 497, 448, 130, 64, 1):
            want = gpu.q4_matmul(w, x[:T], out_dtype=SF)
            y = torch.empty(T, N, device="cuda")
            check(lib().cx_q4_matmul(gpu.handle, C.byref(w.desc), x.data_ptr(), BF16, None, T, None, 1, None, T, y.data_ptr(), F32,
                                     scratch.data_ptr(), size, gpu.stream()))
            torch.cuda.synchronize()
            assert torch.equal(y, want), T
    finally:
        torch.cuda.synchronize()
        w.free()
