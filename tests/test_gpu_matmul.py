"""Products of a program's own experts in 16 bits and in 8-bit integers, and the gradients
of the 16-bit ones, against their formulas in 64 bits on the CPU.

Tolerances count roundings.  A product of two 16-bit values is exact in fp32 and a sum of n of
them off by at most n 2^-24 of the sum of their sizes; the output's rounding adds half a
step.  A sum of products of 8-bit integers is exact; its conversion to fp32 and the two
scales round three times.
"""
from __future__ import annotations

import pytest
import torch

from test_gpu_q4 import BF, HALF, HF, SF, U, near, product_ref, rand, rounded, split

pytestmark = pytest.mark.gpu

I8 = torch.int8


def own(t, odd=False):
    """t on the GPU; odd: at an address that is no multiple of 16 bytes."""
    if not odd:
        return t.cuda()
    room = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
    room[1:] = t.reshape(-1).cuda()
    return room[1:].view(t.shape)


# rows, weight rows, columns: a token; widths that pieces of 16 bytes do and do not divide; tiles that end inside
# their rows, their outputs and their last step; more than one step, odd and even counts of them
ONE = [(1, 32, 64), (1, 1, 1), (1, 512, 7168), (2, 18, 130), (5, 100, 129), (16, 64, 1000), (17, 130, 384), (33, 34, 8), (40, 66, 72), (64, 256, 640),
       (65, 250, 512), (129, 1024, 256), (300, 160, 2048), (513, 96, 72), (1000, 333, 411), (257, 514, 328), (200, 2050, 96)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("T,N,K", ONE)
def test_one_matrix(gpu, T, N, K, gated, dtype):
    if gated:
        N += N % 2
    x, w = rand(T, T, K, dtype=dtype), rand(N, N, K, dtype=dtype, std=0.1)
    y64, e = product_ref(x.double(), w.double(), False)
    want, tol = product_ref(x.double(), w.double(), gated)
    for odd in (False, True):
        for out in (dtype, SF) if not odd else (dtype,):
            print(f"[mm] {T}x{K} by {N} gated {gated} {dtype} to {out} odd {odd}", flush=True)
            y = gpu.matmul(own(x, odd), own(w, odd), gated=gated, keep=gated, out_dtype=out)
            torch.cuda.synchronize()
            if gated:
                y, pre = y
                assert pre.dtype == dtype
                near(pre, y64, rounded(y64, e, dtype), "pre")
            assert y.dtype == out
            near(y, want, rounded(want, tol, out), (odd, out))


def poisoned(x, rows):
    """x with NaN from row `rows` on: rows that belong to no matrix."""
    x = x.clone()
    x[rows:] = float("nan")
    return x


# pairs, matrices, weight rows, columns: one row a matrix, many rows a matrix, more matrices than rows,
# as many as there can be, tiles over several items
STACK = [(1, 1, 32, 64), (7, 5, 50, 200), (40, 64, 48, 256), (64, 200, 130, 136), (300, 6, 144, 520), (1200, 4, 256, 384), (5, 1024, 16, 33),
         (2000, 130, 96, 72), (900, 3, 514, 328), (3000, 9, 260, 100)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("P,E,N,K", STACK)
def test_stack(gpu, P, E, N, K, gated, dtype):
    """Rows dealt by offsets, as they lie and through an order with entries that are negative or past x;
    rows behind the last matrix hold NaN and come out as zeros."""
    off = split(P, E, P)
    held = int(off[-1])
    w = rand(N, E, N, K, dtype=dtype, std=0.1)
    g = torch.Generator().manual_seed(P)
    top_k = 3
    n_x = -(-P // top_k)
    order = torch.randperm(P, generator=g)
    order[held:] = ~order[held:]
    lost = torch.randperm(max(held, 1), generator=g)[:held // 20]
    order[lost[::2]] = ~order[lost[::2]]
    order[lost[1::2]] = n_x * top_k + order[lost[1::2]]
    for ordered, out in ((False, dtype), (True, SF)):
        print(f"[mm] stack {P} over {E} {N}x{K} gated {gated} {dtype} ordered {ordered}", flush=True)
        n = n_x if ordered else P
        x = rand(3, n, K, dtype=dtype)
        if not ordered:
            x = poisoned(x, held)
        src = torch.where(order < 0, n, order // top_k).clamp(max=n) if ordered else torch.arange(P)
        rows = torch.cat((x.double(), torch.zeros(1, K, dtype=torch.float64)))[src]
        cols = N // 2 if gated else N
        want, tol = torch.zeros(P, cols, dtype=torch.float64), torch.zeros(P, cols, dtype=torch.float64)
        sums, stol = torch.zeros(P, N, dtype=torch.float64), torch.zeros(P, N, dtype=torch.float64)
        for e in range(E):
            a, b = int(off[e]), int(off[e + 1])
            if a < b:
                want[a:b], tol[a:b] = product_ref(rows[a:b], w[e].double(), gated)
                sums[a:b], stol[a:b] = product_ref(rows[a:b], w[e].double(), False)
        torch.full((P * N * 2,), float("nan"), device="cuda")  # goes back to the allocator
        y = gpu.matmul(x.cuda(), w.cuda(), gated=gated, keep=gated, offsets=off.cuda(), order=order.to(torch.int32).cuda() if ordered else None,
                       top_k=top_k, out_dtype=out)
        torch.cuda.synchronize()
        if gated:
            y, pre = y
            near(pre, sums, rounded(sums, stol, dtype), "pre")
            assert not pre[held:].any()
        near(y, want, rounded(want, tol, out), ordered)
        assert not y[held:].any()
        if ordered:
            assert not y[lost.cuda()].any()
    gpu.sync()


def int8s(seed, *shape):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-128, 128, shape, generator=g).to(I8)


def i8_ref(x, xs, w, ws, gated):
    y = (x.double() @ w.double().T) * xs.double()[:, None] * ws.double()
    e = y.abs() * 4 * U
    if not gated:
        return y, e
    h = w.shape[0] // 2
    g, u, eg, eu = y[:, :h], y[:, h:], e[:, :h], e[:, h:]
    s = g * torch.sigmoid(g)
    return s * u, 1.1 * eg * (u.abs() + eu) + s.abs() * eu + (s * u).abs() * (g.abs() + 16) * 2 * U


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("T,N,K", ONE + [(3, 32, 131071)])
def test_int8_one_matrix(gpu, T, N, K, gated):
    if gated:
        N += N % 2
    x, w = int8s(T, T, K), int8s(N, N, K)
    xs, ws = torch.rand(T, generator=torch.Generator().manual_seed(1)) * 1e-3 + 1e-4, torch.randn(N, generator=torch.Generator().manual_seed(2)) * 0.1
    want, tol = i8_ref(x, xs, w, ws, gated)
    for odd, out in ((False, BF), (False, SF), (True, HF)):
        print(f"[mm] int8 {T}x{K} by {N} gated {gated} to {out} odd {odd}", flush=True)
        if out == HF and float(want.abs().max()) > 60000:
            continue
        y = gpu.i8_matmul(own(x, odd), own(xs, odd), own(w, odd), own(ws, odd), gated=gated, out_dtype=out)
        torch.cuda.synchronize()
        near(y, want, rounded(want, tol, out), (odd, out))


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("P,E,N,K", STACK)
def test_int8_stack(gpu, P, E, N, K, gated):
    off = split(P, E, P)
    held = int(off[-1])
    w, ws = int8s(N, E, N, K), torch.rand(E, N, generator=torch.Generator().manual_seed(2)) * 0.1
    top_k = 3
    n_x = -(-P // top_k)
    order = torch.randperm(P, generator=torch.Generator().manual_seed(P))
    order[held:] = ~order[held:]
    for ordered in (False, True):
        print(f"[mm] int8 stack {P} over {E} {N}x{K} gated {gated} ordered {ordered}", flush=True)
        n = n_x if ordered else P
        x, xs = int8s(3, n, K), torch.rand(n, generator=torch.Generator().manual_seed(1)) * 1e-3
        src = torch.where(order < 0, ~order, order) // top_k if ordered else torch.arange(P)
        cols = N // 2 if gated else N
        want, tol = torch.zeros(P, cols, dtype=torch.float64), torch.zeros(P, cols, dtype=torch.float64)
        for e in range(E):
            a, b = int(off[e]), int(off[e + 1])
            if a < b:
                want[a:b], tol[a:b] = i8_ref(x[src[a:b]], xs[src[a:b]], w[e], ws[e], gated)
        y = gpu.i8_matmul(x.cuda(), xs.cuda(), w.cuda(), ws.cuda(), gated=gated, offsets=off.cuda(),
                          order=order.to(torch.int32).cuda() if ordered else None, top_k=top_k, out_dtype=SF)
        torch.cuda.synchronize()
        near(y, want, rounded(want, tol, SF), ordered)
        assert not y[held:].any()
    gpu.sync()


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("T,K", [(1, 1), (1, 7168), (3, 130), (17, 1411), (40, 8200), (2, 70000), (700, 64)])
def test_quantize(gpu, T, K, dtype):
    """Both quotients are correctly rounded, so that codes and scales are the formula's, bit by bit."""
    print(f"[mm] quantize {T}x{K} {dtype}", flush=True)
    x = rand(T, T, K, dtype=dtype)
    x[0] *= 0.0
    if T > 2:
        x[1] = 3.0
        x[2, : K // 2] *= -100.0
    for odd in (False, True):
        q, s = gpu.quantize_i8(own(x, odd))
        torch.cuda.synchronize()
        scale = (x.float().abs().amax(1) / torch.tensor(127.0)).clamp_min(1e-12)
        assert torch.equal(s.cpu(), scale)
        assert torch.equal(q.cpu(), torch.round(x.float() / scale[:, None]).to(I8))


@pytest.mark.parametrize("dtype", [BF, SF])
@pytest.mark.parametrize("T,K", [(2050, 2048), (2049, 1001), (5, 512), (6, 513)])
def test_quantize_many_rows(gpu, T, K, dtype):
    test_quantize(gpu, T, K, dtype)


def test_quantize_rows_that_are_not_finite(gpu):
    x = rand(1, 5, 200)
    x[1, 3], x[2, 199], x[3, 0] = float("nan"), float("inf"), -float("inf")
    q, s = gpu.quantize_i8(x.cuda())
    torch.cuda.synchronize()
    assert bool(torch.isnan(s[1])) and bool(torch.isinf(s[2:4]).all()) and bool(torch.isfinite(s[[0, 4]]).all())
    # a product with such a row is not finite, and its neighbours are
    w = torch.ones(3, 200, dtype=I8, device="cuda")
    y = gpu.i8_matmul(q, s, w, torch.ones(3, device="cuda"), out_dtype=SF)
    assert bool(torch.isfinite(y[[0, 4]]).all()) and not bool(torch.isfinite(y[1:4]).any())


def grad_ref(dy, x, w, off):
    """dx, dw and how far fp32 sums of them may be off."""
    E, N, K = w.shape
    dx, ex = torch.zeros(x.shape, dtype=torch.float64), torch.zeros(x.shape, dtype=torch.float64)
    dw, ew = torch.zeros(w.shape, dtype=torch.float64), torch.zeros(w.shape, dtype=torch.float64)
    for e in range(E):
        a, b = int(off[e]), int(off[e + 1])
        if a == b:
            continue
        d, xx, ww = dy[a:b].double(), x[a:b].double(), w[e].double()
        dx[a:b], ex[a:b] = d @ ww, (d.abs() @ ww.abs()) * (N + 8) * U
        dw[e], ew[e] = d.T @ xx, (d.abs().T @ xx.abs()) * (b - a + 8) * U
    return dx, ex, dw, ew


GRADS = [(1, 0, 32, 64), (1, 0, 512, 2048), (130, 0, 34, 72), (257, 0, 130, 411), (1000, 0, 256, 136), (5, 3, 18, 33), (40, 64, 48, 136),
         (300, 6, 145, 520), (1200, 4, 258, 384), (3000, 9, 264, 96), (64, 200, 40, 24), (0, 3, 16, 24), (600, 2, 520, 328)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("P,E,N,K", GRADS)
def test_gradients(gpu, P, E, N, K, dtype):
    """E 0: one matrix, without offsets.  Rows behind the last matrix hold NaN; matrices without rows have zeros."""
    off = split(P, E, P) if E else torch.tensor([0, P])
    held = int(off[-1])
    x, dy, w = poisoned(rand(1, P, K, dtype=dtype), held), poisoned(rand(2, P, N, dtype=dtype, std=0.1), held), rand(3, max(1, E), N, K, dtype=dtype, std=0.1)
    dx, ex, dw, ew = grad_ref(dy, x, w, off)
    for odd, out in ((False, dtype), (False, SF), (True, dtype)):
        print(f"[mm] gradients {P} over {E} {N}x{K} {dtype} dw {out} odd {odd}", flush=True)
        torch.full((P * N * 2 + w.numel() * 4,), float("nan"), device="cuda")  # goes back to the allocator
        wd = own(w if E else w[0], odd)
        gx, gw = gpu.matmul_grad(own(dy, odd), own(x, odd), wd, offsets=off.to(torch.int32).cuda() if E else None, dw_dtype=out)
        torch.cuda.synchronize()
        assert gx.dtype == dtype and gw.dtype == out and gw.shape == wd.shape
        near(gx, dx, rounded(dx, ex, dtype), "dx")
        near(gw.view(w.shape), dw, rounded(dw, ew, out), "dw")
        assert not gx[held:].any()
    if held > P:  # offsets that leave the rows
        from constellation_amd._lib import CxError
        with pytest.raises(CxError, match="offset"):
            gpu.sync()
    else:
        gpu.sync()
    only, none = gpu.matmul_grad(dy.cuda(), x.cuda(), wd, offsets=off.to(torch.int32).cuda() if E else None, want_dw=False)
    assert none is None and torch.equal(only, gx)
    none, only = gpu.matmul_grad(dy.cuda(), x.cuda(), wd, offsets=off.to(torch.int32).cuda() if E else None, want_dx=False, dw_dtype=SF)
    assert none is None
    near(only.view(w.shape), dw, rounded(dw, ew, SF), "dw alone")
    if held > P:
        with pytest.raises(CxError, match="offset"):
            gpu.sync()


def gate_grad_ref(dh, pre):
    """The gradient at pre of silu(g) u, and how far fp32 may be off before the rounding: each factor rounds
    a few times, the exponential's argument moves it by up to |g| units, and 1 + g (1 - s) may cancel."""
    g, u = pre.double().chunk(2, 1)
    d, s = dh.double(), torch.sigmoid(pre.double().chunk(2, 1)[0])
    out = torch.cat((d * u * s * (1 + g * (1 - s)), d * g * s), 1)
    size = torch.cat(((d * u * s).abs() * (1 + g.abs()), (d * g * s).abs()), 1)
    return out, size * (torch.cat((g, g), 1).abs() + 16) * 2 * U


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("P,E,I,K", [(1, 0, 16, 64), (130, 0, 17, 72), (300, 6, 80, 264), (1200, 4, 128, 129), (64, 200, 24, 24)])
def test_gated_gradients(gpu, P, E, I, K, dtype):
    """The gradient at pre is rounded to the type, half a step of each value, and enters the products as it is."""
    off = split(P, E, P) if E else torch.tensor([0, P])
    held = int(off[-1])
    x, dh, w = poisoned(rand(1, P, K, dtype=dtype), held), poisoned(rand(2, P, I, dtype=dtype), held), rand(3, max(1, E), 2 * I, K, dtype=dtype, std=0.1)
    pre = poisoned(rand(4, P, 2 * I, dtype=dtype, std=2.0), held)
    d, ed = gate_grad_ref(dh, pre)
    d[held:], ed[held:] = 0, 0
    ed = rounded(d, ed, dtype)
    dx, ex, dw, ew = grad_ref(d, torch.nan_to_num(x), w, off)
    for e in range(max(1, E)):
        a, b = int(off[e]), int(off[e + 1])
        ex[a:b] += ed[a:b] @ w[e].double().abs() * (1 + 2 * I * U)
        ew[e] += ed[a:b].T @ torch.nan_to_num(x[a:b]).double().abs() * (1 + P * U)
    for odd in (False, True):
        print(f"[mm] gated gradients {P} over {E} {I}x{K} {dtype} odd {odd}", flush=True)
        gx, gw = gpu.matmul_grad(own(dh, odd), own(x, odd), own(w if E else w[0], odd), pre=own(pre, odd),
                                 offsets=off.to(torch.int32).cuda() if E else None)
        torch.cuda.synchronize()
        near(gx, dx, rounded(dx, ex, dtype), "dx")
        near(gw.view(w.shape), dw, rounded(dw, ew, dtype), "dw")
        assert not gx[held:].any()


def test_gradients_against_differences(gpu):
    """d loss along a direction, from the gradients and from two forward passes, in a gated product.  fp32 outputs, and a
    step so long that their rounding is small beside the difference; what is left is the third derivative's part, h^2 / 6 of
    it, and the 16-bit rounding of inputs: steps are powers of two on values of few bits, so that x + h v is exact."""
    P, I, K = 48, 24, 40
    g = torch.Generator().manual_seed(0)
    pick = lambda *s: (torch.randint(-8, 9, s, generator=g).float() / 16)  # noqa: E731
    x, w, vx, vw = pick(P, K), pick(2 * I, K), pick(P, K), pick(2 * I, K)
    dh = pick(P, I)
    h = 2.0 ** -6  # x + h v has values of 2^-10 up to 1: 11 bits, exact in fp16
    run = lambda t: gpu.matmul((x + t * vx).to(HF).cuda(), (w + t * vw).to(HF).cuda(), gated=True, out_dtype=SF).double()  # noqa: E731
    slope = float(((run(h) - run(-h)) / (2 * h) * dh.cuda().double()).sum())
    y, pre = gpu.matmul(x.to(HF).cuda(), w.to(HF).cuda(), gated=True, keep=True)
    dx, dw = gpu.matmul_grad(dh.to(HF).cuda(), x.to(HF).cuda(), w.to(HF).cuda(), pre=pre, dw_dtype=SF)
    got = float((dx.double() * vx.cuda().double()).sum() + (dw.double() * vw.cuda().double()).sum())
    # along t, g and u are g0 + t a + t^2 b: the third derivative of silu(g) u in t by the chain rule, with
    # |silu'| <= 1.1, |silu''| <= 0.5 and |silu'''| <= 0.31
    d64 = lambda a, b: a.double() @ b.double().T  # noqa: E731
    g0, u0 = d64(x, w).chunk(2, 1)
    ga, ua = (d64(x, vw) + d64(vx, w)).abs().chunk(2, 1)
    gb, ub = d64(vx, vw).abs().chunk(2, 1)
    ga, ua = ga + 2 * h * gb, ua + 2 * h * ub
    uh = u0.abs() + h * ua
    third = (0.31 * ga ** 3 + 3 * 0.5 * ga * 2 * gb) * uh + 3 * (0.5 * ga ** 2 + 1.1 * 2 * gb) * ua + 3 * 1.1 * ga * 2 * ub
    # and the roundings: pre and dpre to half a step of fp16 each (pre's moves dpre by its slope, at most 1.1 + |u|),
    # dx to half a step
    d = dh.double().abs()
    moved = (0.5 * u0.abs() * g0.abs() + 1.1 * u0.abs() + 1.1 * g0.abs() + g0.abs() * 1.1 + u0.abs() * 1.1) * HALF[HF] * d
    tol = float((third * d).sum() * h * h / 6) + float((moved * (ga + ua)).sum()) + float((dx.double().abs().cpu() * vx.double().abs()).sum()) * HALF[HF]
    size = float((run(0).abs() * dh.cuda().double().abs()).sum())
    tol += size * (K + 30) * U / h
    assert abs(slope - got) <= tol and tol < 0.05 * abs(got) + 1.0, (slope, got, tol)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_nan_and_infinities_stay_in_their_rows(gpu, dtype):
    """A row of x or of the weights that is not finite, also the last one of its tile and one whose neighbour's
    tail reads past its end."""
    for K in (70, 72, 130):
        x, w = rand(1, 70, K, dtype=dtype), rand(2, 40, K, dtype=dtype)
        x[3, 5], x[69, K - 1], w[7, 0], w[39, K - 1] = float("nan"), float("inf"), float("nan"), -float("inf")
        y = gpu.matmul(x.cuda(), w.cuda())
        bad = torch.zeros(70, 40, dtype=torch.bool)
        bad[[3, 69]] = True
        bad[:, [7, 39]] = True
        assert torch.equal(~torch.isfinite(y).cpu(), bad)
        dy = rand(3, 70, 40, dtype=dtype)
        dx, dw = gpu.matmul_grad(dy.cuda(), torch.nan_to_num(x, nan=1.0, posinf=1.0).cuda(), w.cuda())
        bad = torch.zeros(70, K, dtype=torch.bool)
        bad[:, [0, K - 1]] = True
        assert torch.equal(~torch.isfinite(dx).cpu(), bad) and bool(torch.isfinite(dw).all())


def test_offsets_out_of_order_are_cut_and_reported(gpu):
    from constellation_amd._lib import CxError
    E, N, K, P = 4, 40, 64, 100
    x, w = rand(1, P, K, dtype=BF), rand(2, E, N, K, dtype=BF, std=0.1)
    for off, cut in (([0, 30, 20, 60, 400], [0, 30, 30, 60, 100]), ([0, -5, 50, 50, 90], [0, 0, 50, 50, 90]), ([7, 10, 20, 30, 40], [0, 10, 20, 30, 40])):
        print(f"[mm] offsets {off}", flush=True)
        y = gpu.matmul(x.cuda(), w.cuda(), offsets=torch.tensor(off, dtype=torch.int32, device="cuda"))
        with pytest.raises(CxError, match="offset"):
            gpu.sync()
        dx, dw = gpu.matmul_grad(y, x.cuda(), w.cuda(), offsets=torch.tensor(off, dtype=torch.int32, device="cuda"))
        with pytest.raises(CxError, match="offset"):
            gpu.sync()
        good = torch.tensor(cut, dtype=torch.int32, device="cuda")
        assert torch.equal(y, gpu.matmul(x.cuda(), w.cuda(), offsets=good))
        gx, gw = gpu.matmul_grad(y, x.cuda(), w.cuda(), offsets=good)
        assert torch.equal(dx, gx) and torch.equal(dw, gw)
        gpu.sync()


def test_offsets_of_odd_rows(gpu):
    """Rows that are copied first: a first offset past the second gives matrix 0 the rows from 0 on; and a captured call, whose
    matrices with rows are others at each replay."""
    from constellation_amd._lib import CxError
    E, N, K, P = 4, 41, 67, 100
    x, w, dy = rand(1, P, K, dtype=BF).cuda(), rand(2, E, N, K, dtype=BF, std=0.1).cuda(), rand(3, P, N, dtype=BF).cuda()
    off = torch.tensor([0, 5, 20, 30, 40], dtype=torch.int32, device="cuda")

    def step():
        return (gpu.matmul(x, w, offsets=off), *gpu.matmul_grad(dy, x, w, offsets=off))
    want = step()
    gpu.sync()
    off[0] = 7
    bad = step()
    with pytest.raises(CxError, match="offset"):
        gpu.sync()
    assert all(torch.equal(a, b) for a, b in zip(bad, want))
    off[0] = 0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for cut in ([0, 0, 100, 100, 100], [0, 100, 100, 100, 100], [0, 25, 25, 25, 99], [0, 0, 0, 0, 0], [0, 5, 20, 30, 40]):
        print(f"[mm] offsets {cut}", flush=True)
        off.copy_(torch.tensor(cut, dtype=torch.int32))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), cut
        y = torch.zeros(P, N, dtype=torch.float64)
        for e in range(E):
            y[cut[e]:cut[e + 1]] = x[cut[e]:cut[e + 1]].cpu().double() @ w[e].cpu().double().T
        assert torch.allclose(want[0].cpu().double(), y, rtol=2.0 ** -8, atol=2.0 ** -12)
    gpu.sync()


def test_replays_and_streams(gpu):
    """A captured forward and backward, replayed over new values of the same buffers between eager work, and the
    same calls on another stream: the eager results, bit by bit."""
    E, N, K, P = 5, 96, 136, 300
    off = split(P, E, 1).cuda()
    w, v = rand(2, E, N, K, dtype=BF, std=0.1).cuda(), rand(3, E, K, N // 2, dtype=BF, std=0.1).cuda()
    x, dy = torch.empty(P, K, dtype=BF, device="cuda"), torch.empty(P, K, dtype=BF, device="cuda")
    q, ws = gpu.quantize_i8(w)

    def step():
        h, pre = gpu.matmul(x, w, gated=True, keep=True, offsets=off)
        y = gpu.matmul(h, v, offsets=off)
        dh, dv = gpu.matmul_grad(dy, h, v, offsets=off)
        dx, dw = gpu.matmul_grad(dh, x, w, pre=pre, offsets=off)
        xq, xs = gpu.quantize_i8(x)
        return h, pre, y, dh, dv, dx, dw, gpu.i8_matmul(xq, xs, q, ws, gated=True, offsets=off)

    def fill(seed):
        x.copy_(rand(seed, P, K, dtype=BF))
        dy.copy_(rand(seed + 50, P, K, dtype=BF))
    fill(0)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(4):
        fill(seed)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), seed
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step()
        again = step()  # beside it
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, other, again)), seed
    gpu.sync()


def test_no_rows(gpu):
    w = torch.ones(3, 8, 16, dtype=BF, device="cuda")
    x = torch.empty(0, 16, dtype=BF, device="cuda")
    off = torch.zeros(4, dtype=torch.int32, device="cuda")
    assert gpu.matmul(x, w, offsets=off).shape == (0, 8) and gpu.quantize_i8(x)[0].shape == (0, 16)
    dx, dw = gpu.matmul_grad(x[:, :8], x, w, offsets=off)
    assert dx.shape == (0, 16) and not dw.any()
