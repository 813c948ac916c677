"""The rows around the experts: RMS norm with the residual's addition and an e4m3
output, pairs sorted by expert, rows gathered, summed back, and the sum's gradient,
against their formulas in 64 bits on the CPU.

Tolerances count roundings: a result of n fp32 additions and m other fp32 steps is
off by at most (n + m) 2^-24 of the sum of its terms' sizes, and a rounding to the
output type by half a step of it.
"""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF, HF, SF = torch.bfloat16, torch.float16, torch.float32
HALF = {BF: 2.0 ** -8, HF: 2.0 ** -11, SF: 2.0 ** -24}   # relative half step
TINY = {BF: 2.0 ** -134, HF: 2.0 ** -25, SF: 2.0 ** -150}  # half of the smallest value


def rand(seed, *shape, std=1.0, dtype=SF):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g, dtype=torch.float64) * std).to(dtype)


def near(got, want, tol, what):
    got, want = got.cpu().double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), what
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), what
    ok = ~nan & ~inf
    over = ((got - want).abs() - tol)[ok]
    assert over.numel() == 0 or float(over.max()) <= 0, (what, float(over.max()))


def off_by(x, n):
    """x (of any storage) as a view whose data starts n elements after an allocation's start."""
    flat = torch.empty(x.numel() + n, dtype=x.dtype, device="cuda")
    flat[n:] = x.reshape(-1).cuda()
    return flat[n:].view(x.shape)


# ---------------------------------------------------------------------------- norm

def check_norm(gpu, x, r, w, eps, out_dtype, quantize, shift=0, what=""):
    T, H = x.shape
    n = gpu.rms_norm(off_by(x, shift), None if w is None else off_by(w, shift), eps=eps,
                     residual=None if r is None else off_by(r, shift), out_dtype=out_dtype, quantize=quantize)
    torch.cuda.synchronize()
    s = x
    if r is not None:
        s = (x.double() + r.double()).to(SF).to(x.dtype)  # fp32 holds the sum, or is within 2^-24 of it
        assert n.sum.dtype == x.dtype
        near(n.sum, s, s.double().abs() * 2 * HALF[x.dtype] * (x.double() + r.double() != s.double()) + TINY[x.dtype], what + " sum")
        s = n.sum.cpu()
    else:
        assert n.sum is None
    v = s.double()
    y = v / torch.sqrt((v ** 2).mean(1, keepdim=True) + eps)
    if w is not None:
        y = y * w.double()
    # squares of H values summed by up to 1024 threads (at most 64 each), 6 + 16 joins; half of it in the root
    e = (64 + 22 + 12) * U
    fin = torch.where(torch.isfinite(y), y.abs(), 0.0)
    near(n.y, y.to(out_dtype) if out_dtype == SF else y, fin * (e + HALF[out_dtype]) + TINY[out_dtype], what + " y")
    if not quantize:
        assert n.q is None and n.scale is None
        return
    B = -(-H // 128)
    pad = torch.zeros(T, B * 128, dtype=torch.float64)
    pad[:, :H] = y
    amax = pad.view(T, B, 128).abs().amax(2)
    scale = torch.where(torch.isnan(amax), amax, (amax / 448).clamp_min(1e-12))
    near(n.scale, scale, torch.where(torch.isfinite(scale), scale, 0.0) * (e + 2 * U), what + " scale")
    got_s = n.scale.cpu().double()[:, torch.arange(H) // 128]
    q = n.q.cpu().double()
    fin = torch.isfinite(y) & torch.isfinite(got_s)
    assert torch.equal(torch.isnan(q), torch.isnan(y / got_s)), what
    # e4m3: half a step is 2^-4 of the value, or 2^-10 below the normal range (2^-6)
    tol = torch.maximum(y.abs() * 2.0 ** -4, got_s * 2.0 ** -10) + y.abs() * 2 * e
    assert bool(((q * got_s - y).abs() <= tol)[fin].all()), what


@pytest.mark.parametrize("dtype,out,wdt", [(BF, BF, BF), (HF, HF, SF), (SF, SF, SF), (BF, SF, HF), (SF, BF, BF)])
@pytest.mark.parametrize("T,H", [(1, 7168), (3, 1), (5, 127), (2, 1411), (7, 2048), (1, 8200), (2, 16392), (1, 65536)])
def test_rms_norm(gpu, T, H, dtype, out, wdt):
    print(f"[rows] norm {T}x{H} {dtype} {out} {wdt}", flush=True)
    x, r = rand(1, T, H, dtype=dtype), rand(2, T, H, std=3.0, dtype=dtype)
    w = (1 + rand(3, H, std=0.1)).to(wdt)
    check_norm(gpu, x, r, w, 1e-6, out, True, what="full")
    check_norm(gpu, x, None, None, 0.0, out, False, what="bare")


def test_rms_norm_addresses_and_values(gpu):
    """Rows at odd addresses, zero rows and blocks, tiny and huge values, NaN and infinities."""
    print("[rows] norm addresses and values", flush=True)
    for dtype in (BF, HF, SF):
        x, r, w = rand(4, 6, 640, dtype=dtype), rand(5, 6, 640, dtype=dtype), rand(6, 640, dtype=dtype)
        for shift in (1, 2, 4):
            check_norm(gpu, x, r, w, 1e-6, dtype, True, shift=shift, what=f"shift {shift}")
        x[0] = 0
        x[1, 128:256] = 0
        x[2] *= 2.0 ** -10
        x[3, 7] = float("nan")
        x[4, 300] = float("inf")
        check_norm(gpu, x, None, w, 1e-6, dtype, True, what="values")
        check_norm(gpu, torch.zeros_like(x), None, w, 0.0, dtype, True, what="zeros over no eps")


def test_rms_norm_in_place_and_alone(gpu):
    """The sum may be written over the residual; an 8-bit output alone; no tokens."""
    import ctypes as C  # noqa: F401
    from constellation_amd._lib import BF16, CX_OK, lib
    print("[rows] norm in place", flush=True)
    x, r, w = (rand(i, 4, 1024, dtype=BF).cuda() for i in (1, 2, 3))
    w = w[0].contiguous()
    n = gpu.rms_norm(x, w, residual=r, quantize=True)
    for over in (0, 1):
        a, b = x.clone(), r.clone()
        q, sc = torch.empty_like(n.q), torch.empty_like(n.scale)
        assert lib().cx_rms_norm(gpu.handle, a.data_ptr(), BF16, b.data_ptr(), w.data_ptr(), BF16, 4, 1024, 1e-6,
                                 (a, b)[over].data_ptr(), None, BF16, q.data_ptr(), sc.data_ptr(), gpu.stream()) == CX_OK
        torch.cuda.synchronize()
        assert torch.equal((a, b)[over], n.sum) and torch.equal(q.view(torch.uint8), n.q.view(torch.uint8))
        assert torch.equal(sc, n.scale)
    m = gpu.rms_norm(x, w, residual=r, want_y=False, quantize=True)
    assert m.y is None and torch.equal(m.q.view(torch.uint8), n.q.view(torch.uint8))
    e = gpu.rms_norm(x[:0], w, residual=r[:0], quantize=True)
    assert e.y.shape == (0, 1024) and e.q.shape == (0, 1024) and e.scale.shape == (0, 8)


# ---------------------------------------------------------------------------- sort, gather, combine

def sorted_ref(ids, E):
    """(order, offsets, place) by the definition, in Python."""
    flat = ids.reshape(-1).tolist()
    key = [e if 0 <= e < E else E for e in flat]
    order = sorted(range(len(flat)), key=lambda i: key[i])
    place = [0] * len(flat)
    for row, i in enumerate(order):
        place[i] = row if key[i] < E else ~row
    offsets = [sum(k < e for k in key) for e in range(E + 1)]
    i32 = torch.int32
    return (torch.tensor([i if key[i] < E else ~i for i in order], dtype=i32), torch.tensor(offsets, dtype=i32),
            torch.tensor(place, dtype=i32).view(ids.shape))


def some_ids(seed, T, K, E, drop):
    g = torch.Generator().manual_seed(seed)
    ids = torch.rand(T, E, generator=g).topk(K, dim=1).indices.to(torch.int32) if K <= E else \
        torch.randint(0, E, (T, K), generator=g).to(torch.int32)
    return torch.where(torch.rand(T, K, generator=g) < drop, -1, ids)


SORTS = [(1, 1, 1, 0.0), (1, 8, 256, 0.0), (29, 8, 256, 0.0), (64, 8, 8, 0.3), (65, 1, 1024, 0.0), (513, 3, 60, 0.75),
         (200, 64, 5, 0.1), (4099, 8, 256, 0.0), (9001, 8, 64, 0.2), (40, 6, 64, 1.0)]


@pytest.mark.parametrize("T,K,E,drop", SORTS)
def test_sort_tokens(gpu, T, K, E, drop):
    print(f"[rows] sort {T}x{K} of {E}", flush=True)
    ids = some_ids(T + K, T, K, E, drop)
    got = gpu.sort_tokens(ids.cuda(), E)
    torch.cuda.synchronize()
    for g, w, what in zip(got, sorted_ref(ids, E), ("order", "offsets", "place")):
        assert torch.equal(g.cpu(), w), what


def test_sort_tokens_empty_one_expert_and_bad_id(gpu):
    from constellation_amd._lib import CxError
    print("[rows] sort edges", flush=True)
    order, offsets, place = gpu.sort_tokens(torch.empty((0, 8), dtype=torch.int32, device="cuda"), 16)
    assert order.numel() == 0 and place.shape == (0, 8) and offsets.cpu().tolist() == [0] * 17
    ids = torch.full((700, 2), 3, dtype=torch.int32)  # the same expert twice for each token
    for g, w in zip(gpu.sort_tokens(ids.cuda(), 4), sorted_ref(ids, 4)):
        assert torch.equal(g.cpu(), w)
    ids[5, 1] = 4
    got = gpu.sort_tokens(ids.cuda().long(), 4)
    with pytest.raises(CxError, match="out of range"):
        gpu.sync()
    for g, w in zip(got, sorted_ref(ids, 4)):
        assert torch.equal(g.cpu(), w)
    gpu.sync()


@pytest.mark.parametrize("dtype", [BF, HF, SF, torch.float8_e4m3fn, torch.uint8])
@pytest.mark.parametrize("T,K,H", [(1, 8, 7168), (33, 3, 1411), (5, 64, 130), (130, 2, 1), (17, 4, 12)])
def test_gather_rows(gpu, T, K, H, dtype):
    print(f"[rows] gather {T}x{K}x{H} {dtype}", flush=True)
    ids = some_ids(H, T, K, 16, 0.25)
    order, _, place = sorted_ref(ids, 16)
    x = torch.randint(0, 255, (T, H * dtype.itemsize), dtype=torch.uint8, generator=torch.Generator().manual_seed(H))
    want = torch.where(order[:, None] < 0, torch.tensor(0, dtype=torch.uint8), x[torch.where(order < 0, ~order, order).long() // K])
    for shift in (0, 1):
        got = gpu.gather_rows(off_by(x.view(dtype), shift), place.cuda())
        torch.cuda.synchronize()
        assert got.dtype == dtype and torch.equal(got.cpu().view(torch.uint8), want), shift


def combine_ref(ys, place, w, add):
    held = place >= 0
    rows = torch.where(held, place, ~place).long()
    terms = torch.where(held[:, :, None], ys.double()[rows], 0.0) * torch.where(held, w.double(), 0.0)[:, :, None]
    extra = 0.0 if add is None else add.double()
    size = terms.abs().sum(1) + (0.0 if add is None else add.double().abs())
    return terms.sum(1) + extra, size


@pytest.mark.parametrize("dtype,out", [(BF, BF), (HF, SF), (SF, SF), (SF, BF), (BF, HF)])
@pytest.mark.parametrize("T,K,H,drop", [(1, 8, 7168, 0.0), (33, 3, 1411, 0.3), (3, 64, 136, 0.2), (130, 1, 1, 0.5), (9, 9, 2056, 1.0)])
def test_combine_rows(gpu, T, K, H, drop, dtype, out):
    print(f"[rows] combine {T}x{K}x{H} {dtype} {out}", flush=True)
    place = sorted_ref(some_ids(H, T, K, 16, drop), 16)[2]
    ys, w, add = rand(1, T * K, H, dtype=dtype), rand(2, T, K).abs(), rand(3, T, H, dtype=out)
    ys[torch.where(place < 0, ~place, 0).max()] = float("nan") if drop else 0.0  # a row without an expert, when there is one
    if bool((place >= 0).any()) and drop:
        row = int(torch.where(place < 0, ~place, 0).max())
        if bool((place == row).any()):
            ys[row] = 0.0
    for ww, aa, shift in ((w, None, 0), (w, add, 0), (None, add, 1), (None, None, 0)):
        want, size = combine_ref(ys, place, torch.ones(T, K) if ww is None else ww, aa)
        got = gpu.combine_rows(off_by(ys, shift), place.cuda(), None if ww is None else ww.cuda(),
                               add=None if aa is None else off_by(aa, shift), out_dtype=out)
        torch.cuda.synchronize()
        assert got.dtype == out
        # K products and K + 1 additions in fp32, then the rounding
        near(got, want, size * (K + 2) * U + want.abs() * HALF[out] * (1 + 2.0 ** -10) + TINY[out], f"{ww is None} {aa is None}")


def test_combine_leaves_out_bad_rows_and_weights(gpu):
    """NaN and infinite weights and rows of pairs without an expert change nothing."""
    print("[rows] combine, NaN behind the rows", flush=True)
    ids = some_ids(5, 20, 4, 8, 0.4)
    place = sorted_ref(ids, 8)[2]
    ys, w = rand(1, 80, 256, dtype=BF), rand(2, 20, 4).abs()
    clean = gpu.combine_rows(ys.cuda(), place.cuda(), w.cuda())
    ys[(~place[place < 0]).long()] = float("inf")
    w[place < 0] = float("nan")
    got = gpu.combine_rows(ys.cuda(), place.cuda(), w.cuda())
    dys, dw = gpu.combine_rows_grad(clean, ys.cuda(), place.cuda(), w.cuda())
    torch.cuda.synchronize()
    assert torch.equal(got, clean)
    assert bool(torch.isfinite(dys).all()) and bool(torch.isfinite(dw).all())
    assert not dys[(~place[place < 0]).long().cuda()].any() and not dw.cpu()[place < 0].any()


@pytest.mark.parametrize("dtype,dodt", [(BF, BF), (HF, SF), (SF, SF), (SF, BF)])
@pytest.mark.parametrize("T,K,H,drop", [(1, 8, 7168, 0.0), (33, 3, 1411, 0.3), (3, 64, 136, 0.2), (130, 1, 1, 0.5), (447, 9, 72, 0.1), (448, 10, 72, 0.1), (1030, 9, 72, 0.1)])
def test_combine_rows_grad(gpu, T, K, H, drop, dtype, dodt):
    print(f"[rows] grad {T}x{K}x{H} {dtype} {dodt}", flush=True)
    place = sorted_ref(some_ids(H, T, K, 16, drop), 16)[2]
    held = place >= 0
    rows = torch.where(held, place, ~place).long()
    ys, w, d = rand(1, T * K, H, dtype=dtype), rand(2, T, K).abs(), rand(3, T, H, dtype=dodt)
    for ww, shift in ((w, 0), (None, 1)):
        w64 = torch.where(held, torch.ones(T, K, dtype=torch.float64) if ww is None else ww.double(), 0.0)
        want = torch.empty(T * K, H, dtype=torch.float64)
        want[rows.reshape(-1)] = (w64[:, :, None] * d.double()[:, None]).reshape(-1, H)
        prod = d.double()[:, None] * ys.double()[rows]
        dys, dw = gpu.combine_rows_grad(off_by(d, shift), off_by(ys, shift), place.cuda(), None if ww is None else ww.cuda())
        torch.cuda.synchronize()
        assert dys.dtype == dtype and dw.dtype == SF
        near(dys, want, want.abs() * (U + HALF[dtype] * (1 + 2.0 ** -10)) + TINY[dtype], "dys")
        # 8 columns of each 2048 a thread, then 6 + 4 joins; a product and an addition each
        steps = 8 * -(-H // 2048) + 12
        near(dw, torch.where(held, prod.sum(2), 0.0), prod.abs().sum(2) * steps * U, "dw")


def test_gradients_are_those_of_the_forward(gpu):
    """<d out, v> of the gather and the sum, by differences: both are linear in the
    rows and in the weights, so a step of 1 is exact up to the roundings of fp32."""
    print("[rows] gradients against differences", flush=True)
    T, K, H = 24, 3, 96
    place = sorted_ref(some_ids(7, T, K, 8, 0.2), 8)[2].cuda()
    x, vx = rand(1, T, H).cuda(), rand(2, T, H).cuda()
    ys, vy = rand(3, T * K, H).cuda(), rand(4, T * K, H).cuda()
    w, vw = rand(5, T, K).abs().cuda(), rand(6, T, K).abs().cuda()
    gx, go = rand(7, T * K, H).cuda().double(), rand(8, T, H).cuda()

    def diff(a, b):
        return a.double() - b.double()

    def same(a, b):
        assert abs(float(a) - float(b)) <= 1e-4 * (1 + abs(float(b))), (float(a), float(b))

    same((gx * diff(gpu.gather_rows(x + vx, place), gpu.gather_rows(x, place))).sum(),
         (gpu.combine_rows(gx.float(), place).double() * vx).sum())
    dys, dw = gpu.combine_rows_grad(go, ys, place, w)
    base = gpu.combine_rows(ys, place, w)
    same((go * diff(gpu.combine_rows(ys + vy, place, w), base)).sum(), (dys.double() * vy).sum())
    same((go * diff(gpu.combine_rows(ys, place, w + vw), base)).sum(), (dw.double() * vw).sum())


def test_places_outside_the_rows_are_reported(gpu):
    """A place that names no row is skipped, whichever call reads it."""
    from constellation_amd._lib import CxError
    print("[rows] places outside", flush=True)
    T, K, H = 6, 2, 64
    place = sorted_ref(some_ids(3, T, K, 4, 0.0), 4)[2]
    x, ys = rand(1, T, H).cuda(), rand(2, T * K, H).cuda()
    for bad in (T * K, -T * K - 1, 2 ** 31 - 1, -2 ** 31):
        p = place.clone()
        p[2, 1] = bad
        gpu.gather_rows(x, p.cuda())
        with pytest.raises(CxError, match="outside the rows"):
            gpu.sync()
        out = gpu.combine_rows(ys, p.cuda())
        if bad > 0:
            with pytest.raises(CxError, match="outside the rows"):
                gpu.sync()
        want = combine_ref(ys.cpu(), torch.where(p == bad, -1, p), torch.ones(T, K), None)[0]
        near(out, want, 1e-5, "combine")
        gpu.combine_rows_grad(out, ys, p.cuda())
        with pytest.raises(CxError, match="outside the rows"):
            gpu.sync()
    gpu.sync()


def test_rows_in_graphs_and_streams(gpu):
    """norm -> sort -> gather -> combine -> gradient as one captured graph, replayed on
    new inputs with eager calls between, equal to eager bit for bit."""
    print("[rows] graph", flush=True)
    T, K, H, E = 77, 4, 1024, 32
    w = rand(9, H, dtype=BF).cuda()

    def inputs(i):
        return (rand(i, T, H, dtype=BF).cuda(), rand(i + 50, T, H, dtype=BF).cuda(),
                some_ids(i, T, K, E, 0.2).cuda(), rand(i + 99, T, K).abs().cuda())

    def chain(x, r, ids, wt):
        n = gpu.rms_norm(x, w, residual=r, quantize=True)
        order, offsets, place = gpu.sort_tokens(ids, E)
        xs = gpu.gather_rows(n.y, place)
        out = gpu.combine_rows(xs, place, wt, add=n.sum)
        dys, dw = gpu.combine_rows_grad(out, xs, place, wt)
        return [n.sum, n.y, n.q.view(torch.uint8), n.scale, order, offsets, place, xs, out, dys, dw,
                gpu.combine_rows(dys, place)]

    held = [t.clone() for t in inputs(1)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain(*held)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side, capture_error_mode="thread_local"):
        got = chain(*held)
    for i in (2, 3, 4):
        new = inputs(i)
        for h, t in zip(held, new):
            h.copy_(t)
        torch.cuda.synchronize()
        g.replay()
        want = chain(*new)
        torch.cuda.synchronize()
        for k, (a, b) in enumerate(zip(got, want)):
            assert torch.equal(a, b), (i, k)
    del g


@pytest.mark.parametrize("E", [1, 510, 511, 600, 1024])
def test_sort_no_tokens(gpu, E):
    """No pairs at all, on both sides of the sort's limits for one workgroup."""
    print(f"[rows] sort nothing over {E}", flush=True)
    for K in (1, 8):
        order, offsets, place = gpu.sort_tokens(torch.empty((0, K), dtype=torch.int32, device="cuda"), E)
        assert order.numel() == 0 and place.shape == (0, K) and offsets.cpu().tolist() == [0] * (E + 1)
    gpu.sync()
