"""Products with 4-bit weights and layers of 4-bit experts against their formulas in
64 bits on the CPU.

Tolerances count roundings.  The products of codes, scales and x are exact in fp32 up
to the scale's (one rounding), and a sum of n of them is off by at most n 2^-24 of the
sum of their sizes; the output's rounding adds half a step.
"""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF, HF, SF, F8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
HALF = {BF: 2.0 ** -8, HF: 2.0 ** -11, SF: 2.0 ** -24}
TINY = {BF: 2.0 ** -134, HF: 2.0 ** -25, SF: 2.0 ** -150}
# h takes part in the down product as fp16 times a power of two per row: 11 significant bits, whose
# half step is at most 2^-11 of the value (1 + 2^-11 lies between 1 and its neighbour 1 + 2^-10)
H_HALF = 2.0 ** -11
E2M1 = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)


def make(seed, E, N, K, group):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (E, N, (K + 1) // 2), generator=g, dtype=torch.uint8)  # an odd width's last nibble is not zero
    scales = ((torch.rand(E, N, -(-K // group), generator=g) + 0.5) * 0.02 *
              torch.where(torch.rand(E, N, 1, generator=g) < 0.1, -1.0, 1.0)).to(BF)
    return codes, scales


def dense(codes, scales, K, group):
    nib = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)[..., :K]
    return E2M1[nib.long()] * scales.double().repeat_interleave(group, -1)[..., :K]


def rand(seed, *shape, dtype=SF, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g, dtype=torch.float64) * std).to(dtype)


def make_x(seed, T, K, dtype):
    """(x, scale or None, its values in 64 bits)"""
    x = rand(seed, T, K, dtype=SF if dtype == F8 else dtype)
    if dtype != F8:
        return x, None, x.double()
    s = torch.rand(T, -(-K // 128), generator=torch.Generator().manual_seed(seed)) + 0.01
    q = (x * 40).to(F8)
    return q, s, q.double() * s.double().repeat_interleave(128, 1)[:, :K]


def product_ref(x, W, gated):
    """(y, how far fp32 sums may be off) of x W^T, before the output's rounding."""
    K = W.shape[1]
    y, size = x @ W.T, x.abs() @ W.abs().T
    e = size * (K + 8) * U
    if not gated:
        return y, e
    h = W.shape[0] // 2
    g, u, eg, eu = y[:, :h], y[:, h:], e[:, :h], e[:, h:]
    s = g * torch.sigmoid(g)
    out = s * u
    # |silu'| <= 1.1; an exponential in fp32 is off by a few units and its argument's, |g|, more
    return out, 1.1 * eg * (u.abs() + eu) + s.abs() * eu + out.abs() * (g.abs() + 16) * 2 * U


def near(got, want, tol, what):
    got = got.cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    over = (got - want).abs() - tol
    assert not bool(torch.isnan(over).any()), what
    assert over.numel() == 0 or float(over.max()) <= 0, (what, float(over.max()))


def rounded(want, e, out):
    return e + (want.abs() + e) * HALF[out] + TINY[out]


SHAPES = [(1, 32, 32), (1, 512, 7168), (2, 18, 130), (5, 100, 129), (16, 64, 1000), (17, 130, 384), (33, 34, 1), (70, 256, 640),
          (128, 258, 512), (129, 1024, 256), (300, 160, 2048), (513, 96, 72)]


@pytest.mark.parametrize("dtype", [BF, HF, F8])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("T,N,K", SHAPES)
def test_q4_matmul(gpu, T, N, K, gated, dtype):
    from constellation_amd.engine import Q4Matrix
    for group in (32, 64, 128):
        print(f"[q4] {T}x{K} by {N} group {group} gated {gated} {dtype}", flush=True)
        codes, scales = make(T + N, 1, N, K, group)
        w = Q4Matrix.pack(codes.cuda(), scales.cuda(), K, group=group, gated=gated)
        try:
            x, xs, x64 = make_x(K, T, K, dtype)
            want, e = product_ref(x64, dense(codes, scales, K, group)[0], gated)
            if dtype == F8:
                e = e * 2  # the row's scale is a factor of its own
            for out in ({BF: (BF, SF), HF: (HF, BF), F8: (BF, SF)}[dtype] if group == 128 else (None,)):
                y = gpu.q4_matmul(w, x.cuda(), x_scale=None if xs is None else xs.cuda(), out_dtype=out)
                torch.cuda.synchronize()
                near(y, want, rounded(want, e, y.dtype), out)
        finally:
            w.free()


def split(T, E, seed):
    """offsets of E matrices over T rows, some matrices without rows, some rows behind the last."""
    g = torch.Generator().manual_seed(seed)
    cut = torch.sort(torch.randint(0, max(1, T - T // 8) + 1, (E,), generator=g)).values
    return torch.cat((torch.zeros(1, dtype=torch.long), cut)).to(torch.int32)


@pytest.mark.parametrize("dtype,gated", [(BF, False), (HF, True), (F8, False), (F8, True)])
@pytest.mark.parametrize("P,E,N,K,group", [(1, 1, 32, 64, 32), (7, 5, 50, 200, 64), (40, 64, 48, 256, 128), (300, 6, 144, 520, 32),
                                           (1200, 4, 256, 384, 128), (5, 1024, 16, 33, 32)])
def test_q4_matmul_stack(gpu, P, E, N, K, group, dtype, gated):
    """Rows dealt to the matrices by offsets, as they lie and through an order; rows behind the last are zeros."""
    from constellation_amd.engine import Q4Matrix
    print(f"[q4] stack {P} over {E} {N}x{K} group {group} {dtype} {gated}", flush=True)
    codes, scales = make(P + E, E, N, K, group)
    w = Q4Matrix.pack(codes.cuda(), scales.cuda(), K, group=group, gated=gated)
    W = dense(codes, scales, K, group)
    off = split(P, E, P)
    try:
        x, xs, x64 = make_x(3, P, K, dtype)
        top_k = 3
        n_x = -(-P // top_k)
        order = torch.randperm(P, generator=torch.Generator().manual_seed(1)).to(torch.int32)
        order[int(off[-1]):] = ~order[int(off[-1]):]
        for ordered in (False, True):
            want, tol = torch.zeros(P, w.out_cols, dtype=torch.float64), torch.zeros(P, w.out_cols, dtype=torch.float64)
            src = torch.where(order < 0, ~order, order).long() // top_k if ordered else torch.arange(P)
            for e in range(E):
                a, b = int(off[e]), int(off[e + 1])
                if a < b:
                    want[a:b], tol[a:b] = product_ref(x64[src[a:b]], W[e], gated)
            n = n_x if ordered else P
            y = gpu.q4_matmul(w, x[:n].cuda(), x_scale=None if xs is None else xs[:n].cuda(), offsets=off.cuda(),
                              order=order.cuda() if ordered else None, top_k=top_k)
            torch.cuda.synchronize()
            near(y, want, rounded(want, 2 * tol, y.dtype) * (want != 0), ordered)
    finally:
        w.free()


def test_q4_matmul_rows_at_any_address_and_bad_offsets(gpu):
    from constellation_amd._lib import CxError
    from constellation_amd.engine import Q4Matrix
    print("[q4] addresses and offsets", flush=True)
    codes, scales = make(1, 3, 40, 256, 64)
    w = Q4Matrix.pack(codes.cuda(), scales.cuda(), 256, group=64)
    W = dense(codes, scales, 256, 64)
    try:
        for P in (20, 200):
            x = rand(2, P, 256, dtype=BF)
            off = torch.tensor([0, P // 3, P // 2, P], dtype=torch.int32)
            want = torch.cat([x[a:b].double() @ W[e].T for e, (a, b) in enumerate(zip(off[:-1], off[1:]))])
            tol = torch.cat([x[a:b].double().abs() @ W[e].abs().T for e, (a, b) in enumerate(zip(off[:-1], off[1:]))]) * 264 * U
            for shift in (1, 3, 4):
                flat = torch.empty(x.numel() + shift, dtype=BF, device="cuda")
                flat[shift:] = x.reshape(-1).cuda()
                y = gpu.q4_matmul(w, flat[shift:].view(P, 256), offsets=off.cuda())
                near(y, want, rounded(want, tol, BF), shift)
            gpu.sync()
            bad = torch.tensor([0, P // 3, P // 4, 10 * P], dtype=torch.int32)  # goes back, and past the rows
            y = gpu.q4_matmul(w, x.cuda(), offsets=bad.cuda())
            with pytest.raises(CxError, match="outside the rows"):
                gpu.sync()
            near(y[:P // 3], want[:P // 3], rounded(want, tol, BF)[:P // 3], "before the fault")
            order = torch.arange(P, dtype=torch.int32)
            order[3], order[4] = -5, P + 7  # no pair, and one past x: rows of zeros
            y = gpu.q4_matmul(w, x.cuda(), offsets=off.cuda(), order=order.cuda())
            assert not y[3:5].any()
            near(y[5:], want[5:], rounded(want, tol, BF)[5:], "order")
            assert gpu.q4_matmul(w, x[:0].cuda(), offsets=torch.zeros(4, dtype=torch.int32, device="cuda")).shape == (0, 40)
    finally:
        w.free()


def test_q4_values(gpu):
    """Every code, a NaN row among others, infinite and zero scales."""
    from constellation_amd.engine import Q4Matrix
    print("[q4] values", flush=True)
    K = 128
    codes = torch.zeros(1, 16, K // 2, dtype=torch.uint8)
    for r in range(16):
        codes[0, r] = r | (r << 4)
    scales = torch.ones(1, 16, 1, dtype=BF)
    w = Q4Matrix.pack(codes.cuda(), scales.cuda(), K)
    try:
        for T in (3, 80):
            x = torch.zeros(T, K, dtype=BF)
            x[0, 5] = 1.0
            x[1, 7] = float("nan")
            x[2] = 0.25
            y = gpu.q4_matmul(w, x.cuda(), out_dtype=SF).cpu().double()
            assert torch.equal(y[0], E2M1) and bool(torch.isnan(y[1]).all()) and torch.equal(y[2], 32 * E2M1)
            assert T == 3 or not y[3:].any()
    finally:
        w.free()


def layer_ref(x64, ids, w, gu, dn, h_half, shared=None):
    """(y, tolerance before the output's rounding) of a layer on given routes; h_half: relative rounding of h."""
    T = x64.shape[0]
    y, tol = torch.zeros(T, dn.shape[1], dtype=torch.float64), torch.zeros(T, dn.shape[1], dtype=torch.float64)
    picks = [(t, int(e), float(w[t, k]), gu, dn) for t in range(T) for k, e in enumerate(ids[t].tolist()) if e >= 0]
    if shared is not None:
        picks += [(t, 0, 1.0, *shared) for t in range(T)]
    for t, e, wt, g, d in picks:
        h, eh = product_ref(x64[t:t + 1], g[e], True)
        eh = eh + h.abs() * h_half
        o, size = h @ d[e].T, h.abs() @ d[e].abs().T
        eo = size * (d.shape[2] + 8) * U + eh @ d[e].abs().T
        y[t] += wt * o[0]
        tol[t] += wt * (eo[0] + 4 * U * o[0].abs()) + ids.shape[1] * U * wt * o[0].abs()
    return y, tol


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("T,K,E,H,I,group,dtype", [(1, 8, 32, 512, 256, 128, BF), (3, 2, 4, 300, 70, 32, HF), (40, 4, 8, 256, 128, 64, BF),
                                                   (130, 8, 8, 256, 130, 128, BF), (300, 2, 3, 384, 192, 32, HF), (2, 1, 1, 33, 17, 32, BF)])
def test_q4_layer(gpu, T, K, E, H, I, group, dtype, shared):
    from constellation_amd.engine import Q4Layer, Q4Matrix
    print(f"[q4] layer {T}x{K} of {E} {H}x{I} group {group} {dtype} shared {shared}", flush=True)
    gu, dn, sg, sd = (make(i + T, n, *s, group) for i, (n, s) in
                      enumerate(((E, (2 * I, H)), (E, (H, I)), (1, (2 * I, H)), (1, (H, I)))))
    mats = [Q4Matrix.pack(c.cuda(), s.cuda(), k, group=group, gated=gt)
            for (c, s), k, gt in ((gu, H, True), (dn, I, False), (sg, H, True), (sd, I, False))]
    try:
        layer = Q4Layer(gpu, mats[0], mats[1], (mats[2], mats[3]) if shared else None)
        x = rand(5, T, H, dtype=dtype)
        g = torch.Generator().manual_seed(6)
        ids = torch.rand(T, E, generator=g).topk(K, dim=1).indices.to(torch.int32)
        ids[torch.rand(T, K, generator=g) < 0.15] = -1
        ids[T // 2] = -1  # a token without a route
        w = torch.rand(T, K, generator=g)
        y, yf = gpu.moe(layer, x.cuda(), ids.cuda(), w.cuda(), want_f32=True)
        torch.cuda.synchronize()
        gpu.sync()
        D = [dense(c, s, k, group) for (c, s), k in ((gu, H), (dn, I), (sg, H), (sd, I))]
        want, tol = layer_ref(x.double(), ids, w, D[0], D[1], H_HALF, (D[2], D[3]) if shared else None)
        near(yf, want, tol, "fp32")
        near(y, want, rounded(want, tol, dtype), "rounded")
        if not shared:
            assert not yf[T // 2].any()
        again = gpu.moe(layer, x.cuda(), ids.cuda(), w.cuda())
        assert torch.equal(again, y)
        assert gpu.moe(layer, x[:0].cuda(), ids[:0].cuda(), w[:0].cuda()).shape == (0, H)
    finally:
        for m in mats:
            m.free()


def test_q4_layer_bad_routes(gpu):
    """A repeated expert, an id past the experts and a bad weight are left out and reported, as in cx_moe_decode."""
    from constellation_amd._lib import CxError
    from constellation_amd.engine import Q4Layer, Q4Matrix
    print("[q4] bad routes", flush=True)
    E, H, I = 6, 128, 64
    gu, dn = make(1, E, 2 * I, H, 32), make(2, E, H, I, 32)
    mats = [Q4Matrix.pack(gu[0].cuda(), gu[1].cuda(), H, group=32, gated=True), Q4Matrix.pack(dn[0].cuda(), dn[1].cuda(), I, group=32)]
    try:
        layer = Q4Layer(gpu, *mats)
        x = rand(3, 4, H, dtype=BF).cuda()
        good = torch.tensor([[0, 1, 2], [3, -1, -1], [4, -1, 5], [-1, 2, 0]], dtype=torch.int32)
        w = torch.full((4, 3), 0.5)
        want = gpu.moe(layer, x, good.cuda(), w.cuda())
        for put, weight, text in (((1, 1, 3), 0.5, "twice"), ((1, 1, 6), 0.5, "out of range"), ((1, 1, 2), float("nan"), "weight"),
                                  ((2, 1, 0), -1.0, "weight")):
            ids, ww = good.clone(), w.clone()
            ids[put[0], put[1]], ww[put[0], put[1]] = put[2], weight
            got = gpu.moe(layer, x, ids.cuda(), ww.cuda())
            with pytest.raises(CxError, match=text):
                gpu.sync()
            assert torch.equal(got, want), text
        gpu.sync()
    finally:
        for m in mats:
            m.free()


def test_q4_run_together_as_served(gpu):
    """norm -> 8 bits -> sort -> gathered products -> sum, and the layer call on the same
    routes: two ways through the operators that agree up to the 8-bit rounding of x;
    and moe_dispatch on a local node that holds the layer."""
    from constellation_amd import moe_dispatch as D
    from constellation_amd.engine import Q4Layer, Q4Matrix
    print("[q4] together", flush=True)
    T, K, E, H, I = 21, 4, 16, 512, 256
    gu, dn = make(1, E, 2 * I, H, 32), make(2, E, H, I, 64)
    mats = [Q4Matrix.pack(gu[0].cuda(), gu[1].cuda(), H, group=32, gated=True), Q4Matrix.pack(dn[0].cuda(), dn[1].cuda(), I, group=64)]
    try:
        layer = Q4Layer(gpu, *mats)
        x, r = rand(3, T, H, dtype=BF).cuda(), rand(4, T, H, dtype=BF).cuda()
        nw = (1 + rand(5, H, std=0.1)).to(BF).cuda()
        wr, bias = rand(6, E, H, dtype=BF, std=0.02).cuda(), rand(7, E, std=0.01).cuda()
        opt = dict(n_group=4, topk_group=2, top_k=K, norm_topk_prob=True, routed_scaling_factor=2.5)
        n = gpu.rms_norm(x, nw, residual=r, quantize=True)
        ids, w = gpu.route(n.y, wr, bias, **opt)
        order, offsets, place = gpu.sort_tokens(ids, E)
        h = gpu.q4_matmul(mats[0], n.q, x_scale=n.scale, offsets=offsets, order=order, top_k=K)
        ys = gpu.q4_matmul(mats[1], h, offsets=offsets, out_dtype=SF)
        y8 = gpu.combine_rows(ys, place, w, add=n.sum.float(), out_dtype=SF).double() - n.sum.double()
        y, yf, ids2, w2 = gpu.moe_layer(layer, n.y, wr, bias, want_f32=True, **opt)
        assert torch.equal(ids, ids2) and torch.equal(w, w2)
        rel = float((y8 - yf.double()).norm() / yf.double().norm())
        assert rel < 0.1, rel  # x in e4m3: each value within 2^-4
        # the same rows in 16 bits: h is rounded to bf16 here, kept finer in the layer call
        h = gpu.q4_matmul(mats[0], gpu.gather_rows(n.y, place), offsets=offsets)
        y16 = gpu.combine_rows(gpu.q4_matmul(mats[1], h, offsets=offsets, out_dtype=SF), place, w).double()
        rel = float((y16 - yf.double()).norm() / yf.double().norm())
        assert rel < 2.0 ** -7, rel
        with gpu.__class__(0) as other:  # another context, another stream
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                z = other.moe(layer, n.y, ids, w)
            side.synchronize()
            assert torch.equal(z, y)
        out, stream, ids3, w3 = D.run_moe_block([D.LocalNode({0: layer})], x, r, 0, nw, wr, bias, shared=False, **opt)
        torch.cuda.synchronize()
        assert torch.equal(out, y) and torch.equal(stream, n.sum) and torch.equal(ids3, ids) and torch.equal(w3, w)
        one = D.run_moe_block([D.LocalNode({0: layer})], x[3], None, 0, nw, wr, bias, shared=False, **opt)
        assert one[0].shape == (H,) and torch.equal(one[1], x[3])
    finally:
        torch.cuda.synchronize()
        for m in mats:
            m.free()


def test_q4_layer_graphs(gpu):
    """Two captured layer calls of different sizes, replayed in turn with eager calls between: each keeps its own scratch."""
    from constellation_amd.engine import Q4Layer, Q4Matrix
    print("[q4] graphs", flush=True)
    K, E, H, I = 4, 16, 512, 256
    gu, dn = make(1, E, 2 * I, H, 128), make(2, E, H, I, 128)
    mats = [Q4Matrix.pack(gu[0].cuda(), gu[1].cuda(), H, gated=True), Q4Matrix.pack(dn[0].cuda(), dn[1].cuda(), I)]
    try:
        layer = Q4Layer(gpu, *mats)
        g = torch.Generator().manual_seed(1)

        def inputs(T, i):
            return (rand(i, T, H, dtype=BF).cuda(), torch.rand(T, E, generator=g).topk(K, dim=1).indices.to(torch.int32).cuda(),
                    torch.rand(T, K, generator=g).cuda())

        side, graphs = torch.cuda.Stream(), {}
        for T in (1, 150):
            held = inputs(T, T)
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                gpu.moe(layer, *held)
            torch.cuda.synchronize()
            cg = torch.cuda.CUDAGraph()
            with torch.cuda.graph(cg, stream=side, capture_error_mode="thread_local"):
                out = gpu.moe(layer, *held)
            graphs[T] = (cg, held, out)
        for i in range(3):
            for T, (cg, held, out) in graphs.items():
                new = inputs(T, 10 * i + T)
                for h, t in zip(held, new):
                    h.copy_(t)
                torch.cuda.synchronize()
                cg.replay()
                want = gpu.moe(layer, *new)
                torch.cuda.synchronize()
                assert torch.equal(out, want), (i, T)
        graphs.clear()
    finally:
        torch.cuda.synchronize()
        for m in mats:
            m.free()


def test_refusals(gpu):
    """Each bad argument is refused with a message, before any launch."""
    import ctypes as C
    from constellation_amd._lib import BF16, CX_EINVAL, CX_OK, E4M3, F32, Q4Desc, lib
    from constellation_amd.engine import Q4Layer, Q4Matrix
    print("[q4] refusals", flush=True)
    codes, scales = make(1, 2, 32, 64, 32)
    w = Q4Matrix.pack(codes.cuda(), scales.cuda(), 64, group=32, gated=True)
    L, s = lib(), gpu.stream()
    try:
        x = rand(1, 4, 64, dtype=BF).cuda()
        y = torch.empty(4, 16, dtype=BF, device="cuda")
        i32 = torch.zeros(64, dtype=torch.int32, device="cuda")
        buf = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")

        def refused(rc, text):
            assert rc == CX_EINVAL and text.encode() in L.cx_last_error(), (rc, text, L.cx_last_error())

        def norm(ctx=gpu.handle, dt=BF16, T=4, H=64, eps=1e-6, xp=x.data_ptr(), yp=y.data_ptr(), q=None, sc=None, ydt=BF16):
            return L.cx_rms_norm(ctx, xp, dt, None, None, BF16, T, H, eps, None, yp, ydt, q, sc, s)

        refused(norm(ctx=None), "NULL context")
        refused(norm(dt=E4M3), "dtypes must be")
        refused(norm(ydt=9), "dtypes must be")
        refused(norm(T=-1), "bad n_tokens")
        refused(norm(H=0), "must not be empty")
        refused(norm(H=65537), "hidden must be 1..65536")
        refused(norm(eps=-1.0), "eps must be")
        refused(norm(eps=float("nan")), "eps must be")
        refused(norm(xp=None), "NULL buffer")
        refused(norm(yp=None), "NULL buffer")
        refused(norm(yp=None, q=buf.data_ptr()), "NULL buffer")
        refused(norm(T=1 << 30, H=8), "too many rows")

        def sort(ctx=gpu.handle, T=4, K=2, E=8, ids=i32.data_ptr(), off=i32.data_ptr()):
            return L.cx_sort_tokens(ctx, ids, T, K, E, buf.data_ptr(), off, buf.data_ptr(), s)

        refused(sort(ctx=None), "NULL context")
        refused(sort(K=0), "bad n_tokens/top_k")
        refused(sort(K=65), "bad n_tokens/top_k")
        refused(sort(E=0), "n_experts must be 1..1024")
        refused(sort(E=1025), "n_experts must be 1..1024")
        refused(sort(T=1 << 30, K=4), "too many pairs")
        refused(sort(ids=None), "NULL buffer")
        refused(sort(off=None), "NULL buffer")
        refused(L.cx_gather_rows(gpu.handle, x.data_ptr(), 0, i32.data_ptr(), 4, 1, buf.data_ptr(), s), "must not be empty")
        refused(L.cx_gather_rows(gpu.handle, x.data_ptr(), 128, None, 4, 1, buf.data_ptr(), s), "NULL buffer")
        refused(L.cx_gather_rows(gpu.handle, x.data_ptr(), 1 << 30, i32.data_ptr(), 1 << 20, 1, buf.data_ptr(), s), "too many rows")
        refused(L.cx_combine_rows(gpu.handle, x.data_ptr(), E4M3, i32.data_ptr(), None, None, 4, 1, 64, y.data_ptr(), BF16, None, s),
                "dtypes must be")
        refused(L.cx_combine_rows(gpu.handle, x.data_ptr(), BF16, i32.data_ptr(), None, None, 4, 1, 64, None, BF16, None, s), "NULL buffer")
        refused(L.cx_combine_rows_grad(gpu.handle, x.data_ptr(), BF16, x.data_ptr(), BF16, i32.data_ptr(), None, 4, 1, 64, None, None, s),
                "NULL buffer")

        d = Q4Desc()

        def pack(E=1, N=32, K=64, g=32, gated=0, c=codes.cuda().data_ptr(), dev=0):
            return L.cx_q4_pack(dev, c, buf.data_ptr(), E, N, K, g, gated, s, C.byref(d))

        refused(pack(dev=99), "invalid device")
        refused(pack(g=16), "group must be")
        refused(pack(E=0), "bad 4-bit shape")
        refused(pack(E=1025), "bad 4-bit shape")
        refused(pack(N=1 << 25), "bad 4-bit shape")
        refused(pack(N=31, gated=1), "even number of rows")
        refused(pack(c=None), "NULL buffer")
        need = L.cx_q4_scratch(C.byref(w.desc), BF16, 4, 4, 1)

        def mm(desc=w.desc, dt=BF16, xs=None, n_x=4, off=i32.data_ptr(), order=None, P=4, odt=BF16, scr=buf.data_ptr(), sz=need, K=1):
            return L.cx_q4_matmul(gpu.handle, C.byref(desc) if desc is not None else None, x.data_ptr(), dt, xs, n_x, order, K, off, P,
                                  y.data_ptr(), odt, scr, sz, s)

        refused(mm(desc=None), "descriptor")
        refused(mm(desc=Q4Desc()), "descriptor")
        refused(mm(dt=F32), "x must be")
        refused(mm(dt=E4M3), "NULL buffer")
        refused(mm(odt=E4M3), "y must be")
        refused(mm(P=-1), "bad n_rows")
        refused(mm(n_x=3), "same rows")
        refused(mm(n_x=0, order=i32.data_ptr()), "x has no rows")
        refused(mm(off=None), "needs offsets")
        refused(mm(sz=need - 1), "scratch must be")
        refused(mm(scr=buf.data_ptr() + 4), "scratch must be")
        refused(mm(order=i32.data_ptr(), K=0), "top_k")

        def moe(g=w.desc, dn=w.desc, sg=None, T=4, K=2, sz=1 << 20):
            return L.cx_q4_moe(gpu.handle, C.byref(g), C.byref(dn), sg, None, x.data_ptr(), BF16, T, i32.data_ptr(), buf.data_ptr(), K,
                               y.data_ptr(), BF16, None, buf.data_ptr(), sz, s)

        refused(moe(), "must be gated")
        refused(moe(sg=C.byref(w.desc)), "both of its matrices")
        with pytest.raises(ValueError, match="gated"):
            Q4Layer(gpu, w, w)
        with pytest.raises(ValueError, match="columns"):
            gpu.q4_matmul(w, x[:, :32])
        with pytest.raises(ValueError, match="x_scale"):
            gpu.q4_matmul(w, x, x_scale=torch.ones(4, 1, device="cuda"))
        with pytest.raises(ValueError, match="offsets"):
            gpu.q4_matmul(w, x, offsets=i32[:2])
        with pytest.raises(ValueError, match="do not hold"):
            Q4Matrix.pack(codes.cuda(), scales.cuda(), 66, group=32)
        with pytest.raises(TypeError, match="uint8"):
            Q4Matrix.pack(codes.cuda().int(), scales.cuda(), 64, group=32)
        with pytest.raises(ValueError, match="context on cuda"):
            gpu.rms_norm(x.cpu())
        with pytest.raises(ValueError, match="residual"):
            gpu.rms_norm(x, residual=x[:2])
        with pytest.raises(TypeError, match="fp8"):
            gpu.moe_layer_request(w, b"")
        with pytest.raises(ValueError, match="nothing to compute"):
            gpu.rms_norm(x, want_y=False)
        with pytest.raises(ValueError, match="place"):
            gpu.gather_rows(x, i32[:8].view(2, 4))
        with pytest.raises(ValueError, match="sorted rows"):
            gpu.combine_rows(x, i32[:4].view(2, 2)[:1])
        assert norm() == CX_OK  # the context still serves
        torch.cuda.synchronize()
    finally:
        w.free()


def test_q4_two_streams_and_ragged_stacks(gpu):
    """Two products of one context on two streams at once, each with its own scratch; and a
    stack through each kernel with row counts about its item sizes."""
    from constellation_amd.engine import Q4Matrix
    print("[q4] two streams", flush=True)
    K, N, E = 320, 80, 3
    codes, scales = make(5, E, N, K, 64)
    w = Q4Matrix.pack(codes.cuda(), scales.cuda(), K, group=64)
    W = dense(codes, scales, K, 64)
    try:
        for cuts in ((0, 1, 1, 2), (0, 16, 33, 34), (0, 17, 20, 48), (0, 129, 129, 130), (0, 256, 400, 401), (0, 113, 210, 467)):
            off = torch.tensor(cuts, dtype=torch.int32)
            P = cuts[-1]
            x = rand(P, P, K, dtype=BF)
            want = torch.cat([x[a:b].double() @ W[e].T for e, (a, b) in enumerate(zip(cuts, cuts[1:]))])
            tol = torch.cat([x[a:b].double().abs() @ W[e].abs().T for e, (a, b) in enumerate(zip(cuts, cuts[1:]))]) * (K + 8) * U
            xs = [x.cuda(), (2 * x).cuda()]  # exact: a power of two
            offs, out = off.cuda(), [None, None]
            torch.cuda.synchronize()
            streams = [torch.cuda.Stream(), torch.cuda.Stream()]
            for _ in range(3):
                for i, s in enumerate(streams):
                    with torch.cuda.stream(s):
                        out[i] = gpu.q4_matmul(w, xs[i], offsets=offs)
            torch.cuda.synchronize()
            for i in (0, 1):
                near(out[i], (i + 1) * want, rounded((i + 1) * want, (i + 1) * tol, BF), cuts)
    finally:
        w.free()


def test_q4_layer_against_single_expert_calls(gpu):
    """A layer of 70 tokens with every token on the same experts equals the products called one after another
    in fp32, and one token alone (its own kernels) equals its row up to the roundings of h."""
    from constellation_amd.engine import Q4Layer, Q4Matrix
    print("[q4] layer against products", flush=True)
    E, H, I, T = 4, 384, 256, 70
    gu, dn = make(1, E, 2 * I, H, 32), make(2, E, H, I, 128)
    mats = [Q4Matrix.pack(gu[0].cuda(), gu[1].cuda(), H, group=32, gated=True), Q4Matrix.pack(dn[0].cuda(), dn[1].cuda(), I)]
    try:
        layer = Q4Layer(gpu, *mats)
        x, w = rand(3, T, H, dtype=BF), torch.rand(T, 2, generator=torch.Generator().manual_seed(4))
        ids = torch.tensor([[2, 0]] * T, dtype=torch.int32)
        _, yf = gpu.moe(layer, x.cuda(), ids.cuda(), w.cuda(), want_f32=True)
        want, tol = layer_ref(x.double(), ids, w, dense(gu[0], gu[1], H, 32), dense(dn[0], dn[1], I, 128), H_HALF)
        near(yf, want, tol, "layer")
        for t in (0, 33):
            _, one = gpu.moe(layer, x[t:t + 1].cuda(), ids[t:t + 1].cuda(), w[t:t + 1].cuda(), want_f32=True)
            near(one, want[t:t + 1], tol[t:t + 1], t)
    finally:
        for m in mats:
            m.free()


def test_q4_layer_of_the_shared_expert_alone(gpu):
    """Tokens without routes (top_k 0) through a layer of 600 experts: the shared one takes them all."""
    from constellation_amd.engine import Q4Layer, Q4Matrix
    print("[q4] shared expert alone", flush=True)
    E, H, I = 600, 40, 24
    stacks = [make(i, n, *s, 32) for i, (n, s) in enumerate(((E, (2 * I, H)), (E, (H, I)), (1, (2 * I, H)), (1, (H, I))))]
    mats = [Q4Matrix.pack(c.cuda(), s.cuda(), k, group=32, gated=gt) for (c, s), k, gt in zip(stacks, (H, I, H, I), (True, False) * 2)]
    try:
        layer = Q4Layer(gpu, mats[0], mats[1], (mats[2], mats[3]))
        D = [dense(c, s, k, 32) for (c, s), k in zip(stacks, (H, I, H, I))]
        for T in (1, 2, 150):
            x, ids, w = rand(T, T, H, dtype=BF), torch.empty(T, 0, dtype=torch.int32), torch.empty(T, 0)
            _, yf = gpu.moe(layer, x.cuda(), ids.cuda(), w.cuda(), want_f32=True)
            gpu.sync()
            want, tol = layer_ref(x.double(), ids, w, D[0], D[1], H_HALF, (D[2], D[3]))
            near(yf, want, tol, T)
    finally:
        for m in mats:
            m.free()


@pytest.mark.parametrize("E,shared", [(5, True), (200, False), (1024, True)])
def test_q4_layer_skewed_routes(gpu, E, shared):
    """Experts of no, one and hundreds of rows in one call: items of every length, from one and from
    several workgroups of the sort, and of two experts a thread."""
    from constellation_amd.engine import Q4Layer, Q4Matrix
    print(f"[q4] skewed over {E} shared {shared}", flush=True)
    H, I, T, K = 72, 32, 700, 3
    stacks = [make(i + E, n, *s, 32) for i, (n, s) in enumerate(((E, (2 * I, H)), (E, (H, I)), (1, (2 * I, H)), (1, (H, I))))]
    mats = [Q4Matrix.pack(c.cuda(), s.cuda(), k, group=32, gated=gt) for (c, s), k, gt in zip(stacks, (H, I, H, I), (True, False) * 2)]
    try:
        layer = Q4Layer(gpu, mats[0], mats[1], (mats[2], mats[3]) if shared else None)
        g = torch.Generator().manual_seed(E)
        lean = torch.randn(E, generator=g) * 2
        ids = (torch.randn(T, E, generator=g) + lean).topk(K, dim=1).indices.to(torch.int32)
        x, w = rand(1, T, H, dtype=BF), torch.rand(T, K, generator=g)
        _, yf = gpu.moe(layer, x.cuda(), ids.cuda(), w.cuda(), want_f32=True)
        gpu.sync()
        D = [dense(c, s, k, 32) for (c, s), k in zip(stacks, (H, I, H, I))]
        want, tol = layer_ref(x.double(), ids, w, D[0], D[1], H_HALF, (D[2], D[3]) if shared else None)
        near(yf, want, tol, E)
        # the same rows as a stack's: some matrices without rows, rows behind the last one
        order, offsets, _ = gpu.sort_tokens(ids.cuda(), E)
        for gap in (0, 37):
            off = offsets.cpu().clamp(max=T * K - gap)
            got = gpu.q4_matmul(mats[1], x.cuda()[:, :I].contiguous(), offsets=off.cuda(), order=order, top_k=K, out_dtype=SF).cpu().double()
            gpu.sync()
            e_of = torch.searchsorted(off[1:].long(), torch.arange(T * K), right=True)
            src = x.double()[(order.cpu() // K).long(), :I]
            rows = torch.stack([D[1][min(int(e), E - 1)] @ v if e < E else torch.zeros(H, dtype=torch.float64) for e, v in zip(e_of, src)])
            size = torch.stack([D[1][min(int(e), E - 1)].abs() @ v.abs() for e, v in zip(e_of, src)])
            near(got, rows, size * (I + 8) * U + TINY[SF], (E, gap))
    finally:
        for m in mats:
            m.free()


@pytest.mark.parametrize("dtype", [BF, HF, F8])
@pytest.mark.parametrize("E,N,K,group,counts", [(1, 70, 1023, 64, (1, 4, 5, 16, 17)), (1, 70, 1025, 64, (4, 5, 16, 17)), (1, 70, 1032, 64, (1, 16, 17, 65)),
                                                (1, 4200, 256, 32, (1, 3, 16)), (1, 600, 1024, 64, (129, 1740, 1760)), (5, 48, 136, 32, (5, 6, 80, 81)), (5, 2048, 2048, 128, (5, 6, 81))])
def test_q4_matmul_on_both_sides_of_its_rules(gpu, E, N, K, group, counts, dtype):
    """Each kernel at the sizes where another takes over, eager and from a graph replayed between eager calls."""
    from constellation_amd.engine import Q4Matrix
    print(f"[q4] rules {E}x{N}x{K} {dtype}", flush=True)
    codes, scales = make(E + K, E, N, K, group)
    w = Q4Matrix.pack(codes.cuda(), scales.cuda(), K, group=group)
    W = dense(codes, scales, K, group)
    try:
        for P in counts:
            x, xs, x64 = make_x(P, P, K, dtype)
            off = torch.tensor([0] + sorted(torch.randint(0, P + 1, (E - 1,), generator=torch.Generator().manual_seed(P)).tolist()) + [P], dtype=torch.int32)
            want = torch.cat([x64[a:b] @ W[e].T for e, (a, b) in enumerate(zip(off[:-1].tolist(), off[1:].tolist()))])
            size = torch.cat([x64[a:b].abs() @ W[e].abs().T for e, (a, b) in enumerate(zip(off[:-1].tolist(), off[1:].tolist()))])
            xd, sd, offd = x.cuda(), None if xs is None else xs.cuda(), off.cuda() if E > 1 else None

            def call():
                return gpu.q4_matmul(w, xd, x_scale=sd, offsets=offd, out_dtype=SF)
            eager = call()
            near(eager, want, size * (K + 8) * U + TINY[SF], P)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                y = call()
            for _ in range(3):
                y.zero_()
                graph.replay()
                again = call()
                torch.cuda.synchronize()
                assert torch.equal(y, eager) and torch.equal(again, eager), P
        gpu.sync()
    finally:
        w.free()


def test_q4_matmul_after_free(gpu):
    """A freed matrix, and a layer that holds one, are refused."""
    from constellation_amd.engine import Q4Layer, Q4Matrix
    H, I, E = 64, 32, 2
    gu, dn = make(1, E, 2 * I, H, 32), make(2, E, H, I, 32)
    g = Q4Matrix.pack(gu[0].cuda(), gu[1].cuda(), H, group=32, gated=True)
    d = Q4Matrix.pack(dn[0].cuda(), dn[1].cuda(), I, group=32)
    layer = Q4Layer(gpu, g, d)
    x = rand(1, 3, H, dtype=BF).cuda()
    g.free()
    g.free()  # once more does nothing
    with pytest.raises(ValueError, match="freed"):
        gpu.q4_matmul(g, x, offsets=torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="freed"):
        gpu.moe(layer, x, torch.zeros(3, 1, dtype=torch.int32, device="cuda"), torch.ones(3, 1, device="cuda"))
    d.free()
