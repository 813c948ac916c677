"""A program's own experts as they are used: a training step through sorted rows, the gated block, the product after it and their
gradients as autograd.Functions; then the same experts in 8-bit integers as a layer, through Context.moe, moe_layer and the
server-side dispatch.  Against the formulas in 64 bits."""
from __future__ import annotations

import pytest
import torch

from test_gpu_matmul import gate_grad_ref, i8_ref, rounded
from test_gpu_q4 import BF, HALF, HF, SF, TINY, U, near, product_ref, rand

pytestmark = pytest.mark.gpu


class Gather(torch.autograd.Function):
    @staticmethod
    def forward(fn, ctx, x, place):
        fn.engine = ctx
        fn.save_for_backward(place)
        return ctx.gather_rows(x, place)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(fn, dxs):
        return None, fn.engine.combine_rows(dxs, fn.saved_tensors[0]), None


class Block(torch.autograd.Function):
    @staticmethod
    def forward(fn, ctx, x, w, offsets):
        h, pre = ctx.matmul(x, w, gated=True, keep=True, offsets=offsets)
        fn.engine = ctx
        fn.save_for_backward(x, w, pre, offsets)
        return h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(fn, dh):
        x, w, pre, offsets = fn.saved_tensors
        return None, *fn.engine.matmul_grad(dh, x, w, pre=pre, offsets=offsets), None


class Product(torch.autograd.Function):
    @staticmethod
    def forward(fn, ctx, x, w, offsets):
        fn.engine = ctx
        fn.save_for_backward(x, w, offsets)
        return ctx.matmul(x, w, offsets=offsets)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(fn, dy):
        x, w, offsets = fn.saved_tensors
        return None, *fn.engine.matmul_grad(dy, x, w, offsets=offsets), None


class Combine(torch.autograd.Function):
    @staticmethod
    def forward(fn, ctx, ys, place, weights):
        fn.engine = ctx
        fn.save_for_backward(ys, place, weights)
        return ctx.combine_rows(ys, place, weights)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(fn, dout):
        dys, dw = fn.engine.combine_rows_grad(dout, *fn.saved_tensors)
        return None, dys, None, dw


def routes(seed, T, E, K, drop=0.2):
    g = torch.Generator().manual_seed(seed)
    ids = torch.rand(T, E, generator=g).topk(K, dim=1).indices.to(torch.int32)
    ids[torch.rand(T, K, generator=g) < drop] = -1
    return ids, torch.rand(T, K, generator=g) + 0.1


class Bound:
    """A value in 64 bits and how far what stands for it may be off; each operation adds its own."""

    def __init__(self, v, e=None):
        self.v, self.e = v, torch.zeros_like(v) if e is None else e

    def product(self, other):
        n = self.v.shape[-1]
        a, b = self.v.abs() + self.e, other.v.abs() + other.e
        return Bound(self.v @ other.v.T, a @ other.e.T + self.e @ b.T + (a @ b.T) * (n + 8) * U)

    def rows(self, at):
        return Bound(self.v[at], self.e[at])

    def T(self):
        return Bound(self.v.T, self.e.T)

    def to(self, dtype):
        return Bound(self.v, rounded(self.v, self.e, dtype))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T,K,E,H,I", [(1, 1, 1, 24, 8), (37, 3, 9, 130, 34), (300, 2, 6, 64, 40), (500, 4, 5, 264, 144)])
def test_a_training_step(gpu, T, K, E, H, I, dtype):
    """Forward and gradients of every leaf.  The bound follows each rounding through the step; what the gradient at pre
    takes from pre's own rounding goes by its slope, |d dpre / d pre| <= 0.5 |dh| (|u| + 1) + 1.1 |dh| for each of both."""
    print(f"[own] step {T}x{K} over {E} {H} {I} {dtype}", flush=True)
    ids, wts = routes(T, T, E, K)
    x, gu, dn, dout = rand(1, T, H, dtype=dtype), rand(2, E, 2 * I, H, dtype=dtype, std=0.1), rand(3, E, H, I, dtype=dtype, std=0.1), rand(4, T, H, dtype=dtype)
    order, offsets, place = gpu.sort_tokens(ids.cuda(), E)
    leaves = [t.cuda().requires_grad_() for t in (x, gu, dn, wts)]
    out = Combine.apply(gpu, Product.apply(gpu, Block.apply(gpu, Gather.apply(gpu, leaves[0], place), leaves[1], offsets), leaves[2], offsets), place, leaves[3])
    out.backward(dout.cuda())
    torch.cuda.synchronize()
    gpu.sync()
    held, at = (ids >= 0), [(ids == e).nonzero() for e in range(E)]
    w = wts.double() * held
    y = [Bound(torch.zeros(T, H, dtype=torch.float64)) for _ in range(5)]
    sums, dx = y[0], y[1]
    dgu, ddn = Bound(torch.zeros(E, 2 * I, H, dtype=torch.float64)), Bound(torch.zeros(E, H, I, dtype=torch.float64))
    dw = Bound(torch.zeros(T, K, dtype=torch.float64))
    for e in range(E):
        t, k = at[e][:, 0], at[e][:, 1]
        if t.numel() == 0:
            continue
        xe, ge, de = Bound(x[t].double()), Bound(gu[e].double()), Bound(dn[e].double())
        pre = xe.product(ge)
        v, h_tol = product_ref(x[t].double(), gu[e].double(), True)
        h = Bound(v, h_tol).to(dtype)
        ys = h.product(de).to(dtype)
        f = w[t, k][:, None]
        sums.v.index_add_(0, t, f * ys.v)
        sums.e.index_add_(0, t, f * (ys.e + (ys.v.abs() + ys.e) * (K + 2) * U))
        d = dout[t].double()
        dys = Bound(f * d, (f * d).abs() * U).to(dtype)
        dw.v[t, k] = (d * ys.v).sum(1)
        dw.e[t, k] = (d.abs() * (ys.e + (ys.v.abs() + ys.e) * (H + 8) * U)).sum(1)
        dh = dys.product(de.T()).to(dtype)
        p = pre.to(dtype)
        at64, calc = gate_grad_ref(dh.v, p.v)
        g, u = p.v.chunk(2, 1)
        eg, eu = p.e.chunk(2, 1)
        size = dh.v.abs() + dh.e
        slope = size * ((0.5 * (u.abs() + eu) + 1.1) * eg + 1.1 * eu)
        dpre = Bound(at64, 2 * calc + torch.cat((slope + 1.1 * dh.e * (u.abs() + eu), slope + dh.e * (g.abs() + eg)), 1)).to(dtype)
        dxs = dpre.product(ge.T()).to(dtype)
        dx.v.index_add_(0, t, dxs.v)
        dx.e.index_add_(0, t, dxs.e + (dxs.v.abs() + dxs.e) * (K + 2) * U)
        for into, a, b in ((dgu, dpre, xe), (ddn, dys, h)):
            r = a.T().product(b.T())
            into.v[e], into.e[e] = r.v, r.e
    for got, ref, out_type, what in ((out.detach(), sums, dtype, "out"), (leaves[0].grad, dx, dtype, "dx"), (leaves[1].grad, dgu, dtype, "dgate_up"),
                                     (leaves[2].grad, ddn, dtype, "ddown"), (leaves[3].grad, dw, SF, "dweights")):
        near(got, ref.v, rounded(ref.v, ref.e, out_type), what)


def layer_ref(x, ids, wts, gu, gs, dn, ds, shared, dtype):
    """(y, how far it may be off) of a layer of 8-bit experts: rows of x become codes exactly as the formula says; of h, a
    code may be one off where its quotient lies within h's own error of a border."""
    T, K = ids.shape
    E, H, I = dn.shape
    xs = (x.float().abs().amax(1) / torch.tensor(127.0)).clamp_min(1e-12)
    q = torch.round(x.float() / xs[:, None])
    y, tol = torch.zeros(T, H, dtype=torch.float64), torch.zeros(T, H, dtype=torch.float64)
    for e in range(E):
        if shared and e == E - 1:
            t, f = torch.arange(T), torch.ones(T, 1, dtype=torch.float64)
        else:
            t, k = (ids == e).nonzero(as_tuple=True)
            f = wts[t, k].double()[:, None]
        if t.numel() == 0:
            continue
        h, eh = i8_ref(q[t], xs[t], gu[e], gs[e], True)
        hs = (h.abs().amax(1) / 127).clamp_min(1e-12)
        r = h / hs[:, None]
        off = eh / hs[:, None] + r.abs() * (eh.amax(1) / h.abs().amax(1).clamp_min(1e-300) + 4 * U)[:, None]  # of the quotient, with the scale's own
        code = torch.round(r)
        border = ((r - torch.floor(r) - 0.5).abs() <= off).double()
        rel = (eh.amax(1) / h.abs().amax(1).clamp_min(1e-300) + 4 * U)[:, None]
        W = dn[e].double() * ds[e].double()[:, None]
        ys = (code @ W.T) * hs[:, None]
        ey = (border @ W.abs().T) * hs[:, None] + ys.abs() * (rel + 4 * U)
        y.index_add_(0, t, f * ys)
        tol.index_add_(0, t, f * ey + (f * ys).abs() * (K + 3) * U)
    return y, tol


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T,K,E,H,I,shared", [(1, 2, 4, 64, 32, True), (1, 1, 1, 30, 7, False), (37, 3, 9, 130, 34, False), (300, 2, 6, 256, 48, True),
                                              (64, 0, 2, 48, 16, True), (700, 4, 12, 96, 80, True)])
def test_a_layer_of_8_bit_experts(gpu, T, K, E, H, I, shared, dtype):
    from constellation_amd.engine import I8Layer
    print(f"[own] 8-bit layer {T}x{K} over {E} {H} {I} shared {shared} {dtype}", flush=True)
    routed = E - int(shared)
    ids, wts = routes(T, T, max(routed, K), K) if K else (torch.zeros(T, 0, dtype=torch.int32), torch.zeros(T, 0))
    ids = torch.where(ids >= routed, -1, ids)
    x, gu, dn = rand(1, T, H, dtype=dtype), rand(2, E, 2 * I, H, dtype=dtype, std=0.1), rand(3, E, H, I, dtype=dtype, std=0.1)
    layer = I8Layer.quantize(gpu, gu.cuda(), dn.cuda(), shared=shared)
    want, tol = layer_ref(x, ids, wts, layer.gate_up.cpu(), layer.gate_up_scale.cpu(), layer.down.cpu(), layer.down_scale.cpu(), shared, dtype)
    y, yf = gpu.moe(layer, x.cuda(), ids.cuda(), wts.cuda(), want_f32=True)
    torch.cuda.synchronize()
    near(yf, want, rounded(want, tol, SF), "y_f32")
    near(y, want, rounded(want, tol, dtype), "y")
    gpu.sync()
    # captured and replayed over other tokens
    buf, b_ids, b_w = x.cuda(), ids.cuda(), wts.cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = gpu.moe(layer, buf, b_ids, b_w)
    for seed in (5, 6):
        buf.copy_(rand(seed, T, H, dtype=dtype))
        eager = gpu.moe(layer, buf, b_ids, b_w)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, eager)


def test_routes_are_checked(gpu):
    """As a layer of 4-bit experts does: a repeated expert, a bad weight and an expert that is not there are left out and
    reported; the other routes count."""
    from constellation_amd._lib import CxError
    from constellation_amd.engine import I8Layer
    T, K, E, H, I = 5, 3, 4, 64, 32
    x = rand(1, T, H, dtype=BF).cuda()
    layer = I8Layer.quantize(gpu, rand(2, E, 2 * I, H, dtype=BF, std=0.1).cuda(), rand(3, E, H, I, dtype=BF, std=0.1).cuda())
    ids, w = torch.tensor([[0, 1, 2]] * T, dtype=torch.int32), torch.full((T, K), 0.5)
    good = gpu.moe(layer, x, torch.where(torch.arange(K) == 1, -1, ids).cuda(), w.cuda())
    for bad_id, bad_w in ((0, 0.5), (4, 0.5), (1, -1.0), (1, float("nan"))):
        i, v = ids.clone(), w.clone()
        i[:, 1], v[:, 1] = bad_id, bad_w
        y = gpu.moe(layer, x, i.cuda(), v.cuda())
        with pytest.raises(CxError):
            gpu.sync()
        assert torch.equal(y, good), (bad_id, bad_w)


def test_through_the_dispatch(gpu):
    """One node with all experts, two nodes with half of them each, and the block with residual and norm before it."""
    from constellation_amd.engine import I8Layer
    from constellation_amd.moe_dispatch import LocalNode, run_moe_block, run_topk_moe_layer
    T, E, K, H, I = 40, 8, 2, 128, 48
    x, gu, dn = rand(1, T, H, dtype=BF).cuda(), rand(2, E, 2 * I, H, dtype=BF, std=0.1).cuda(), rand(3, E, H, I, dtype=BF, std=0.1).cuda()
    whole = LocalNode({0: I8Layer.quantize(gpu, gu, dn)})
    ids, wts = routes(1, T, E, K, drop=0.0)
    one = run_topk_moe_layer([whole], x, 0, ids, wts, n_experts=E, shared=False)
    assert torch.equal(one, gpu.moe(whole.layers[0], x, ids.cuda(), wts.cuda()))
    halves = [LocalNode({0: I8Layer.quantize(gpu, gu[a:b], dn[a:b], experts=range(a, b), n_experts=E)}) for a, b in ((0, 4), (4, 8))]
    two = run_topk_moe_layer(halves, x, 0, ids, wts, n_experts=E, shared=False)
    # the same routes' values added in another order: sums of K values in fp32, then one rounding
    _, yf = gpu.moe(whole.layers[0], x, ids.cuda(), wts.cuda(), want_f32=True)
    big = sum(gpu.moe(whole.layers[0], x, ids[:, k:k + 1].cuda(), wts[:, k:k + 1].cuda(), want_f32=True)[1].double().abs() for k in range(K))
    assert bool(((two.double() - yf.double()).abs() <= big * (2 * K + 2) * U + (yf.double().abs() + big * 2 * K * U) * HALF[BF] + TINY[BF]).all())
    w_r, bias = rand(4, E, H, dtype=BF).cuda(), torch.zeros(E, device="cuda")
    y, stream, got_ids, got_w = run_moe_block([whole], x, x, 0, torch.ones(H, dtype=BF, device="cuda"), w_r, bias, n_group=2, topk_group=2, top_k=K,
                                              norm_topk_prob=True, routed_scaling_factor=1.0, shared=False)
    n = gpu.rms_norm(x, torch.ones(H, dtype=BF, device="cuda"), residual=x)
    assert torch.equal(stream, n.sum) and torch.equal(y, gpu.moe(whole.layers[0], n.y, got_ids, got_w))
    gpu.sync()
