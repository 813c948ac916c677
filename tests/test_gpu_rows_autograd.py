"""The sorted rows in a training step: a router's and the experts' gradients through
autograd.Functions around gather_rows, combine_rows and combine_rows_grad, against the
formulas in 64 bits."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


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


@pytest.mark.parametrize("T,K,H", [(1, 1, 8), (37, 3, 130), (500, 4, 64)])
def test_gradients_through_functions(gpu, T, K, H):
    print(f"[rows] functions {T}x{K} of {H}", flush=True)
    g = torch.Generator().manual_seed(T)
    E = 9
    x, w, dout = (torch.randn(*s, generator=g) for s in ((T, H), (T, K), (T, H)))
    scale = torch.rand(E, generator=g) + 0.5  # the experts: a factor each
    ids = torch.rand(T, E, generator=g).topk(K, dim=1).indices.to(torch.int32)
    ids[torch.rand(T, K, generator=g) < 0.2] = -1
    order, offsets, place = gpu.sort_tokens(ids.cuda(), E)
    xd, wd = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    rows = torch.arange(T * K, device="cuda")
    factor = scale.cuda()[torch.searchsorted(offsets[1:].long(), rows, right=True).clamp(max=E - 1)][:, None]
    out = Combine.apply(gpu, Gather.apply(gpu, xd, place) * factor, place, wd)
    out.backward(dout.cuda())
    torch.cuda.synchronize()
    held = (ids >= 0).double()
    f = scale.double()[ids.clamp(min=0).long()] * held
    dot = (dout.double() * x.double()).sum(1, keepdim=True)
    size = (dout.double() * x.double()).abs().sum(1, keepdim=True)
    want = [((w.double() * f).sum(1, keepdim=True) * x.double(), (w.double() * f).abs().sum(1, keepdim=True) * x.double().abs()),
            ((w.double() * f).sum(1, keepdim=True) * dout.double(), (w.double() * f).abs().sum(1, keepdim=True) * dout.double().abs()),
            (f * dot, f * size)]
    for got, (ref, big), n in zip((out.detach(), xd.grad, wd.grad), want, (K, K, H)):
        assert bool(((got.cpu().double() - ref).abs() <= (n + 6) * U * big + 2.0 ** -140).all())
