"""The products of a program's own experts record no graph: tensors that require grad are refused where one is being
recorded, rather than answered with a result that has none.  No GPU: a context of "device -1", where CPU tensors are at home,
and a library that says that it was called."""
from __future__ import annotations

import pytest
import torch

from constellation_amd.engine import I8Layer
from test_q4_layer_checks import Called, ctx  # noqa: F401  (ctx is a fixture)

T, K, N, E = 4, 16, 8, 3


def z(*s, dtype=torch.bfloat16):
    return torch.zeros(*s, dtype=dtype)


def quantize(c):
    t = {"x": z(T, K)}
    return t, lambda: c.quantize_i8(t["x"])


def i8(c):
    t = {"x_scale": torch.ones(T), "w_scale": torch.ones(N)}
    return t, lambda: c.i8_matmul(z(T, K, dtype=torch.int8), t["x_scale"], z(N, K, dtype=torch.int8), t["w_scale"])


def refuses(call, t, which):
    with pytest.raises(Called):  # reaches the library
        call()
    t[which].requires_grad_()
    with pytest.raises(ValueError, match="records no graph"):
        call()
    with torch.no_grad(), pytest.raises(Called):
        call()

    class Own(torch.autograd.Function):  # whose forward records nothing
        @staticmethod
        def forward(fn, _):
            with pytest.raises(Called):
                call()
            return torch.zeros(())
    Own.apply(t[which])


@pytest.mark.parametrize("make,which", [(quantize, "x"), (i8, "x_scale"), (i8, "w_scale")])
def test_a_graph_is_not_lost_in_8_bits(ctx, make, which):  # noqa: F811
    t, call = make(ctx)
    refuses(call, t, which)


def test_a_layer_takes_trained_weights(ctx):  # noqa: F811
    """Served weights are a program's parameters: the layer's codes are theirs at that moment, and no step of a graph."""
    with pytest.raises(Called, match="cx_quantize_i8"):
        I8Layer.quantize(ctx, z(E, 2 * N, K).requires_grad_(), z(E, K, N).requires_grad_())


@pytest.mark.parametrize("which", ["dy", "x", "w", "pre"])
def test_no_second_gradient_is_lost(ctx, which):  # noqa: F811
    """In a backward that is itself recorded (create_graph) or outside of one."""
    t = {"dy": z(T, N // 2), "x": z(T, K), "w": z(N, K), "pre": z(T, N)}
    refuses(lambda: ctx.matmul_grad(t["dy"], t["x"], t["w"], pre=t["pre"]), t, which)


@pytest.mark.parametrize("make,which", [(quantize, "x"), (i8, "x_scale"), (i8, "w_scale"),
                                        (lambda c: (t := {"x": z(T, K), "w": z(N, K)}, lambda: c.matmul(t["x"], t["w"])), "x"),
                                        (lambda c: (t := {"x": z(T, K), "w": z(N, K)}, lambda: c.matmul(t["x"], t["w"])), "w"),
                                        (lambda c: (t := {"dy": z(T, N), "x": z(T, K)}, lambda: c.matmul_grad(t["dy"], t["x"], z(N, K))), "dy"),
                                        (lambda c: (t := {"x": z(T, K)}, lambda: c.gather_rows(t["x"], torch.arange(T, dtype=torch.int32).view(T, 1))), "x")])
def test_no_tangent_is_lost(ctx, make, which):  # noqa: F811
    """Forward mode: a tensor with a tangent, at any mode of the backward one."""
    fwd = torch.autograd.forward_ad
    t, call = make(ctx)
    plain = t[which]
    with fwd.dual_level():
        with pytest.raises(Called):  # a level alone is no tangent
            call()
        t[which] = fwd.make_dual(plain, torch.ones_like(plain))
        with pytest.raises(ValueError, match="records no graph"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="records no graph"):
            call()

        class Own(torch.autograd.Function):  # whose jvp has the tangents
            @staticmethod
            def forward(fn, v):
                t[which] = v
                with pytest.raises(Called):
                    call()
                return v.clone()

            @staticmethod
            def jvp(fn, dv):
                return dv.clone()
        Own.apply(t[which])
    t[which] = plain
    with pytest.raises(Called):
        call()
