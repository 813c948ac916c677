"""Arguments that the products of a program's own experts refuse, before anything touches a device.  No GPU: of the C ABI the
context is memory that none of these calls reads; of the Python side it is one of "device -1", where CPU tensors are at
home, and a library that says that it was called."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from constellation_amd._lib import BF16, CX_EINVAL, CX_OK, E4M3, F32, FP16, I8LayerDesc, lib
from constellation_amd.engine import I8Layer
from test_q4_layer_checks import Called, ctx  # noqa: F401  (ctx is a fixture)


@pytest.fixture(scope="module")
def at():
    """Host memory in the place of device buffers: 16-byte aligned, never read."""
    raw = C.create_string_buffer(1 << 16)
    yield (C.addressof(raw) + 255) // 256 * 256


def refused(rc, text):
    assert rc == CX_EINVAL and text.encode() in lib().cx_last_error(), (rc, text, lib().cx_last_error())


def matmul(at, **k):
    a = dict(ctx=at, x=at, n_x=4, w=at, dtype=BF16, n_mats=1, rows=64, cols=128, gated=0, order=None, top_k=1, offsets=None, n_rows=4, y=at, y_dtype=BF16,
             pre=None, scratch=at, size=1 << 40, stream=None)
    a.update(k)
    return lib().cx_matmul(*a.values())


def grad(at, **k):
    a = dict(ctx=at, dy=at, x=at, w=at, dtype=BF16, pre=None, n_mats=1, rows=64, cols=128, offsets=None, n_rows=4, dx=at, dw=at, dw_dtype=BF16, scratch=at,
             size=1 << 40, stream=None)
    a.update(k)
    return lib().cx_matmul_grad(*a.values())


def i8(at, **k):
    a = dict(ctx=at, x=at, x_scale=at, n_x=4, w=at, w_scale=at, n_mats=1, rows=64, cols=128, gated=0, order=None, top_k=1, offsets=None, n_rows=4, y=at,
             y_dtype=BF16, scratch=at, size=1 << 40, stream=None)
    a.update(k)
    return lib().cx_i8_matmul(*a.values())


SIZES = [(dict(n_mats=0), "n_mats must be"), (dict(n_mats=1025, offsets=1), "n_mats must be"), (dict(rows=0), "rows must be"), (dict(cols=-1), "rows must be"),
         (dict(rows=(1 << 22) + 1), "rows must be"), (dict(rows=1 << 22, cols=1 << 16), "2^32 bytes"), (dict(n_rows=-1, n_x=-1), "bad n_rows"),
         (dict(n_mats=2), "needs offsets"), (dict(n_rows=(1 << 30) + 1, n_x=(1 << 30) + 1), "too many rows"), (dict(ctx=None), "NULL context")]


@pytest.mark.parametrize("call", [matmul, grad, i8])
@pytest.mark.parametrize("change,text", SIZES)
def test_sizes(at, call, change, text):
    change = {k: at if k == "offsets" else v for k, v in change.items() if not (k == "n_x" and call is grad)}
    refused(call(at, **change), text)


@pytest.mark.parametrize("call", [matmul, i8])
def test_forward(at, call):
    refused(call(at, gated=1, rows=63), "even number")
    refused(call(at, n_x=5), "the same rows")
    refused(call(at, order=at, top_k=0), "bad n_x or top_k")
    refused(call(at, order=at, n_x=0), "x has no rows")
    refused(call(at, y_dtype=E4M3), "y must be")
    refused(call(at, y=None), "NULL buffer")
    refused(call(at, w=None), "NULL buffer")
    refused(call(at, x=at + 2), "start on 16 bytes")
    refused(call(at, w=at + 2), "start on 16 bytes")
    refused(call(at, order=at, n_x=1 << 30, cols=512), "2^32 bytes in all")
    assert call(at, n_rows=0, n_x=0, x=None, y=None, w=None) == CX_OK


def test_of_one_kind(at):
    refused(matmul(at, dtype=F32), "fp16 or bf16")
    refused(matmul(at, dtype=E4M3), "fp16 or bf16")
    refused(matmul(at, pre=at), "gated product only")
    refused(i8(at, x_scale=None), "NULL buffer")
    refused(i8(at, cols=131072), "cols 1..131071")
    refused(grad(at, dtype=F32), "fp16 or bf16")
    refused(grad(at, dw_dtype=FP16), "x's type or fp32")
    refused(grad(at, dx=None, dw=None), "nothing to compute")
    refused(grad(at, dy=None), "NULL buffer")
    refused(grad(at, pre=at, rows=63), "even number")
    refused(grad(at, dy=at + 8), "start on 16 bytes")
    refused(grad(at, pre=at, size=16), "scratch must be")
    assert grad(at, n_rows=0, dw=None, dx=None, x=None, dy=None) == CX_OK


def test_scratch(at):
    """What the size call asks for is asked of the caller, whole and aligned."""
    need = lib().cx_matmul_scratch(BF16, 256, 1, 4096, 7168, 256, 0)
    assert need > 0
    for bad in (dict(scratch=None), dict(size=need - 1), dict(scratch=at + 8)):
        refused(matmul(at, rows=4096, cols=7168, n_rows=256, n_x=256, **{**dict(size=need), **bad}), f"scratch must be {need} bytes")
    assert lib().cx_matmul_scratch(BF16, 1, 0, 1, 1, 1, 0) == 0 and lib().cx_matmul_scratch(BF16, 1, 1, 1, 1, 0, 0) == 0
    # rows of x and of the weights that are no whole pieces of 16 bytes: copies of both
    assert lib().cx_matmul_scratch(BF16, 4000, 1, 100, 9, 4000, 0) >= (4000 + 100) * 16 * 2


def test_quantize_refuses(at):
    q = lib().cx_quantize_i8
    refused(q(None, at, BF16, 1, 1, at, at, None), "NULL context")
    refused(q(at, at, BF16, -1, 1, at, at, None), "bad n_tokens")
    refused(q(at, at, BF16, 1, 0, at, at, None), "rows must not be empty")


def desc(at, **k):
    d = I8LayerDesc(at, at, at, at, 4, 64, 32, 0)
    for n, v in k.items():
        setattr(d, n, v)
    return d


@pytest.mark.parametrize("change,call,text", [
    (dict(down=None), {}, "NULL or empty"), (dict(n_mats=0), {}, "routed expert"), (dict(n_mats=1, shared=1), {}, "routed expert"), (dict(n_mats=1025), {}, "n_mats must be"),
    (dict(hidden=131072), {}, "cols 1..131071"), (dict(inter=0), {}, "inter must be"), (dict(inter=1 << 30), {}, "inter must be"), ({}, dict(dt=F32), "fp16/bf16"),
    ({}, dict(T=-1), "bad n_tokens"), ({}, dict(K=65), "bad n_tokens"), ({}, dict(K=0), "bad n_tokens"), ({}, dict(T=1 << 30, K=2), "too many pairs"),
    ({}, dict(x=None), "NULL buffer"), ({}, dict(size=64), "scratch must be")])
def test_layer_descriptor(at, change, call, text):
    a = dict(x=at, dt=BF16, T=3, K=2, size=1 << 40)
    a.update(call)
    refused(lib().cx_i8_moe(at, C.byref(desc(at, **change)), a["x"], a["dt"], a["T"], at, at, a["K"], at, BF16, None, at, a["size"], None), text)
    assert lib().cx_i8_moe_scratch(C.byref(desc(at, n_mats=0)), 3, 2) == 0


T, K, N, E = 6, 16, 8, 3
OFF = torch.zeros(E + 1, dtype=torch.int32)


def z(*s, dtype=torch.bfloat16):
    return torch.zeros(*s, dtype=dtype)


@pytest.mark.parametrize("x,w,kw,error", [
    (z(T, K), z(N, K + 1), {}, ValueError), (z(T, K), z(N, K, dtype=torch.float16), {}, TypeError), (z(T, K, dtype=torch.float32), z(N, K, dtype=torch.float32), {}, TypeError),
    (z(T, K), z(E, N, K), {}, ValueError), (z(T, K), z(E, N, K), {"offsets": OFF[:-1]}, ValueError), (z(T, K), z(E, N, K), {"offsets": OFF.long()}, ValueError),
    (z(T, K), z(N + 1, K), {"gated": True}, ValueError), (z(T, K), z(N, K), {"keep": True}, ValueError), (z(T, K), z(N, K), {"order": OFF.long()}, ValueError),
    (z(T, K), z(K, N).T, {}, ValueError), (z(T * K), z(N, K), {}, ValueError), (z(T, K), z(1, 1, N, K), {}, ValueError)])
def test_matmul_arguments(ctx, x, w, kw, error):  # noqa: F811
    with pytest.raises(error):
        ctx.matmul(x, w, **kw)


def test_good_calls_reach_the_library(ctx):  # noqa: F811
    for call in (lambda: ctx.matmul(z(T, K), z(N, K)), lambda: ctx.matmul(z(K, T).T, z(E, N, K), offsets=OFF, gated=True, keep=True),
                 lambda: ctx.matmul_grad(z(T, N), z(T, K), z(N, K)), lambda: ctx.matmul_grad(z(T, N // 2), z(T, K), z(E, N, K), pre=z(T, N), offsets=OFF),
                 lambda: ctx.quantize_i8(z(2, 3, K)), lambda: ctx.i8_matmul(z(T, K, dtype=torch.int8), torch.ones(T), z(N, K, dtype=torch.int8), torch.ones(N))):
        with pytest.raises(Called, match="cx_(matmul|quantize|i8)"):
            call()


def test_a_recorded_graph_is_not_lost(ctx):  # noqa: F811
    for x, w in ((z(T, K).requires_grad_(), z(N, K)), (z(T, K), z(N, K).requires_grad_())):
        with pytest.raises(ValueError, match="records no graph"):
            ctx.matmul(x, w)
        with torch.no_grad(), pytest.raises(Called):
            ctx.matmul(x, w)


@pytest.mark.parametrize("kw,error", [
    ({"dy": z(T, N + 1)}, ValueError), ({"pre": z(T, N)}, ValueError), ({"dy": z(T, N // 2), "pre": z(T, N - 1)}, ValueError), ({"dw_dtype": torch.float16}, TypeError),
    ({"want_dx": False, "want_dw": False}, ValueError), ({"dy": z(T, N, dtype=torch.float16)}, TypeError)])
def test_matmul_grad_arguments(ctx, kw, error):  # noqa: F811
    a = {"dy": z(T, N), **kw}
    with pytest.raises(error):
        ctx.matmul_grad(a.pop("dy"), z(T, K), z(N, K), **a)


@pytest.mark.parametrize("change,error", [(("x", z(T, K)), TypeError), (("xs", torch.ones(T + 1)), ValueError), (("xs", torch.ones(T).double()), ValueError),
                                          (("ws", torch.ones(N + 1)), ValueError), (("w", z(N, K)), TypeError)])
def test_i8_arguments(ctx, change, error):  # noqa: F811
    a = {"x": z(T, K, dtype=torch.int8), "xs": torch.ones(T), "w": z(N, K, dtype=torch.int8), "ws": torch.ones(N)}
    a[change[0]] = change[1]
    with pytest.raises(error):
        ctx.i8_matmul(a["x"], a["xs"], a["w"], a["ws"])


def test_layer_arguments(ctx):  # noqa: F811
    q = torch.int8
    good = dict(gate_up=z(E, 2 * N, K, dtype=q), gate_up_scale=torch.ones(E, 2 * N), down=z(E, K, N, dtype=q), down_scale=torch.ones(E, K))
    layer = I8Layer(ctx, **good)
    assert (layer.n_experts, layer.hidden, layer.inter, layer.shared) == (E, K, N, None)
    assert I8Layer(ctx, **good, shared=True).n_experts == E - 1 and I8Layer(ctx, **good, experts=[5, 1, 2]).n_experts == 6
    for change, error in (({"gate_up": z(E, N, K, dtype=q)}, ValueError), ({"down": z(E, K, N)}, TypeError), ({"down_scale": torch.ones(E, N)}, ValueError),
                          ({"gate_up": z(E, K, 2 * N, dtype=q).transpose(1, 2)}, ValueError), ({"experts": [0, 1]}, ValueError), ({"experts": [0, 1, 1]}, ValueError)):
        with pytest.raises(error):
            I8Layer(ctx, **{**good, **change})
    with pytest.raises(ValueError):  # the shared expert alone
        I8Layer(ctx, *(t[:1] for t in good.values()), shared=True)
    with pytest.raises(Called, match="cx_i8_moe_scratch"):
        ctx.moe(layer, z(T, K), torch.zeros(T, 2), torch.ones(T, 2))
    with pytest.raises(ValueError):  # another width
        ctx.moe(layer, z(T, K + 1), torch.zeros(T, 2), torch.ones(T, 2))
    with pytest.raises(TypeError):
        ctx.moe_layer_request(layer, b"")


@pytest.mark.parametrize("name", ["gate_up", "gate_up_scale", "down", "down_scale"])
def test_a_layer_whose_tensors_were_replaced(ctx, name):  # noqa: F811
    """Its descriptor points to those that it was made of, whose memory may be another's by then."""
    q = torch.int8
    layer = I8Layer(ctx, z(E, 2 * N, K, dtype=q), torch.ones(E, 2 * N), z(E, K, N, dtype=q), torch.ones(E, K))
    call = lambda: ctx.moe(layer, z(T, K), torch.zeros(T, 2), torch.ones(T, 2))  # noqa: E731
    getattr(layer, name).copy_(torch.ones_like(getattr(layer, name)))  # values in place are the layer's own
    with pytest.raises(Called, match="cx_i8_moe_scratch"):
        call()
    old = getattr(layer, name)
    setattr(layer, name, old.clone())
    with pytest.raises(ValueError, match="replaced"):
        call()
    setattr(layer, name, old)
    with pytest.raises(Called, match="cx_i8_moe_scratch"):
        call()
    old.data = old.data.clone()
    with pytest.raises(ValueError, match="replaced"):
        call()
