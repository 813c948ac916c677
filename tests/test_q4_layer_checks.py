"""What Context.moe and Context.moe_layer refuse on a layer of 4-bit experts, before any
call into the library.  No GPU: a context of "device -1", where CPU tensors are at home,
and a library that fails the test when it is called."""
from __future__ import annotations

import pytest
import torch

from constellation_amd import engine
from constellation_amd._lib import Q4Desc

E, H, I, T, K = 4, 64, 32, 3, 2


class Called(Exception):
    pass


class NoLibrary:
    """The library's rules for scratch, and no other call."""

    def __getattr__(self, name):
        def call(*args):
            raise Called(name)
        return call


def matrix(n, rows, cols, gated, device=-1):
    d = Q4Desc()
    d.codes, d.scales, d.n_mats, d.rows, d.cols, d.group, d.gated = 256, 256, n, rows, cols, 32, int(gated)
    return engine.Q4Matrix(device, d)


@pytest.fixture()
def ctx(monkeypatch):
    monkeypatch.setattr(engine, "lib", lambda: NoLibrary())
    monkeypatch.setattr(engine, "_stream", lambda device: 0)
    monkeypatch.setattr(engine, "_device", lambda index: torch.device("cpu"))
    c = engine.Context.__new__(engine.Context)
    c.device, c.handle = -1, 1
    return c


@pytest.fixture()
def layer(ctx):
    return engine.Q4Layer(ctx, matrix(E, 2 * I, H, True), matrix(E, H, I, False))


def router(**kw):
    a = dict(x=torch.zeros(T, H, dtype=torch.bfloat16), w_router=torch.zeros(E, H, dtype=torch.bfloat16), bias=torch.zeros(E),
             n_group=2, topk_group=1, top_k=K)
    return {**a, **kw}


def test_a_good_call_reaches_the_router(ctx, layer):
    for kw in ({}, {"w_router": torch.zeros(H, E, dtype=torch.bfloat16).T}, {"resident": torch.ones(E, dtype=torch.bool)},
               {"out": (torch.zeros(T, H, dtype=torch.float16), None, torch.zeros(T, K, dtype=torch.int32), torch.zeros(T, K))}):
        with pytest.raises(Called, match="cx_route"):
            ctx.moe_layer(layer, **router(**kw))


@pytest.mark.parametrize("kw,text", [
    ({"x": torch.zeros(T, H - 1, dtype=torch.bfloat16)}, "columns"),
    ({"x": torch.zeros(T, H + 64, dtype=torch.bfloat16)}, "columns"),
    ({"x": torch.zeros(H, dtype=torch.bfloat16)}, "columns"),
    ({"w_router": torch.zeros(E - 1, H, dtype=torch.bfloat16)}, "w_router"),
    ({"w_router": torch.zeros(H, E, dtype=torch.bfloat16)}, "w_router"),
    ({"bias": torch.zeros(E - 1)}, "bias"),
    ({"bias": torch.zeros(E, dtype=torch.bfloat16)}, "bias"),
    ({"resident": torch.ones(E - 1, dtype=torch.uint8)}, "resident"),
    ({"resident": torch.ones(E)}, "resident"),
    ({"out": (torch.zeros(T, H - 1, dtype=torch.bfloat16), None, torch.zeros(T, K, dtype=torch.int32), torch.zeros(T, K))}, "out must"),
    ({"out": (torch.zeros(T, H), None, torch.zeros(T, K, dtype=torch.int32), torch.zeros(T, K))}, "out must"),
    ({"out": (torch.zeros(T, H, dtype=torch.bfloat16), torch.zeros(T, H, dtype=torch.bfloat16), torch.zeros(T, K, dtype=torch.int32), torch.zeros(T, K))}, "out must"),
    ({"out": (torch.zeros(T, H, dtype=torch.bfloat16), None, torch.zeros(T, K, dtype=torch.int64), torch.zeros(T, K))}, "out must"),
    ({"out": (torch.zeros(T, H, dtype=torch.bfloat16), None, torch.zeros(T, K, dtype=torch.int32), torch.zeros(T, K + 1))}, "out must"),
])
def test_bad_router_calls_launch_nothing(ctx, layer, kw, text):
    with pytest.raises(ValueError, match=text):
        ctx.moe_layer(layer, **router(**kw))


def test_tensors_elsewhere_launch_nothing(ctx, layer):
    ctx.device = 0
    with pytest.raises(ValueError, match="tensor on cpu, context on cuda:0"):
        ctx.moe_layer(layer, **router())


def test_a_freed_or_foreign_layer_launches_nothing(ctx, layer):
    x, ids, w = torch.zeros(T, H, dtype=torch.bfloat16), torch.zeros(T, K, dtype=torch.int32), torch.ones(T, K)
    layer.down._live = False
    for call in (lambda: ctx.moe_layer(layer, **router()), lambda: ctx.moe(layer, x, ids, w)):
        with pytest.raises(ValueError, match="freed"):
            call()
    far = engine.Context.__new__(engine.Context)
    far.device, far.handle = 1, 1
    there = engine.Q4Layer(far, matrix(E, 2 * I, H, True, 1), matrix(E, H, I, False, 1))
    for call in (lambda: ctx.moe_layer(there, **router()), lambda: ctx.moe(there, x, ids, w)):
        with pytest.raises(ValueError, match="layer on cuda:1"):
            call()


@pytest.mark.parametrize("ids,w", [(torch.zeros(K, dtype=torch.int32), torch.ones(K)), (torch.zeros(T, K, dtype=torch.int32), torch.ones(T, K + 1)),
                                   (torch.zeros(T - 1, K, dtype=torch.int32), torch.ones(T - 1, K)), (torch.zeros(T, K, dtype=torch.int32), torch.ones(T)),
                                   (torch.zeros(T, 0, dtype=torch.int32), torch.ones(T, K))])
def test_routes_of_another_shape_launch_nothing(ctx, ids, w):
    """A shared expert beside them does not make them a call without routes."""
    shared = (matrix(1, 2 * I, H, True), matrix(1, H, I, False))
    layer = engine.Q4Layer(ctx, matrix(E, 2 * I, H, True), matrix(E, H, I, False), shared)
    with pytest.raises(ValueError, match="routes must be"):
        ctx.moe(layer, torch.zeros(T, H, dtype=torch.bfloat16), ids, w)
