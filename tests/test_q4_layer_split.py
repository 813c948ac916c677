"""A layer of 4-bit experts whose stacks hold some of the layer's experts.  No GPU: what the
library would be given is read from a stand-in for it."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from constellation_amd import engine
from constellation_amd import moe_dispatch as D
from test_q4_layer_checks import E, H, I, ctx, matrix  # noqa: F401  (ctx is a fixture)


def layer(ctx, **kw):
    return engine.Q4Layer(ctx, matrix(E, 2 * I, H, True), matrix(E, H, I, False), **kw)


def test_who_holds_what(ctx):  # noqa: F811
    whole, some = layer(ctx), layer(ctx, experts=[5, 2, 9, 0], n_experts=12)
    assert whole.n_experts == E and all(e is whole for e in whole.experts) and whole._slots is None
    assert some.n_experts == 12 and [i for i, e in enumerate(some.experts) if e is some] == [0, 2, 5, 9]
    assert layer(ctx, experts=[5, 2, 9, 0]).n_experts == 10
    assert layer(ctx, experts=range(E), n_experts=E)._slots is None
    node = D.LocalNode({0: some})
    assert node.resident(0, 12).nonzero()[0].tolist() == [0, 2, 5, 9] and not node.resident(1, 12).any()
    assert node.resident(0, 4).nonzero()[0].tolist() == [0, 2] and node.resident(0, 20).nonzero()[0].tolist() == [0, 2, 5, 9]


@pytest.mark.parametrize("kw", [{"experts": []}, {"experts": [0, 1, 2]}, {"experts": [0, 1, 2, 2]}, {"experts": [0, 1, 2, -1]},
                                {"experts": [0, 1, 2, 7], "n_experts": 7}, {"n_experts": E - 1}, {"n_experts": 0}])
def test_bad_ids(ctx, kw):  # noqa: F811
    with pytest.raises(ValueError, match="different ids below n_experts"):
        layer(ctx, **kw)


def test_ids_reach_the_library_as_slots(ctx, monkeypatch):  # noqa: F811
    seen = []

    class Library:
        def cx_q4_moe_scratch(self, *a):
            return 16

        def cx_q4_moe(self, *a):
            seen.append(torch.tensor(list((C.c_int32 * (a[7] * a[10])).from_address(a[8]))).view(a[7], a[10]).tolist())
            return 0

        def __getattr__(self, name):  # cx_moe_decode, ..., looked up and not called
            return None
    monkeypatch.setattr(engine, "lib", lambda: Library())
    some = layer(ctx, experts=[5, 2, 9, 0], n_experts=12)
    ids = torch.tensor([[5, 2, -1], [0, 9, 1], [11, 12, 1 << 30], [-7, 5, 0]], dtype=torch.int32)
    x, w = torch.zeros(4, H, dtype=torch.bfloat16), torch.ones(4, 3)
    ctx.moe(some, x, ids, w)
    ctx.moe(layer(ctx), x, ids, w)
    # an expert that is not held is one past the stacks, which the library reports
    assert seen[0] == [[0, 1, -1], [3, 2, E], [E, E, E], [-1, 0, 3]] and seen[1] == ids.tolist()
    assert ids[0, 0] == 5
