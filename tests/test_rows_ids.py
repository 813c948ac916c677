"""Ids that Context.sort_tokens is given, and what the library gets of them.  No GPU."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from constellation_amd import engine
from test_q4_layer_checks import ctx  # noqa: F401  (a fixture)


@pytest.fixture()
def seen(monkeypatch, ctx):  # noqa: F811
    got = []

    class Library:
        def cx_sort_tokens(self, handle, ids, T, K, *_):
            got.append(list((C.c_int32 * (T * K)).from_address(ids)))
            return 0
    monkeypatch.setattr(engine, "lib", lambda: Library())
    return got


def test_ids_past_32_bits_name_no_expert(ctx, seen):  # noqa: F811
    ctx.sort_tokens(torch.tensor([[3, 2 ** 32 + 3], [-1, -2 ** 32 + 1], [2 ** 31, 7]]), 8)
    assert seen[0] == [3, 2 ** 31 - 1, -1, -1, 2 ** 31 - 1, 7]


@pytest.mark.parametrize("dtype", [torch.int32, torch.int16, torch.int8, torch.uint8, torch.uint16, torch.uint32, torch.uint64, torch.int64])
def test_smaller_integers(ctx, seen, dtype):  # noqa: F811
    ctx.sort_tokens(torch.tensor([[3, 120]]).to(dtype), 8)
    assert seen[0] == [3, 120]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bool, torch.bfloat16, torch.complex64])
def test_other_types_are_refused(ctx, seen, dtype):  # noqa: F811
    with pytest.raises(TypeError, match="ids must be integers"):
        ctx.sort_tokens(torch.ones(2, 2).to(dtype), 8)
    assert not seen
