"""Arguments of the 4-bit entry points that are refused before anything touches a
device.  No GPU: the context is memory that none of these calls reads."""
from __future__ import annotations

import ctypes as C

import pytest

from constellation_amd._lib import BF16, CX_EINVAL, E4M3, FP16, Q4Desc, lib


@pytest.fixture(scope="module")
def held():
    """Host memory in the place of device buffers: 16-byte aligned, never read."""
    raw = C.create_string_buffer(1 << 16)
    return raw, (C.addressof(raw) + 255) // 256 * 256


def desc(at, n_mats=1, rows=64, cols=128, group=128, gated=0):
    d = Q4Desc()
    d.codes, d.scales = at, at
    d.n_mats, d.rows, d.cols, d.group, d.gated = n_mats, rows, cols, group, gated
    return d


def refused(rc, text):
    assert rc == CX_EINVAL and text.encode() in lib().cx_last_error(), (rc, text, lib().cx_last_error())


def matmul(at, d, dt=BF16, xs=None, n_x=4, P=4, offsets=None, size=1 << 16):
    return lib().cx_q4_matmul(at, C.byref(d), at, dt, xs, n_x, None, 1, offsets, P, at, BF16, at, size, None)


@pytest.mark.parametrize("dt", [BF16, FP16])
@pytest.mark.parametrize("rows", [1, 16, 4000])
def test_x_scale_without_e4m3(held, dt, rows):
    """Refused for any number of rows: some kernels would read it as a factor of the row."""
    _, at = held
    refused(matmul(at, desc(at), dt=dt, xs=at, n_x=rows, P=rows, size=1 << 40), "x_scale comes with e4m3 x only")
    refused(matmul(at, desc(at), dt=E4M3, xs=None), "NULL buffer")


@pytest.mark.parametrize("field,value", [("n_mats", 1025), ("n_mats", 0), ("n_mats", 1 << 20), ("rows", (1 << 24) + 16), ("cols", (1 << 24) + 128),
                                         ("rows", 0), ("cols", -1), ("group", 48)])
def test_descriptors_past_what_is_packed(held, field, value):
    """A descriptor that cx_q4_pack would not have made: a stack of more than 1024 matrices has no plan."""
    _, at = held
    d = desc(at, 4)
    setattr(d, field, value)
    refused(matmul(at, d, offsets=at, size=1 << 40), "bad 4-bit descriptor")
    gu, dn = desc(at, 4, 128, 128, gated=1), desc(at, 4, 128, 64)
    for w in (gu, dn):
        keep = getattr(w, field)
        setattr(w, field, value)
        refused(lib().cx_q4_moe(at, C.byref(gu), C.byref(dn), None, None, at, BF16, 4, at, at, 2, at, BF16, None, at, 1 << 40, None),
                "bad 4-bit descriptor")
        setattr(w, field, keep)


@pytest.mark.parametrize("hidden", [2 ** 31 - 1, 2 ** 31 - 2048])
def test_rows_whose_columns_do_not_fit_an_int(held, hidden):
    """A thread looks at up to 2048 columns from its first one on."""
    _, at = held
    L = lib()
    refused(L.cx_combine_rows(at, at, BF16, at, None, None, 1, 1, hidden, at, BF16, None, None), "at most 2147481599 columns")
    refused(L.cx_combine_rows_grad(at, at, BF16, at, BF16, at, None, 1, 1, hidden, at, None, None), "at most 2147481599 columns")
    refused(L.cx_gather_rows(at, at, hidden + 2048, at, 1, 1, at, None), "fewer than 2^31 bytes")
