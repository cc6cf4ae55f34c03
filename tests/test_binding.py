"""Arguments of the Python calls for long contexts in a small cache, on the CPU (the host layer over a HIP runtime that runs
nothing, see test_serving_refusals.py): addresses as every other call takes them, the axes of the pairs in any form."""
import numpy as np
import pytest

import tmac_attn
from test_serving_refusals import P, fake  # noqa: F401  (the fixture)

CALLS = {  # positions of the addresses, arguments
    "kv_append_axes_paged": ((0, 2, 3, 5, 7, 8, 10, 12, 13, 14),
                             [P, 896, 2 * P, 3 * P, 128, 4 * P, 128, 5 * P, 6 * P, 9, 7 * P, 4, 8 * P, 9 * P, 10 * P, 3, None, 3,
                              5, 14, 2, 64, 64]),
    "decode_weighted": ((0, 1, 2, 4, 6, 7, 8, 10), [P, 2 * P, 3 * P, 9, 4 * P, 40, 5 * P, 6 * P, 8 * P, 640, 10 * P, 3, 14, 2, 64,
                                                    640]),
    "select_rows": ((0, 2, 3), [P, 640, 2 * P, 3 * P, 3, 2, 640, 100]),
    "kv_compact_paged": ((0, 1, 3, 5, 6, 8, 10, 11), [P, 2 * P, 9, 3 * P, 40, 4 * P, 5 * P, 100, 6 * P, 7, 7 * P, 9 * P, 640, 3, 2,
                                                      64]),
    "kv_widen_pages": ((0, 1, 2, 3), [P, 2 * P, 3 * P, 4 * P, 9, 2, 64]),
}


@pytest.fixture
def ctx(fake):  # noqa: F811
    c = tmac_attn.Context.__new__(tmac_attn.Context)
    c.lib, c.handle = fake.lib, fake.handle
    return c


def array_at(address):
    a = tmac_attn.DeviceArray.__new__(tmac_attn.DeviceArray)
    a.ptr = address
    return a


@pytest.mark.parametrize("name", sorted(CALLS))
@pytest.mark.parametrize("form", [int, np.int64, np.uint64, array_at], ids=["int", "int64", "uint64", "array"])
def test_addresses_in_every_form(ctx, name, form):
    places, good = CALLS[name]
    assert getattr(ctx, name)(*[form(x) if i in places else x for i, x in enumerate(good)]) == 0


@pytest.mark.parametrize("name", sorted(CALLS))
def test_host_objects_are_no_addresses(ctx, name):
    """Bytes, text, host arrays: none is taken as a device address."""
    places, good = CALLS[name]
    for i in places:
        for bad in (b"\x00" * 16, "text", bytearray(16), np.zeros(4, np.float32), [P], 1.5j):
            with pytest.raises((TypeError, ValueError)):
                getattr(ctx, name)(*good[:i], bad, *good[i + 1:])


@pytest.mark.parametrize("make", [list, tuple, bytes, bytearray, lambda x: np.array(x, np.uint8), lambda x: np.array(x, np.int8),
                                  lambda x: np.array(x, np.int32), lambda x: np.array(x, np.int64), iter,
                                  lambda x: np.repeat(np.array(x, np.uint8), 2)[::2]],
                         ids=["list", "tuple", "bytes", "bytearray", "uint8", "int8", "int32", "int64", "iterator", "strided"])
def test_axes_of_the_pairs_in_every_form(ctx, monkeypatch, make):
    """32 values, whatever holds them, reach the library as 32 bytes."""
    seen, lib, axes = [], ctx.lib, [0] * 8 + [1] * 12 + [2] * 12

    class Library:
        def __getattr__(self, name):
            fn = getattr(lib, name)
            return lambda *a: seen.append(a[19]) or fn(*a)

    ctx.lib = Library()
    good = list(CALLS["kv_append_axes_paged"][1])
    good[16] = make(axes)
    assert ctx.kv_append_axes_paged(*good) == 0
    assert seen == [bytes(axes)]


@pytest.mark.parametrize("bad", [[0] * 31, [0] * 33, b"\x00" * 31, np.zeros(4, np.int64), np.zeros(8, np.int32),
                                 np.zeros(128, np.uint8), [0.5] * 32, [-1] * 32, [300] * 32, np.zeros(32, np.float32)])
def test_axes_that_are_not_32_bytes(ctx, bad):
    good = list(CALLS["kv_append_axes_paged"][1])
    good[16] = bad
    with pytest.raises((TypeError, ValueError)):
        ctx.kv_append_axes_paged(*good)


@pytest.mark.parametrize("bad", [[3] * 32, np.full(32, -1, np.int8), np.full(32, 255, np.uint8)])
def test_axes_beyond_n_axes(ctx, bad):
    good = list(CALLS["kv_append_axes_paged"][1])
    good[16] = bad
    with pytest.raises(tmac_attn.TmacError):
        ctx.kv_append_axes_paged(*good)
