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
