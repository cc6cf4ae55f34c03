"""Refusals and grids of the calls for long contexts in a small cache, on the CPU: the host layer over a HIP runtime that
runs nothing (see test_serving_refusals.py), and the helpers' 4-bit pages against the format's definition."""
import ctypes

import numpy as np
import pytest

import budget
import tmac_attn
from budget import Q4
from test_serving_refusals import P, fake  # noqa: F401  (the fixture)
from tmac_attn import (TMAC_ERR_CAPTURE, TMAC_ERR_INVALID_ARG, TMAC_ERR_MISALIGNED, TMAC_ERR_NULL_POINTER,
                       TMAC_ERR_UNSUPPORTED, TMAC_OK)

AXES = ctypes.create_string_buffer(bytes([0] * 8 + [1] * 12 + [2] * 12), 32)
GOOD = {
    "tmac_kv_append_axes_paged": dict(kv_dtype=Q4, q=P, q_stride=896, q_out=2 * P, k=3 * P, k_stride=128, v=4 * P,
                                      v_stride=128, k_pages=5 * P, v_pages=6 * P, n_pages=9, block_table=7 * P,
                                      max_pages=4, row_starts=8 * P, first_rows=9 * P, positions=10 * P, n_axes=3,
                                      pair_axis=ctypes.addressof(AXES), n_seq=3, n_rows=5, n_head=14, n_kv_head=2,
                                      head_dim=64, max_pos=64, base=1e6),
    "tmac_attention_decode_weighted": dict(kv_dtype=Q4, q=P, k_pages=2 * P, v_pages=3 * P, n_pages=9, block_table=4 * P,
                                           max_pages=40, lengths=5 * P, weights_in=6 * P, weights_out=8 * P,
                                           weight_stride=640, out=10 * P, n_seq=3, n_head=14, n_kv_head=2, head_dim=64,
                                           max_len=640),
    "tmac_select_rows": dict(weights=P, weight_stride=640, lengths=2 * P, kept=3 * P, n_seq=3, n_kv_head=2, max_len=640,
                             keep=100, first=4, last=64),
    "tmac_kv_compact_paged": dict(kv_dtype=Q4, k_pages=P, v_pages=2 * P, n_pages=9, block_table=3 * P, max_pages=40,
                                  lengths=4 * P, kept=5 * P, keep=100, to_table=6 * P, to_pages=7, weights_in=7 * P,
                                  weights_out=9 * P, weight_stride=640, n_seq=3, n_kv_head=2, head_dim=64),
    "tmac_kv_widen_pages": dict(kv_dtype=Q4, k_pages=P, v_pages=2 * P, k_out=3 * P, v_out=4 * P, n_pages=9, n_kv_head=2,
                                head_dim=64),
}
MAY_BE_NULL = {("tmac_kv_append_axes_paged", "pair_axis"), ("tmac_attention_decode_weighted", "weights_in")}
POINTERS = [(n, k) for n, kw in GOOD.items() for k, v in kw.items() if isinstance(v, int) and v >= P]
ALIGN16 = {"q", "q_out", "k", "v", "k_pages", "v_pages", "out", "k_out", "v_out"}


def call(fake, name, **kw):  # noqa: F811
    args = dict(GOOD[name])
    assert set(kw) <= set(args), kw
    args.update(kw)
    fake.lib.fake_clear()
    rc = getattr(fake.lib, name)(fake.handle, None, *args.values())
    return rc, [(fake.lib.fake_launch_name(i).decode(), fake.lib.fake_launch_grid(i, 0)) for i in range(fake.lib.fake_launches())]


@pytest.mark.parametrize("name", sorted(GOOD))
def test_accepted_by_type(fake, name):  # noqa: F811
    types = {0: "f32", 1: "bf16", 2: "f16", 3: "q8", Q4: "q4"} if "kv_dtype" in GOOD[name] else {None: ""}
    for dt, text in types.items():
        rc, launches = call(fake, name, **({} if dt is None else {"kv_dtype": dt}))
        assert rc == TMAC_OK and launches and text in launches[0][0]
    if "kv_dtype" in GOOD[name]:
        for bad in (-1, 4, 5, 15, 17):
            assert call(fake, name, kv_dtype=bad) == (TMAC_ERR_INVALID_ARG, [])


@pytest.mark.parametrize("name,arg", POINTERS)
def test_null_and_misaligned_pointers(fake, name, arg):  # noqa: F811
    if arg == "pair_axis":
        assert call(fake, name, pair_axis=None)[0] == TMAC_OK
        return
    rc, launches = call(fake, name, **{arg: None})
    if (name, arg) in MAY_BE_NULL:
        assert rc == TMAC_OK
    else:
        assert rc == TMAC_ERR_NULL_POINTER and not launches
    for off in (4, 8) if arg in ALIGN16 else (1, 2):
        rc, launches = call(fake, name, **{arg: GOOD[name][arg] + off})
        assert rc == TMAC_ERR_MISALIGNED and not launches, off


@pytest.mark.parametrize("name", sorted(GOOD))
def test_shapes_outside_the_domain(fake, name):  # noqa: F811
    good = GOOD[name]
    if "head_dim" in good:
        for head_dim in (0, 32, 63, 128):
            assert call(fake, name, head_dim=head_dim) == (TMAC_ERR_UNSUPPORTED, [])
    for bad in (0, -2):
        assert call(fake, name, n_kv_head=bad) == (TMAC_ERR_INVALID_ARG, [])
    if "n_head" in good:
        for bad in (0, -14, 13):
            assert call(fake, name, n_head=bad) == (TMAC_ERR_INVALID_ARG, [])
        rc, _ = call(fake, name, n_head=34, **({"q_stride": 34 * 64} if "q_stride" in good else {}))
        assert rc == (TMAC_OK if name == "tmac_kv_append_axes_paged" else TMAC_ERR_UNSUPPORTED)
    for arg in ("n_pages", "max_pages"):
        for bad in (0, -1):
            if arg in good and (name != "tmac_kv_widen_pages" or bad):
                assert call(fake, name, **{arg: bad}) == (TMAC_ERR_INVALID_ARG, []), (arg, bad)
    if "n_seq" in good:
        assert call(fake, name, n_seq=-1) == (TMAC_ERR_INVALID_ARG, [])
        assert call(fake, name, n_seq=0) == (TMAC_OK, [])


BIG = 2 ** 31 - 1


@pytest.mark.parametrize("name,kw", [
    ("tmac_kv_append_axes_paged", dict(max_pos=0)),
    ("tmac_kv_append_axes_paged", dict(n_rows=-1)),
    ("tmac_kv_append_axes_paged", dict(n_axes=0)),
    ("tmac_kv_append_axes_paged", dict(n_axes=5)),
    ("tmac_kv_append_axes_paged", dict(n_axes=2)),  # pairs on axis 2
    ("tmac_kv_append_axes_paged", dict(q_stride=892)),
    ("tmac_kv_append_axes_paged", dict(k_stride=124)),
    ("tmac_kv_append_axes_paged", dict(v_stride=0)),
    ("tmac_kv_append_axes_paged", dict(base=0.0)),
    ("tmac_kv_append_axes_paged", dict(base=float("nan"))),
    ("tmac_kv_append_axes_paged", dict(q_out=P + 896 * 4)),
    ("tmac_kv_append_axes_paged", dict(q_out=3 * P + 4 * 127 * 4)),
    ("tmac_kv_append_axes_paged", dict(q_out=4 * P - 5 * 896 * 4 + 16)),
    ("tmac_kv_append_axes_paged", dict(q=None, q_out=None, n_rows=2 ** 30)),
    ("tmac_attention_decode_weighted", dict(max_len=0)),
    ("tmac_attention_decode_weighted", dict(max_len=641)),
    ("tmac_attention_decode_weighted", dict(weight_stride=639)),
    ("tmac_attention_decode_weighted", dict(weights_out=6 * P + 4)),  # over weights_in, not it
    ("tmac_attention_decode_weighted", dict(weights_out=6 * P + (5 * 640 + 639) * 4)),
    ("tmac_attention_decode_weighted", dict(n_seq=BIG)),
    ("tmac_select_rows", dict(max_len=0)),
    ("tmac_select_rows", dict(max_len=641)),
    ("tmac_select_rows", dict(keep=0, first=0, last=0)),
    ("tmac_select_rows", dict(first=-1)),
    ("tmac_select_rows", dict(last=-1)),
    ("tmac_select_rows", dict(first=37)),
    ("tmac_select_rows", dict(first=BIG, last=BIG)),
    ("tmac_select_rows", dict(n_seq=BIG, n_kv_head=BIG)),
    ("tmac_kv_compact_paged", dict(keep=0)),
    ("tmac_kv_compact_paged", dict(keep=113)),
    ("tmac_kv_compact_paged", dict(weight_stride=99)),
    ("tmac_kv_compact_paged", dict(weights_out=7 * P)),
    ("tmac_kv_compact_paged", dict(weights_out=7 * P + (6 * 640 - 1) * 4)),
    ("tmac_kv_compact_paged", dict(n_seq=BIG, n_kv_head=BIG)),
    ("tmac_kv_widen_pages", dict(n_pages=-1)),
    ("tmac_kv_widen_pages", dict(n_pages=2 ** 24)),
])
def test_refused(fake, name, kw):  # noqa: F811
    assert call(fake, name, **kw) == (TMAC_ERR_INVALID_ARG, [])


def test_legal_edges(fake):  # noqa: F811
    ok = lambda name, **kw: call(fake, name, **kw)[0] == TMAC_OK  # noqa: E731
    assert ok("tmac_kv_append_axes_paged", q=None, q_out=None)
    assert ok("tmac_kv_append_axes_paged", q_out=P)
    assert call(fake, "tmac_kv_append_axes_paged", n_rows=0) == (TMAC_OK, [])
    assert ok("tmac_attention_decode_weighted", weights_out=6 * P)  # in place
    assert ok("tmac_attention_decode_weighted", weights_in=None, weights_out=None, weight_stride=0)
    assert ok("tmac_attention_decode_weighted", weights_out=6 * P + (5 * 640 + 640) * 4)  # right behind
    assert call(fake, "tmac_attention_decode_weighted", weights_out=None)[0] == TMAC_ERR_NULL_POINTER
    assert ok("tmac_kv_compact_paged", weights_in=None, weights_out=None, weight_stride=0)
    assert ok("tmac_kv_compact_paged", weights_out=7 * P + 6 * 640 * 4)
    assert call(fake, "tmac_kv_compact_paged", weights_out=None)[0] == TMAC_ERR_NULL_POINTER
    assert ok("tmac_kv_widen_pages", k_pages=None, k_out=None) and ok("tmac_kv_widen_pages", v_pages=None, v_out=None)
    assert call(fake, "tmac_kv_widen_pages", k_pages=None, k_out=None, v_pages=None, v_out=None)[0] == TMAC_ERR_NULL_POINTER
    assert call(fake, "tmac_kv_widen_pages", n_pages=0) == (TMAC_OK, [])


def test_growth_is_refused_while_capturing(fake):  # noqa: F811
    fake.lib.fake_set_capturing(1)
    try:
        assert call(fake, "tmac_attention_decode_weighted", n_seq=4096, max_pages=8192, max_len=131072,
                    weight_stride=131072, weights_in=None) == (TMAC_ERR_CAPTURE, [])
        assert call(fake, "tmac_kv_append_axes_paged", max_pos=65536, base=54321.0) == (TMAC_ERR_CAPTURE, [])
    finally:
        fake.lib.fake_set_capturing(0)


def test_largest_numbers_overflow_nothing(fake):  # noqa: F811
    """Strides and counts at their largest: refused or launched, with no crash."""
    for kw in (dict(k_stride=2 ** 62), dict(q_stride=2 ** 62, v_stride=2 ** 62)):
        call(fake, "tmac_kv_append_axes_paged", **kw)
    for name in ("tmac_attention_decode_weighted", "tmac_select_rows", "tmac_kv_compact_paged"):
        call(fake, name, weight_stride=2 ** 62)
    assert call(fake, "tmac_attention_decode_weighted", weight_stride=2 ** 62)[0] == TMAC_ERR_INVALID_ARG


# ---- the 4-bit pages of the helpers ----

def test_every_code_has_a_place_of_its_own():
    for key in (True, False):
        byte, high, scale = budget.places(key)
        assert sorted((2 * byte + high).reshape(-1)) == list(range(1024))
        assert sorted(scale.reshape(-1)) == list(range(256, 288))
        for r in range(16):  # a byte holds two dims of one row
            assert len(np.unique(byte[r])) == 32


def test_codes_are_the_nearest():
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((2, 16, 3, 64)) * np.exp2(rng.uniform(-8, 8, (2, 16, 3, 1)))).astype(np.float32)
    q, d = budget.codes4(x)
    step = np.abs(np.repeat(d, 32, -1))
    for key in (True, False):
        y = budget.widen4(budget.pack4(x, key), key)
        np.testing.assert_array_equal(y, (q.astype(np.float32) - 8) * np.repeat(d, 32, -1))
        # half a step; beyond code 15 (the side that the largest magnitude is not on) up to a step, and what the scale's
        # rounding to 7 bits (2^-7 of it) leaves out at the ends
        assert (np.abs(y - x) <= step * (1 + 8 * 2.0 ** -7)).all()
        inside = (q > 0) & (q < 15)
        assert (np.abs(y - x)[inside] <= step[inside] * (0.5 + 2.0 ** -20)).all()
    m = d.view(np.uint32) & 0x1FFFF
    assert not m.any() and (d.astype(np.float16).astype(np.float32) == d).all()


def test_blocks_at_the_ends_of_the_scale():
    x = np.zeros((7, 64), np.float32)
    x[1, 5] = 2.0 ** -12           # scale 2^-15: 0
    x[2, 5] = -2.0 ** -11          # 2^-14 kept
    x[3, 5] = 8 * 8128.0
    x[4, 5] = 8 * 8500.0
    x[5, 5], x[6, 40] = np.nan, np.inf
    q, d = budget.codes4(x)
    assert d[0].tolist() == [0, 0] and d[1, 0] == 0 and d[2, 0] == 2.0 ** -14 and d[3, 0] == -8128
    assert d[4, 0] == -np.inf and np.isnan(d[5, 0]) and d[6].tolist() == [0, -np.inf]
    assert (q[0] == 8).all() and (q[1] == 8).all() and q[2, 5] == 0
    assert q[3, 5] == 0


def test_workgroups_by_length_and_number(fake):  # noqa: F811
    """The splits that the rules give on a card of 256 CUs: whole sequences in one launch, long ones dealt, then joined."""
    d = "tmac_attention_decode_weighted"
    long = dict(max_len=6400, max_pages=400, weight_stride=6400, weights_out=6 * P)
    assert call(fake, d) == (TMAC_OK, [("tmac_rows_q4_pair", 6)])
    assert call(fake, d, n_head=18) == (TMAC_OK, [("tmac_rows_q4", 6)])
    assert call(fake, d, weights_in=None, weights_out=None) == (TMAC_OK, [("tmac_rows_q4_pair", 6)])
    assert call(fake, d, **long) == (TMAC_OK, [("tmac_rows_q4_pair", 156), ("tmac_rows_finish", 6 * (7 + 7))])
    assert call(fake, d, **{**long, "weights_in": None, "weights_out": None}) == (
        TMAC_OK, [("tmac_rows_q4_pair", 156), ("tmac_rows_finish", 6 * 7)])
    assert call(fake, d, **long, n_seq=100) == (TMAC_OK, [("tmac_rows_q4_pair", 301), ("tmac_rows_finish", 200 * (2 + 7))])
    assert call(fake, d, **{**long, "max_len": 4096}, n_seq=100) == (TMAC_OK, [("tmac_rows_q4_pair", 200)])
    wide = dict(max_len=4097, weight_stride=4097)
    assert call(fake, "tmac_select_rows", **{**wide, "max_len": 4096}) == (TMAC_OK, [("tmac_select_rows_256", 6)])
    assert call(fake, "tmac_select_rows", **wide) == (TMAC_OK, [("tmac_select_rows_1024", 6)])
    assert call(fake, "tmac_kv_compact_paged") == (TMAC_OK, [("tmac_compact_q4", 11)])
