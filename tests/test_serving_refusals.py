"""Refusals and grids of the serving operators on paged caches, on the CPU: the host layer
linked with a HIP runtime that runs nothing and writes every launch down
(tests/cpp/fake_hip.cpp).  A refused call launches nothing; an accepted one launches grids
that cover the work its kernels look for."""
import ctypes
import os

import pytest

import tmac_attn
from tmac_attn import (TMAC_ERR_CAPTURE, TMAC_ERR_INVALID_ARG, TMAC_ERR_MISALIGNED, TMAC_ERR_NULL_POINTER,
                       TMAC_ERR_UNSUPPORTED, TMAC_OK)

FAKE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "build", "libtmac_fake.so")
P = 0x10000  # an aligned address; nothing reads it


class Fake:
    def __init__(self):
        self.lib = ctypes.CDLL(FAKE)
        for name, (res, args) in tmac_attn.SIGNATURES.items():
            fn = getattr(self.lib, name)
            fn.restype, fn.argtypes = res, args
        self.lib.fake_launch_name.restype = ctypes.c_char_p
        h = ctypes.c_void_p()
        assert self.lib.tmac_init(ctypes.byref(h), 0) == TMAC_OK
        self.handle = h.value

    def call(self, name, **kw):
        """(status, [(kernel, grid)]) of entry point `name` with its good arguments but for kw."""
        args = dict(GOOD[name])
        assert set(kw) <= set(args), kw
        args.update(kw)
        self.lib.fake_clear()
        rc = getattr(self.lib, name)(self.handle, None, *args.values())
        return rc, [(self.lib.fake_launch_name(i).decode(), self.lib.fake_launch_grid(i, 0))
                    for i in range(self.lib.fake_launches())]


GOOD = {
    "tmac_kv_append_paged": dict(kv_dtype=0, q=P, q_stride=896, q_out=2 * P, k=3 * P, k_stride=128, v=4 * P,
                                 v_stride=128, k_pages=5 * P, v_pages=6 * P, n_pages=9, block_table=7 * P, max_pages=4,
                                 row_starts=8 * P, positions=9 * P, n_seq=3, n_rows=5, n_head=14, n_kv_head=2,
                                 head_dim=64, max_len=64, base=1e6),
    "tmac_kv_page_bounds": dict(kv_dtype=0, k_pages=P, n_pages=9, block_table=2 * P, max_pages=4, first_rows=3 * P,
                                lengths=4 * P, bounds=5 * P, n_seq=3, n_kv_head=2, head_dim=64, max_new=20),
    "tmac_select_pages": dict(q=P, bounds=2 * P, n_pages=9, block_table=3 * P, max_pages=40, lengths=4 * P,
                              selected=5 * P, n_seq=3, n_head=14, n_kv_head=2, head_dim=64, max_len=640, top=5, first=1,
                              last=2),
    "tmac_attention_decode_selected": dict(kv_dtype=0, q=P, k_pages=2 * P, v_pages=3 * P, n_pages=9, block_table=4 * P,
                                           max_pages=4, lengths=5 * P, selected=6 * P, top=5, out=7 * P, n_seq=3,
                                           n_head=14, n_kv_head=2, head_dim=64),
    "tmac_attention_decode_shared": dict(kv_dtype=0, q=P, k_pages=2 * P, v_pages=3 * P, n_pages=9, block_table=4 * P,
                                         max_pages=40, lengths=5 * P, group_starts=6 * P, prefix_lens=7 * P, n_groups=2,
                                         out=8 * P, n_seq=30, n_head=14, n_kv_head=2, head_dim=64, max_prefix=300,
                                         max_tail=100),
}
# null is a legal value of these
MAY_BE_NULL = {("tmac_kv_page_bounds", "first_rows")}
POINTERS = [(n, k) for n, kw in GOOD.items() for k, v in kw.items() if isinstance(v, int) and v >= P]
ALIGN16 = {"q", "q_out", "k", "v", "k_pages", "v_pages", "bounds", "out"}


@pytest.fixture(scope="module")
def fake():
    if not os.path.exists(FAKE):
        pytest.skip("tests/cpp is not built")
    return Fake()


@pytest.mark.parametrize("name", sorted(GOOD))
def test_accepted(fake, name):
    rc, launches = fake.call(name)
    assert rc == TMAC_OK and launches


@pytest.mark.parametrize("name,arg", POINTERS)
def test_null_and_misaligned_pointers(fake, name, arg):
    rc, launches = fake.call(name, **{arg: None})
    if (name, arg) in MAY_BE_NULL:
        assert rc == TMAC_OK
    else:
        assert rc == TMAC_ERR_NULL_POINTER and not launches
    for off in (4, 8) if arg in ALIGN16 else (1, 2):
        rc, launches = fake.call(name, **{arg: GOOD[name][arg] + off})
        assert rc == TMAC_ERR_MISALIGNED and not launches, off


@pytest.mark.parametrize("name", sorted(GOOD))
def test_shapes_outside_the_domain(fake, name):
    good = GOOD[name]
    for head_dim in (0, 32, 63, 128):
        assert fake.call(name, head_dim=head_dim) == (TMAC_ERR_UNSUPPORTED, [])
    for bad in (0, -2):
        assert fake.call(name, n_kv_head=bad) == (TMAC_ERR_INVALID_ARG, [])
    if "n_head" in good:
        for bad in (0, -14, 13):
            assert fake.call(name, n_head=bad) == (TMAC_ERR_INVALID_ARG, [])
        rc, launches = fake.call(name, n_head=34, **({"q_stride": 34 * 64} if "q_stride" in good else {}))
        assert rc == (TMAC_OK if name == "tmac_kv_append_paged" else TMAC_ERR_UNSUPPORTED)
        assert fake.call(name, n_head=16, n_kv_head=1, **({"q_stride": 1024} if "q_stride" in good else {}))[0] == TMAC_OK
    for arg in ("n_pages", "max_pages"):
        for bad in (0, -1):
            assert fake.call(name, **{arg: bad}) == (TMAC_ERR_INVALID_ARG, [])
    assert fake.call(name, n_seq=-1) == (TMAC_ERR_INVALID_ARG, [])
    assert fake.call(name, n_seq=0) == (TMAC_OK, [])
    if "kv_dtype" in good:
        for bad in (-1, 4):
            assert fake.call(name, kv_dtype=bad) == (TMAC_ERR_INVALID_ARG, [])


@pytest.mark.parametrize("name,kw,status", [
    ("tmac_kv_append_paged", dict(max_len=0), TMAC_ERR_INVALID_ARG),
    ("tmac_kv_append_paged", dict(max_len=65), TMAC_ERR_INVALID_ARG),
    ("tmac_kv_append_paged", dict(n_rows=-1), TMAC_ERR_INVALID_ARG),
    ("tmac_kv_append_paged", dict(q_stride=892), TMAC_ERR_INVALID_ARG),
    ("tmac_kv_append_paged", dict(k_stride=124), TMAC_ERR_INVALID_ARG),
    ("tmac_kv_append_paged", dict(v_stride=0), TMAC_ERR_INVALID_ARG),
    ("tmac_kv_append_paged", dict(q_stride=898), TMAC_ERR_MISALIGNED),
    ("tmac_kv_append_paged", dict(k_stride=130), TMAC_ERR_MISALIGNED),
    ("tmac_kv_append_paged", dict(base=0.0), TMAC_ERR_INVALID_ARG),
    ("tmac_kv_append_paged", dict(base=float("nan")), TMAC_ERR_INVALID_ARG),
    ("tmac_kv_append_paged", dict(base=float("inf")), TMAC_ERR_INVALID_ARG),
    # q_out one row behind q, q_out = q with rows further apart than q_out's
    ("tmac_kv_append_paged", dict(q_out=P + 896 * 4), TMAC_ERR_INVALID_ARG),
    ("tmac_kv_append_paged", dict(q_out=P, q_stride=1152), TMAC_ERR_INVALID_ARG),
    ("tmac_kv_append_paged", dict(q_out=3 * P + 4 * 127 * 4), TMAC_ERR_INVALID_ARG),  # over k, over v
    ("tmac_kv_append_paged", dict(q_out=4 * P - 5 * 896 * 4 + 16), TMAC_ERR_INVALID_ARG),
    ("tmac_kv_page_bounds", dict(max_new=-1), TMAC_ERR_INVALID_ARG),
    ("tmac_select_pages", dict(max_len=0), TMAC_ERR_INVALID_ARG),
    ("tmac_select_pages", dict(max_len=641), TMAC_ERR_INVALID_ARG),
    ("tmac_select_pages", dict(top=0, first=0, last=0), TMAC_ERR_INVALID_ARG),
    ("tmac_select_pages", dict(first=-1), TMAC_ERR_INVALID_ARG),
    ("tmac_select_pages", dict(last=-1), TMAC_ERR_INVALID_ARG),
    ("tmac_select_pages", dict(first=3, last=3), TMAC_ERR_INVALID_ARG),
    ("tmac_select_pages", dict(first=2 ** 31 - 1, last=2 ** 31 - 1), TMAC_ERR_INVALID_ARG),
    ("tmac_attention_decode_selected", dict(top=0), TMAC_ERR_INVALID_ARG),
    ("tmac_attention_decode_shared", dict(n_groups=-1), TMAC_ERR_INVALID_ARG),
    ("tmac_attention_decode_shared", dict(max_prefix=-1), TMAC_ERR_INVALID_ARG),
    ("tmac_attention_decode_shared", dict(max_tail=-1), TMAC_ERR_INVALID_ARG),
    # more units of work than a grid can number
    ("tmac_kv_page_bounds", dict(n_seq=2 ** 31 - 1, max_pages=2 ** 27, max_new=2 ** 31 - 1), TMAC_ERR_INVALID_ARG),
    ("tmac_select_pages", dict(n_seq=2 ** 31 - 1, max_pages=2 ** 27, max_len=2 ** 31 - 1), TMAC_ERR_INVALID_ARG),
    ("tmac_attention_decode_selected", dict(n_seq=2 ** 31 - 1), TMAC_ERR_INVALID_ARG),
    ("tmac_attention_decode_shared", dict(n_seq=2 ** 31 - 1), TMAC_ERR_INVALID_ARG),
    # more threads than 32 bits
    ("tmac_kv_append_paged", dict(q=None, q_out=None, n_rows=2 ** 30), TMAC_ERR_INVALID_ARG),
    ("tmac_kv_page_bounds", dict(n_seq=2 ** 25), TMAC_ERR_INVALID_ARG),
    ("tmac_select_pages", dict(n_seq=2 ** 24, top=40), TMAC_ERR_INVALID_ARG),
    ("tmac_attention_decode_selected", dict(n_seq=2 ** 24), TMAC_ERR_INVALID_ARG),
])
def test_refused(fake, name, kw, status):
    assert fake.call(name, **kw) == (status, [])


def test_legal_edges(fake):
    ok = lambda name, **kw: fake.call(name, **kw)[0] == TMAC_OK  # noqa: E731
    assert ok("tmac_kv_append_paged", q=None, q_out=None)
    assert ok("tmac_kv_append_paged", q_out=P)                       # in place
    assert ok("tmac_kv_append_paged", n_rows=1, q_out=P, q_stride=0, k_stride=0, v_stride=0)  # strides of one row
    assert fake.call("tmac_kv_append_paged", n_rows=0) == (TMAC_OK, [])
    assert fake.call("tmac_kv_page_bounds", max_new=0) == (TMAC_OK, [])
    assert ok("tmac_attention_decode_shared", n_groups=0, group_starts=None, prefix_lens=None)
    # bounds beyond the table are the table's
    assert fake.call("tmac_attention_decode_shared", max_prefix=2 ** 31 - 1, max_tail=2 ** 31 - 1) == fake.call(
        "tmac_attention_decode_shared", max_prefix=640, max_tail=640)
    # no rows possible: the last launch alone writes the zero outputs
    rc, launches = fake.call("tmac_attention_decode_shared", max_prefix=0, max_tail=0)
    assert rc == TMAC_OK and [k for k, _ in launches] == ["tmac_tail_finish_f32"]
    # every list holds all pages: no scores
    rc, launches = fake.call("tmac_select_pages", top=40)
    assert rc == TMAC_OK and [k for k, _ in launches] == ["tmac_select_pages_256"]


def test_growth_is_refused_while_capturing(fake):
    """A workspace that would have to grow under a capture: no launch."""
    fake.lib.fake_set_capturing(1)
    try:
        big = dict(n_seq=4096, max_pages=4096)
        assert fake.call("tmac_select_pages", max_len=65536, **big) == (TMAC_ERR_CAPTURE, [])
        assert fake.call("tmac_attention_decode_shared", max_prefix=65536, max_tail=65536, **big) == (TMAC_ERR_CAPTURE, [])
        assert fake.call("tmac_kv_append_paged", max_pages=4096, max_len=65536, base=12345.0) == (TMAC_ERR_CAPTURE, [])
    finally:
        fake.lib.fake_set_capturing(0)


def test_bounds_grid_covers_every_start_in_a_page(fake):
    """max_new rows from any row of a page on touch at most the pages the grid holds."""
    for new in list(range(1, 40)) + [1000, 1001]:
        _, [(_, grid)] = fake.call("tmac_kv_page_bounds", max_new=new, max_pages=4096, n_seq=1, n_kv_head=4)
        pages = max((first + new - 1) // 16 + 1 for first in range(16))
        assert pages <= grid < pages + 1  # 4 kv heads: one page a workgroup of 4 waves
        _, [(_, grid)] = fake.call("tmac_kv_page_bounds", max_new=new, max_pages=4096, n_seq=1, n_kv_head=4, first_rows=None)
        assert grid == -(-new // 16)


def test_shared_grid(fake):
    """The prefix kernel's workgroups share the units of any grouping: a multiple of the eight dies, no more than one
    per CU (256) and, where every grouping has fewer units, no more than those."""
    for n_seq, n_groups in ((1, 1), (9, 1), (10, 1), (30, 2), (30, 30), (200, 7), (2000, 1)):
        cuts = [[i * n_seq // n_groups for i in range(n_groups + 1)], [0] * n_groups + [n_seq],
                list(range(n_groups)) + [n_seq], [0] + [n_seq - n_groups + i for i in range(1, n_groups + 1)]]
        need = max(sum(-(-(b - a) * 7 // 64) for a, b in zip(c, c[1:])) for c in cuts)
        args = dict(n_seq=n_seq, n_groups=n_groups, max_tail=0, max_pages=16384)
        room = (9 * 2 ** 15 if n_seq >= 64 else 3 * 2 ** 16) // (2 * n_seq)  # 2 kv heads: rows that every sequence reads itself
        rc, launches = fake.call("tmac_attention_decode_shared", max_prefix=min(room, 384), **args)
        assert rc == TMAC_OK and launches[0][0].startswith("tmac_tail_")
        rc, launches = fake.call("tmac_attention_decode_shared", max_prefix=max(room, 384) + 1, **args)
        assert rc == TMAC_OK and launches[0][0] == "tmac_prefix_f32"
        assert launches[0][1] % 8 == 0 and min(2 * need, 256) <= launches[0][1] <= 256


def test_append_heads_of_a_workgroup(fake):
    """A workgroup numbers the heads of its rows in 32 bits: more are refused."""
    big = dict(q=None, q_out=None, n_rows=1, k_stride=0, v_stride=0, n_seq=1)
    assert fake.call("tmac_kv_append_paged", n_head=2 ** 30, n_kv_head=2 ** 30, **big) == (TMAC_ERR_INVALID_ARG, [])
    assert fake.call("tmac_kv_append_paged", n_head=2 ** 30 - 16, n_kv_head=2 ** 30 - 16, **big) == (TMAC_ERR_INVALID_ARG, [])
    assert fake.call("tmac_kv_append_paged", n_head=2 ** 30 - 17, n_kv_head=2 ** 30 - 17, **big)[0] == TMAC_OK


def test_most_sequences(fake):
    """The limits the header names: 65,535 sequences, and kv heads where a grid numbers them."""
    for name in ("tmac_select_pages", "tmac_attention_decode_shared"):
        assert fake.call(name, n_seq=65535)[0] == TMAC_OK
        assert fake.call(name, n_seq=65536) == (TMAC_ERR_INVALID_ARG, [])
    assert fake.call("tmac_attention_decode_shared", n_head=65535, n_kv_head=65535)[0] == TMAC_OK
    assert fake.call("tmac_attention_decode_shared", n_head=65536, n_kv_head=65536) == (TMAC_ERR_INVALID_ARG, [])
    # the others have no such limit
    assert fake.call("tmac_kv_append_paged", n_seq=65536)[0] == TMAC_OK
    assert fake.call("tmac_kv_page_bounds", n_seq=65536)[0] == TMAC_OK
    assert fake.call("tmac_attention_decode_selected", n_seq=65536)[0] == TMAC_OK


def lists(fake, n_sk, top, dt):
    """(kernel, workgroups a list) of an attention over n_sk lists."""
    rc, launches = fake.call("tmac_attention_decode_selected", kv_dtype=dt, n_seq=n_sk, n_head=7, n_kv_head=1, top=top)
    assert rc == TMAC_OK and launches[0][1] % n_sk == 0
    return launches[0][0], launches[0][1] // n_sk


@pytest.mark.parametrize("dt", range(4))
def test_split_lists_fit_the_card_at_once(fake, dt):
    """A split list has no more workgroups than all lists find room for at once (two a CU, 256 CUs): one more each would
    be a second round.  From 341 lists on no list is split, and up to one a CU a split one has two at least."""
    for n_sk in list(range(1, 260)) + [300, 340, 342, 400, 511, 512, 600]:
        for top in (1, 16, 64, 100, 500, 2000, 100000):
            kernel, each = lists(fake, n_sk, top, dt)
            assert each == 1 or each * n_sk <= 512 or (n_sk > 256 and each == 2 and 3 * n_sk <= 1024)


@pytest.mark.parametrize("dt", range(4))
def test_long_lists_are_split_where_cus_would_be_idle(fake, dt):
    """No step at half the CUs: a long list is split below and above it, a short one is not, and the length between
    grows with the lists."""
    for n_sk in (1, 60, 127, 128, 129, 130, 144, 160, 170):
        assert lists(fake, n_sk, 2000, dt)[1] >= 3
        assert lists(fake, n_sk, 8, dt)[1] == 1
    most = []
    for n_sk in (64, 96, 112, 128, 129, 150, 170):
        most.append(max(top for top in range(8, 1200, 4) if lists(fake, n_sk, top, dt)[1] == 1))
    assert most == sorted(most) and most[4] < 1.1 * most[3] + 4
    # own rows by the same rule
    for n_seq in (72, 85):
        rc, launches = fake.call("tmac_attention_decode_shared", kv_dtype=dt, n_seq=n_seq, n_groups=0, max_pages=1024,
                                 max_prefix=0, max_tail=16384)
        assert rc == TMAC_OK and launches[0][0].startswith("tmac_tail_") and launches[0][1] == 3, launches


def test_q8_prefixes_of_many_sequences_are_read_once(fake):
    """More Q8_0 readers than CUs convert a prefix of 700 rows slower than one launch more; other types do not."""
    for dt, n_seq, n_kv, rows, first in ((3, 200, 2, 700, "prefix"), (3, 45, 8, 800, "prefix"), (3, 200, 2, 500, "tail"),
                                         (3, 128, 2, 1100, "tail"), (1, 200, 2, 700, "tail"), (2, 45, 8, 800, "tail")):
        rc, launches = fake.call("tmac_attention_decode_shared", kv_dtype=dt, n_seq=n_seq, n_head=n_kv, n_kv_head=n_kv,
                                 n_groups=1, max_pages=1024, max_prefix=rows, max_tail=64)
        assert rc == TMAC_OK and launches[0][0].startswith("tmac_" + first), (dt, n_seq, rows, launches)
