"""The serving operators on paged caches (tmac_kv_append_paged, tmac_kv_page_bounds,
tmac_select_pages, tmac_attention_decode_selected, tmac_attention_decode_shared) against plain
64-bit forms.

Appended rows, bounds and selections are compared bit for bit: rotation and storage are the
oracle's, a maximum rounded outward has one value, and scores are summed in 64 bits and rounded
once.  Attention outputs meet the framework's contract |gpu - ref| <= 2e-5 + 1e-4 |ref| on the
widened cache, and their 2-norm is within 2e-6 of the reference's: a score of 64 products of
N(0, 1) values carries 64 * 2^-24 * |q| |k| / 8 at most, about 8 |q||k| 2^-24 < 4e-6 * 64 / 8 in the
worst case and its square root, 5e-7, at random; the weights and the sums add three roundings of
2^-24 each, and a 2-norm over thousands of values sees the random size (the worst case of all
64-term sums at once would be 3e-5, inside the elementwise contract)."""
import numpy as np
import pytest

import oracle
import tmac_attn
from conftest import assert_close
from serving import (ALL_DT, BF16, F16, F32, PR, Q8, attend64, bounds_ref, decode64, make_pool, outward, select_ref,
                     store, tables, widen)

pytestmark = pytest.mark.gpu
FAULT = tmac_attn.TMAC_ERR_DEVICE_FAULT
HEADS = [(14, 2), (1, 1), (8, 8), (16, 1), (12, 4), (33, 3)]  # groups of 7, 1, 1, 16, 3, 11


def close(got, ref, what):
    assert_close(got, ref, what)
    norm = np.linalg.norm(ref)
    if norm:
        off = np.linalg.norm(got.astype(np.float64) - ref) / norm
        assert off <= 2e-6, (what, off)


def no_fault(ctx):
    assert ctx.check_device_error() == 0


# ---- append ---------------------------------------------------------------------------------

def append_ref(q, k, v, kp, vp, table, starts, pos, n_kv, dt, n_pages, max_len, q_out, base=1e6):
    """(q_out, k pool, v pool) as the definition gives them, bit for bit, on copies."""
    kp, vp, q_out = kp.copy(), vp.copy(), q_out.copy()
    for s in range(len(pos)):
        for t in range(starts[s], starts[s + 1]):
            p = int(pos[s]) + t - starts[s]
            if not 0 <= p < max_len:
                continue
            if q is not None:
                q_out[t] = oracle.rope_heads(q[t], q.shape[1], 64, p, base).reshape(q.shape[1], 64)
            page = table[s, p // PR]
            if 0 <= page < n_pages:
                kp[page, p % PR] = store(oracle.rope_heads(k[t], n_kv, 64, p, base).reshape(n_kv, 64), dt)
                vp[page, p % PR] = store(v[t], dt)
    return q_out, kp, vp


def run_append(ctx, dt, nh, nkv, counts, pos, seed, fused=False, in_place=False, with_q=True, lead=0, behind=0,
               table=None, n_pages=None, max_len=None, base=1e6, width=0, stream=None):
    rng = np.random.default_rng(seed)
    counts, pos = np.asarray(counts), np.asarray(pos)
    if table is None:
        table, n_pages = tables(rng, np.where(counts > 0, pos + counts, 0), extra_pages=2, width=width)
    max_len = max_len or table.shape[1] * PR
    starts = (lead + np.concatenate([[0], np.cumsum(counts)])).astype(np.int32)
    rows = int(starts[-1]) + behind
    x = oracle.normal(seed, (rows, nh + 2 * nkv, 64))
    x *= np.exp2(rng.uniform(-3, 3, (rows, 1, 1))).astype(np.float32)
    q, k, v = x[:, :nh], x[:, nh:nh + nkv], x[:, nh + nkv:]
    kp, _ = make_pool(seed + 1, n_pages, nkv, dt)
    vp, _ = make_pool(seed + 2, n_pages, nkv, dt)
    before = q if in_place else np.full((rows, nh, 64), 7.5, np.float32)
    dk_p, dv_p = ctx.upload(kp), ctx.upload(vp)
    dt_, ds, dp = ctx.upload(table), ctx.upload(starts), ctx.upload(pos.astype(np.int32))
    row = (nh + 2 * nkv) * 64
    if fused:
        dx = ctx.upload(x)
        dq, dk, dv, qs, ks = dx.ptr, dx.at(nh * 64), dx.at((nh + nkv) * 64), row, row
    else:
        dq, dk, dv = (ctx.upload(np.ascontiguousarray(y)) for y in (q, k, v))
        qs, ks = nh * 64, nkv * 64
    dout = dq if in_place else ctx.upload(before)
    ctx.kv_append_paged(dq if with_q else None, qs, dout if with_q else None, dk, ks, dv, ks, dk_p, dv_p, n_pages, dt_,
                        table.shape[1], ds, dp, len(counts), rows, nh, nkv, 64, max_len, base, stream=stream,
                        kv_dtype=dt)
    if stream is not None:
        ctx.synchronize(stream)
    ref = append_ref(q if with_q else None, k, v, kp, vp, table, starts, pos, nkv, dt, n_pages, max_len, before, base)
    got = dout.numpy().reshape(before.shape), dk_p.numpy(), dv_p.numpy()
    for name, a, b in zip(("q", "k", "v"), got, ref):
        np.testing.assert_array_equal(a.view(np.uint8), np.ascontiguousarray(b).view(np.uint8), err_msg=name)


@pytest.mark.parametrize("dt", ALL_DT)
@pytest.mark.parametrize("nh,nkv", HEADS)
def test_append_shapes(ctx, dt, nh, nkv):
    run_append(ctx, dt, nh, nkv, [1, 0, 37, 16, 0, 0, 5, 1], [0, 3, 11, 16, 0, 9, 255, 15], 100 + nh, fused=dt % 2 == 1)
    no_fault(ctx)


@pytest.mark.parametrize("dt", ALL_DT)
def test_append_one_row(ctx, dt):
    for pos in (0, 15, 16, 4000):
        run_append(ctx, dt, 14, 2, [1], [pos], 110 + pos)
    no_fault(ctx)


@pytest.mark.parametrize("dt", [F32, Q8])
def test_append_many_rows_per_workgroup(ctx, dt):
    """More rows than eight per CU: workgroups of several rows, sequences that begin and end inside one,
    padding before and behind."""
    rng = np.random.default_rng(5)
    counts = rng.integers(0, 40, 700)
    counts[rng.random(700) < 0.3] = 0
    run_append(ctx, dt, 2, 1, counts, rng.integers(0, 200, 700), 120, lead=5, behind=9, fused=True)
    no_fault(ctx)


def test_append_in_place_and_without_queries(ctx):
    run_append(ctx, BF16, 14, 2, [3, 20], [7, 100], 130, in_place=True)
    run_append(ctx, F32, 14, 2, [3, 20], [7, 100], 131, with_q=False)
    run_append(ctx, F32, 14, 2, [3, 20], [7, 100], 132, base=10000.0)
    no_fault(ctx)


def test_append_skips_bad_positions_and_pages(ctx):
    """Positions outside [0, max_len) are skipped (bit 0), rows of pages outside the pool are rotated but not
    stored (bit 2); everything else is written, nothing else is touched."""
    table = np.array([[0, 1, 2], [3, 4, 5]], np.int32)
    run_append(ctx, F32, 14, 2, [20, 4], [-3, 46], 140, table=table, n_pages=6, max_len=48)
    assert ctx.check_device_error() == FAULT
    run_append(ctx, Q8, 14, 2, [48, 4], [0, 30], 141, table=table, n_pages=6, max_len=33)
    assert ctx.check_device_error() == FAULT
    bad = table.copy()
    bad[0, 1], bad[1, 0] = -1, 6
    run_append(ctx, BF16, 14, 2, [40, 20], [2, 4], 142, table=bad, n_pages=6)
    assert ctx.check_device_error() == FAULT
    no_fault(ctx)


def test_append_equals_the_layer_step(ctx):
    """The bytes a layer step writes for a token are the bytes an append writes, for every cache type."""
    n, nh, nkv = 5, 14, 2
    rng = np.random.default_rng(9)
    pos = np.array([0, 15, 16, 77, 300], np.int32)
    table, n_pages = tables(rng, pos + 1)
    q, k, v = oracle.normal(150, (n, nh * 64)), oracle.normal(151, (n, nkv * 64)), oracle.normal(152, (n, nkv * 64))
    for dt in ALL_DT:
        kp, _ = make_pool(153, n_pages, nkv, dt)
        one = [ctx.upload(kp), ctx.upload(kp)]
        two = [ctx.upload(kp), ctx.upload(kp)]
        dq, dk, dv, dtab, dpos, dout = *(ctx.upload(x) for x in (q, k, v, table, pos)), ctx.empty((n, nh * 64))
        starts = ctx.upload(np.arange(n + 1, dtype=np.int32))
        ctx.layer_attention_paged(dq, dk, dv, *one, n_pages, dtab, table.shape[1], dpos, dout, n, nh, nkv, 64, 304,
                                  kv_dtype=dt)
        ctx.kv_append_paged(None, 0, None, dk, 128, dv, 128, *two, n_pages, dtab, table.shape[1], starts, dpos, n, n, nh,
                            nkv, 64, 304, kv_dtype=dt)
        for a, b in zip(one, two):
            np.testing.assert_array_equal(a.numpy().view(np.uint8), b.numpy().view(np.uint8))
    no_fault(ctx)


# ---- page bounds ----------------------------------------------------------------------------

def bf16_values(u):
    return (u.astype(np.uint32) << 16).view(np.float32)


@pytest.mark.parametrize("dt", ALL_DT)
@pytest.mark.parametrize("nkv", [1, 2, 5])
def test_bounds(ctx, dt, nkv):
    rng = np.random.default_rng(20 + nkv)
    lens = np.array([1, 16, 17, 0, 250, 33, 64], np.int32)
    table, n_pages = tables(rng, lens, extra_pages=3)
    kp, kw = make_pool(200 + nkv, n_pages, nkv, dt, spread=6)
    before = outward(oracle.normal(201, (n_pages, nkv, 2, 64)), True)
    for first in (None, np.zeros(7, np.int32), np.array([0, 15, 16, 0, 100, 40, -5], np.int32), lens - 1):
        db = ctx.upload((before.view(np.uint32) >> 16).astype(np.uint16))
        df = None if first is None else ctx.upload(first.astype(np.int32))
        new = int((lens - (0 if first is None else np.maximum(first, 0))).max())
        ctx.kv_page_bounds(ctx.upload(kp), n_pages, ctx.upload(table), table.shape[1], df, ctx.upload(lens), db, len(lens),
                           nkv, 64, new, kv_dtype=dt)
        np.testing.assert_array_equal(bf16_values(db.numpy()), bounds_ref(kw, before, table, first, lens, nkv))
    no_fault(ctx)


@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_bounds_of_infinities_nan_and_borders(ctx, dt):
    """Values on and next to bf16 borders, signed zeros, tiny and huge values, infinities and NaN; what lies behind the
    length is not looked at."""
    kp, _ = make_pool(210, 2, 1, F32)
    x = kp.copy()
    x[0, 3, 0, :8] = [np.inf, -np.inf, np.nan, 3.4e38, -3.4e38, 1e-40, -1e-40, 0.0]
    x[0, :, 0, 8] = 1.0
    x[0, :, 0, 9] = np.nextafter(np.float32(1), np.float32(2))
    x[0, :, 0, 10] = -np.nextafter(np.float32(1), np.float32(2))
    x[0, :, 0, 11] = -0.0
    x[1, 5:, 0, :] = np.nan  # behind the length
    x[1, 7, 0, 5] = np.inf
    with np.errstate(over="ignore"):
        s = store(x, dt)
        w = widen(s, dt)
    table, lens = np.array([[0, 1]], np.int32), np.array([21], np.int32)
    db = ctx.upload(np.zeros((2, 1, 2, 64), np.uint16))
    ctx.kv_page_bounds(ctx.upload(s), 2, ctx.upload(table), 2, None, ctx.upload(lens), db, 1, 1, 64, 21, kv_dtype=dt)
    got = bf16_values(db.numpy())
    assert np.isfinite(got).all()
    np.testing.assert_array_equal(got, bounds_ref(w, np.zeros((2, 1, 2, 64), np.float32), table, None, lens, 1))
    no_fault(ctx)


def test_bounds_errors(ctx):
    table, lens = np.array([[0, 1], [2, 9], [3, 4]], np.int32), np.array([30, 30, 40], np.int32)
    kp, kw = make_pool(220, 5, 2, F32)
    before = np.zeros((5, 2, 2, 64), np.float32)
    db = ctx.upload(np.zeros((5, 2, 2, 64), np.uint16))
    # sequence 1's second page is outside the pool, sequence 2 is longer than its table
    ctx.kv_page_bounds(ctx.upload(kp), 5, ctx.upload(table), 2, None, ctx.upload(lens), db, 3, 2, 64, 40)
    ref = bounds_ref(kw, before, table[:1], None, lens[:1], 2)
    ref = bounds_ref(kw, ref, table[1:2], None, [16], 2)
    np.testing.assert_array_equal(bf16_values(db.numpy()), ref)
    assert ctx.check_device_error() == FAULT
    # more new rows than max_new: that sequence is skipped
    db = ctx.upload(np.zeros((5, 2, 2, 64), np.uint16))
    ctx.kv_page_bounds(ctx.upload(kp), 5, ctx.upload(table), 2, ctx.upload(np.array([10, 0, 0], np.int32)),
                       ctx.upload(np.array([15, 6, 0], np.int32)), db, 3, 2, 64, 5)
    np.testing.assert_array_equal(bf16_values(db.numpy()), bounds_ref(kw, before, table, [10], [15], 2))
    assert ctx.check_device_error() == FAULT
    no_fault(ctx)


# ---- selection ------------------------------------------------------------------------------

def run_select(ctx, q, b, table, lens, nkv, top, first, last, max_len=None):
    n, nh = q.shape[:2]
    n_pages = b.shape[0]
    dsel = ctx.upload(np.full((n, nkv, top), 77, np.int32))
    ctx.select_pages(ctx.upload(q), ctx.upload((b.view(np.uint32) >> 16).astype(np.uint16)), n_pages, ctx.upload(table),
                     table.shape[1], ctx.upload(np.asarray(lens, np.int32)), dsel, n, nh, nkv, 64,
                     max_len or table.shape[1] * PR, top, first, last)
    got = dsel.numpy()
    if not max_len and table.shape[1] <= 512 and (np.asarray(lens) <= table.shape[1] * PR).all():
        # short lists are scored and selected by one workgroup each: the same from a table too long for that
        wide = np.pad(table, ((0, 0), (0, 513 - table.shape[1])), constant_values=2 ** 30)
        np.testing.assert_array_equal(run_select(ctx, q, b, wide, lens, nkv, top, first, last), got)
    return got


def random_bounds(seed, n_pages, nkv):
    mid, half = oracle.normal(seed, (n_pages, nkv, 64)), np.abs(oracle.normal(seed + 1, (n_pages, nkv, 64))) + 1
    return np.stack([outward(mid + half, True), outward(mid - half, False)], 2)


@pytest.mark.parametrize("nh,nkv", HEADS + [(4, 2), (6, 2), (10, 2), (12, 2), (8, 1), (26, 2)])
def test_select_groups(ctx, nh, nkv):
    rng = np.random.default_rng(nh)
    lens = np.array([2000, 0, 5, 161, 160, 176, 1023], np.int32)
    table, n_pages = tables(rng, lens)
    q, b = oracle.normal(300 + nh, (len(lens), nh, 64)), random_bounds(301 + nh, n_pages, nkv)
    for top, first, last in ((10, 1, 1), (10, 0, 0), (3, 1, 2), (64, 2, 5), (1, 0, 0), (200, 1, 1)):
        got = run_select(ctx, q, b, table, lens, nkv, top, first, last)
        np.testing.assert_array_equal(got, select_ref(q, b, table, lens, nkv, top, first, last))
    no_fault(ctx)


def test_select_long(ctx):
    """More pages than one workgroup scores or one pass of the list holds, an odd count, a large budget."""
    rng = np.random.default_rng(3)
    lens = np.array([50001, 32768, 20000], np.int32)
    table, n_pages = tables(rng, lens)
    q, b = oracle.normal(310, (3, 14, 64)), random_bounds(311, n_pages, 2)
    for top in (7, 513, 3000):
        np.testing.assert_array_equal(run_select(ctx, q, b, table, lens, 2, top, 1, 1),
                                      select_ref(q, b, table, lens, 2, top, 1, 1))
    no_fault(ctx)


@pytest.mark.parametrize("n,longest", [(70, 4000), (256, 1100), (300, 1100), (1030, 300)])
def test_select_many_lists(ctx, n, longest):
    """More steps of pages than waves that fit the card, dealt out over a wave's sequences; more sequences than are
    dealt out.  The lengths are ragged and the first, the last and a run of others are empty."""
    rng = np.random.default_rng(n)
    lens = rng.integers(1, longest + 1, n).astype(np.int32)
    lens[[0, 40, 41, 42, n - 1]] = 0
    lens[50] = longest
    table, n_pages = tables(rng, lens)
    q, b = oracle.normal(312 + n, (n, 6, 64)), random_bounds(313 + n, n_pages, 2)
    np.testing.assert_array_equal(run_select(ctx, q, b, table, lens, 2, 9, 1, 1),
                                  select_ref(q, b, table, lens, 2, 9, 1, 1))
    no_fault(ctx)


def test_select_more_pages_than_registers_hold(ctx):
    rng = np.random.default_rng(4)
    lens = np.array([140001, 131073], np.int32)
    table, n_pages = tables(rng, lens)
    q, b = oracle.normal(316, (2, 7, 64)), random_bounds(317, n_pages, 1)
    for top, first, last in ((1000, 1, 1), (1, 0, 0), (8700, 0, 3)):
        np.testing.assert_array_equal(run_select(ctx, q, b, table, lens, 1, top, first, last),
                                      select_ref(q, b, table, lens, 1, top, first, last))
    no_fault(ctx)


def test_select_ties_go_to_the_lower_page(ctx):
    """A zero query (all scores 0), equal bounds on many pages, and scores that differ only beyond fp32."""
    rng = np.random.default_rng(4)
    lens = np.array([1600, 1600, 1600], np.int32)
    table, n_pages = tables(rng, lens)
    b = random_bounds(320, n_pages, 2)
    b[table[1, 10:90]] = b[table[1, 10]]
    b[table[2]] = b[table[2, 0]]
    b[table[2, 50:], :, :, 0] *= np.float32(1 + 2.0 ** -7)  # a bf16 step in one dim, weighed by a tiny query value
    q = oracle.normal(321, (3, 14, 64))
    q[0] = 0
    q[2, :, 0] = 1e-9
    for top in (5, 40, 99):
        got = run_select(ctx, q, b, table, lens, 2, top, 0, 0)
        np.testing.assert_array_equal(got, select_ref(q, b, table, lens, 2, top, 0, 0))
        assert (got[0] == np.arange(top)).all()
    no_fault(ctx)


def test_select_extreme_values(ctx):
    """Scores that overflow fp32 become infinities of their order; negative scores sort below positive ones; a query
    that is not finite still gives valid distinct pages."""
    rng = np.random.default_rng(5)
    lens = np.array([800, 800], np.int32)
    table, n_pages = tables(rng, lens)
    b = random_bounds(330, n_pages, 2)
    b[table[0, ::3]] *= np.float32(1e38)
    b[table[0, 1::3]] = -np.abs(b[table[0, 1::3]])[:, :, ::-1]
    b = outward(b, True)
    q = oracle.normal(331, (2, 14, 64)) * np.float32(10)
    with np.errstate(over="ignore"):
        np.testing.assert_array_equal(run_select(ctx, q, b, table, lens, 2, 12, 1, 1),
                                      select_ref(q, b, table, lens, 2, 12, 1, 1))
    q[1, 3, 5], q[1, 9, 1] = np.nan, np.inf
    got = run_select(ctx, q, b, table, lens, 2, 12, 1, 1)
    for h in range(2):
        assert len(set(got[1, h])) == 12 and got[1, h].min() == 0 and got[1, h].max() == 49
    no_fault(ctx)


def test_select_errors(ctx):
    rng = np.random.default_rng(6)
    lens = np.array([400, 400], np.int32)
    table, n_pages = tables(rng, lens)
    q, b = oracle.normal(340, (2, 14, 64)), random_bounds(341, n_pages, 2)
    got = run_select(ctx, q, b, table, [400, 320], 2, 5, 1, 1, max_len=320)
    assert (got[0] == -1).all()
    np.testing.assert_array_equal(got[1:], select_ref(q[1:], b, table[1:], [320], 2, 5, 1, 1))
    assert ctx.check_device_error() == FAULT
    bad = table.copy()
    bad[0, 7], bad[1, 3] = -4, n_pages  # clamped to the pool's first and last page
    got = run_select(ctx, q, b, bad, lens, 2, 5, 1, 1)
    bad[0, 7], bad[1, 3] = 0, n_pages - 1
    np.testing.assert_array_equal(got, select_ref(q, b, bad, lens, 2, 5, 1, 1))
    assert ctx.check_device_error() == FAULT
    no_fault(ctx)


# ---- attention over selected pages ----------------------------------------------------------

def rows_of_list(table, lens, sel):
    def rows(s, h):
        r = [PR * j + i for j in sel[s, h] if j >= 0 for i in range(PR) if PR * j + i < lens[s]]
        r = np.array(r, np.int64)
        return table[s, r // PR], r % PR
    return rows


def run_selected(ctx, q, kp, vp, table, lens, sel, nkv, dt, stream=None):
    n, nh = q.shape[:2]
    dout = ctx.upload(np.full(q.shape, 9.0, np.float32))
    ctx.decode_selected(ctx.upload(q), ctx.upload(kp), ctx.upload(vp), kp.shape[0], ctx.upload(table), table.shape[1],
                        ctx.upload(np.asarray(lens, np.int32)), ctx.upload(sel), sel.shape[2], dout, n, nh, nkv, 64,
                        stream=stream, kv_dtype=dt)
    if stream is not None:
        ctx.synchronize(stream)
    return dout.numpy()


def random_lists(rng, lens, nkv, top, shuffle=False):
    sel = np.full((len(lens), nkv, top), -1, np.int32)
    for s, n in enumerate(lens):
        m = -(-int(n) // PR)
        for h in range(nkv):
            pick = rng.permutation(m)[:top]
            sel[s, h, :len(pick)] = pick if shuffle else np.sort(pick)
            if shuffle:
                rng.shuffle(sel[s, h])
    return sel


@pytest.mark.parametrize("dt", ALL_DT)
@pytest.mark.parametrize("nh,nkv", HEADS)
def test_selected_shapes(ctx, dt, nh, nkv):
    rng = np.random.default_rng(30 + nh)
    lens = np.array([1, 16, 0, 500, 337, 15, 31], np.int32)
    table, n_pages = tables(rng, lens)
    kp, kw = make_pool(400 + nh, n_pages, nkv, dt)
    vp, vw = make_pool(401 + nh, n_pages, nkv, dt)
    q = oracle.normal(402 + nh, (len(lens), nh, 64))
    for top, shuffle in ((1, False), (3, True), (9, False), (40, True)):
        sel = random_lists(rng, lens, nkv, top, shuffle)
        got = run_selected(ctx, q, kp, vp, table, lens, sel, nkv, dt)
        close(got, decode64(q, kw, vw, rows_of_list(table, lens, sel), nkv), f"top {top}")
    no_fault(ctx)


@pytest.mark.parametrize("dt", ALL_DT)
def test_selected_long_lists(ctx, dt):
    """Lists that fill several lookups of a wave (over 64 pages each), in many splits, in eight waves and in four."""
    rng = np.random.default_rng(31)
    for n, top in ((1, 700), (130, 600), (300, 300)):
        lens = np.full(n, 16 * 710 - 3, np.int32)
        table = rng.integers(0, 900, (n, 710)).astype(np.int32)
        kp, kw = make_pool(410, 900, 1, dt)
        vp, vw = make_pool(411, 900, 1, dt)
        q = oracle.normal(412, (n, 7, 64)) * np.float32(2)
        sel = random_lists(rng, lens, 1, top)
        sel[0, 0, -1] = 709
        got = run_selected(ctx, q, kp, vp, table, lens, sel, 1, dt)
        close(got, decode64(q, kw, vw, rows_of_list(table, lens, sel), 1), f"{n} x {top}")
    no_fault(ctx)


@pytest.mark.parametrize("dt", ALL_DT)
def test_selected_all_pages_is_the_paged_decode(ctx, dt):
    rng = np.random.default_rng(32)
    lens = np.array([700, 33, 1, 512], np.int32)
    table, n_pages = tables(rng, lens)
    kp, kw = make_pool(420, n_pages, 2, dt)
    vp, vw = make_pool(421, n_pages, 2, dt)
    q = oracle.normal(422, (4, 14, 64))
    sel = np.broadcast_to(np.arange(table.shape[1], dtype=np.int32), (4, 2, table.shape[1])).copy()  # past the length too
    got = run_selected(ctx, q, kp, vp, table, lens, sel, 2, dt)
    dout = ctx.empty((4, 14, 64))
    ctx.decode_paged(ctx.upload(q), ctx.upload(kp), ctx.upload(vp), n_pages, ctx.upload(table), table.shape[1],
                     ctx.upload(lens), dout, 4, 14, 2, 64, 704, kv_dtype=dt)
    assert_close(got, dout.numpy(), "against decode_paged", atol=4e-5, rtol=2e-4)  # both within the contract
    no_fault(ctx)


@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_selected_ignores_what_lies_outside(ctx, dt):
    """NaN and infinities in unselected pages and behind the last row change nothing."""
    rng = np.random.default_rng(33)
    lens = np.array([200, 37], np.int32)
    table, n_pages = tables(rng, lens, extra_pages=1)
    x, y = oracle.normal(430, (n_pages, PR, 2, 64)), oracle.normal(431, (n_pages, PR, 2, 64))
    sel = np.array([[[0, 4, 12], [0, 4, 12]], [[1, 2, -1], [1, 2, -1]]], np.int32)
    q = oracle.normal(432, (2, 14, 64))
    ref = decode64(q, widen(store(x, dt), dt), widen(store(y, dt), dt), rows_of_list(table, lens, sel), 2)
    used = np.zeros((n_pages, PR), bool)
    for s in range(2):
        pg, at = rows_of_list(table, lens, sel)(s, 0)
        used[pg, at] = True
    for bad in (np.nan, np.inf, -np.inf):
        a, b = x.copy(), y.copy()
        a[~used] = bad
        b[~used] = bad
        close(run_selected(ctx, q, store(a, dt), store(b, dt), table, lens, sel, 2, dt), ref, f"{bad}")
    no_fault(ctx)


def test_selected_late_maximum_and_large_scores(ctx):
    """Scores that climb by more than the lazy threshold page after page, and one that outweighs all others."""
    rng = np.random.default_rng(34)
    lens = np.array([16 * 64], np.int32)
    table, n_pages = tables(rng, lens)
    kp, _ = make_pool(440, n_pages, 1, F32)
    vp, vw = make_pool(441, n_pages, 1, F32)
    q = np.ones((1, 4, 64), np.float32) + 0.01 * oracle.normal(442, (1, 4, 64))
    for p in range(64):
        kp[table[0, p]] *= np.float32(0.1)
        kp[table[0, p], p % 16] += np.float32(0.9 * p)
    sel = np.arange(64, dtype=np.int32).reshape(1, 1, 64)
    got = run_selected(ctx, q, kp, vp, table, lens, sel, 1, F32)
    # |score| up to 64 * 57 / 8 = 456: 2^-24 * 456 * 8 in the exponent, 2.2e-4 relative in a weight that matters
    ref = decode64(q, kp, vw, rows_of_list(table, lens, sel), 1)
    assert_close(got, ref, "staircase", atol=3e-4, rtol=3e-4)
    no_fault(ctx)


def test_selected_errors(ctx):
    """Entries outside the table are skipped, block-table entries outside the pool clamped; both raise bit 2."""
    rng = np.random.default_rng(35)
    lens = np.array([100, 100], np.int32)
    table, n_pages = tables(rng, lens)
    kp, kw = make_pool(450, n_pages, 2, F32)
    vp, vw = make_pool(451, n_pages, 2, F32)
    q = oracle.normal(452, (2, 14, 64))
    sel = random_lists(rng, lens, 2, 4)
    bad = sel.copy()
    bad[0, 0, 1], bad[0, 1, 3], bad[1, 0, 0] = table.shape[1], -2, 2 ** 31 - 1
    ok = np.where((bad < 0) | (bad >= table.shape[1]), -1, bad)
    got = run_selected(ctx, q, kp, vp, table, lens, bad, 2, F32)
    close(got, decode64(q, kw, vw, rows_of_list(table, lens, ok), 2), "list entries")
    assert ctx.check_device_error() == FAULT
    t2 = table.copy()
    t2[0, sel[0, 0, 0]], t2[1, sel[1, 0, 1]] = -1, n_pages + 5
    t3 = np.clip(t2, 0, n_pages - 1)
    got = run_selected(ctx, q, kp, vp, t2, lens, sel, 2, F32)
    close(got, decode64(q, kw, vw, rows_of_list(t3, lens, sel), 2), "table entries")
    assert ctx.check_device_error() == FAULT
    no_fault(ctx)


# ---- attention over shared prefixes ----------------------------------------------------------

def shared_tables(rng, starts, prefix, lens):
    """Tables in which the pages wholly inside a group's prefix are real in its first sequence only."""
    n = len(lens)
    own = [-(-int(x) // PR) for x in lens]
    width = max(max(own), max([-(-int(p) // PR) for p in prefix], default=0), 1)
    total = sum(own) + sum(-(-int(p) // PR) for p in prefix) + 1
    perm = iter(rng.permutation(total).astype(np.int32))
    table = np.full((n, width), 2 ** 30, np.int32)  # never to be read
    of = np.full(n, -1)
    for g in range(len(prefix)):
        of[starts[g]:starts[g + 1]] = g
    for s in range(n):
        p = int(prefix[of[s]]) if of[s] >= 0 else 0
        first = of[s] >= 0 and s == starts[of[s]]
        a, b = (0 if first else p // PR), own[s]
        if first:
            b = max(b, -(-p // PR))  # the prefix is there whatever the length of this sequence
        for j in range(a, b):
            table[s, j] = next(perm)
    return table, total, of


def rows_shared(table, starts, prefix, of, lens):
    def rows(s, h):
        r = np.arange(int(lens[s]))
        pg = table[s, r // PR].copy()
        if of[s] >= 0:
            p = int(prefix[of[s]])
            pg[:p] = table[starts[of[s]], r[:p] // PR]
        return pg, r % PR
    return rows


def run_shared(ctx, q, kp, vp, table, lens, starts, prefix, nkv, dt, max_prefix=None, max_tail=None, stream=None):
    n, nh = q.shape[:2]
    dout = ctx.upload(np.full(q.shape, 9.0, np.float32))
    i32 = lambda x: ctx.upload(np.asarray(x, np.int32))  # noqa: E731
    ctx.decode_shared(ctx.upload(q), ctx.upload(kp), ctx.upload(vp), kp.shape[0], ctx.upload(table), table.shape[1],
                      i32(lens), i32(starts) if len(prefix) else None, i32(prefix) if len(prefix) else None, len(prefix),
                      dout, n, nh, nkv, 64, max(prefix, default=0) if max_prefix is None else max_prefix,
                      table.shape[1] * PR if max_tail is None else max_tail, stream=stream, kv_dtype=dt)
    if stream is not None:
        ctx.synchronize(stream)
    return dout.numpy()


def once_for_all(table, nkv, longest):
    """(table, max_prefix) with room for a prefix so long that it is read once for all sequences."""
    room = max(longest, (9 << 15) // (len(table) * nkv) + 1)
    wide = np.full((len(table), max(table.shape[1], -(-room // PR))), 2 ** 30, np.int32)
    wide[:, :table.shape[1]] = table
    return wide, room


def shared_case(ctx, dt, nh, nkv, starts, prefix, tails, seed, zero=(), scale=1.0, **kw):
    """The call as it is, and with room for a prefix so long that it is read once for all (short ones every sequence
    reads itself)."""
    rng = np.random.default_rng(seed)
    of = np.full(len(tails), -1)
    for g in range(len(prefix)):
        of[starts[g]:starts[g + 1]] = g
    lens = np.array([t + (prefix[of[s]] if of[s] >= 0 else 0) for s, t in enumerate(tails)], np.int32)
    lens[list(zero)] = 0
    table, total, of = shared_tables(rng, starts, prefix, lens)
    kp, kwd = make_pool(seed + 1, total, nkv, dt)
    vp, vwd = make_pool(seed + 2, total, nkv, dt)
    q = oracle.normal(seed + 3, (len(tails), nh, 64)) * np.float32(scale)
    ref = decode64(q, kwd, vwd, rows_shared(table, starts, prefix, of, lens), nkv)
    close(run_shared(ctx, q, kp, vp, table, lens, starts, prefix, nkv, dt, **kw), ref, f"{nh}/{nkv} {prefix}")
    if prefix:
        wide, room = once_for_all(table, nkv, max(prefix))
        kw.setdefault("max_tail", table.shape[1] * PR)
        close(run_shared(ctx, q, kp, vp, wide, lens, starts, prefix, nkv, dt, max_prefix=room, **kw), ref,
              f"{nh}/{nkv} {prefix}, once for all")
    no_fault(ctx)


@pytest.mark.parametrize("dt", ALL_DT)
@pytest.mark.parametrize("nh,nkv", HEADS)
def test_shared_shapes(ctx, dt, nh, nkv):
    # one group, a whole batch of groups with odd prefixes, sequences outside any group, a group of none
    shared_case(ctx, dt, nh, nkv, [0, 5], [333], [1, 40, 16, 0, 100], 500 + nh)
    shared_case(ctx, dt, nh, nkv, [1, 4, 4, 11], [17, 90, 128], [20, 3, 70, 0, 5, 0, 1, 1, 0, 33, 16, 50], 510 + nh)


@pytest.mark.parametrize("dt", ALL_DT)
@pytest.mark.parametrize("prefix", [0, 1, 15, 16, 17, 64, 255, 1000])
def test_shared_prefix_lengths(ctx, dt, prefix):
    shared_case(ctx, dt, 14, 2, [0, 11], [prefix], [0 if prefix else 1, 1, 2, 15, 16, 17, 64, 200, 0, 31, 5], 520 + prefix,
                scale=2.0)


@pytest.mark.parametrize("dt", ALL_DT)
def test_shared_many_sequences(ctx, dt):
    """Many column blocks, column blocks that end inside a sequence's heads, 70 groups (more than a wave looks at once)."""
    rng = np.random.default_rng(6)
    shared_case(ctx, dt, 14, 2, [0, 77], [2000], list(rng.integers(0, 60, 77)), 540)
    cuts = np.sort(rng.integers(0, 201, 69))
    starts = [0] + list(cuts) + [200]
    shared_case(ctx, dt, 4, 1, [int(x) for x in starts], [int(x) for x in rng.integers(1, 120, 70)],
                list(rng.integers(0, 40, 200)), 541, zero=(3, 50, 199))


@pytest.mark.parametrize("dt", ALL_DT)
@pytest.mark.parametrize("nh,nkv", [(4, 1), (14, 2)])
def test_shared_few_sequences_long_rows(ctx, dt, nh, nkv):
    """A prefix in more runs than one workgroup merges, own rows that are split, and one of them without the other."""
    shared_case(ctx, dt, nh, nkv, [0, 2], [6011], [30, 5], 560, max_tail=64)
    shared_case(ctx, dt, nh, nkv, [1, 3], [6011], [40, 2999, 1], 561, max_tail=3000)
    shared_case(ctx, dt, nh, nkv, [0, 2], [33], [2100, 1030], 562)
    shared_case(ctx, dt, nh, nkv, [], [], [2100, 0, 1030], 563)


@pytest.mark.parametrize("dt", ALL_DT)
def test_shared_more_blocks_than_workgroups(ctx, dt):
    """Groups of one sequence each on 8 kv heads: a workgroup takes several (block, kv head, run) units."""
    rng = np.random.default_rng(7)
    shared_case(ctx, dt, 32, 8, list(range(91)), [int(x) for x in rng.integers(0, 150, 90)],
                list(rng.integers(0, 20, 90)), 570, zero=(0, 44))


def test_shared_without_groups_or_tails(ctx):
    shared_case(ctx, F32, 14, 2, [], [], [40, 1, 300, 17], 550)
    shared_case(ctx, BF16, 14, 2, [0, 3], [160], [0, 0, 0], 551, max_tail=0)
    # a padded batch: lengths of zero, the group's first sequence among them (its table still holds the prefix)
    shared_case(ctx, Q8, 14, 2, [0, 5], [100], [5, 6, 7, 8, 9], 552, zero=(0, 3))
    shared_case(ctx, F32, 14, 2, [0, 3], [100], [5, 6, 7], 553, zero=(0, 1, 2))
    # bounds that are more than the table holds
    shared_case(ctx, BF16, 14, 2, [0, 3], [100], [5, 6, 7], 554, max_tail=10 ** 6)


@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_shared_ignores_what_lies_outside(ctx, dt):
    """NaN and infinities behind the prefix in its last page, before a sequence's own rows in that page, and behind the
    lengths change nothing."""
    rng = np.random.default_rng(36)
    starts, prefix, lens = [0, 3], [37], np.array([37, 41, 90], np.int32)
    table, total, of = shared_tables(rng, starts, prefix, lens)
    x, y = oracle.normal(560, (total, PR, 2, 64)), oracle.normal(561, (total, PR, 2, 64))
    q = oracle.normal(562, (3, 14, 64))
    rows = rows_shared(table, starts, prefix, of, lens)
    ref = decode64(q, widen(store(x, dt), dt), widen(store(y, dt), dt), rows, 2)
    used = np.zeros((total, PR), bool)
    for s in range(3):
        used[rows(s, 0)] = True
    for bad in (np.nan, np.inf, -np.inf):
        a, b = x.copy(), y.copy()
        a[~used] = bad
        b[~used] = bad
        close(run_shared(ctx, q, store(a, dt), store(b, dt), table, lens, starts, prefix, 2, dt), ref, f"{bad}")
        wide, room = once_for_all(table, 2, 37)
        close(run_shared(ctx, q, store(a, dt), store(b, dt), wide, lens, starts, prefix, 2, dt, max_prefix=room), ref,
              f"{bad}, once for all")
    no_fault(ctx)


@pytest.mark.parametrize("more", [0, 400])
def test_shared_errors(ctx, more):
    """Lengths and prefixes outside the call's bounds: NaN for those sequences and bit 1, the others unharmed;
    prefixes that every sequence reads itself, and longer ones that are read once."""
    rng = np.random.default_rng(37)
    starts, prefix = [0, 3, 5], [50 + more, 80 + more]
    # the second is shorter than its prefix, the last's own rows are more than max_tail
    lens = np.array([60 + more, 49 + more, 0, 85 + more, 400 + more], np.int32)
    table, total, of = shared_tables(rng, starts, prefix, lens)
    kp, kw = make_pool(570, total, 2, F32)
    vp, vw = make_pool(571, total, 2, F32)
    q = oracle.normal(572, (5, 14, 64))
    ok = lens.copy()
    ok[[1, 4]] = 0
    ref = decode64(q, kw, vw, rows_shared(table, starts, prefix, of, ok), 2)
    got = run_shared(ctx, q, kp, vp, table, lens, starts, prefix, 2, F32, max_prefix=80 + more, max_tail=300)
    assert np.isnan(got[[1, 4]]).all()
    close(got[[0, 2, 3]], ref[[0, 2, 3]], "others")
    assert ctx.check_device_error() == FAULT
    # the second group's prefix is too long
    got = run_shared(ctx, q, kp, vp, table, ok, starts, prefix, 2, F32, max_prefix=79 + more)
    assert np.isnan(got[3]).all()
    close(got[[0, 1, 2, 4]], ref[[0, 1, 2, 4]], "others")
    assert ctx.check_device_error() == FAULT
    # a length beyond the table, and negative lengths and prefixes (as 0)
    long = ok.copy()
    long[0], long[2] = table.shape[1] * PR + 1, -7
    got = run_shared(ctx, q, kp, vp, table, long, starts, prefix, 2, F32)
    assert np.isnan(got[0]).all() and not got[2].any()
    assert ctx.check_device_error() == FAULT
    t2 = np.where(table == 2 ** 30, 0, table)
    t2[0, 1], t2[3, 5] = -3, total + 9  # clamped
    t3 = np.clip(t2, 0, total - 1)
    got = run_shared(ctx, q, kp, vp, t2, ok, starts, prefix, 2, F32)
    close(got, decode64(q, kw, vw, rows_shared(t3, starts, prefix, of, ok), 2), "clamped pages")
    assert ctx.check_device_error() == FAULT
    no_fault(ctx)


# ---- together --------------------------------------------------------------------------------

@pytest.mark.parametrize("dt", ALL_DT)
def test_prompt_then_sparse_decode(ctx, dt):
    """A prompt and a few tokens appended, bounds, selection and attention as a serving loop runs them: the whole chain
    against the plain forms on the cache that the append left."""
    nh, nkv, n, top = 14, 2, 3, 9
    rng = np.random.default_rng(40)
    final = np.array([700, 333, 95], np.int32)
    table, n_pages = tables(rng, final)
    kp, _ = make_pool(600, n_pages, nkv, dt)
    dkp, dvp, dtab = ctx.upload(kp), ctx.upload(kp), ctx.upload(table)
    db = ctx.upload(np.zeros((n_pages, nkv, 2, 64), np.uint16))
    dsel, dout = ctx.empty((n, nkv, top), np.int32), ctx.empty((n, nh, 64))
    have = np.zeros(n, np.int32)
    for step, add in enumerate([final - 3, [1, 1, 1], [1, 1, 1], [1, 1, 1]]):
        add = np.asarray(add, np.int32)
        rows = int(add.sum())
        x = ctx.upload(oracle.normal(610 + step, (rows, nh + 2 * nkv, 64)))
        stride = (nh + 2 * nkv) * 64
        dq = ctx.empty((rows, nh, 64))
        starts = np.concatenate([[0], np.cumsum(add)]).astype(np.int32)
        dlen = ctx.upload(have + add)
        ctx.kv_append_paged(x.ptr, stride, dq, x.at(nh * 64), stride, x.at((nh + nkv) * 64), stride, dkp, dvp, n_pages,
                            dtab, table.shape[1], ctx.upload(starts), ctx.upload(have), n, rows, nh, nkv, 64, 704,
                            kv_dtype=dt)
        ctx.kv_page_bounds(dkp, n_pages, dtab, table.shape[1], ctx.upload(have), dlen, db, n, nkv, 64, int(add.max()),
                           kv_dtype=dt)
        have += add
        if step == 0:
            continue
        ctx.select_pages(dq, db, n_pages, dtab, table.shape[1], dlen, dsel, n, nh, nkv, 64, 704, top, 1, 1)
        ctx.decode_selected(dq, dkp, dvp, n_pages, dtab, table.shape[1], dlen, dsel, top, dout, n, nh, nkv, 64,
                            kv_dtype=dt)
        q, kw, vw = dq.numpy(), widen(dkp.numpy(), dt), widen(dvp.numpy(), dt)
        b = bounds_ref(kw, np.zeros((n_pages, nkv, 2, 64), np.float32), table, None, have, nkv)
        np.testing.assert_array_equal(bf16_values(db.numpy()), b)
        sel = select_ref(q, b, table, have, nkv, top, 1, 1)
        np.testing.assert_array_equal(dsel.numpy(), sel)
        close(dout.numpy(), decode64(q, kw, vw, rows_of_list(table, have, sel), nkv), f"step {step}")
    no_fault(ctx)


@pytest.mark.parametrize("dt", ALL_DT)
def test_selected_pages_hold_the_largest_scores(ctx, dt):
    """What the selection is for: no key of a page scores above the page's bound, so a key planted far above all
    others is always in the list."""
    rng = np.random.default_rng(41)
    lens = np.array([1600], np.int32)
    table, n_pages = tables(rng, lens)
    q = oracle.normal(620, (1, 14, 64))
    x = oracle.normal(621, (n_pages, PR, 2, 64))
    for h in range(2):
        x[table[0, 57], 6, h] = 3 * q[0, 7 * h + 2]
    kp = store(x, dt)
    db = ctx.empty((n_pages, 2, 2, 64), np.uint16)
    dt_, dl = ctx.upload(table), ctx.upload(lens)
    ctx.kv_page_bounds(ctx.upload(kp), n_pages, dt_, 100, None, dl, db, 1, 2, 64, 1600, kv_dtype=dt)
    dsel = ctx.empty((1, 2, 3), np.int32)
    ctx.select_pages(ctx.upload(q), db, n_pages, dt_, 100, dl, dsel, 1, 14, 2, 64, 1600, 3, 1, 1)
    assert (dsel.numpy()[0, :, 1] == 57).all()
    no_fault(ctx)


def test_captured_step_replays(ctx):
    """Append, bounds, selection, both attentions in one captured step: replayed with new positions, with eager calls
    of other sizes between the replays (they share the context's workspace), each replay equals the eager result."""
    nh, nkv, n, top, dt = 14, 2, 4, 6, BF16
    rng = np.random.default_rng(42)
    base = np.array([300, 200, 250, 490], np.int32)
    table, n_pages = tables(rng, base + 8, width=1540)
    kp, _ = make_pool(630, n_pages, nkv, dt)
    vp, _ = make_pool(631, n_pages, nkv, dt)
    W = table.shape[1]
    s = ctx.stream()
    dkp, dvp, dtab = ctx.upload(kp), ctx.upload(vp), ctx.upload(table)
    b0 = random_bounds(632, n_pages, nkv)
    db = ctx.upload((b0.view(np.uint32) >> 16).astype(np.uint16))
    dx, dq = ctx.empty((n, nh + 2 * nkv, 64)), ctx.empty((n, nh, 64))
    dpos, dlen, dstart = ctx.empty(n, np.int32), ctx.empty(n, np.int32), ctx.upload(np.arange(n + 1, dtype=np.int32))
    dsel, o1, o2, o3 = ctx.empty((n, nkv, top), np.int32), *(ctx.empty((n, nh, 64)) for _ in range(3))
    dg, dpre = ctx.upload(np.array([0, 2, 4], np.int32)), ctx.upload(np.array([150, 64], np.int32))
    stride = (nh + 2 * nkv) * 64

    def step():
        ctx.kv_append_paged(dx.ptr, stride, dq, dx.at(nh * 64), stride, dx.at((nh + nkv) * 64), stride, dkp, dvp, n_pages,
                            dtab, W, dstart, dpos, n, n, nh, nkv, 64, 500, stream=s, kv_dtype=dt)
        ctx.kv_page_bounds(dkp, n_pages, dtab, W, dpos, dlen, db, n, nkv, 64, 1, stream=s, kv_dtype=dt)
        ctx.select_pages(dq, db, n_pages, dtab, W, dlen, dsel, n, nh, nkv, 64, 500, top, 1, 1, stream=s)
        ctx.decode_selected(dq, dkp, dvp, n_pages, dtab, W, dlen, dsel, top, o1, n, nh, nkv, 64, stream=s, kv_dtype=dt)
        for o, room in ((o2, 160), (o3, 24600)):  # the prefix read by every sequence, and once for all
            ctx.decode_shared(dq, dkp, dvp, n_pages, dtab, W, dlen, dg, dpre, 2, o, n, nh, nkv, 64, room, 500, stream=s,
                              kv_dtype=dt)

    def results():
        ctx.synchronize(s)
        return [d.numpy() for d in (dq, dkp, dvp, db, dsel, o1, o2, o3)]

    def load(i):
        dx.copy_from(oracle.normal(640 + i, (n, nh + 2 * nkv, 64)), s)
        dpos.copy_from(base + i, s)
        dlen.copy_from(base + i + 1, s)

    def restore():
        dkp.copy_from(kp, s), dvp.copy_from(vp, s), db.copy_from((b0.view(np.uint32) >> 16).astype(np.uint16), s)

    eager = []
    for i in range(5):
        load(i)
        step()
        eager.append(results())
    restore()
    ctx.step_begin(s)
    step()
    graph = ctx.step_end(s)
    try:
        for i in range(5):
            load(i)
            ctx.graph_launch(graph, s)
            got = results()
            for k, (a, b) in enumerate(zip(got, eager[i])):
                np.testing.assert_array_equal(a.view(np.uint8), b.view(np.uint8), err_msg=f"replay {i}, output {k}")
            # eager calls of other shapes, larger than the captured ones, between the replays
            shared_case(ctx, F32, 14, 2, [0, 40], [500 + 100 * i], [3] * 40, 650 + i)
            no_fault(ctx)
    finally:
        ctx.graph_destroy(graph)
        ctx.destroy_stream(s)


def test_same_call_same_bits_and_two_streams_of_two_contexts(ctx):
    """Repeated calls give the same bits; two contexts on their own streams do not disturb each other."""
    rng = np.random.default_rng(43)
    lens = np.full(20, 1500, np.int32)
    table, n_pages = tables(rng, lens)
    kp, _ = make_pool(660, n_pages, 2, Q8)
    vp, _ = make_pool(661, n_pages, 2, Q8)
    q = oracle.normal(662, (20, 14, 64))
    sel = random_lists(rng, lens, 2, 30)
    a = run_selected(ctx, q, kp, vp, table, lens, sel, 2, Q8)
    with tmac_attn.Context(0) as other:
        s1, s2 = ctx.stream(), other.stream()
        devs = []
        for c in (ctx, other):
            devs.append([c.upload(x) for x in (q, kp, vp, table, lens, sel)] + [c.empty(q.shape)])
        for _ in range(10):
            for c, s, d in ((ctx, s1, devs[0]), (other, s2, devs[1])):
                c.decode_selected(d[0], d[1], d[2], n_pages, d[3], table.shape[1], d[4], d[5], 30, d[6], 20, 14, 2, 64,
                                  stream=s, kv_dtype=Q8)
        ctx.synchronize(s1)
        other.synchronize(s2)
        for d in devs:
            np.testing.assert_array_equal(d[6].numpy().view(np.uint32), a.view(np.uint32))
        ctx.destroy_stream(s1)
        other.destroy_stream(s2)
    no_fault(ctx)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_offsets_beyond_32_bits(ctx, dt):
    """A pool of more than 2^32 bytes whose last pages are used: page offsets need 64 bits."""
    kind = np.float32 if dt == F32 else np.uint16
    n_pages = (1 << 32) // (PR * 64 * np.dtype(kind).itemsize) + 40  # one kv head
    dk, dv = ctx.empty((n_pages, PR, 1, 64), kind), ctx.empty((n_pages, PR, 1, 64), kind)
    lens = np.array([40], np.int32)
    table = np.array([[n_pages - 1, 5, n_pages - 20]], np.int32)
    x = oracle.normal(670, (40, 6, 64))
    dx = ctx.upload(x)
    dq = ctx.empty((40, 4, 64))
    dtab = ctx.upload(table)
    ctx.kv_append_paged(dx.ptr, 384, dq, dx.at(256), 384, dx.at(320), 384, dk, dv, n_pages, dtab, 3,
                        ctx.upload(np.array([0, 40], np.int32)), ctx.upload(np.zeros(1, np.int32)), 1, 40, 4, 1, 64, 48,
                        kv_dtype=dt)
    k = np.stack([oracle.rope_heads(x[p, 4], 1, 64, p) for p in range(40)]).reshape(40, 64)
    q = dq.numpy()[39:]
    ref = attend64(q[0], widen(store(k, dt), dt), widen(store(x[:, 5], dt), dt))[None]
    dlen, dout = ctx.upload(lens), ctx.empty((1, 4, 64))
    dsel = ctx.upload(np.array([[[0, 1, 2]]], np.int32))
    ctx.decode_selected(dq.at(39 * 256), dk, dv, n_pages, dtab, 3, dlen, dsel, 3, dout, 1, 4, 1, 64, kv_dtype=dt)
    close(dout.numpy(), ref, "selected")
    wide, room = once_for_all(table, 1, 20)
    for t, most in ((table, 20), (wide, room)):
        ctx.decode_shared(dq.at(39 * 256), dk, dv, n_pages, ctx.upload(t), t.shape[1], dlen,
                          ctx.upload(np.array([0, 1], np.int32)), ctx.upload(np.array([20], np.int32)), 1, dout, 1, 4, 1,
                          64, most, 20, kv_dtype=dt)
        close(dout.numpy(), ref, "shared")
    for d in (dk, dv):
        d.free()
    no_fault(ctx)


def put(ctx, ptr, host):
    host = np.ascontiguousarray(host)
    ctx._check(ctx.lib.tmac_memcpy_h2d(ctx.handle, None, ptr, host.ctypes.data, host.nbytes), "memcpy_h2d")
    ctx.synchronize()


def get(ctx, ptr, shape, kind=np.float32):
    host = np.empty(shape, kind)
    ctx.synchronize()
    ctx._check(ctx.lib.tmac_memcpy_d2h(ctx.handle, None, host.ctypes.data, ptr, host.nbytes), "memcpy_d2h")
    ctx.synchronize()
    return host


@pytest.mark.parametrize("dt", ALL_DT)
def test_selected_rows_of_a_page_beyond_31_bits(ctx, dt):
    """So many kv heads that the last rows of one page lie 2^31 bytes and more behind its first: row offsets inside a
    page need 64 bits.  Of the pools, the queries and the outputs only the first and last three heads are looked at."""
    width, kind = (68, np.uint8) if dt == Q8 else (64, np.float32 if dt == F32 else np.uint16)
    size = width * np.dtype(kind).itemsize
    nkv, some = (1 << 31) // (15 * size) + 60, 3
    heads = (0, nkv - some)
    x, y, q = oracle.normal(680, (PR, 2 * some, 64)), oracle.normal(681, (PR, 2 * some, 64)), oracle.normal(682, (2 * some, 64))
    k, v = store(x, dt), store(y, dt)
    dk, dv = ctx.empty((PR, nkv, width), kind), ctx.empty((PR, nkv, width), kind)
    dq, dout = ctx.empty((nkv, 64)), ctx.empty((nkv, 64))
    dtab, dsel = ctx.upload(np.zeros((1, 1), np.int32)), ctx.upload(np.zeros((1, nkv, 1), np.int32))
    for i, h in enumerate(heads):
        part = slice(some * i, some * (i + 1))
        put(ctx, dq.at(h * 64), q[part])
        for r in range(PR):
            put(ctx, dk.at((r * nkv + h) * width), k[r, part])
            put(ctx, dv.at((r * nkv + h) * width), v[r, part])
    for n in (PR, 13):
        ctx.decode_selected(dq, dk, dv, 1, dtab, 1, ctx.upload(np.array([n], np.int32)), dsel, 1, dout, 1, nkv, nkv, 64,
                            kv_dtype=dt)
        got = np.concatenate([get(ctx, dout.at(h * 64), (some, 64)) for h in heads])
        ref = np.stack([attend64(q[i:i + 1], widen(k[:n, i], dt), widen(v[:n, i], dt))[0] for i in range(2 * some)])
        close(got, ref, f"{n} rows")
    for d in (dk, dv, dq, dout, dsel):
        d.free()
    no_fault(ctx)


def test_append_heads_of_a_row_beyond_31_bits(ctx):
    """One row of 2^25 query heads and a few, 8.6 GB, rotated in place: the last heads' offsets pass 2^31 floats."""
    nh, some, pos = (1 << 25) + 64, 3, 77
    q, kv = oracle.normal(690, (2 * some, 64)), oracle.normal(691, (2, 1, 64))
    dq, dkv = ctx.empty((nh, 64)), ctx.upload(kv)
    heads = (0, nh - some)
    for i, h in enumerate(heads):
        put(ctx, dq.at(h * 64), q[some * i:some * (i + 1)])
    dk, dv = ctx.upload(np.zeros((5, PR, 1, 64), np.float32)), ctx.upload(np.zeros((5, PR, 1, 64), np.float32))
    i32 = lambda x: ctx.upload(np.asarray(x, np.int32))  # noqa: E731
    ctx.kv_append_paged(dq, 0, dq, dkv, 0, dkv.at(64), 0, dk, dv, 5, i32([[4, 3, 2, 1, 0]]), 5, i32([0, 1]), i32([pos]), 1, 1,
                        nh, 1, 64, 80)
    got = np.concatenate([get(ctx, dq.at(h * 64), (some, 64)) for h in heads])
    np.testing.assert_array_equal(got, oracle.rope_heads(q, 2 * some, 64, pos).reshape(got.shape))
    np.testing.assert_array_equal(dk.numpy()[0, pos % PR, 0], oracle.rope_heads(kv[0], 1, 64, pos).reshape(64))
    np.testing.assert_array_equal(dv.numpy()[0, pos % PR], kv[1])
    dq.free()
    no_fault(ctx)


# ---- stored rows that are not finite and are read -----------------------------------------------

def spoil(pool, dt, page, row, dim, bad):
    """Copy of a stored pool with one value of kv head 0 set to `bad` (Q8_0: the scale of its 32 dims)."""
    p = pool.copy()
    if dt == Q8:
        at = 64 + 2 * (dim // 32)
        p[page, row, 0, at:at + 2] = np.array([bad], np.float16).view(np.uint8)
    else:
        p[page, row, 0, dim] = store(np.array([bad], np.float32), dt)[0]
    return p


def check_spoilt(got, ref, without, what, key=None, value=None):
    """One (sequence, kv head)'s outputs [heads][64] over a row with a key or a value that is not finite; ref: with
    the row as it was, without: without the row.  key: its score; value: the dims that it spoils."""
    if value is not None:
        rest = np.setdiff1d(np.arange(64), value)
        assert not np.isfinite(got[:, value]).any(), what
        close(got[:, rest], ref[:, rest], what)
    elif key == -np.inf:  # weight 0, or nothing finite
        for h in range(len(got)):
            if np.isfinite(got[h]).any():
                close(got[h], without[h], what)
    else:
        assert not np.isfinite(got).any(), what


@pytest.mark.parametrize("route", ["whole list", "split list", "own", "prefix, read by each", "prefix, once for all"])
@pytest.mark.parametrize("dt", ALL_DT)
def test_rows_that_are_read_and_not_finite(ctx, dt, route):
    """NaN and infinities in one stored row that is read: what they do to the outputs that read it, and that the other
    kv head and a sequence that does not read it keep their values."""
    rng = np.random.default_rng(38)
    nh, nkv, row, dim = 14, 2, 333, 5
    lens = np.array([700, 690], np.int32)
    shared = route.startswith("prefix") or route == "own"
    if shared:
        starts, prefix = [0, 2], [600 if route != "own" else 40]
        table, total, of = shared_tables(rng, starts, prefix, lens)
        rows = rows_shared(table, starts, prefix, of, lens)
    else:
        table, total = tables(rng, lens)
        n = 12 if route == "whole list" else 44
        sel = np.full((2, nkv, n), -1, np.int32)
        sel[:, :, 0], sel[:, :, 1:] = row // PR, [j for j in range(44) if j != row // PR][:n - 1]
        rows = rows_of_list(table, lens, sel)
    kp, kw = make_pool(700, total, nkv, dt)
    vp, vw = make_pool(701, total, nkv, dt)
    q = oracle.normal(702, (2, nh, 64))
    q[:, :, dim] = np.abs(q[:, :, dim]) + np.float32(0.3)
    if dt == Q8:  # a scale spoils 32 keys: their integers decide the sign of the score
        kp[:, :, :, :32] = (rng.integers(1, 120, kp[..., :32].shape) * 1).astype(np.int8).view(np.uint8)
        kw = widen(kp, dt)
        q[:, :, :32] = np.abs(q[:, :, :32]) + np.float32(0.01)
    pages, at = rows(0, 0)
    logical = np.concatenate([PR * j + np.arange(PR) for j in sel[0, 0] if j >= 0]) if not shared else np.arange(lens[0])
    logical = logical[logical < lens[0]]
    i = int(np.flatnonzero(logical == row)[0])
    page, r = int(pages[i]), int(at[i])
    readers = [0, 1] if route.startswith("prefix") else [0]

    def run(a, b):
        if not shared:
            return run_selected(ctx, q, a, b, table, lens, sel, nkv, dt)
        if route != "prefix, once for all":
            return run_shared(ctx, q, a, b, table, lens, starts, prefix, nkv, dt)
        wide, room = once_for_all(table, nkv, prefix[0])
        return run_shared(ctx, q, a, b, wide, lens, starts, prefix, nkv, dt, max_prefix=room)

    ref = decode64(q, kw, vw, rows, nkv)

    def others(s, h):
        pg, x = rows(s, h)
        keep = ~((pg == page) & (x == r))
        return pg[keep], x[keep]
    without = decode64(q, kw, vw, others, nkv)
    close(run(kp, vp), ref, "finite")
    for name, bad in (("NaN", np.nan), ("+inf", np.inf), ("-inf", -np.inf)):
        for what, a, b in ((f"key {name}", spoil(kp, dt, page, r, dim, bad), vp),
                           (f"value {name}", kp, spoil(vp, dt, page, r, dim, bad))):
            got = run(a, b)
            value = None if b is vp else (np.arange(32) if dt == Q8 else np.array([dim]))
            for s in range(2):
                if s in readers:
                    check_spoilt(got[s, :7], ref[s, :7], without[s, :7], what, key=bad, value=value)
                else:
                    close(got[s, :7], ref[s, :7], f"{what}, another sequence")
                close(got[s, 7:], ref[s, 7:], f"{what}, the other kv head")
    no_fault(ctx)


@pytest.mark.parametrize("bits", [0x7FC0, 0xFFFF, 0x7F80, 0xFF80, 0x7F7F])
def test_select_bounds_of_pages_that_are_taken_anyway(ctx, bits):
    """Bounds of a sequence's first and last pages may hold anything: NaN, infinities, stale values."""
    rng = np.random.default_rng(7)
    for lens, top, first, last in (([1600, 333], 12, 2, 3), ([40000, 33000], 40, 1, 2)):
        lens = np.array(lens, np.int32)
        table, n_pages = tables(rng, lens)
        q, b = oracle.normal(350, (2, 14, 64)), random_bounds(351, n_pages, 2)
        ref = select_ref(q, b, table, lens, 2, top, first, last)
        for s, n in enumerate(-(-lens // PR)):
            forced = np.r_[table[s, :first], table[s, n - last:n]]
            b.view(np.uint32)[forced] = np.uint32(bits) << 16
        np.testing.assert_array_equal(run_select(ctx, q, b, table, lens, 2, top, first, last), ref)
    no_fault(ctx)


@pytest.mark.parametrize("dt", ALL_DT)
def test_selected_long_lists_of_many_sequences(ctx, dt):
    """Around 2/3 of the CUs, above and below one list a CU: lists split in three or two and whole ones of eight waves
    and of four, long enough that a wave looks its pages up twice."""
    rng = np.random.default_rng(39)
    for n, top in ((168, 790), (180, 600), (260, 300)):
        lens = np.full(n, 16 * 800 - 5, np.int32)
        table = rng.integers(0, 500, (n, 800)).astype(np.int32)
        kp, kw = make_pool(490, 500, 1, dt)
        vp, vw = make_pool(491, 500, 1, dt)
        q = oracle.normal(492, (n, 4, 64))
        sel = random_lists(rng, lens, 1, top)
        sel[1, 0, 5:] = -1
        got = run_selected(ctx, q, kp, vp, table, lens, sel, 1, dt)
        close(got, decode64(q, kw, vw, rows_of_list(table, lens, sel), 1), f"{n} x {top}")
    no_fault(ctx)


@pytest.mark.parametrize("dt", ALL_DT)
def test_selected_pages_listed_twice(ctx, dt):
    """A page listed twice counts twice, the last, partly filled one too, in one workgroup and in several; a length beyond
    the table leaves the listed pages whole."""
    rng = np.random.default_rng(47)
    lens = np.array([700, 693, 2 ** 31 - 1], np.int32)
    table, n_pages = tables(rng, [700, 693, 704])
    kp, kw = make_pool(493, n_pages, 2, dt)
    vp, vw = make_pool(494, n_pages, 2, dt)
    q = oracle.normal(495, (3, 14, 64))
    for top in (7, 90):
        sel = rng.integers(0, 44, (3, 2, top)).astype(np.int32)
        sel[..., 0], sel[..., top // 2], sel[..., -1], sel[1, 0, 2:4] = 43, 43, 43, -1
        got = run_selected(ctx, q, kp, vp, table, lens, sel, 2, dt)
        close(got, decode64(q, kw, vw, rows_of_list(table, lens.astype(np.int64), sel), 2), f"top {top}")
    no_fault(ctx)


def test_two_captured_steps_share_the_workspace(ctx):
    """Two captured calls of one context, whose partials lie in the same workspace, replayed in turn: each gives its eager
    result every time."""
    rng = np.random.default_rng(48)
    s, steps = ctx.stream(), []
    for i, (n, top, dt) in enumerate(((3, 60, BF16), (5, 90, F32))):
        lens = np.full(n, 1600, np.int32)
        table, n_pages = tables(rng, lens)
        kp, _ = make_pool(496 + i, n_pages, 2, dt)
        sel = random_lists(rng, lens, 2, top)
        d = [ctx.upload(x) for x in (oracle.normal(498 + i, (n, 14, 64)), kp, kp, table, lens, sel)] + [ctx.empty((n, 14, 64))]

        def call(d=d, n=n, n_pages=n_pages, width=table.shape[1], top=top, dt=dt):
            ctx.decode_selected(d[0], d[1], d[2], n_pages, d[3], width, d[4], d[5], top, d[6], n, 14, 2, 64, stream=s,
                                kv_dtype=dt)
        call()
        eager = d[6].numpy(s)
        steps.append([call, d[6], eager, None])
    for step in steps:
        ctx.step_begin(s)
        step[0]()
        step[3] = ctx.step_end(s)
    for _ in range(4):
        for _, out, _, graph in steps:
            out.fill_bytes(0xFF, s)
            ctx.graph_launch(graph, s)
        for _, out, eager, _ in steps:
            np.testing.assert_array_equal(out.numpy(s).view(np.uint32), eager.view(np.uint32))
    for step in steps:
        ctx.graph_destroy(step[3])
    ctx.destroy_stream(s)
    no_fault(ctx)
