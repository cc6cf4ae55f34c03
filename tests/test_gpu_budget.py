"""Long contexts in a small cache (tmac_kv_append_axes_paged, tmac_attention_decode_weighted, tmac_select_rows,
tmac_kv_compact_paged, tmac_kv_widen_pages) against plain 64-bit forms.

Stored rows, lists and moved rows are compared bit for bit.  Attention outputs and weights are held to bounds that
budget.attend64 derives from the sizes of the products, element by element."""
import numpy as np
import pytest

import budget
import oracle
import serving
import tmac_attn
from budget import Q4, TYPES, compact_ref, keep_ref, make_pool, put4, rope_axes
from serving import BF16, F16, F32, PR, Q8, store, tables

pytestmark = pytest.mark.gpu
FAULT = tmac_attn.TMAC_ERR_DEVICE_FAULT
HEADS = [(14, 2), (1, 1), (8, 8), (16, 1), (12, 4), (33, 3)]  # groups of 7, 1, 1, 16, 3, 11
SECTIONS = [0] * 8 + [1] * 12 + [2] * 12
NAMES = {F32: "f32", BF16: "bf16", F16: "f16", Q8: "q8", Q4: "q4"}
by_type = pytest.mark.parametrize("dt", TYPES, ids=[NAMES[t] for t in TYPES])


def no_fault(ctx):
    assert ctx.check_device_error() == 0


def faults(ctx):
    assert ctx.check_device_error() == FAULT
    no_fault(ctx)  # reading cleared it


def same_bits(got, ref, what):
    np.testing.assert_array_equal(np.ascontiguousarray(got).view(np.uint8), np.ascontiguousarray(ref).view(np.uint8),
                                  err_msg=what)


# ---- pages ----------------------------------------------------------------------------------

@by_type
@pytest.mark.parametrize("n_pages,nkv", [(1, 1), (5, 3), (70, 2)])
def test_widen(ctx, dt, n_pages, nkv):
    (kp, kw), (vp, vw) = (make_pool(900 + i, n_pages, nkv, dt, i == 0) for i in (0, 1))
    out = [ctx.upload(np.full(kw.shape, 7.5, np.float32)) for _ in range(3)]
    dk, dv = ctx.upload(kp), ctx.upload(vp)
    ctx.kv_widen_pages(dk, dv, out[0], out[1], n_pages, nkv, 64, kv_dtype=dt)
    ctx.kv_widen_pages(None, dv, None, out[2], n_pages, nkv, 64, kv_dtype=dt)
    for got, ref, what in zip(out, (kw, vw, vw), ("k", "v", "v alone")):
        same_bits(got.numpy(), ref, what)
    no_fault(ctx)


def test_widen_all_bytes(ctx):
    """Any bytes, every scale of 16 bits that is a number: code and scale as the format says."""
    rng = np.random.default_rng(5)
    pages = rng.integers(0, 256, (300, 2, 576), dtype=np.uint8)
    s = pages.view(np.uint16)[..., 256:]
    s[(s & 0x7C00) == 0x7C00] &= 0xBFFF
    for i, key in enumerate((True, False)):
        d, out = ctx.upload(pages), ctx.empty((300, 16, 2, 64))
        args = [d, None, out, None] if key else [None, d, None, out]
        ctx.kv_widen_pages(*args, 300, 2, 64, kv_dtype=Q4)
        np.testing.assert_array_equal(out.numpy(), budget.widen4(pages, key))


# ---- append ---------------------------------------------------------------------------------

def append_ref(q, k, v, kp, vp, table, starts, at, pos, axis, dt, n_pages, max_pos, q_out, base=1e6):
    kp, vp, q_out = kp.copy(), vp.copy(), q_out.copy()
    for s in range(len(at)):
        for t in range(int(starts[s]), int(starts[s + 1])):
            row, p = int(at[s]) + t - int(starts[s]), pos[:, t]
            if not 0 <= row < table.shape[1] * PR or (p < 0).any() or (p >= max_pos).any():
                continue
            if q is not None:
                q_out[t] = rope_axes(q[t], p, axis, base)
            page = table[s, row // PR]
            if 0 <= page < n_pages:
                kr = rope_axes(k[t], p, axis, base)
                if dt == Q4:
                    for h in range(k.shape[1]):
                        put4(kp[page, h], row % PR, kr[h], True)
                        put4(vp[page, h], row % PR, v[t, h], False)
                else:
                    kp[page, row % PR], vp[page, row % PR] = store(kr, dt), store(v[t], dt)
    return q_out, kp, vp


def run_append(ctx, dt, nh, nkv, counts, at, seed, axis=SECTIONS, n_axes=3, fused=False, in_place=False, with_q=True,
               lead=0, behind=0, table=None, n_pages=None, max_pos=5000, pos=None, width=0, values=None):
    rng = np.random.default_rng(seed)
    counts, at = np.asarray(counts), np.asarray(at)
    if table is None:
        table, n_pages = tables(rng, np.where(counts > 0, at + counts, 0), extra_pages=2, width=width)
    starts = (lead + np.concatenate([[0], np.cumsum(counts)])).astype(np.int32)
    rows = int(starts[-1]) + behind
    x = oracle.normal(seed, (rows, nh + 2 * nkv, 64))
    x *= np.exp2(rng.uniform(-3, 3, (rows, 1, 1))).astype(np.float32)
    if values is not None:
        values(x)
    q, k, v = x[:, :nh], x[:, nh:nh + nkv], x[:, nh + nkv:]
    if pos is None:
        pos = rng.integers(0, max_pos, (n_axes, rows))
    pos = pos.astype(np.int32)
    kp, vp = (make_pool(seed + 1 + i, n_pages, nkv, dt, i == 0)[0] for i in (0, 1))
    before = q if in_place else np.full((rows, nh, 64), 7.5, np.float32)
    dkp, dvp = ctx.upload(kp), ctx.upload(vp)
    dtab, ds, da, dp = ctx.upload(table), ctx.upload(starts), ctx.upload(at.astype(np.int32)), ctx.upload(pos)
    row = (nh + 2 * nkv) * 64
    if fused:
        dx = ctx.upload(x)
        dq, dk, dv, qs, ks = dx.ptr, dx.at(nh * 64), dx.at((nh + nkv) * 64), row, row
    else:
        dq, dk, dv = (ctx.upload(np.ascontiguousarray(y)) for y in (q, k, v))
        qs, ks = nh * 64, nkv * 64
    dout = dq if in_place else ctx.upload(before)
    ctx.kv_append_axes_paged(dq if with_q else None, qs, dout if with_q else None, dk, ks, dv, ks, dkp, dvp, n_pages, dtab,
                             table.shape[1], ds, da, dp, n_axes, axis, len(counts), rows, nh, nkv, 64, max_pos, 1e6,
                             kv_dtype=dt)
    ref = append_ref(q if with_q else None, k, v, kp, vp, table, starts, at, pos, [0] * 32 if axis is None else axis, dt,
                     n_pages, max_pos, before)
    for name, a, b in zip(("q", "k", "v"), (dout.numpy().reshape(before.shape), dkp.numpy(), dvp.numpy()), ref):
        same_bits(a, b, name)


@by_type
@pytest.mark.parametrize("nh,nkv", HEADS)
def test_append_shapes(ctx, dt, nh, nkv):
    run_append(ctx, dt, nh, nkv, [1, 0, 37, 16, 0, 0, 5, 1], [0, 3, 11, 16, 0, 9, 255, 15], 1000 + nh, fused=nh % 2 == 0)
    no_fault(ctx)


@pytest.mark.parametrize("axis,n_axes", [(None, 1), (None, 3), ([i % 3 for i in range(32)], 3), ([3 - i // 8 for i in range(32)], 4),
                                         ([1] * 32, 2)])
def test_append_axes(ctx, axis, n_axes):
    for dt in (F32, Q4):
        run_append(ctx, dt, 6, 2, [3, 20], [7, 30], 1040, axis=axis, n_axes=n_axes)
    no_fault(ctx)


@by_type
def test_append_many_rows_per_workgroup(ctx, dt):
    """More rows than eight per CU: workgroups of several rows, sequences that begin and end inside one."""
    run_append(ctx, dt, 2, 1, [700, 1, 0, 2300, 15, 1500, 3], [5, 0, 4, 1, 800, 17, 31], 1050, fused=True)
    no_fault(ctx)


@by_type
def test_append_in_place_padding_and_keys_alone(ctx, dt):
    run_append(ctx, dt, 14, 2, [2, 9], [40, 6], 1060, in_place=True)
    run_append(ctx, dt, 14, 2, [2, 9], [40, 6], 1061, with_q=False)
    run_append(ctx, dt, 14, 2, [2, 0, 9], [40, 0, 6], 1062, lead=3, behind=21)
    no_fault(ctx)


@by_type
def test_append_skips_bad_rows(ctx, dt):
    rng = np.random.default_rng(7)
    table, n_pages = tables(rng, [64, 64, 64])
    table[1, 1], table[2, 0] = n_pages, -1
    pos = rng.integers(0, 100, (3, 30))
    pos[1, 4], pos[2, 5], pos[0, 6] = 100, -1, 2 ** 31 - 1
    for at in ([2, 10, 0], [60, -3, 2 ** 31 - 4]):
        run_append(ctx, dt, 4, 2, [10, 10, 10], at, 1070, table=table, n_pages=n_pages, pos=pos, max_pos=100)
        faults(ctx)


@pytest.mark.parametrize("dt", [F32, BF16, F16, Q8])
def test_append_equals_the_append_of_one_position(ctx, dt):
    """One axis, places that are the positions: the bits of tmac_kv_append_paged."""
    rng = np.random.default_rng(8)
    nh, nkv, counts, at = 14, 2, np.array([5, 40, 1]), np.array([3, 100, 16])
    table, n_pages = tables(rng, at + counts)
    starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    n = int(starts[-1])
    x = oracle.normal(1080, (n, nh + 2 * nkv, 64))
    pos = np.concatenate([a + np.arange(c) for a, c in zip(at, counts)]).astype(np.int32)
    row, got = (nh + 2 * nkv) * 64, []
    dx, dtab, ds, da, dp = (ctx.upload(y) for y in (x, table, starts, at.astype(np.int32), pos))
    for axes in (False, True):
        dk, dv = (ctx.upload(make_pool(1081, n_pages, nkv, dt, True)[0]) for _ in range(2))
        dq = ctx.empty((n, nh, 64))
        head = (dx.ptr, row, dq, dx.at(nh * 64), row, dx.at((nh + nkv) * 64), row, dk, dv, n_pages, dtab, table.shape[1], ds)
        if axes:
            ctx.kv_append_axes_paged(*head, da, dp, 1, None, 3, n, nh, nkv, 64, 200, kv_dtype=dt)
        else:
            ctx.kv_append_paged(*head, da, 3, n, nh, nkv, 64, table.shape[1] * PR, kv_dtype=dt)
        got.append([d.numpy() for d in (dq, dk, dv)])
    for a, b in zip(*got):
        same_bits(a, b, "append")


def test_append_4_bit_blocks_at_the_ends(ctx):
    """Zeros, magnitudes on both sides of the smallest and the largest scale, equal magnitudes of both signs, NaN and
    infinities: codes and scales as the format says.  (Position 0 turns nothing.)"""
    def values(x):
        x[:] = 0
        x[0, :, 3] = 2.0 ** -12
        x[1, :, 3], x[1, :, 9] = -2.0 ** -11, 2.0 ** -11
        x[2, :, 40], x[2, :, 41] = 3.0, -3.0
        x[3, :, 7], x[3, :, 8] = 8 * 8128.0, 1.0
        x[4, :, 7], x[4, :, 8] = 8 * 8200.0, 1.0
        x[5, :, 50] = np.nan
        x[6, :, 33], x[6, :, 34] = -np.inf, np.inf
        x[7] = np.random.default_rng(1).integers(-8, 8, x[7].shape)  # codes that are halves of a step off
    # (keys and values alone: the sign of a NaN in a rotated query is nobody's)
    run_append(ctx, Q4, 2, 1, [8], [5], 1090, pos=np.zeros((3, 8), int), values=values, with_q=False)


# ---- attention and weights ------------------------------------------------------------------

def run_weighted(ctx, dt, nh, nkv, lens, seed, weights=True, in_place=False, max_len=None, stride=None, before=True,
                 poison=True, q=None, pools=None, table=None, n_pages=None):
    rng = np.random.default_rng(seed)
    lens = np.asarray(lens, np.int32)
    n = len(lens)
    if table is None:
        table, n_pages = tables(rng, lens, extra_pages=1, width=1)
    max_len = max_len or max(1, int(lens.max()))
    width = max(table.shape[1], -(-max_len // PR))
    table = np.pad(table, ((0, 0), (0, width - table.shape[1])))
    stride = stride or max_len
    (kp, kw), (vp, vw) = pools or (make_pool(seed + 1 + i, n_pages, nkv, dt, i == 0) for i in (0, 1))
    if poison:  # rows behind the last one hold anything
        kp, vp = kp.copy(), vp.copy()
        for s in range(n):
            for r in range(int(lens[s]), -(-int(lens[s]) // PR) * PR):
                page = table[s, r // PR]
                for pool, key in ((kp, True), (vp, False)):
                    if dt == Q4:
                        byte, _, scale = budget.places(key)
                        pool[page][:, byte[r % PR]] = 0xFF
                        pool[page].view(np.uint16)[:, scale[r % PR]] = 0x7E00
                    else:
                        pool[page, r % PR] = np.nan if dt == F32 else 0xFF if dt == Q8 else 0x7FFF
    if q is None:
        q = oracle.normal(seed + 3, (n, nh, 64))
    w0 = np.abs(oracle.normal(seed + 4, (n, nkv, stride))) if before else None
    after = (w0 if in_place else np.full((n, nkv, stride), 7.5, np.float32)).copy()
    dout = ctx.upload(np.full((n, nh, 64), 7.5, np.float32))
    dwo = ctx.upload(after) if weights else None
    dwi = dwo if in_place else (ctx.upload(w0) if weights and before else None)
    ctx.decode_weighted(ctx.upload(q), ctx.upload(kp), ctx.upload(vp), n_pages, ctx.upload(table), width, ctx.upload(lens), dwi,
                        dwo, stride, dout, n, nh, nkv, 64, max_len, kv_dtype=dt)
    out, w, tol, w_tol = budget.attend64(q, kw, vw, table, lens, nkv)
    got = dout.numpy()
    bad = np.abs(got - out) > tol
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], out[bad][:4], tol[bad][:4])
    if weights:
        gw = dwo.numpy()
        for s in range(n):
            m = int(lens[s])
            ref = w[s, :, :m] + (w0[s, :, :m] if before else 0.0)
            lim = w_tol[s, :, :m] + 2.0 ** -24 * np.abs(ref) * 1.01
            assert (np.abs(gw[s, :, :m] - ref) <= lim).all(), (s, np.abs(gw[s, :, :m] - ref).max())
            same_bits(gw[s, :, m:], after[s, :, m:], "behind the rows")
            if m:  # every query head gives a weight of 1 in all
                total = w[s, :, :m].sum(-1)
                np.testing.assert_allclose(total, nh // nkv, rtol=1e-12)
    return got, dwo.numpy() if weights else None


@by_type
@pytest.mark.parametrize("nh,nkv", HEADS)
def test_weighted_shapes(ctx, dt, nh, nkv):
    run_weighted(ctx, dt, nh, nkv, [0, 1, 15, 16, 17, 31, 32, 33, 200, 0, 513], 1100 + nh)
    no_fault(ctx)


@by_type
def test_weighted_without_weights(ctx, dt):
    a, _ = run_weighted(ctx, dt, 14, 2, [700, 1, 0, 129], 1130, weights=False)
    b, _ = run_weighted(ctx, dt, 14, 2, [700, 1, 0, 129], 1130)
    same_bits(a, b, "with and without weights")


@by_type
@pytest.mark.parametrize("lens", [[1], [9], [2049], [5000], [4096] * 3 + [1, 3000]])
def test_weighted_lengths(ctx, dt, lens):
    run_weighted(ctx, dt, 14, 2, lens, 1140, in_place=True, max_len=max(lens) + 7, stride=max(lens) + 19)
    no_fault(ctx)


@by_type
def test_weighted_many_sequences(ctx, dt):
    rng = np.random.default_rng(12)
    run_weighted(ctx, dt, 7, 1, rng.integers(0, 300, 700), 1150, before=False)
    run_weighted(ctx, dt, 4, 2, rng.integers(0, 900, 150), 1151)
    no_fault(ctx)


@pytest.mark.parametrize("dt", [F32, BF16, Q4])
def test_weighted_late_maximum(ctx, dt):
    """Keys whose scores rise all along the sequence, and large queries: the running maximum moves at every step."""
    rng = np.random.default_rng(13)
    lens = np.array([1000, 333], np.int32)
    table, n_pages = tables(rng, lens)
    x = oracle.normal(1160, (n_pages, PR, 2, 64))
    u = np.sign(oracle.normal(1161, 64)).astype(np.float32)
    for s in range(2):
        for r in range(lens[s]):
            x[table[s, r // PR], r % PR] = x[table[s, r // PR], r % PR] * 0.1 + u * (r / 200)
    st = budget.pack4(x, True) if dt == Q4 else store(x, dt)
    q = np.tile(u, (2, 14, 1)) * 3
    run_weighted(ctx, dt, 14, 2, lens, 1162, q=q, pools=((st, budget.widen(st, dt, True)), make_pool(1163, n_pages, 2, dt, False)),
                 table=table, n_pages=n_pages)


@by_type
def test_weighted_equals_the_paged_decode(ctx, dt):
    """Both within the framework's contract of the same 64-bit result."""
    if dt == Q4:
        pytest.skip("no other call reads 4-bit pages")
    rng = np.random.default_rng(14)
    lens = np.array([900, 37, 2000], np.int32)
    table, n_pages = tables(rng, lens)
    pools = [make_pool(1170 + i, n_pages, 2, dt, i == 0) for i in (0, 1)]
    q = oracle.normal(1172, (3, 14, 64))
    got, _ = run_weighted(ctx, dt, 14, 2, lens, 1173, q=q, pools=pools, table=table, n_pages=n_pages, poison=False)
    out = ctx.empty((3, 14, 64))
    ctx.decode_paged(ctx.upload(q), ctx.upload(pools[0][0]), ctx.upload(pools[1][0]), n_pages, ctx.upload(table), table.shape[1],
                     ctx.upload(lens), out, 3, 14, 2, 64, 2000, kv_dtype=dt)
    assert np.abs(out.numpy() - got).max() <= 4e-5 + 2e-4 * np.abs(got).max()


@by_type
def test_weighted_errors(ctx, dt):
    """A sequence that is too long: NaN, its weights left alone; a page outside the pool: clamped; both reported."""
    rng = np.random.default_rng(15)
    lens = np.array([40, 90, 64], np.int32)
    table, n_pages = tables(rng, lens)
    (kp, _), (vp, _) = (make_pool(1180 + i, n_pages, 2, dt, i == 0) for i in (0, 1))
    q = oracle.normal(1182, (3, 4, 64))
    w = ctx.upload(np.full((3, 2, 80), 7.5, np.float32))
    out = ctx.empty((3, 4, 64))
    args = lambda t, n_len: (ctx.upload(q), ctx.upload(kp), ctx.upload(vp), n_pages, ctx.upload(t), t.shape[1],  # noqa: E731
                             ctx.upload(n_len), None, w, 80, out, 3, 4, 2, 64, 80)
    ctx.decode_weighted(*args(table, lens), kv_dtype=dt)
    got, gw = out.numpy(), w.numpy()
    assert np.isnan(got[1]).all() and np.isfinite(got[[0, 2]]).all()
    assert (gw[1] == 7.5).all() and (gw[0, :, 40:] == 7.5).all() and (gw[0, :, :40] < 7.5).all()
    faults(ctx)
    t = table.copy()
    t[0, 1], t[2, 3] = n_pages + 5, -9
    lens[1] = 80
    ctx.decode_weighted(*args(t, lens), kv_dtype=dt)
    a = out.numpy()
    faults(ctx)
    t[0, 1], t[2, 3] = n_pages - 1, 0
    ctx.decode_weighted(*args(t, lens), kv_dtype=dt)
    same_bits(a, out.numpy(), "clamped")
    no_fault(ctx)
    ctx.decode_weighted(*args(t, np.array([-5, 80, 0], np.int32)), kv_dtype=dt)  # a negative length is 0
    assert (out.numpy()[[0, 2]] == 0).all()
    no_fault(ctx)


# ---- rows to keep ---------------------------------------------------------------------------

def run_rows(ctx, w, lens, keep, first, last, max_len=None):
    n, nkv, stride = w.shape
    kept = ctx.upload(np.full((n, nkv, keep), 99, np.int32))
    ctx.select_rows(ctx.upload(w), stride, ctx.upload(np.asarray(lens, np.int32)), kept, n, nkv, max_len or stride, keep, first,
                    last)
    return kept.numpy()


@pytest.mark.parametrize("n,nkv,longest,keep,first,last", [
    (1, 1, 1, 1, 0, 0), (1, 2, 2048, 512, 4, 64), (9, 3, 700, 68, 4, 64), (5, 2, 5000, 1, 0, 0), (5, 2, 5000, 1, 0, 1),
    (3, 1, 17001, 5003, 4, 64), (2, 1, 40000, 1000, 0, 500), (2, 2, 33000, 32000, 0, 0), (300, 2, 100, 40, 1, 1),
    (4, 1, 1025, 1024, 3, 5), (3, 2, 300, 100, 40, 60)])
def test_rows(ctx, n, nkv, longest, keep, first, last):
    rng = np.random.default_rng(n + longest)
    w = np.exp(rng.normal(0, 3, (n, nkv, longest))).astype(np.float32)
    w[rng.random(w.shape) < 0.1] = 0
    lens = rng.integers(0, longest + 1, n)
    lens[0] = longest
    np.testing.assert_array_equal(run_rows(ctx, w, lens, keep, first, last), keep_ref(w, lens, keep, first, last))
    no_fault(ctx)


def test_rows_ties_and_extremes(ctx):
    rng = np.random.default_rng(21)
    for values in ([0.0], [1.0], [0.0, 1.0], [0.0, -0.0, 1e-45, 2e-45], [-np.inf, -1.0, 0.0, 1.0, np.inf, np.nan],
                   [3.4e38, np.inf, -3.4e38], [1.0, 1.0000001, 1.0000002]):
        for n, keep in ((3000, 700), (20000, 12345)):
            w = rng.choice(np.array(values, np.float32), (2, 2, n))
            ref = keep_ref(np.where(w == 0, np.float32(0), w) if -0.0 not in values[1:2] else w, [n, n - 1], keep, 4, 64)
            got = run_rows(ctx, w, [n, n - 1], keep, 4, 64)
            if values[:2] == [0.0, -0.0]:  # -0 counts as below +0
                order = np.where((w == 0) & np.signbit(w), np.float32(-1e-45), w)
                ref = keep_ref(order, [n, n - 1], keep, 4, 64)
            np.testing.assert_array_equal(got, ref, err_msg=str(values))
    no_fault(ctx)


def test_rows_that_are_kept_anyway_may_hold_anything(ctx):
    rng = np.random.default_rng(22)
    w = rng.random((2, 1, 900), dtype=np.float32)
    ref = run_rows(ctx, w, [900, 900], 100, 10, 30)
    for x in (np.nan, -np.inf, np.inf, -1.0):
        w[:, :, :10] = x
        w[:, :, 870:] = x
        np.testing.assert_array_equal(run_rows(ctx, w, [900, 900], 100, 10, 30), ref)


def test_rows_errors(ctx):
    w = np.random.default_rng(23).random((3, 2, 500), dtype=np.float32)
    got = run_rows(ctx, w, [500, 401, -7], 50, 4, 8, max_len=400)
    assert (got == -1).all()
    faults(ctx)
    got = run_rows(ctx, w, [400, 401, 30], 50, 4, 8, max_len=400)
    np.testing.assert_array_equal(got[[0, 2]], keep_ref(w, [400, 0, 30], 50, 4, 8)[[0, 2]])
    assert (got[1] == -1).all()
    faults(ctx)


# ---- compaction -----------------------------------------------------------------------------

def run_compact(ctx, dt, nkv, lens, keep, seed, kept=None, weights=True, stride=None, to=None, table=None, n_pages=None):
    rng = np.random.default_rng(seed)
    lens = np.asarray(lens, np.int32)
    n = len(lens)
    per = -(-keep // PR)
    if table is None:
        table, n_pages = tables(rng, lens, extra_pages=n * per, width=1)
        free = np.setdiff1d(np.arange(n_pages), np.concatenate([table[s, :-(-int(lens[s]) // PR)] for s in range(n)]))
        to = rng.permutation(free)[:n * per].reshape(n, per).astype(np.int32)
    kp, vp = (make_pool(seed + 1 + i, n_pages, nkv, dt, i == 0)[0] for i in (0, 1))
    stride = stride or max(int(lens.max()), keep)
    w = rng.random((n, nkv, stride), dtype=np.float32)
    if kept is None:
        kept = keep_ref(w, lens, keep, 0, 0)
    dk, dv = ctx.upload(kp), ctx.upload(vp)
    dwo = ctx.upload(np.full_like(w, 7.5)) if weights else None
    ctx.kv_compact_paged(dk, dv, n_pages, ctx.upload(table), table.shape[1], ctx.upload(lens), ctx.upload(kept), keep,
                         ctx.upload(to), to.shape[1], ctx.upload(w) if weights else None, dwo, stride, n, nkv, 64, kv_dtype=dt)
    rk, rv, rw = compact_ref(kp, vp, dt, table, lens, kept, to, w if weights else None, w)
    same_bits(dk.numpy(), rk, "k")
    same_bits(dv.numpy(), rv, "v")
    if weights:
        same_bits(dwo.numpy(), rw, "weights")


@by_type
@pytest.mark.parametrize("nkv,lens,keep", [(1, [1], 1), (2, [40, 0, 300, 17], 33), (3, [64, 200], 64), (8, [100, 90], 7),
                                           (2, [3000, 2500, 2999], 1001)])
def test_compact(ctx, dt, nkv, lens, keep):
    run_compact(ctx, dt, nkv, lens, keep, 1200 + keep)
    run_compact(ctx, dt, nkv, lens, keep, 1201 + keep, weights=False)
    no_fault(ctx)


@by_type
def test_compact_any_list(ctx, dt):
    """Lists in any order, a row twice, gaps: what lies at a gap stays."""
    rng = np.random.default_rng(31)
    kept = rng.integers(0, 90, (2, 2, 50)).astype(np.int32)
    kept[rng.random(kept.shape) < 0.3] = -1
    kept[0, 0, 16:32] = -1  # a page of gaps
    run_compact(ctx, dt, 2, [90, 95], 50, 1210, kept=kept, stride=200)
    no_fault(ctx)


@by_type
def test_compact_errors(ctx, dt):
    rng = np.random.default_rng(32)
    kept = np.sort(rng.integers(0, 60, (2, 1, 20)).astype(np.int32), -1)
    kept[0, 0, 3], kept[0, 0, 5], kept[1, 0, 0], kept[1, 0, 19] = 60, -2, 2 ** 31 - 1, -2 ** 31
    want = np.where((kept >= 60) | (kept < 0), -1, kept).astype(np.int32)
    table, n_pages = tables(rng, [60, 60], extra_pages=4)
    free = np.setdiff1d(np.arange(n_pages), table)
    to = free.reshape(2, 2).astype(np.int32)
    kp, vp = (make_pool(1220 + i, n_pages, 1, dt, i == 0)[0] for i in (0, 1))
    lens = np.array([60, 60], np.int32)

    def go(lst, tab, dst):
        dk, dv = ctx.upload(kp), ctx.upload(vp)
        ctx.kv_compact_paged(dk, dv, n_pages, ctx.upload(tab), 4, ctx.upload(lens), ctx.upload(lst), 20, ctx.upload(dst), 2, None,
                             None, 0, 2, 1, 64, kv_dtype=dt)
        return dk.numpy(), dv.numpy()

    a = go(kept, table, to)
    faults(ctx)
    b = go(want, table, to)
    no_fault(ctx)
    for x, y in zip(a, b):
        same_bits(x, y, "entries outside are skipped")
    t2 = table.copy()
    t2[0, 1] = n_pages + 3
    a = go(want, t2, to)
    faults(ctx)
    t2[0, 1] = n_pages - 1
    if n_pages - 1 not in to:
        for x, y in zip(a, go(want, t2, to)):
            same_bits(x, y, "clamped")
    d2 = to.copy()
    d2[1, 1] = -1
    a = go(want, table, d2)
    faults(ctx)
    ref = want.copy()
    ref[1, 0, 16:] = -1
    for x, y in zip(a, go(ref, table, to)):
        same_bits(x, y, "a page outside the pool is left out")


# ---- together -------------------------------------------------------------------------------

@by_type
def test_a_session_in_a_budget(ctx, dt):
    """A prompt with a video's positions, decode steps whose weights accumulate, eviction to a budget, and further
    steps at rows that are not their positions: every step against the host's own cache."""
    rng = np.random.default_rng(41)
    nh, nkv, n, budget_rows, sinks, recent = 14, 2, 2, 40, 4, 8
    counts = np.array([70, 45])
    cap = 96
    pages = -(-cap // PR)
    n_pages = 2 * n * pages
    order = rng.permutation(n_pages).astype(np.int32).reshape(2, n, pages)
    table, spare = order[0].copy(), order[1].copy()
    kp, vp = (make_pool(1300 + i, n_pages, nkv, dt, i == 0)[0] for i in (0, 1))
    dk, dv, dtab = ctx.upload(kp), ctx.upload(vp), ctx.upload(table)
    row = (nh + 2 * nkv) * 64
    w = np.zeros((n, nkv, cap), np.float32)
    dw = [ctx.upload(w), ctx.upload(w)]
    lens, pos = np.zeros(n, np.int32), np.zeros(n, np.int64)

    def append(counts, positions, seed):
        nonlocal kp, vp
        starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        x = oracle.normal(seed, (int(starts[-1]), nh + 2 * nkv, 64))
        dx, dq = ctx.upload(x), ctx.empty((len(x), nh, 64))
        ctx.kv_append_axes_paged(dx.ptr, row, dq, dx.at(nh * 64), row, dx.at((nh + nkv) * 64), row, dk, dv, n_pages, dtab, pages,
                                 ctx.upload(starts), ctx.upload(lens), ctx.upload(positions.astype(np.int32)), 3, SECTIONS, n,
                                 len(x), nh, nkv, 64, 1000, kv_dtype=dt)
        q, kp, vp = append_ref(x[:, :nh], x[:, nh:nh + nkv], x[:, nh + nkv:], kp, vp, table, starts, lens, positions, SECTIONS,
                               dt, n_pages, 1000, np.zeros((len(x), nh, 64), np.float32))
        same_bits(dq.numpy(), q, "q")
        return dq, q

    positions = np.concatenate([np.stack([np.minimum(np.arange(c), 9), np.arange(c) // 8, np.arange(c) % 8]) for c in counts], 1)
    append(counts, positions, 1310)
    lens[:] = counts
    pos[:] = 70
    for step in range(12):
        dq, q = append([1, 1], np.tile(pos, (3, 1)), 1320 + step)
        lens += 1
        pos += 1
        out = ctx.empty((n, nh, 64))
        ctx.decode_weighted(dq, dk, dv, n_pages, dtab, pages, ctx.upload(lens), dw[0], dw[0], cap, out, n, nh, nkv, 64, cap,
                            kv_dtype=dt)
        kw, vw = budget.widen(kp, dt, True), budget.widen(vp, dt, False)
        ref, rw, tol, w_tol = budget.attend64(q, kw, vw, table, lens, nkv)
        assert (np.abs(out.numpy() - ref) <= tol).all()
        got = dw[0].numpy()
        for s in range(n):
            m = lens[s]
            assert (np.abs(got[s, :, :m] - w[s, :, :m] - rw[s, :, :m]) <= w_tol[s, :, :m] + 2.0 ** -23 * got[s, :, :m]).all()
        w = got
        if step % 5 == 4:  # over budget: keep 40 rows, in the spare pages; the old ones become the spare ones
            kept = ctx.empty((n, nkv, budget_rows), np.int32)
            ctx.select_rows(dw[0], cap, ctx.upload(lens), kept, n, nkv, cap, budget_rows, sinks, recent)
            np.testing.assert_array_equal(kept.numpy(), keep_ref(w, lens, budget_rows, sinks, recent))
            ctx.kv_compact_paged(dk, dv, n_pages, dtab, pages, ctx.upload(lens), kept, budget_rows, ctx.upload(spare), pages, dw[0],
                                 dw[1], cap, n, nkv, 64, kv_dtype=dt)
            kp, vp, w = compact_ref(kp, vp, dt, table, lens, kept.numpy(), spare, w, w)
            same_bits(dw[1].numpy(), w, "weights")
            dw.reverse()
            table, spare = spare, table
            dtab.copy_from(table)
            lens = np.minimum(lens, budget_rows).astype(np.int32)
    same_bits(dk.numpy(), kp, "k")
    same_bits(dv.numpy(), vp, "v")
    no_fault(ctx)


@pytest.mark.parametrize("dt", [BF16, Q4], ids=["bf16", "q4"])
def test_captured_step_replays(ctx, dt):
    """Append, attention with weights, selection and compaction in one captured step: replayed with new rows, lengths
    and positions, with larger eager calls between the replays, each replay equals the eager result."""
    nh, nkv, n, keep = 14, 2, 3, 100
    rng = np.random.default_rng(51)
    base = np.array([300, 200, 250], np.int32)
    table, n_pages = tables(rng, base + 16, extra_pages=3 * 7)
    free = np.setdiff1d(np.arange(n_pages), np.concatenate([table[s, :-(-(int(base[s]) + 16) // PR)] for s in range(n)]))
    to = free[:21].reshape(3, 7).astype(np.int32)
    pools = [make_pool(1400 + i, n_pages, nkv, dt, i == 0)[0] for i in (0, 1)]
    W, L = table.shape[1], 400
    table = np.pad(table, ((0, 0), (0, max(0, 25 - W))))
    W = table.shape[1]
    s = ctx.stream()
    dk, dv, dtab, dto = ctx.upload(pools[0]), ctx.upload(pools[1]), ctx.upload(table), ctx.upload(to)
    dx, dq, out = ctx.empty((n, nh + 2 * nkv, 64)), ctx.empty((n, nh, 64)), ctx.empty((n, nh, 64))
    dat, dlen, dpos = ctx.empty(n, np.int32), ctx.empty(n, np.int32), ctx.empty((3, n), np.int32)
    dstart = ctx.upload(np.arange(n + 1, dtype=np.int32))
    w0 = np.abs(oracle.normal(1402, (n, nkv, L)))
    dw, dw2, dw3, kept = ctx.upload(w0), ctx.empty((n, nkv, L)), ctx.empty((n, nkv, L)), ctx.empty((n, nkv, keep), np.int32)
    dw2.copy_from(w0)
    row = (nh + 2 * nkv) * 64

    def step():
        ctx.kv_append_axes_paged(dx.ptr, row, dq, dx.at(nh * 64), row, dx.at((nh + nkv) * 64), row, dk, dv, n_pages, dtab, W, dstart,
                                 dat, dpos, 3, SECTIONS, n, n, nh, nkv, 64, 5000, stream=s, kv_dtype=dt)
        ctx.decode_weighted(dq, dk, dv, n_pages, dtab, W, dlen, dw, dw2, L, out, n, nh, nkv, 64, L, stream=s, kv_dtype=dt)
        ctx.select_rows(dw2, L, dlen, kept, n, nkv, L, keep, 4, 20, stream=s)
        ctx.kv_compact_paged(dk, dv, n_pages, dtab, W, dlen, kept, keep, dto, 7, dw2, dw3, L, n, nkv, 64, stream=s, kv_dtype=dt)

    def results():
        ctx.synchronize(s)
        return [d.numpy() for d in (dq, dk, dv, out, dw2, kept, dw3)]

    def load(i):
        dx.copy_from(oracle.normal(1410 + i, (n, nh + 2 * nkv, 64)), s)
        dat.copy_from(base + i, s)
        dlen.copy_from(base + i + 1, s)
        dpos.copy_from(np.array([[9, 8, 7], [100 + i, 5, 3], [4000, i, 2]], np.int32), s)

    eager = []
    for i in range(4):
        load(i)
        step()
        eager.append(results())
    dk.copy_from(pools[0], s), dv.copy_from(pools[1], s), dw2.copy_from(w0, s)
    ctx.step_begin(s)
    step()
    graph = ctx.step_end(s)
    try:
        for i in range(4):
            load(i)
            ctx.graph_launch(graph, s)
            for k, (a, b) in enumerate(zip(results(), eager[i])):
                same_bits(a, b, f"replay {i}, output {k}")
            run_weighted(ctx, F16, 14, 2, [4000 + 1000 * i, 77], 1420 + i)  # a larger workspace
            no_fault(ctx)
    finally:
        ctx.graph_destroy(graph)
        ctx.destroy_stream(s)


@by_type
def test_same_call_same_bits(ctx, dt):
    lens = [2300, 0, 900, 1500, 64] * 4
    a = run_weighted(ctx, dt, 14, 2, lens, 1500)
    b = run_weighted(ctx, dt, 14, 2, lens, 1500)
    for x, y in zip(a, b):
        same_bits(x, y, "repeat")


@pytest.mark.parametrize("dt", [F32, Q4], ids=["f32", "q4"])
def test_offsets_beyond_32_bits(ctx, dt):
    """Pages at both ends of pools of more than 4 GiB: append, attention, compaction."""
    nkv = 8
    page_bytes = nkv * (576 if dt == Q4 else 4096)
    n_pages = (1 << 32) // page_bytes + 40
    k, v = ctx.empty(n_pages * page_bytes, np.uint8), ctx.empty(n_pages * page_bytes, np.uint8)
    table = np.array([[n_pages - 1, 0, n_pages - 3], [n_pages - 2, 1, n_pages - 5]], np.int32)
    to = np.array([[n_pages - 7, 3], [5, n_pages - 8]], np.int32)
    starts, at = np.array([0, 40, 75], np.int32), np.array([0, 5], np.int32)
    x = oracle.normal(1600, (75, 3 * nkv, 64))
    pos = np.arange(75, dtype=np.int32)[None]
    dx, dq, dtab = ctx.upload(x), ctx.empty((75, nkv, 64)), ctx.upload(table)
    # the first rows of the second sequence, which the append does not write
    for p in (n_pages - 2,):
        for d in (k, v):
            ctx._check(ctx.lib.tmac_memset(ctx.handle, None, d.ptr + p * page_bytes, 0, page_bytes), "memset")
    row = 3 * nkv * 64
    ctx.kv_append_axes_paged(dx.ptr, row, dq, dx.at(nkv * 64), row, dx.at(2 * nkv * 64), row, k, v, n_pages, dtab, 3,
                             ctx.upload(starts), ctx.upload(at), ctx.upload(pos), 1, None, 2, 75, nkv, nkv, 64, 100, kv_dtype=dt)
    small = {int(p): i for i, p in enumerate(np.concatenate([table.reshape(-1), to.reshape(-1)]))}
    shape = (10, nkv, 576) if dt == Q4 else (10, PR, nkv, 64)
    zero = np.zeros(shape, np.uint8 if dt == Q4 else np.float32)
    stab = np.array([[small[int(p)] for p in r] for r in table], np.int32)
    sto = np.array([[small[int(p)] for p in r] for r in to], np.int32)
    q, rk, rv = append_ref(x[:, :nkv], x[:, nkv:2 * nkv], x[:, 2 * nkv:], zero, zero, stab, starts, at, pos, [0] * 32, dt, 10, 100,
                           np.zeros((75, nkv, 64), np.float32))

    def fetch(d, p):
        out = np.empty(shape[1:], zero.dtype)
        ctx.synchronize()
        ctx._check(ctx.lib.tmac_memcpy_d2h(ctx.handle, None, out.ctypes.data, d.ptr + int(p) * page_bytes, page_bytes), "d2h")
        ctx.synchronize()
        return out

    lens = np.array([40, 40], np.int32)
    out, w = ctx.empty((2, nkv, 64)), ctx.empty((2, nkv, 48))
    ctx.decode_weighted(ctx.upload(q[[39, 74]]), k, v, n_pages, dtab, 3, ctx.upload(lens), None, w, 48, out, 2, nkv, nkv, 64, 48,
                        kv_dtype=dt)
    ref, rw, tol, w_tol = budget.attend64(q[[39, 74]], budget.widen(rk, dt, True), budget.widen(rv, dt, False), stab, lens, nkv)
    assert (np.abs(out.numpy() - ref) <= tol).all()
    gw = w.numpy()[:, :, :40]
    assert (np.abs(gw - rw) <= w_tol + 2.0 ** -23 * gw).all()
    kept = np.tile(np.arange(9, 39, dtype=np.int32), (2, nkv, 1))
    ctx.kv_compact_paged(k, v, n_pages, dtab, 3, ctx.upload(lens), ctx.upload(kept), 30, ctx.upload(to), 2, None, None, 0, 2, nkv, 64,
                         kv_dtype=dt)
    ck, cv, _ = compact_ref(rk, rv, dt, stab, lens, kept, sto, None, None)
    for d, c in ((k, ck), (v, cv)):
        for s in range(2):
            got = fetch(d, to[s, 0])
            same_bits(got, c[sto[s, 0]], "moved")
    no_fault(ctx)
    k.free(), v.free()


def test_two_streams_of_two_contexts(ctx):
    """A second context on its own stream at the same time: neither disturbs the other."""
    import tmac_attn as tm
    rng = np.random.default_rng(61)
    lens = np.full(12, 1500, np.int32)
    table, n_pages = tables(rng, lens)
    (kp, _), (vp, _) = (make_pool(1700 + i, n_pages, 2, Q4, i == 0) for i in (0, 1))
    with tm.Context(0) as other:
        runs = []
        for c, seed in ((ctx, 1702), (other, 1703)):
            s = c.stream()
            q, out, w = c.upload(oracle.normal(seed, (12, 14, 64))), c.empty((12, 14, 64)), c.empty((12, 2, 1500))
            args = (q, c.upload(kp), c.upload(vp), n_pages, c.upload(table), table.shape[1], c.upload(lens), None, w, 1500, out, 12, 14,
                    2, 64, 1500)
            c.decode_weighted(*args, kv_dtype=Q4)
            runs.append((c, s, args, out, w, out.numpy(), w.numpy()))
        for _ in range(20):
            for c, s, args, *_rest in runs:
                c.decode_weighted(*args, stream=s, kv_dtype=Q4)
        for c, s, _, out, w, a, b in runs:
            c.synchronize(s)
            same_bits(out.numpy(), a, "out")
            same_bits(w.numpy(), b, "weights")
            c.destroy_stream(s)


# ---- workgroups by share of the batch's steps ------------------------------------------------

@pytest.mark.parametrize("n,nkv,group", [(3, 2, 7), (70, 1, 1), (60, 3, 2), (257, 1, 9), (300, 1, 2), (1030, 1, 1)])
@pytest.mark.parametrize("dt", [F32, Q4], ids=["f32", "q4"])
def test_weighted_uneven_batches(ctx, dt, n, nkv, group):
    """A few long sequences among short and empty ones, more sequences than a round of the lengths holds: some have
    many workgroups, most one, and the lengths alone decide."""
    rng = np.random.default_rng(n)
    lens = rng.integers(0, 41, n)
    for i, x in zip((0, n // 2, n - 1), (5003, 4100, 6000)):
        lens[i] = x
    run_weighted(ctx, dt, nkv * group, nkv, lens, 1800 + n, max_len=6016)
    run_weighted(ctx, dt, nkv * group, nkv, lens, 1801 + n, weights=False, max_len=6016)
    no_fault(ctx)


@by_type
def test_weighted_long_bound_short_rows(ctx, dt):
    """max_len far above every length, no rows at all, one row."""
    for lens in ([0, 0, 0], [1, 0, 5], [300, 299, 31]):
        run_weighted(ctx, dt, 14, 2, lens, 1810, max_len=9000)
    no_fault(ctx)


def test_weighted_errors_of_long_batches(ctx):
    """As test_weighted_errors where a batch's steps are dealt: too long a sequence gets NaN, the others their result."""
    rng = np.random.default_rng(16)
    lens = np.array([4500, 6000, 30], np.int32)
    table, n_pages = tables(rng, lens)
    pools = [make_pool(1820 + i, n_pages, 2, Q4, i == 0) for i in (0, 1)]
    q = oracle.normal(1822, (3, 14, 64))
    w, out = ctx.upload(np.full((3, 2, 5000), 7.5, np.float32)), ctx.empty((3, 14, 64))
    ctx.decode_weighted(ctx.upload(q), ctx.upload(pools[0][0]), ctx.upload(pools[1][0]), n_pages, ctx.upload(table),
                        table.shape[1], ctx.upload(lens), None, w, 5000, out, 3, 14, 2, 64, 5000, kv_dtype=Q4)
    faults(ctx)
    got, gw = out.numpy(), w.numpy()
    assert np.isnan(got[1]).all() and (gw[1] == 7.5).all()
    keep = [0, 2]
    ref, rw, tol, w_tol = budget.attend64(q[keep], pools[0][1], pools[1][1], table[keep], lens[keep], 2)
    assert (np.abs(got[keep] - ref) <= tol).all()
    for i, s in enumerate(keep):
        m = lens[s]
        assert (np.abs(gw[s, :, :m] - rw[i, :, :m]) <= w_tol[i, :, :m] + 2.0 ** -23 * gw[s, :, :m]).all()
        assert (gw[s, :, m:] == 7.5).all()


def test_captured_long_batch_replays_with_other_lengths(ctx):
    """The lengths on the device deal the work anew on every replay; eager calls on the same workspace between."""
    nh, nkv, n, L = 14, 2, 5, 7000
    rng = np.random.default_rng(52)
    table, n_pages = tables(rng, [L] * n)
    pools = [make_pool(1830 + i, n_pages, nkv, Q4, i == 0)[0] for i in (0, 1)]
    s = ctx.stream()
    dk, dv, dtab, dlen = ctx.upload(pools[0]), ctx.upload(pools[1]), ctx.upload(table), ctx.empty(n, np.int32)
    dq, out, w = ctx.upload(oracle.normal(1832, (n, nh, 64))), ctx.empty((n, nh, 64)), ctx.empty((n, nkv, L))
    w.copy_from(np.zeros((n, nkv, L), np.float32), s)

    def step():
        ctx.decode_weighted(dq, dk, dv, n_pages, dtab, table.shape[1], dlen, None, w, L, out, n, nh, nkv, 64, L, stream=s,
                            kv_dtype=Q4)

    batches = [np.array(x, np.int32) for x in ([7000, 1, 0, 333, 5000], [0, 0, 0, 0, 0], [64, 6999, 7000, 7000, 31], [7000] * 5)]
    eager = []
    for lens in batches:
        dlen.copy_from(lens, s)
        w.copy_from(np.zeros((n, nkv, L), np.float32), s)
        step()
        ctx.synchronize(s)
        eager.append((out.numpy(), w.numpy()))
    ctx.step_begin(s)
    step()
    graph = ctx.step_end(s)
    try:
        for i, lens in enumerate(batches * 2):
            dlen.copy_from(lens, s)
            w.copy_from(np.zeros((n, nkv, L), np.float32), s)
            ctx.graph_launch(graph, s)
            ctx.synchronize(s)
            for a, b in zip((out.numpy(), w.numpy()), eager[i % len(batches)]):
                same_bits(a, b, f"replay {i}")
            run_weighted(ctx, BF16, 8, 8, [200 + 900 * i, 50], 1840 + i)
    finally:
        ctx.graph_destroy(graph)
        ctx.destroy_stream(s)
    no_fault(ctx)


@pytest.mark.parametrize("nh,nkv", [(8, 1), (9, 1), (16, 2), (18, 2)])
def test_weighted_4_bit_scales_of_all_sizes(ctx, nh, nkv):
    """Rows whose scales go from 2^-14 to 2^9, values and keys: both forms of the 4-bit products (up to 8 query heads a kv
    head, and more) hold the bounds."""
    rng = np.random.default_rng(53)
    lens = np.array([400, 77], np.int32)
    table, n_pages = tables(rng, lens)
    pools = []
    for i in (0, 1):
        x = oracle.normal(1850 + i, (n_pages, PR, nkv, 64))
        x *= np.exp2(rng.uniform(-11, 1 if i == 0 else 9, (n_pages, PR, nkv, 1))).astype(np.float32)
        st = budget.pack4(x, i == 0)
        pools.append((st, budget.widen4(st, i == 0)))
    run_weighted(ctx, Q4, nh, nkv, lens, 1852, pools=pools, table=table, n_pages=n_pages)
    no_fault(ctx)


@pytest.mark.parametrize("dt,nh,nkv,n,max_len", [(BF16, 14, 2, 85, 4384), (BF16, 14, 2, 85, 4385), (BF16, 16, 1, 160, 1920),
                                                 (Q4, 16, 1, 160, 1921), (Q4, 14, 2, 86, 4096), (F32, 16, 1, 172, 1921),
                                                 (Q8, 30, 2, 84, 2049), (Q4, 14, 2, 130, 1600), (Q4, 14, 2, 130, 1601),
                                                 (Q4, 14, 2, 130, 2640)])
def test_weights_on_both_sides_of_the_scores_in_lds(ctx, dt, nh, nkv, n, max_len):
    rng = np.random.default_rng(n)
    lens = rng.integers(0, 70, n)
    lens[[1, n // 2, n - 1]] = max_len, max_len - 33, max_len // 2
    run_weighted(ctx, dt, nh, nkv, lens, 1860, max_len=max_len)
    no_fault(ctx)


@by_type
def test_compact_rows_behind_the_weights(ctx, dt):
    """With weights, an entry at weight_stride or above has none: it is skipped and reported, and nothing behind the last
    row of weights is read (the weights end with their allocation)."""
    rng = np.random.default_rng(33)
    lens = np.array([90, 90], np.int32)
    kept = np.sort(rng.integers(0, 90, (2, 3, 40)).astype(np.int32), -1)
    table, n_pages = tables(rng, lens, extra_pages=6)
    to = np.setdiff1d(np.arange(n_pages), table)[:6].reshape(2, 3).astype(np.int32)
    kp, vp = (make_pool(1870 + i, n_pages, 3, dt, i == 0)[0] for i in (0, 1))
    w = rng.random((2, 3, 50), dtype=np.float32)
    got = []
    for lst in (kept, np.where(kept < 50, kept, -1).astype(np.int32)):
        dk, dv, dw = ctx.upload(kp), ctx.upload(vp), ctx.upload(np.full_like(w, 7.5))
        ctx.kv_compact_paged(dk, dv, n_pages, ctx.upload(table), table.shape[1], ctx.upload(lens), ctx.upload(lst), 40,
                             ctx.upload(to), 3, ctx.upload(w), dw, 50, 2, 3, 64, kv_dtype=dt)
        (faults if lst is kept else no_fault)(ctx)
        got.append((dk.numpy(), dv.numpy(), dw.numpy()))
    for a, b in zip(*got):
        same_bits(a, b, "skipped")
    for a, b in zip(got[1], compact_ref(kp, vp, dt, table, lens, np.where(kept < 50, kept, -1), to, w, w)):
        same_bits(a, b, "the others")


def test_two_graphs_share_the_workspace(ctx):
    """Two captured calls of different shapes, both with parts and scores in the workspace, replayed in turn, weights added
    up in place: as often as that the eager call gives."""
    s = ctx.stream()
    sides = []
    for i, (dt, nh, nkv, lens) in enumerate([(Q4, 14, 2, [7000, 3]), (BF16, 16, 4, [3000, 2999, 0, 1500])]):
        rng = np.random.default_rng(70 + i)
        lens = np.array(lens, np.int32)
        n, L = len(lens), int(lens.max())
        table, n_pages = tables(rng, lens)
        pools = [make_pool(1880 + 2 * i + j, n_pages, nkv, dt, j == 0)[0] for j in (0, 1)]
        q, out, w = ctx.upload(oracle.normal(1890 + i, (n, nh, 64))), ctx.empty((n, nh, 64)), ctx.empty((n, nkv, L))
        args = (q, ctx.upload(pools[0]), ctx.upload(pools[1]), n_pages, ctx.upload(table), table.shape[1], ctx.upload(lens), w, w, L,
                out, n, nh, nkv, 64, L)
        zeros = np.zeros((n, nkv, L), np.float32)
        w.copy_from(zeros, s)
        eager = []
        for _ in range(3):
            ctx.decode_weighted(*args, stream=s, kv_dtype=dt)
            ctx.synchronize(s)
            eager.append((out.numpy(), w.numpy()))
        sides.append((args, dt, out, w, zeros, eager))
    graphs = []
    for args, dt, out, w, zeros, _ in sides:
        w.copy_from(zeros, s)
        out.copy_from(np.zeros(out.shape, np.float32), s)
        ctx.step_begin(s)
        ctx.decode_weighted(*args, stream=s, kv_dtype=dt)
        graphs.append(ctx.step_end(s))
    try:
        for turn in range(3):
            for g in graphs:
                ctx.graph_launch(g, s)
            ctx.synchronize(s)
            for _, _, out, w, _, eager in sides:
                same_bits(out.numpy(), eager[turn][0], f"turn {turn}")
                same_bits(w.numpy(), eager[turn][1], f"turn {turn}")
            run_weighted(ctx, F32, 8, 2, [4000 + turn, 77], 1895 + turn)
    finally:
        for g in graphs:
            ctx.graph_destroy(g)
        ctx.destroy_stream(s)
    no_fault(ctx)
