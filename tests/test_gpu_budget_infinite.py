"""Row weights of heads whose scores are infinite (tmac_attention_decode_weighted): weights say what the output says.  A head
that no row takes part in (every score -infinity) has a zero output and adds nothing; one whose output is NaN adds NaN."""
import numpy as np
import pytest

import budget
import oracle
from budget import Q4, TYPES, make_pool
from serving import F16, F32, PR, Q8, tables
from test_gpu_budget import NAMES, no_fault

pytestmark = pytest.mark.gpu
by_type = pytest.mark.parametrize("dt", TYPES, ids=[NAMES[t] for t in TYPES])
# whole sequences (scores in LDS; in memory, of 172 sequences with a bound beyond it), and one cut into parts
PATHS = pytest.mark.parametrize("n,nh,nkv,length,max_len", [(3, 4, 2, 70, 70), (172, 32, 2, 37, 1921), (2, 14, 2, 5000, 5000)],
                                ids=["lds", "memory", "parts"])


def put_keys(pool, dt, page, rows, value=-np.inf):
    """Keys of `rows` of `page` get an infinity or NaN in every dim."""
    nan = np.isnan(value)
    for r in rows:
        if dt == Q4:
            byte, _, scale = budget.places(True)
            pool[page][:, byte[r]] = 0x44 if value < 0 else 0xCC  # codes 4 or 12: -4 or 4 times the scale
            pool[page].view(np.uint16)[:, scale[r]] = 0x7E00 if nan else 0x7C00
        elif dt == Q8:
            pool[page, r, :, :64] = 0xFF if value < 0 else 1  # -1 or 1
            pool[page, r, :, 64:] = np.array([0, 0x7E if nan else 0x7C] * 2, np.uint8)
        elif dt == F32:
            pool[page, r] = value
        else:
            infinity = 0x7C00 if dt == F16 else 0x7F80
            pool[page, r] = infinity | (0x8000 if value < 0 else 0x40 if nan else 0)


def run(ctx, dt, n, nh, nkv, length, max_len, q, kp, vp, table, n_pages, lens, stride, in_place):
    w0 = np.abs(oracle.normal(2202, (n, nkv, stride)))
    dw = ctx.upload(w0)
    dwo = dw if in_place else ctx.upload(np.full_like(w0, 7.5))
    out = ctx.empty((n, nh, 64))
    ctx.decode_weighted(ctx.upload(q), ctx.upload(kp), ctx.upload(vp), n_pages, ctx.upload(table), table.shape[1],
                        ctx.upload(lens), dw, dwo, stride, out, n, nh, nkv, 64, max_len, kv_dtype=dt)
    return out.numpy(), dwo.numpy(), w0


@by_type
@PATHS
def test_no_row_takes_part(ctx, dt, n, nh, nkv, length, max_len):
    rng = np.random.default_rng(3)
    lens = np.full(n, length, np.int32)
    table, n_pages = tables(rng, lens, width=-(-max_len // PR))
    (kp, _), (vp, _) = (make_pool(2200 + i, n_pages, nkv, dt, i == 0) for i in (0, 1))
    kp = kp.copy()
    for s in (0, n - 1):
        for r in range(0, length, PR):
            put_keys(kp, dt, table[s, r // PR], range(PR))
    q = np.abs(oracle.normal(2203, (n, nh, 64)))
    got, w, w0 = run(ctx, dt, n, nh, nkv, length, max_len, q, kp, vp, table, n_pages, lens, max_len, n == 3)
    G = nh // nkv
    for s in (0, n - 1):
        for h in range(nkv):
            heads = got[s, h * G:(h + 1) * G]
            assert (np.isnan(heads).all(-1) | (heads == 0).all(-1)).all()
            if np.isnan(heads).any():
                assert np.isnan(w[s, h, :length]).all()
            else:
                np.testing.assert_array_equal(w[s, h, :length], w0[s, h, :length])
            if dt == F32:
                assert (heads == 0).all()
    assert np.isfinite(got[1:n - 1]).all() and np.isfinite(w[1:n - 1]).all()
    no_fault(ctx)


@PATHS
def test_one_head_of_a_group_has_no_row(ctx, n, nh, nkv, length, max_len):
    """fp32 scores of the first head of each group pass the largest float on the negative side; the others' weights are
    those of these heads alone."""
    rng = np.random.default_rng(4)
    lens = np.full(n, length, np.int32)
    table, n_pages = tables(rng, lens, width=-(-max_len // PR))
    (kp, kw), (vp, vw) = (make_pool(2210 + i, n_pages, nkv, F32, i == 0) for i in (0, 1))
    kp = kp.copy()
    kp[..., 0] = np.float32(-3e38)
    q = oracle.normal(2212, (n, nh, 64))
    G = nh // nkv
    q[:, :, 0] = 0
    q[:, ::G, 0] = 100
    got, w, w0 = run(ctx, F32, n, nh, nkv, length, max_len, q, kp, vp, table, n_pages, lens, max_len, False)
    assert (got[:, ::G] == 0).all()
    kw = kw.copy()
    kw[..., 0] = 0
    out, _, tol, _ = budget.attend64(q, kw, vw, table, lens, nkv)
    others = np.flatnonzero(np.arange(nh) % G)
    assert (np.abs(got - out) <= tol)[:, others].all()
    rest = q.reshape(n, nkv, G, 64)[:, :, 1:].reshape(n, -1, 64)
    _, rw, _, w_tol = budget.attend64(rest, kw, vw, table, lens, nkv)
    ref = w0[:, :, :length] + rw
    assert (np.abs(w[:, :, :length] - ref) <= w_tol + 2.0 ** -24 * 1.01 * ref).all()
    no_fault(ctx)


@by_type
@PATHS
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf], ids=["nan", "inf", "minus_inf"])
def test_a_row_that_is_not_finite(ctx, dt, n, nh, nkv, length, max_len, value):
    """One row of the first sequence.  NaN or a score of +infinity: outputs and weights are not finite.  -infinity: the row
    takes weight 0, or that."""
    rng = np.random.default_rng(5)
    lens = np.full(n, length, np.int32)
    table, n_pages = tables(rng, lens, width=-(-max_len // PR))
    (kp, _), (vp, _) = (make_pool(2220 + i, n_pages, nkv, dt, i == 0) for i in (0, 1))
    kp = kp.copy()
    at = length - 3
    put_keys(kp, dt, table[0, at // PR], [at % PR], value)
    q = np.abs(oracle.normal(2223, (n, nh, 64)))
    got, w, w0 = run(ctx, dt, n, nh, nkv, length, max_len, q, kp, vp, table, n_pages, lens, max_len, False)
    G = nh // nkv
    for h in range(nkv):
        heads, rows = got[0, h * G:(h + 1) * G], w[0, h, :length]
        if value < 0 and np.isfinite(heads).all():
            assert rows[at] == w0[0, h, at]
            np.testing.assert_allclose((rows - w0[0, h, :length]).sum(dtype=np.float64), G, rtol=1e-3)
        else:
            assert not np.isfinite(heads).any() or value < 0
            assert not np.isfinite(rows).any()
    assert np.isfinite(got[1:]).all() and np.isfinite(w[1:, :, :length]).all()
    no_fault(ctx)


@by_type
@PATHS
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf], ids=["nan", "inf", "minus_inf"])
def test_a_query_that_is_not_finite(ctx, dt, n, nh, nkv, length, max_len, value):
    """One dim of one query head: that head's output and its kv head's weights are not finite, all others are held to their
    bounds.  (Not to the bits of the call without: a step raises the base of all of a wave's heads when one asks for it, and
    NaN asks at every step, which rounds sums elsewhere.  Each call's results are within budget.attend64's bounds, which do
    not depend on where the base stands.)"""
    rng = np.random.default_rng(6)
    lens = np.full(n, length, np.int32)
    table, n_pages = tables(rng, lens, width=-(-max_len // PR))
    (kp, kw), (vp, vw) = (make_pool(2230 + i, n_pages, nkv, dt, i == 0) for i in (0, 1))
    q = oracle.normal(2233, (n, nh, 64))
    out, rw, tol, w_tol = budget.attend64(q, kw, vw, table, lens, nkv)
    q[n - 1, 1, 5] = value
    got, w, w0 = run(ctx, dt, n, nh, nkv, length, max_len, q, kp, vp, table, n_pages, lens, max_len, False)
    w = w[:, :, :length]
    assert not np.isfinite(got[n - 1, 1]).any() and not np.isfinite(w[n - 1, 0]).any()
    others = np.ones((n, nh), bool)
    others[n - 1, 1] = False
    assert (np.abs(got - out) <= tol)[others].all()
    others = np.ones((n, nkv), bool)
    others[n - 1, 0] = False
    ref = w0[:, :, :length] + rw
    assert (np.abs(w - ref) <= w_tol + 2.0 ** -24 * 1.01 * ref)[others].all()
    no_fault(ctx)
