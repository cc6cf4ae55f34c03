"""Shared prefixes whose units the prefix kernel walks in several stages of rows: buffers in
turn, loads a stage ahead, page lookups two ahead, sums and maxima carried over.  On the
CPU: that the cases have such units (the host layer's own arguments).  On the GPU: against
a plain form in 64 bits, with keys whose scores rise past the lazy maximum's threshold
stage after stage in the keys that one wave takes.  The tolerance is the other serving tests':
where a planted key scores 8.5 log2 units above the rest it has nearly all of the weight, so
that an error e of a score (under 118 * 64 * 2^-24 = 4.5e-4 for the largest ones) moves an
output by 2^-8.5 e at most, 1.2e-6 of it in the worst case and far less at random."""
import numpy as np
import pytest

import late_max
import oracle
from serving import (ALL_DT, F32, decode64, make_pool, run_rows, runs_of_prefixes, stage_rows, staged_cases, store, widen)
from test_gpu_serving import close, no_fault, rows_shared, run_shared, shared_tables
from test_serving_refusals import GOOD, fake  # noqa: F401

NAMES = [c[0] for c in staged_cases()]
RUNS = {"one group of 96": 11, "90 groups of one": 1}


@pytest.mark.parametrize("dt", ALL_DT)
@pytest.mark.parametrize("name,nh,nkv,starts,prefix", staged_cases(), ids=NAMES)
def test_cases_have_units_of_several_stages(fake, dt, name, nh, nkv, starts, prefix):  # noqa: F811
    n = starts[-1]
    rc, launches = fake.call("tmac_attention_decode_shared", kv_dtype=dt, n_head=nh, n_kv_head=nkv, n_seq=n,
                             n_groups=len(prefix), max_prefix=max(prefix), max_tail=64, max_pages=1000)
    assert rc == 0 and launches[0][0].startswith("tmac_prefix_")
    fields = [fake.lib.fake_launch_prefix(0, i) for i in range(3)]
    runs = runs_of_prefixes(*fields, starts, nh, nkv)
    assert runs == RUNS[name]
    rows = [b - a for p in prefix for a, b in run_rows(p, runs)]
    stages = [-(-x // stage_rows(dt)) for x in rows]
    assert max(stages) >= 4 and sum(s >= 3 for s in stages) >= len(stages) // 3
    assert any(x % stage_rows(dt) for x, s in zip(rows, stages) if s >= 3)  # the last stage is a part of one


def small_pool(table, _, of):
    """shared_tables' result over a pool of no more than the pages that are in use."""
    real = table < 2 ** 30
    pages, table = np.unique(table[real]), table.copy()
    table[real] = np.searchsorted(pages, table[real])
    return table, len(pages), of


def behind_one_prefix64(q, kw, vw, rows, prefix, nkv):
    """decode64 of sequences that all read the same first `prefix` rows: their scores in one product a kv head."""
    n, nh = q.shape[:2]
    G, out = nh // nkv, np.zeros((n, nh, 64))
    pg, at = (x[:prefix] for x in rows(0, 0))
    for h in range(nkv):
        v = vw[pg, at, h].astype(np.float64)
        x = q[:, h * G:(h + 1) * G].reshape(-1, 64).astype(np.float64) @ kw[pg, at, h].astype(np.float64).T / 8.0
        m = x.max(-1).reshape(n, G)
        e = np.exp(x - m.reshape(-1, 1))
        top, bottom = (e @ v).reshape(n, G, 64), e.sum(-1).reshape(n, G)
        for s in range(n):
            pg1, at1 = (x[prefix:] for x in rows(s, h))
            x1 = q[s, h * G:(h + 1) * G].astype(np.float64) @ kw[pg1, at1, h].astype(np.float64).T / 8.0
            m1 = np.maximum(m[s], x1.max(-1, initial=-np.inf))
            e1, f = np.exp(x1 - m1[:, None]), np.exp(m[s] - m1)
            a = e1 @ vw[pg1, at1, h].astype(np.float64) + f[:, None] * top[s]
            out[s, h * G:(h + 1) * G] = a / (e1.sum(-1) + f * bottom[s])[:, None]
    return out


def staircase(dt, a, b, quarter):
    """Rows of one wave's keys, one in every stage of the run [a, b) but the first."""
    size = stage_rows(dt)
    return [r for r in range(a + size + size // 4 * quarter + 5, b, size)]


@pytest.mark.gpu
@pytest.mark.parametrize("planted", [False, True])
@pytest.mark.parametrize("dt", ALL_DT)
def test_many_sequences_behind_one_long_prefix(ctx, dt, planted):
    """96 sequences, 11 runs of up to 1,120 rows.  Planted: all queries lean to one side and a few keys of two runs lie
    along it, each scoring at least 8.5 log2 units above all rows of its run before it, for every query head."""
    _, nh, nkv, starts, prefix = staged_cases()[0]
    rng = np.random.default_rng(45)
    n, P = starts[-1], prefix[0]
    lens = (P + rng.integers(0, 40, n)).astype(np.int32)
    table, total, of = small_pool(*shared_tables(rng, starts, prefix, lens))
    x, (vp, vw) = oracle.normal(800, (total, 16, nkv, 64)), make_pool(801, total, nkv, dt)
    q = oracle.normal(802, (n, nh, 64))
    rows = rows_shared(table, starts, prefix, of, lens)
    pg, at = rows(0, 0)
    if planted:
        q += np.float32(1)
        for run, quarter, first in ((2, 1, 3.0), (9, 3, 4.0)):
            a, b = run_rows(P, RUNS[NAMES[0]])[run]
            steps = staircase(dt, a, b, quarter)
            for i, r in enumerate(steps):
                x[pg[r], at[r]] = first + 2 * i
            s = np.einsum("shd,rd->shr", q.astype(np.float64)[:, :7], widen(store(x[pg[a:b], at[a:b], 0], dt), dt)) * (
                late_max.LOG2E / 8)
            for r in steps[1:]:
                assert (s[..., r - a] - s[..., :r - a].max(-1) > 8.5).all()
    kp = store(x, dt)
    got = run_shared(ctx, q, kp, vp, table, lens, starts, prefix, nkv, dt, max_tail=64)
    close(got, behind_one_prefix64(q, widen(kp, dt), vw, rows, P, nkv), f"planted {planted}")
    no_fault(ctx)


@pytest.mark.gpu
@pytest.mark.parametrize("planted", [False, True])
@pytest.mark.parametrize("dt", ALL_DT)
def test_groups_of_one_behind_prefixes_of_several_stages(ctx, dt, planted):
    """90 prefixes of 500 to 900 rows on 4 kv heads, one run each, several units a workgroup.  Planted: in every prefix
    a key a stage that scores 9 log2 units above every row that is not planted, 18, 27 and so on."""
    _, nh, nkv, starts, prefix = staged_cases()[1]
    rng = np.random.default_rng(46)
    n = len(prefix)
    lens = (np.array(prefix) + rng.integers(0, 20, n)).astype(np.int32)
    table, total, of = small_pool(*shared_tables(rng, starts, prefix, lens))
    x, (vp, vw) = oracle.normal(810, (total, 16, nkv, 64)), make_pool(811, total, nkv, dt)
    q = oracle.normal(812, (n, nh, 64))
    rows = rows_shared(table, starts, prefix, of, lens)
    if planted:
        for s in range(n):
            pg, at = rows(s, 0)
            steps = staircase(dt, 0, prefix[s], s % 4)
            k = x[pg, at].reshape(len(pg), nkv * 64)
            x[pg, at] = late_max.plant(q[s], k, steps, [9.0 * (i + 1) for i in range(len(steps))], nh, nkv,
                                       64).reshape(len(pg), nkv, 64)
    kp = store(x, dt)
    if planted and dt == F32:  # a stored key of fewer bits scores a little lower or higher
        for s in (0, 1, 50):
            pg, at = rows(s, 0)
            steps = staircase(dt, 0, prefix[s], s % 4)
            assert late_max.rise_margins(q[s], x[pg, at].reshape(len(pg), -1), steps, nh, nkv, 64).min() > 8.5
    got = run_shared(ctx, q, kp, vp, table, lens, starts, prefix, nkv, dt, max_tail=64)
    close(got, decode64(q, widen(kp, dt), vw, rows, nkv), f"planted {planted}")
    no_fault(ctx)
