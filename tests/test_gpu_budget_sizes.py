"""Compaction with lists that are wider than what the sequences hold (tmac_kv_compact_paged behind tmac_select_rows), every
buffer as small as the call takes it, against a plain form, bit for bit."""
import numpy as np
import pytest

from budget import TYPES, compact_ref, keep_ref, make_pool
from serving import PR, tables
from test_gpu_budget import NAMES, faults, no_fault, same_bits

pytestmark = pytest.mark.gpu
by_type = pytest.mark.parametrize("dt", TYPES, ids=[NAMES[t] for t in TYPES])


def setting(rng, lens, nkv, dt, to_pages, seed):
    """(table, pages of the pool, destinations, k pool, v pool): the table as wide as the longest sequence needs."""
    n = len(lens)
    table, n_pages = tables(rng, lens, extra_pages=n * to_pages, width=1)
    used = np.concatenate([table[s, :-(-int(lens[s]) // PR)] for s in range(n)])
    to = rng.permutation(np.setdiff1d(np.arange(n_pages), used))[:n * to_pages].reshape(n, to_pages).astype(np.int32)
    return table, n_pages, to, *(make_pool(seed + i, n_pages, nkv, dt, i == 0)[0] for i in (0, 1))


@by_type
@pytest.mark.parametrize("lens,nkv,keep,stride", [([97, 40, 0], 2, 131, 97), ([97, 112], 2, 131, 112), ([10], 1, 68, 10),
                                                  ([1, 0], 3, 500, 1), ([700, 3, 699], 2, 5000, 700)])
def test_lists_wider_than_the_sequences(ctx, dt, lens, nkv, keep, stride):
    rng = np.random.default_rng(keep + len(lens))
    lens = np.array(lens, np.int32)
    n, to_pages = len(lens), -(-int(lens.max()) // PR)
    table, n_pages, to, kp, vp = setting(rng, lens, nkv, dt, to_pages, 2000 + keep)
    w = rng.random((n, nkv, stride), dtype=np.float32)
    dw, dlens, kept = ctx.upload(w), ctx.upload(lens), ctx.upload(np.full((n, nkv, keep), 99, np.int32))
    ctx.select_rows(dw, stride, dlens, kept, n, nkv, stride, keep, 4, 64)
    lists = kept.numpy()
    np.testing.assert_array_equal(lists, keep_ref(w, lens, keep, 4, 64))
    for weights in (True, False):
        dk, dv, dwo = ctx.upload(kp), ctx.upload(vp), ctx.upload(np.full_like(w, 7.5)) if weights else None
        ctx.kv_compact_paged(dk, dv, n_pages, ctx.upload(table), table.shape[1], dlens, kept, keep, ctx.upload(to), to_pages,
                             dw if weights else None, dwo, stride, n, nkv, 64, kv_dtype=dt)
        rk, rv, rw = compact_ref(kp, vp, dt, table, lens, lists[:, :, :stride], to, w, w)
        same_bits(dk.numpy(), rk, "k")
        same_bits(dv.numpy(), rv, "v")
        if weights:
            same_bits(dwo.numpy(), rw, "weights")
    no_fault(ctx)


@by_type
def test_places_without_a_page_or_a_weight(ctx, dt):
    """A list with rows at places past the destination's pages, or past the weights: those are left out and reported, the
    others move."""
    rng = np.random.default_rng(8)
    lens = np.array([30, 32], np.int32)
    table, n_pages, to, kp, vp = setting(rng, lens, 2, dt, 2, 2100)
    lists = rng.integers(0, 30, (2, 2, 60)).astype(np.int32)
    lists[rng.random(lists.shape) < 0.2] = -1
    for stride in (70, 60, 41, 32, 20, 17):  # rows past 20 and 17 have no weight
        w = rng.random((2, 2, stride), dtype=np.float32)
        dk, dv, dwo = ctx.upload(kp), ctx.upload(vp), ctx.upload(np.full_like(w, 7.5))
        ctx.kv_compact_paged(dk, dv, n_pages, ctx.upload(table), table.shape[1], ctx.upload(lens), ctx.upload(lists), 60,
                             ctx.upload(to), 2, ctx.upload(w), dwo, stride, 2, 2, 64, kv_dtype=dt)
        faults(ctx)
        place = np.arange(60)
        taken = np.where((lists < stride) & (place < stride), lists, -1).astype(np.int32)
        rk, rv, _ = compact_ref(kp, vp, dt, table, lens, np.where(place < 32, taken, -1), to, None, None)
        rw = np.zeros_like(w)
        for s, h, j in zip(*np.nonzero(taken >= 0)):
            rw[s, h, j] = w[s, h, taken[s, h, j]]
        same_bits(dk.numpy(), rk, f"k, {stride}")
        same_bits(dv.numpy(), rv, f"v, {stride}")
        same_bits(dwo.numpy(), rw, f"weights, {stride}")
