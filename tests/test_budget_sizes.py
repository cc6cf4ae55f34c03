"""Sizes that the calls for long contexts in a small cache take, on the CPU: the host layer over a HIP runtime that runs
nothing (see test_serving_refusals.py)."""
import random
import types

import numpy as np
import pytest

import tmac_attn
from test_budget_refusals import call
from test_serving_refusals import P, fake  # noqa: F401  (the fixture)
from tmac_attn import TMAC_ERR_INVALID_ARG, TMAC_OK

COMPACT = "tmac_kv_compact_paged"


@pytest.mark.parametrize("kw", [
    # lists wider than the block table's rows: the pages that those rows take
    dict(max_pages=7, keep=131, to_pages=7, weight_stride=156),
    dict(max_pages=7, keep=131, to_pages=7, weight_stride=97),
    dict(max_pages=1, keep=68, to_pages=1, weight_stride=10),
    dict(max_pages=1, keep=68, to_pages=1, weight_stride=1),
    dict(max_pages=1, keep=2 ** 20, to_pages=1, weights_in=None, weights_out=None, weight_stride=0),
    # lists within them: as many pages as they fill
    dict(keep=112, to_pages=7), dict(keep=100, weight_stride=100), dict(max_pages=7, keep=97, weight_stride=97),
    dict(max_pages=7, keep=96, to_pages=6, weight_stride=96)])
def test_compaction_to_what_the_rows_take(fake, kw):  # noqa: F811
    rc, launches = call(fake, COMPACT, **kw)
    keep = kw["keep"]
    assert rc == TMAC_OK and launches == [("tmac_compact_q4", -(-6 * -(-keep // 16) // 4))]


@pytest.mark.parametrize("kw", [
    dict(max_pages=7, keep=131, to_pages=6), dict(max_pages=7, keep=131, weight_stride=96),
    dict(max_pages=1, keep=68, to_pages=0, weight_stride=16), dict(max_pages=1, keep=68, to_pages=1, weight_stride=0),
    dict(max_pages=1, keep=68, to_pages=1, weight_stride=-1),
    dict(max_pages=7, keep=96, to_pages=5), dict(max_pages=7, keep=96, weight_stride=95),
    dict(max_pages=2 ** 31 - 1, keep=113)])
def test_compaction_to_less_is_refused(fake, kw):  # noqa: F811
    assert call(fake, COMPACT, **kw) == (TMAC_ERR_INVALID_ARG, [])


class Buffer:
    """An address and a shape, in a tensor's place."""
    def __init__(self, at, *shape):
        self.at, self.shape = at, shape

    def data_ptr(self):
        return self.at


def test_every_drawn_case_is_accepted(fake, monkeypatch):  # noqa: F811
    """The arguments of drawn performance cases, as their program makes them (tables as wide as the longest sequence needs,
    destinations as wide as the longest list, lists of `keep` places whatever the lengths): no call is refused."""
    torch = pytest.importorskip("torch")
    cases = pytest.importorskip("perf.more_operators")
    ctx = tmac_attn.Context.__new__(tmac_attn.Context)
    ctx.lib, ctx.handle = fake.lib, fake.handle
    types_of = {"f32": 0, "bf16": 1, "f16": 2, "q8": 3, "q4": tmac_attn.TMAC_KV_Q4_PAGES}
    monkeypatch.setattr(cases, "_held", {"ctx": ctx, "type": types_of})
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: types.SimpleNamespace(cuda_stream=0))
    rng, kinds, wide = random.Random(5), {}, 0
    for case in cases.listed() + [cases.draw(rng) for _ in range(400)]:
        z, kind, n, nkv = cases._sizes(case), case["kind"], case["n_seq"], case["nkv"]
        names = ["q", "kp", "vp", "table", "lens", "out", "weights", "kept", "before", "after", "to", "starts", "at", "pos",
                 "q_out", "qkv"]
        s = types.SimpleNamespace(case=case, **{name: Buffer((i + 1) << 32) for i, name in enumerate(names)})
        s.values = [Buffer(1 << 40), Buffer(1 << 41)] if case.get("cache") in ("q4", "q8") else None
        if kind == "append":
            pages = np.where(z["rows"] > 0, cases._pages_of(z["at"] + z["rows"]) - z["at"] // 16, 0)
            s.t, s.total, s.width, s.axis = int(z["rows"].sum()), int(pages.sum()), cases.MAX_POS // 16, cases._pair_axis(case)
        else:
            pages = cases._pages_of(z["lens"])
            s.width, s.total = int(pages.max()), int(pages.sum())
            if kind == "compact":
                kept = cases._pages_of(np.minimum(z["lens"], case["keep"]))
                s.to.shape, s.total = (n, int(kept.max())), s.total + int(kept.sum())
                wide += case["keep"] > case["max_len"]
        fake.lib.fake_clear()
        cases._run_own(s)  # raises where a call is refused
        assert fake.lib.fake_launches() >= 1, case
        kinds[kind] = kinds.get(kind, 0) + 1
    assert set(kinds) == {"append", "attend", "weigh", "rows", "compact"} and wide > 5, (kinds, wide)


@pytest.mark.parametrize("name,arg,most,more", [
    ("tmac_select_rows", "max_len", 2 ** 31 - 1024, dict(weight_stride=2 ** 31)),
    ("tmac_select_rows", "keep", 2 ** 31 - 1024, {}),
    ("tmac_attention_decode_weighted", "max_len", 2 ** 31 - 1024, dict(max_pages=2 ** 27, weights_in=None, weights_out=None, n_seq=1)),
    ("tmac_kv_append_axes_paged", "n_seq", 2 ** 31 - 1024, {}),
    ("tmac_kv_append_paged", "n_seq", 2 ** 31 - 1024, {})])
def test_counts_that_loops_pass_by_their_steps(fake, name, arg, most, more):  # noqa: F811
    """A kernel's loop adds up to 1,024 to a count behind its end: counts are refused where that would leave 32 bits."""
    def go(n):
        if name == "tmac_kv_append_paged":
            return fake.call(name, **{**more, arg: n})
        return call(fake, name, **{**more, arg: n})
    rc, launches = go(most)
    assert rc == TMAC_OK and launches
    for n in (most + 1, 2 ** 31 - 1):
        assert go(n) == (TMAC_ERR_INVALID_ARG, [])
