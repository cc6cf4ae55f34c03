"""Performance cases of the operators that keep long contexts in a small cache: appending at given rows with rotary
positions of several axes, attention over a cache held in 4 bits, attention that also accumulates the weight of every
row, the choice of the rows to keep by it, and the compaction of the cache to those rows.

Pages hold 16 rows; a pool page row is [kv head][64] in the cache's type (Q8_0: 68 bytes per kv head, int8 q[64] and two
fp16 scales).  A 4-bit page is [kv head][576 bytes]: the codes of 16 rows x 64 dims (512 bytes), then 32 fp16 scales, one a
row and 32 dims; value = (code - 8) * scale.  `_layout` has the places.  The shapes are those of the benchmark
configurations and of the tests (14 query heads over 2 kv heads of 64) and other group sizes.  A case's `lens` number fixes
its lengths, so its work is known without a seed; every value comes from the seed.

Kinds:
  append   rows of a ragged batch at given cache rows: q and k rotated at their positions (1 or 3 axes), k and v stored
  attend   one query token per sequence over its whole 4-bit cache
  weigh    the same over any cache, the softmax weights of every row (summed over a kv head's query heads) accumulated
  rows     per (sequence, kv head) the rows to keep: the first, the last and those of the largest accumulated weight
  compact  the kept rows of k, v and the weights moved to the first rows of other pages
"""
import math
import os
import sys

import numpy as np
import torch

own = False

HD, PAGE, BASE, MAX_POS = 64, 16, 1e6, 32768
HEADS = [(14, 2), (14, 2), (8, 1), (16, 4), (8, 8), (32, 8), (12, 4), (16, 1), (2, 2)]
SINKS, RECENT = 4, 64  # rows kept whatever their weight: the first and the last of a sequence


def listed():
    return [
        # the next token of one session whose cache was compacted: its row is not its position (latency)
        {"name": "append_q4_1x1", "kind": "append", "cache": "q4", "nh": 14, "nkv": 2, "n_seq": 1, "chunk": 1,
         "ragged": False, "first": 600, "axes": 1, "lens": 1},
        # one decode step of a batch of conversations about images
        {"name": "append_bf16_48x1_axes", "kind": "append", "cache": "bf16", "nh": 14, "nkv": 2, "n_seq": 48, "chunk": 1,
         "ragged": False, "first": 9000, "axes": 3, "lens": 2},
        # prompts that hold videos, odd lengths, into the 4-bit cache
        {"name": "append_q4_7x5001_axes", "kind": "append", "cache": "q4", "nh": 14, "nkv": 2, "n_seq": 7, "chunk": 5001,
         "ragged": True, "first": 1000, "axes": 3, "lens": 3},
        # one short conversation (latency)
        {"name": "attend_q4_1x700", "kind": "attend", "cache": "q4", "nh": 14, "nkv": 2, "n_seq": 1, "max_len": 700,
         "lens": 4},
        # a serving batch of long, uneven contexts
        {"name": "attend_q4_45x9001", "kind": "attend", "cache": "q4", "nh": 14, "nkv": 2, "n_seq": 45, "max_len": 9001,
         "lens": 5},
        # the benchmark's batch on a quarter of the bytes
        {"name": "attend_q4_256x4096", "kind": "attend", "cache": "q4", "nh": 14, "nkv": 2, "n_seq": 256,
         "max_len": 4096, "lens": 6},
        # one conversation on the 16-bit cache
        {"name": "weigh_bf16_1x2000", "kind": "weigh", "cache": "bf16", "nh": 14, "nkv": 2, "n_seq": 1, "max_len": 2000,
         "lens": 7},
        # a serving batch on the 4-bit cache
        {"name": "weigh_q4_64x4096", "kind": "weigh", "cache": "q4", "nh": 14, "nkv": 2, "n_seq": 64, "max_len": 4096,
         "lens": 8},
        # one conversation over its budget
        {"name": "rows_1x2048", "kind": "rows", "nh": 14, "nkv": 2, "n_seq": 1, "max_len": 2048, "keep": 512, "lens": 9},
        # a serving batch of long contexts
        {"name": "rows_64x16384", "kind": "rows", "nh": 14, "nkv": 2, "n_seq": 64, "max_len": 16384, "keep": 4096,
         "lens": 10},
        # one conversation over its budget, the 4-bit cache
        {"name": "compact_q4_1x2048", "kind": "compact", "cache": "q4", "nh": 14, "nkv": 2, "n_seq": 1, "max_len": 2048,
         "keep": 512, "lens": 11},
        # a serving batch, odd lengths, the 16-bit cache
        {"name": "compact_bf16_40x8001", "kind": "compact", "cache": "bf16", "nh": 14, "nkv": 2, "n_seq": 40,
         "max_len": 8001, "keep": 4001, "lens": 12},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ranges, no larger than the largest listed one of its kind."""
    most = {}
    for c in listed():
        w = work(c)
        most[c["kind"]] = [max(a, b) for a, b in zip(most.get(c["kind"], (0, 0)), (w["bytes"], w["flops"]))]
    while True:
        kind = rng.choice(["append", "append", "attend", "attend", "weigh", "weigh", "rows", "compact"])
        nh, nkv = rng.choice(HEADS)
        c = {"kind": kind, "nh": nh, "nkv": nkv, "lens": rng.randrange(1 << 30)}
        if kind == "attend":
            c["cache"] = "q4"
        elif kind != "rows":
            c["cache"] = rng.choice(["q4", "q4", "f32", "bf16", "f16", "q8"])
        if kind == "append":
            c.update(n_seq=_log(rng, 1, 512), chunk=rng.choice([1, _log(rng, 1, 8000)]), ragged=rng.random() < 0.7,
                     axes=rng.choice([1, 3]))
            c["first"] = rng.randrange(MAX_POS - c["chunk"])
        else:
            c.update(n_seq=_log(rng, 1, 256), max_len=_log(rng, 1, 32768))
            if kind in ("rows", "compact"):
                c["keep"] = _log(rng, SINKS + RECENT, max(SINKS + RECENT, c["max_len"]))
        w, rows = work(c), c["n_seq"] * c.get("max_len", 0) * c["nkv"]
        if w["bytes"] <= most[kind][0] and w["flops"] <= most[kind][1] and rows <= 1 << 22:
            return c


# ---------------------------------------------------------------- sizes

HEAD_BYTES = {"f32": 256, "bf16": 128, "f16": 128, "q8": 68, "q4": 36}  # one (row, kv head) of 64 dims


def _sizes(case):
    """The lengths a case's `lens` number stands for."""
    r = np.random.default_rng(case["lens"])
    n = case["n_seq"]
    if case["kind"] == "append":
        rows = r.integers(0, case["chunk"] + 1, n) if case["ragged"] else np.full(n, case["chunk"])
        if not rows.sum():
            rows[0] = case["chunk"]
        at = np.full(n, case["first"]) - r.integers(0, min(64, case["first"] + 1), n)
        return {"rows": rows, "at": at, "pos": r.integers(at, MAX_POS - case["chunk"] + 1)}
    return {"lens": r.integers(max(1, case["max_len"] // 2), case["max_len"] + 1, n)}


def _pages_of(lens):
    return (np.asarray(lens, np.int64) + PAGE - 1) // PAGE


def work(case):
    """Bytes (each input once, each output once) and operations of one pass."""
    k, z, nh, nkv, n = case["kind"], _sizes(case), case["nh"], case["nkv"], case["n_seq"]
    if k == "append":
        t = int(z["rows"].sum())
        return {"bytes": t * (4 * HD * (2 * nh + 2 * nkv) + 2 * nkv * HEAD_BYTES[case["cache"]] + 4 * HD
                              + 4 * case["axes"]) + 8 * n, "flops": 3 * HD * t * (nh + nkv)}
    rows = int(z["lens"].sum())
    if k in ("attend", "weigh"):
        b = rows * nkv * 2 * HEAD_BYTES[case["cache"]] + n * (8 * nh * HD + 4) + rows // 4
        return {"bytes": b + (8 * nkv * rows if k == "weigh" else 0),
                "flops": 4 * HD * nh * rows + (3 * nh * rows if k == "weigh" else 0)}
    kept = int(np.minimum(z["lens"], case["keep"]).sum())
    if k == "rows":
        return {"bytes": 4 * nkv * (rows + n * case["keep"]) + 4 * n, "flops": nkv * rows}
    return {"bytes": nkv * (kept * (4 * HEAD_BYTES[case["cache"]] + 4 + 8)) + kept // 2 + 4 * n, "flops": nkv * kept}


# ---------------------------------------------------------------- the 4-bit page

def _layout(what, device):
    """Of the codes of a page's head: byte [16 rows][32], and the two dims whose codes that byte holds (low, high)
    [32]; and byte / 2 of the scales [16 rows][2]."""
    r, j = np.arange(16)[:, None], np.arange(32)[None, :]
    h = np.arange(2)[None, :]
    if what == "k":  # 16 lanes a quarter of the dims, 8 bytes each: dims 16 g + 8 m + ..
        g, m, c = j // 8, j // 4 % 2, j % 4
        byte, low = 8 * (16 * g + r) + 4 * m + c, 16 * g + 8 * m + 4 * (c & 1) + (c >> 1)
        high, scale = low + 2, 256 + 16 * h + r
    else:            # 16 lanes four rows, 8 bytes each: dims i, 16 + i of four rows, then 32 + i, 48 + i
        i, p = j % 16, j // 16
        byte = 8 * (16 * (r // 4) + i) + 4 * p + np.array([0, 2, 1, 3])[r % 4]
        low = 32 * p + i
        high, scale = low + 16, 256 + 8 * (r // 4) + 4 * h + r % 4
    t = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(device)  # noqa: E731
    return t(byte + 0 * j), t(low[0]), t(high[0]), t(scale + 0 * h)


def _codes(x):
    """Head rows [..., 64] fp32 -> codes (uint8) and scales (fp16, [..., 2]).  The scale is the value of the largest
    magnitude over -8, kept to 7 bits so that code times scale is exact in 16; magnitudes below 2^-14 are 0."""
    y = x.unflatten(-1, (2, 32))
    hi, lo = y.amax(-1, keepdim=True), y.amin(-1, keepdim=True)
    u = (torch.where(hi > -lo, hi, lo) * -0.125).view(torch.int32)
    d = ((u + 0xFFFF + ((u >> 17) & 1)) & ~0x1FFFF).view(torch.float32)
    d = torch.where(d.abs() < 2.0 ** -14, torch.zeros_like(d), torch.where(d.abs() > 8128.0, d * math.inf, d))
    q = torch.where(d == 0, torch.full_like(y, 8.0), (torch.round(y / d) + 8).clamp(0, 15))
    return q.to(torch.uint8).flatten(-2), d.squeeze(-1).to(torch.float16)


def _put4(pool, what, page, at, head, x):
    """Rows x [n][64] to row `at` of head `head` of pool pages [page][head][576]."""
    byte, low, high, scale = _layout(what, pool.device)
    q, d = _codes(x)
    pool[page[:, None], head[:, None], byte[at]] = q[:, low] | (q[:, high] << 4)
    pool.view(torch.float16)[page[:, None], head[:, None], scale[at]] = d


def _get4(block, what):
    """Values [..., 16, 64] of page heads [..., 576]."""
    byte, low, high, scale = _layout(what, block.device)
    b = block[..., byte.flatten()].unflatten(-1, (16, 32))
    q = torch.empty(*b.shape[:-1], 64, device=block.device, dtype=torch.float32)
    q[..., low], q[..., high] = (b & 15).float(), (b >> 4).float()
    d = block.view(torch.float16)[..., scale.flatten()].unflatten(-1, (16, 2)).float()
    return ((q - 8).unflatten(-1, (2, 32)) * d.unsqueeze(-1)).flatten(-2)


# ---------------------------------------------------------------- inputs

class _State:
    def __init__(self, case, **tensors):
        self.case = case
        self.__dict__.update(tensors)


def _i32(x):
    return torch.from_numpy(np.ascontiguousarray(x, np.int32)).cuda()


def _pool(g, n_pages, nkv, cache, what):
    """A pool of pages of N(0, 1) rows whose channels differ in size, as trained keys' do."""
    x = torch.randn(n_pages * PAGE * nkv, HD, generator=g, device="cuda")
    x *= torch.exp2(torch.rand(HD, generator=g, device="cuda") - 0.5)
    if cache == "f32":
        return x.view(n_pages, PAGE, nkv, HD)
    if cache == "q4":
        out = torch.empty(n_pages, nkv, 576, device="cuda", dtype=torch.uint8)
        byte, low, high, scale = _layout(what, "cuda")
        q, d = _codes(x)
        q = q.view(n_pages, PAGE, nkv, HD).transpose(1, 2)
        out[..., byte.flatten()] = (q[..., low] | (q[..., high] << 4)).flatten(-2)
        out.view(torch.float16)[..., scale.flatten()] = d.view(n_pages, PAGE, nkv, 2).transpose(1, 2).flatten(-2)
        return out
    if cache != "q8":
        return x.to(torch.bfloat16 if cache == "bf16" else torch.float16).view(n_pages, PAGE, nkv, HD)
    y = x.view(-1, 2, 32)
    d = (y.abs().amax(-1, keepdim=True) / 127).to(torch.float16)
    out = torch.empty(y.shape[0], 68, device="cuda", dtype=torch.uint8)
    out[:, :64] = torch.round(y / d.float()).clamp_(-127, 127).to(torch.int8).view(-1, 64).view(torch.uint8)
    out[:, 64:] = d.view(-1, 2).view(torch.uint8)
    return out.view(n_pages, PAGE, nkv, 68)


def _table(g, pages, total, spare=0):
    """Block table over pages dealt at random out of `total`, none twice; `spare` pages stay free, returned too."""
    width = int(pages.max())
    table = torch.zeros(len(pages), width, device="cuda", dtype=torch.int32)
    used = torch.arange(width, device="cuda")[None, :] < torch.from_numpy(pages).cuda()[:, None]
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table[used] = order[:total - spare]
    return table, width, order[total - spare:]


def _pair_axis(case):
    """The axis that each of the 32 pairs turns by: one, or runs of pairs for time, height and width."""
    return np.array([0] * 32 if case["axes"] == 1 else [0] * 8 + [1] * 12 + [2] * 12, np.uint8)


def _positions(z, axes):
    """[axes][rows]: text counts up on every axis; with three, rows past each sequence's first 16 are a video of frames
    of 8 x 16, whose rows share a time and have a height and a width."""
    out = []
    for p, n in zip(z["pos"], z["rows"]):
        i = np.arange(n)
        if axes == 1:
            out.append(p + i[None])
            continue
        f = np.maximum(i - 16, 0)
        text = np.minimum(i, 16)
        out.append(p + np.stack([text + f // 128, text + f % 128 // 16, text + f % 16]))
    return np.concatenate(out, 1)


def _values(g, case, total):
    """Buffers that stored rows of a narrow type are read back to."""
    if case["cache"] not in ("q4", "q8"):
        return None
    return [torch.empty(total, PAGE, case["nkv"], HD, device="cuda") for _ in range(2)]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    k, nh, nkv, n, z = case["kind"], case["nh"], case["nkv"], case["n_seq"], _sizes(case)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    if k == "append":
        # rows as a fused projection leaves them, [q | k | v], and a table in which only the pages written to are real
        t, lo = int(z["rows"].sum()), z["at"] // PAGE
        pages = np.where(z["rows"] > 0, _pages_of(z["at"] + z["rows"]) - lo, 0)
        width, total = MAX_POS // PAGE, int(pages.sum())
        slot = torch.arange(width, device="cuda")[None, :] - torch.from_numpy(lo).cuda()[:, None]
        table = torch.zeros(n, width, device="cuda", dtype=torch.int32)
        table[(slot >= 0) & (slot < torch.from_numpy(pages).cuda()[:, None])] = torch.randperm(
            total, generator=g, device="cuda").to(torch.int32)
        return _State(case, qkv=rand(t, (nh + 2 * nkv) * HD), q_out=torch.empty(t, nh, HD, device="cuda"), t=t,
                      kp=_pool(g, total, nkv, case["cache"], "k"), vp=_pool(g, total, nkv, case["cache"], "v"),
                      table=table, width=width, total=total, starts=_i32(np.concatenate([[0], np.cumsum(z["rows"])])),
                      at=_i32(z["at"]), pos=_i32(_positions(z, case["axes"])), axis=_pair_axis(case),
                      values=_values(g, case, total))
    pages = _pages_of(z["lens"])
    if k in ("attend", "weigh"):
        total = int(pages.sum())
        table, width, _ = _table(g, pages, total)
        s = _State(case, q=rand(n, nh, HD), kp=_pool(g, total, nkv, case["cache"], "k"),
                   vp=_pool(g, total, nkv, case["cache"], "v"), table=table, width=width, total=total,
                   lens=_i32(z["lens"]), out=torch.empty(n, nh, HD, device="cuda"))
        if k == "weigh":  # what earlier steps left
            s.before = torch.exp(2 * rand(n, nkv, case["max_len"])) * 0.01
            s.after = torch.zeros_like(s.before)
        return s
    # accumulated weights: a few rows hold most, some rows nothing at all
    w = torch.exp(3 * rand(n, nkv, case["max_len"])) * 0.001
    w *= torch.rand(n, nkv, case["max_len"], generator=g, device="cuda") > 0.1
    if k == "rows":
        return _State(case, weights=w, lens=_i32(z["lens"]),
                      kept=torch.empty(n, nkv, case["keep"], device="cuda", dtype=torch.int32))
    kept_pages = _pages_of(np.minimum(z["lens"], case["keep"]))
    total, spare = int(pages.sum() + kept_pages.sum()), int(kept_pages.sum())
    table, width, free = _table(g, pages, total, spare)
    to = torch.zeros(n, int(kept_pages.max()), device="cuda", dtype=torch.int32)
    to[torch.arange(to.shape[1], device="cuda")[None, :] < torch.from_numpy(kept_pages).cuda()[:, None]] = free
    s = _State(case, weights=w, lens=_i32(z["lens"]), kp=_pool(g, total, nkv, case["cache"], "k"),
               vp=_pool(g, total, nkv, case["cache"], "v"), table=table, width=width, total=total, to=to,
               after=torch.empty_like(w), values=_values(g, case, total))
    s.kept = _keep(s)
    return s


# ---------------------------------------------------------------- one pass: the framework's operators

_held = {}


def _ctx():
    """The program's one context."""
    if not _held:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(root, "tmac_gguf.cpp_amd"))
        import tmac_attn as tm
        _held["ctx"] = tm.Context(0)
        _held["ctx"].rope_prepare(HD, BASE, MAX_POS)
        _held["type"] = {"f32": tm.TMAC_KV_F32, "bf16": tm.TMAC_KV_BF16, "f16": tm.TMAC_KV_F16, "q8": tm.TMAC_KV_Q8_0,
                         "q4": tm.TMAC_KV_Q4_PAGES}
    return _held["ctx"], _held["type"]


def _run_own(s):
    ctx, types = _ctx()
    c = s.case
    k, nh, nkv, n = c["kind"], c["nh"], c["nkv"], c["n_seq"]
    stream = torch.cuda.current_stream().cuda_stream
    p = lambda t: t.data_ptr()  # noqa: E731
    dt = types[c.get("cache", "f32")]
    if k == "append":
        row = (nh + 2 * nkv) * HD
        x = p(s.qkv)
        ctx.kv_append_axes_paged(x, row, p(s.q_out), x + 4 * nh * HD, row, x + 4 * (nh + nkv) * HD, row, p(s.kp), p(s.vp),
                                 s.total, p(s.table), s.width, p(s.starts), p(s.at), p(s.pos), c["axes"], s.axis, n, s.t,
                                 nh, nkv, HD, MAX_POS, BASE, stream=stream, kv_dtype=dt)
        return {"q": s.q_out, **_pools_own(s, ctx, dt, stream)}
    if k == "rows":
        ctx.select_rows(p(s.weights), c["max_len"], p(s.lens), p(s.kept), n, nkv, c["max_len"], c["keep"], SINKS, RECENT,
                        stream=stream)
        return s.kept
    if k == "compact":
        ctx.kv_compact_paged(p(s.kp), p(s.vp), s.total, p(s.table), s.width, p(s.lens), p(s.kept), c["keep"], p(s.to),
                             s.to.shape[1], p(s.weights), p(s.after), c["max_len"], n, nkv, HD, stream=stream,
                             kv_dtype=dt)
        return {"weights": s.after, **_pools_own(s, ctx, dt, stream)}
    w = k == "weigh"
    ctx.decode_weighted(p(s.q), p(s.kp), p(s.vp), s.total, p(s.table), s.width, p(s.lens), p(s.before) if w else None,
                        p(s.after) if w else None, c["max_len"], p(s.out), n, nh, nkv, HD,
                        min(c["max_len"], s.width * PAGE), stream=stream, kv_dtype=dt)
    return {"out": s.out, "weights": s.after} if w else s.out


def _pools_own(s, ctx, dt, stream):
    """Both pools; quantized ones as the values they stand for."""
    if s.values is None:
        return {"k": s.kp, "v": s.vp}
    ctx.kv_widen_pages(s.kp.data_ptr(), s.vp.data_ptr(), s.values[0].data_ptr(), s.values[1].data_ptr(), s.total,
                       s.case["nkv"], HD, stream=stream, kv_dtype=dt)
    return {"k": s.values[0], "v": s.values[1]}


# ---------------------------------------------------------------- one pass: the plain forms

def _wide(x, what):
    """Pool pages [..., 16, kv heads, 64 values or 68 bytes] or [..., kv heads, 576] as [..., 16, kv heads, 64] in 32
    bits, exactly."""
    if x.dtype != torch.uint8:
        return x.float()
    if x.shape[-1] == 576:
        return _get4(x, what).transpose(-2, -3)
    q = x[..., :64].view(torch.int8).float().unflatten(-1, (2, 32))
    return (q * x[..., 64:].contiguous().view(torch.float16).float().unsqueeze(-1)).flatten(-2)


def _pools(s):
    if s.values is None:
        return {"k": s.kp, "v": s.vp}
    return {"k": _wide(s.kp, "k"), "v": _wide(s.vp, "v")}


def _angles(pos, axis):
    """cos and sin of the engine's angles, each pair's by the position on its axis: frequency and angle rounded to 32
    bits, as in every row that is in a cache already; of far positions only the values are computed in 64."""
    e = torch.arange(0, HD, 2, device=pos.device, dtype=torch.float32) / HD
    theta = 1.0 / torch.pow(torch.tensor(BASE, device=pos.device, dtype=torch.float64), e.double()).float()
    at = pos[torch.from_numpy(axis.astype(np.int64)).to(pos.device)].T.float()  # [rows][pairs]
    a = (at * theta).double()
    return a.cos().float()[:, None, :], a.sin().float()[:, None, :]


def _rotated(x, c, s):
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)


def _stored(x, like):
    """32-bit rows [t, nkv, 64] in the cache's type."""
    if like.dtype != torch.uint8:
        return x.to(like.dtype)
    y = x.unflatten(-1, (2, 32))
    m = y.abs().amax(-1, keepdim=True)
    d = torch.where(m < 1e-10, 1.0, m / 127)
    b = d.contiguous().view(torch.int32)  # the converter's fp16: mantissa cut, small values 0, large ones infinity
    ex = (b >> 23) & 0xFF
    h = torch.where(ex >= 0x8F, 31 << 10, torch.where(ex <= 0x70, 0, ((ex - 112) << 10) | ((b & 0x7FFFFF) >> 13)))
    q = torch.round(y / d).to(torch.int8).flatten(-2).view(torch.uint8)
    return torch.cat([q, h.to(torch.int16).squeeze(-1).contiguous().view(torch.uint8)], -1)


def _run_append(s):
    nh, nkv = s.case["nh"], s.case["nkv"]
    q, k, v = s.qkv.view(s.t, -1, HD).split([nh, nkv, nkv], 1)
    row = torch.arange(s.t, device=q.device)
    seq = torch.searchsorted(s.starts, row, right=True, out_int32=False) - 1
    cell = s.at[seq] + row - s.starts[seq]
    c, sn = _angles(s.pos, s.axis)
    s.q_out.copy_(_rotated(q, c, sn))
    page, at = s.table[seq, cell // PAGE].long(), (cell % PAGE).long()
    for pool, what, x in ((s.kp, "k", _rotated(k, c, sn)), (s.vp, "v", v)):
        if s.case["cache"] == "q4":
            head = torch.arange(nkv, device=q.device).repeat(s.t)
            _put4(pool, what, page.repeat_interleave(nkv), at.repeat_interleave(nkv), head, x.reshape(-1, HD))
        else:
            pool[page, at] = _stored(x, pool)
    return {"q": s.q_out, **_pools(s)}


def _run_attend(s):
    c = s.case
    n, nh, nkv = c["n_seq"], c["nh"], c["nkv"]
    page = s.table.long()
    k, v = (_wide(t[page], w).flatten(1, 2).transpose(1, 2) for t, w in ((s.kp, "k"), (s.vp, "v")))  # [n][nkv][row][64]
    out = (torch.arange(k.shape[2], device=k.device) >= s.lens[:, None])[:, None, None, :]
    x = torch.matmul(s.q.view(n, nkv, nh // nkv, HD), k.transpose(-1, -2).contiguous()) * 0.125
    x = x.masked_fill(out, -math.inf)
    e = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-3e38))
    e = e / e.sum(-1, keepdim=True).clamp(min=1e-38)
    s.out.copy_(torch.matmul(e, v).view(n, nh, HD))
    if c["kind"] == "attend":
        return s.out
    w = s.before + torch.nn.functional.pad(e.sum(2), (0, max(0, c["max_len"] - e.shape[-1])))[..., :c["max_len"]]
    s.after = torch.where((torch.arange(c["max_len"], device=k.device) < s.lens[:, None])[:, None], w, s.after)
    return {"out": s.out, "weights": s.after}


def _keep(s):
    """Rows to keep [n][nkv][keep], ascending, -1 behind: the first and last, then the largest weights, ties to the
    lower row."""
    n, nkv, keep = s.case["n_seq"], s.case["nkv"], s.case["keep"]
    j = torch.arange(s.case["max_len"], device=s.weights.device)
    lens = s.lens[:, None, None]
    w = s.weights.masked_fill(((j < SINKS) | (j >= lens - RECENT)) & (j < lens), math.inf).masked_fill(j >= lens, -math.inf)
    pick = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :keep]
    pick = torch.where(pick < lens, pick, s.case["max_len"]).sort(-1).values
    kept = torch.full((n, nkv, keep), -1, device=w.device, dtype=torch.int32)
    kept[..., :pick.shape[-1]] = torch.where(pick < s.case["max_len"], pick, -1)
    return kept


def _run_rows(s):
    s.kept.copy_(_keep(s))
    return s.kept


def _run_compact(s):
    n, nkv, keep = s.case["n_seq"], s.case["nkv"], s.case["keep"]
    seq, head, j = (s.kept >= 0).nonzero(as_tuple=True)
    row = s.kept[seq, head, j].long()
    page, at = s.table[seq, row // PAGE].long(), row % PAGE
    to_page, to_at = s.to[seq, j // PAGE].long(), j % PAGE
    for pool, what in ((s.kp, "k"), (s.vp, "v")):
        if s.case["cache"] == "q4":
            byte, _, _, scale = _layout(what, pool.device)
            f = pool.view(torch.float16)
            pool[to_page[:, None], head[:, None], byte[to_at]] = pool[page[:, None], head[:, None], byte[at]]
            f[to_page[:, None], head[:, None], scale[to_at]] = f[page[:, None], head[:, None], scale[at]]
        else:
            pool[to_page, to_at, head] = pool[page, at, head]
    s.after.zero_()
    s.after[seq, head, j] = s.weights[seq, head, row]
    return {"weights": s.after, **_pools(s)}


def run(s):
    if own:
        return _run_own(s)
    return {"append": _run_append, "attend": _run_attend, "weigh": _run_attend, "rows": _run_rows,
            "compact": _run_compact}[s.case["kind"]](s)


# ---------------------------------------------------------------- the same in 64 bits

def _exact_rows(pool, cache, what, h, page, at):
    """float64 values of rows `at` of pool pages `page`, kv head h."""
    if cache == "q4":
        x = pool[page, h].cpu().numpy()
        r, d = at.cpu().numpy()[:, None], np.arange(64)[None, :]
        if what == "k":
            e = d % 8
            byte = 8 * (16 * (d // 16) + r) + 4 * (d % 16 // 8) + e // 4 + 2 * (e % 2)
            high, scale = e // 2 % 2, 512 + 32 * (d // 32) + 2 * r
        else:
            byte = 8 * (16 * (r // 4) + d % 16) + 4 * (d // 32) + np.array([0, 2, 1, 3])[r % 4]
            high, scale = d // 16 % 2, 512 + 16 * (r // 4) + 8 * (d // 32) + 2 * (r % 4)
        n = np.arange(len(x))[:, None]
        code = (x[n, byte + 0 * d].astype(np.int64) >> (4 * high)) & 15
        bits = x[n, scale + 0 * d].astype(np.uint16) | (x[n, scale + 1 + 0 * d].astype(np.uint16) << 8)
        return torch.from_numpy((code - 8) * bits.view(np.float16).astype(np.float64)).to(pool.device)
    x = pool[page, at, h]
    if cache != "q8":
        return x.double()
    x = x.cpu().numpy()
    d = np.ascontiguousarray(x[..., 64:]).view(np.float16).astype(np.float64)
    return torch.from_numpy(np.ascontiguousarray(x[..., :64]).view(np.int8) * np.repeat(d, 32, -1)).to(pool.device)


def exact(case, seed):
    k, n, nh, nkv = case["kind"], case["n_seq"], case["nh"], case["nkv"]
    if k in ("rows", "compact"):
        return None  # whole numbers, and stored rows as they are
    s = prepare(case, seed)
    g, z = nh // nkv, _sizes(case)
    if k == "append":
        cell = np.concatenate([p + np.arange(r) for p, r in zip(z["at"], z["rows"])])
        seq = np.repeat(np.arange(n), z["rows"])
        theta = np.array([np.float32(1) / np.float32(math.pow(BASE, d / HD)) for d in range(0, HD, 2)], np.float32)
        pos = s.pos.cpu().numpy()[s.axis].T
        turn = np.exp(1j * (pos.astype(np.float32) * theta).astype(np.float64))  # the definition's angle
        turn = torch.from_numpy(turn).cuda()[:, None, :]
        spin = lambda x: torch.view_as_real(torch.view_as_complex(x.double().unflatten(-1, (32, 2))) * turn).flatten(-2)  # noqa: E731
        x = s.qkv.view(s.t, -1, HD)
        page = s.table[torch.from_numpy(seq).cuda(), torch.from_numpy(cell // PAGE).cuda()].long()
        at = torch.from_numpy(cell % PAGE).cuda()
        pools = []
        for pool, rows in ((s.kp, spin(x[:, nh:nh + nkv])), (s.vp, x[:, nh + nkv:].double())):
            if s.values is not None:  # what a quantized row holds is no value of its own in 64 bits
                pools.append(None)
                continue
            y = pool.double()
            y[page, at] = rows
            pools.append(y)
        return {"q": spin(x[:, :nh]), "k": pools[0], "v": pools[1]}
    if int(z["lens"].sum()) * nkv > 1 << 21:
        return None
    out = torch.zeros(n, nh, HD, device="cuda", dtype=torch.float64)
    weights = s.after.double() if k == "weigh" else None
    table = s.table.long()
    for i in range(n):
        rows = torch.arange(int(z["lens"][i]), device="cuda")
        page = table[i, rows // PAGE]
        for h in range(nkv):
            heads = slice(h * g, (h + 1) * g)
            kk, vv = (_exact_rows(t, case["cache"], w, h, page, rows % PAGE) for t, w in ((s.kp, "k"), (s.vp, "v")))
            w = torch.softmax(s.q[i, heads].double() @ kk.T / 8.0, -1)
            out[i, heads] = w @ vv
            if k == "weigh":
                weights[i, h, :len(rows)] = s.before[i, h, :len(rows)].double() + w.sum(0)
    return {"out": out, "weights": weights} if k == "weigh" else out
