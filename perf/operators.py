"""Performance cases of the serving operators on paged caches: appending rotated rows, attention over
shared prefixes, and page-sparse attention (page bounds, page selection, attention over the selection).

Pages hold 16 rows; a pool page row is [kv head][64] in the cache's type (Q8_0: 68 bytes per kv head, int8 q[64]
and two fp16 scales).  The shapes are those of the benchmark configurations and of the tests (14 query heads over
2 kv heads of 64) and other group sizes.  A case's `lens` number fixes its lengths, so its work is known without a
seed; every value comes from the seed.

Kinds:
  append    rows of a ragged batch: q and k rotated at their positions, k and v written to the pages
  bounds    per (page, kv head) the largest and smallest stored key of every dim, bf16 rounded outward
  select    per (sequence, kv head) the pages whose bounds allow the largest q . k
  selected  one query token per sequence over the pages of a list
  shared    one query token per sequence, groups of sequences sharing a prefix
"""
import math
import os
import sys

import numpy as np
import torch

own = False

HD, PAGE, BASE, MAX_POS = 64, 16, 1e6, 32768
BF16_MAX = 3.3895313892515355e38
HEADS = [(14, 2), (14, 2), (8, 1), (16, 4), (8, 8), (32, 8), (12, 4), (16, 1), (2, 2)]


def listed():
    return [
        # the next token of one interactive session (latency)
        {"name": "append_f32_1x1", "kind": "append", "cache": "f32", "nh": 14, "nkv": 2, "n_seq": 1, "chunk": 1,
         "ragged": False, "first": 200, "lens": 1},
        # one decode step of a serving batch, far positions
        {"name": "append_bf16_64x1", "kind": "append", "cache": "bf16", "nh": 14, "nkv": 2, "n_seq": 64, "chunk": 1,
         "ragged": False, "first": 30000, "lens": 2},
        # prompt chunks of several sequences in one batch, odd lengths
        {"name": "append_f16_7x5001", "kind": "append", "cache": "f16", "nh": 14, "nkv": 2, "n_seq": 7, "chunk": 5001,
         "ragged": True, "first": 1000, "lens": 3},
        # after a decode step: the page that each sequence's new row lies in
        {"name": "bounds_bf16_64x1", "kind": "bounds", "cache": "bf16", "nh": 14, "nkv": 2, "n_seq": 64, "new": 1,
         "max_len": 4096, "lens": 4},
        # after a prompt: every page of it
        {"name": "bounds_f32_8x16000", "kind": "bounds", "cache": "f32", "nh": 14, "nkv": 2, "n_seq": 8, "new": 16000,
         "max_len": 16000, "lens": 5},
        # one long document
        {"name": "select_1x16384", "kind": "select", "nh": 14, "nkv": 2, "n_seq": 1, "max_len": 16384, "top": 64,
         "lens": 6},
        # a serving batch with long contexts
        {"name": "select_64x32768", "kind": "select", "nh": 14, "nkv": 2, "n_seq": 64, "max_len": 32768, "top": 128,
         "lens": 7},
        # one long document, a small budget
        {"name": "selected_f32_1x64", "kind": "selected", "cache": "f32", "nh": 14, "nkv": 2, "n_seq": 1, "top": 64,
         "max_len": 16384, "lens": 8},
        # a serving batch on the 16-bit cache
        {"name": "selected_bf16_64x128", "kind": "selected", "cache": "bf16", "nh": 14, "nkv": 2, "n_seq": 64,
         "top": 128, "max_len": 8192, "lens": 9},
        # a few requests on a quantized cache behind a short system prompt
        {"name": "shared_q8_5_700", "kind": "shared", "cache": "q8", "nh": 14, "nkv": 2, "n_seq": 5, "groups": 1,
         "prefix": 700, "tail": 90, "lens": 10},
        # three different few-shot prompts, odd lengths, a wide model
        {"name": "shared_f32_3g45_2500", "kind": "shared", "cache": "f32", "nh": 32, "nkv": 8, "n_seq": 45, "groups": 3,
         "prefix": 2500, "tail": 300, "lens": 11},
        # a serving batch behind one long document
        {"name": "shared_bf16_96_16384", "kind": "shared", "cache": "bf16", "nh": 14, "nkv": 2, "n_seq": 96,
         "groups": 1, "prefix": 16384, "tail": 512, "lens": 12},
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
        kind = rng.choice(["append", "append", "bounds", "select", "selected", "selected", "shared", "shared"])
        nh, nkv = rng.choice(HEADS)
        c = {"kind": kind, "nh": nh, "nkv": nkv, "lens": rng.randrange(1 << 30)}
        if kind != "select":
            c["cache"] = rng.choice(["f32", "bf16", "f16", "q8"])
        if kind == "append":
            c.update(n_seq=_log(rng, 1, 512), chunk=rng.choice([1, _log(rng, 1, 8000)]), ragged=rng.random() < 0.7)
            c["first"] = rng.randrange(MAX_POS - c["chunk"])
        elif kind == "bounds":
            n = _log(rng, 16, MAX_POS)
            c.update(n_seq=_log(rng, 1, 256), max_len=n, new=rng.choice([1, n, _log(rng, 1, n)]))
        elif kind == "select":
            n = _log(rng, 16, MAX_POS)
            c.update(n_seq=_log(rng, 1, 256), max_len=n, top=_log(rng, 2, 512))
        elif kind == "selected":
            c.update(n_seq=_log(rng, 1, 256), top=_log(rng, 1, 512), max_len=_log(rng, 16, 16384))
        else:
            n = _log(rng, 1, 256)
            c.update(n_seq=n, groups=rng.choice([1, min(n, _log(rng, 1, 12))]), prefix=_log(rng, 16, 16384),
                     tail=_log(rng, 1, 2048))
        w, rows = work(c), c["n_seq"] * (c["prefix"] + c["tail"] if kind == "shared" else c.get("max_len", 0)) * c["nkv"]
        if kind in ("selected", "select"):
            rows = min(rows, c["n_seq"] * c["nkv"] * 16 * c["top"]) if kind == "selected" else rows // 8
        if w["bytes"] <= most[kind][0] and w["flops"] <= most[kind][1] and rows <= 1 << 22:
            return c


# ---------------------------------------------------------------- sizes

HEAD_BYTES = {"f32": 256, "bf16": 128, "f16": 128, "q8": 68}  # one (row, kv head) of 64 dims


def _sizes(case):
    """The lengths a case's `lens` number stands for."""
    r = np.random.default_rng(case["lens"])
    n, k = case["n_seq"], case["kind"]
    if k == "append":
        rows = r.integers(0, case["chunk"] + 1, n) if case["ragged"] else np.full(n, case["chunk"])
        if not rows.sum():
            rows[0] = case["chunk"]
        return {"rows": rows, "pos": np.full(n, case["first"]) - r.integers(0, min(64, case["first"] + 1), n)}
    if k == "bounds":
        lens = r.integers(max(1, case["max_len"] // 2), case["max_len"] + 1, n)
        return {"lens": lens, "first": np.maximum(0, lens - case["new"])}
    if k in ("select", "selected"):
        return {"lens": r.integers(max(1, case["max_len"] // 2), case["max_len"] + 1, n)}
    cut = np.sort(r.choice(np.arange(1, n), case["groups"] - 1, replace=False)) if case["groups"] > 1 else []
    starts = np.concatenate([[0], cut, [n]]).astype(np.int64)
    prefix = r.integers(max(1, case["prefix"] * 3 // 4), case["prefix"] + 1, case["groups"])
    prefix[0] = case["prefix"]
    of = np.repeat(np.arange(case["groups"]), np.diff(starts))
    return {"starts": starts, "prefix": prefix, "of": of, "lens": prefix[of] + r.integers(1, case["tail"] + 1, n)}


def _pages_of(lens):
    return (np.asarray(lens, np.int64) + PAGE - 1) // PAGE


def work(case):
    """Bytes (each input once, each output once) and operations of one pass."""
    k, z, nh, nkv, n = case["kind"], _sizes(case), case["nh"], case["nkv"], case["n_seq"]
    if k == "append":
        t = int(z["rows"].sum())
        return {"bytes": t * (4 * HD * (2 * nh + 2 * nkv) + 2 * nkv * HEAD_BYTES[case["cache"]] + 4 * HD) + 8 * n,
                "flops": 3 * HD * t * (nh + nkv)}
    if k == "bounds":
        first = z["first"] // PAGE * PAGE
        pages = int((_pages_of(z["lens"]) - first // PAGE).sum())
        rows = int((z["lens"] - first).sum())
        return {"bytes": rows * nkv * HEAD_BYTES[case["cache"]] + pages * (4 + nkv * 256) + 8 * n,
                "flops": 2 * HD * rows * nkv}
    pages = _pages_of(z["lens"])
    if k == "select":
        p = int(pages.sum())
        return {"bytes": p * (4 + nkv * 256) + n * (4 * nh * HD + 4 * nkv * case["top"] + 4), "flops": 4 * HD * p * nh}
    if k == "selected":
        rows = int((np.minimum(pages, case["top"]) * PAGE).sum())
        return {"bytes": rows * nkv * 2 * HEAD_BYTES[case["cache"]] + n * (8 * nh * HD + 4 * nkv * case["top"] + 4),
                "flops": 4 * HD * nh * rows}
    read = int(z["prefix"].sum() + (z["lens"] - z["prefix"][z["of"]]).sum())
    return {"bytes": read * nkv * 2 * HEAD_BYTES[case["cache"]] + n * (8 * nh * HD + 4) + read // 4,
            "flops": 4 * HD * nh * int(z["lens"].sum())}


# ---------------------------------------------------------------- inputs

class _State:
    def __init__(self, case, **tensors):
        self.case = case
        self.__dict__.update(tensors)


def _i32(x):
    return torch.from_numpy(np.ascontiguousarray(x, np.int32)).cuda()


def _pool(g, n_pages, nkv, cache):
    """A pool of pages of N(0, 1) rows whose channels differ in size, as trained keys' do."""
    x = torch.randn(n_pages * PAGE * nkv, HD, generator=g, device="cuda")
    x *= torch.exp2(torch.rand(HD, generator=g, device="cuda") - 0.5)
    if cache == "f32":
        return x.view(n_pages, PAGE, nkv, HD)
    if cache != "q8":
        return x.to(torch.bfloat16 if cache == "bf16" else torch.float16).view(n_pages, PAGE, nkv, HD)
    y = x.view(-1, 2, 32)
    d = (y.abs().amax(-1, keepdim=True) / 127).to(torch.float16)
    out = torch.empty(y.shape[0], 68, device="cuda", dtype=torch.uint8)
    out[:, :64] = torch.round(y / d.float()).clamp_(-127, 127).to(torch.int8).view(-1, 64).view(torch.uint8)
    out[:, 64:] = d.view(-1, 2).view(torch.uint8)
    return out.view(n_pages, PAGE, nkv, 68)


def _table(g, pages):
    """Block table over a pool of just these pages, in random order; (table, pages per row, pool pages)."""
    total, width = int(pages.sum()), int(pages.max())
    table = torch.zeros(len(pages), width, device="cuda", dtype=torch.int32)
    used = torch.arange(width, device="cuda")[None, :] < torch.from_numpy(pages).cuda()[:, None]
    table[used] = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    return table, width, total


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    k, nh, nkv, n, z = case["kind"], case["nh"], case["nkv"], case["n_seq"], _sizes(case)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    if k == "append":
        # rows as a fused projection leaves them, [q | k | v], and a table in which only the pages written to are real
        t, lo = int(z["rows"].sum()), z["pos"] // PAGE
        pages = np.where(z["rows"] > 0, _pages_of(z["pos"] + z["rows"]) - lo, 0)
        width, total = MAX_POS // PAGE, int(pages.sum())
        slot = torch.arange(width, device="cuda")[None, :] - torch.from_numpy(lo).cuda()[:, None]
        table = torch.zeros(n, width, device="cuda", dtype=torch.int32)
        table[(slot >= 0) & (slot < torch.from_numpy(pages).cuda()[:, None])] = torch.randperm(
            total, generator=g, device="cuda").to(torch.int32)
        return _State(case, qkv=rand(t, (nh + 2 * nkv) * HD), q_out=torch.empty(t, nh, HD, device="cuda"), t=t,
                      kp=_pool(g, total, nkv, case["cache"]), vp=_pool(g, total, nkv, case["cache"]), table=table,
                      width=width, total=total, starts=_i32(np.concatenate([[0], np.cumsum(z["rows"])])),
                      pos=_i32(z["pos"]))
    if k == "shared":
        # a group's pages: the prefix's, then each sequence's own from the page that the prefix ends in
        own_first = z["prefix"][z["of"]] // PAGE
        own_pages, shared = _pages_of(z["lens"]) - own_first, _pages_of(z["prefix"])
        width, total = int(_pages_of(z["lens"]).max()), int(own_pages.sum() + shared.sum())
        order = torch.randperm(total, generator=g, device="cuda").to(torch.int32).cpu().numpy()
        table, at, head = np.zeros((n, width), np.int32), 0, []
        for p in shared:
            head.append(order[at:at + p])
            at += p
        for s in range(n):
            table[s, :own_first[s]] = head[z["of"][s]][:own_first[s]]
            if s == z["starts"][z["of"][s]]:
                # the group's first sequence keeps the page that the prefix ends in and writes on in it
                m = len(head[z["of"][s]])
                table[s, :m] = head[z["of"][s]]
                table[s, m:own_first[s] + own_pages[s]] = order[at + m - own_first[s]:at + own_pages[s]]
            else:
                table[s, own_first[s]:own_first[s] + own_pages[s]] = order[at:at + own_pages[s]]
            at += own_pages[s]
        return _State(case, q=rand(n, nh, HD), kp=_pool(g, total, nkv, case["cache"]),
                      vp=_pool(g, total, nkv, case["cache"]), table=_i32(table), width=width, total=total,
                      lens=_i32(z["lens"]), starts=_i32(z["starts"]), prefix=_i32(z["prefix"]),
                      out=torch.empty(n, nh, HD, device="cuda"))
    if k == "bounds":
        table, width, total = _table(g, _pages_of(z["lens"]))
        return _State(case, kp=_pool(g, total, nkv, case["cache"]), table=table, width=width, total=total,
                      lens=_i32(z["lens"]), first=_i32(z["first"]),
                      bounds=torch.zeros(total, nkv, 2, HD, device="cuda", dtype=torch.bfloat16))
    pages = _pages_of(z["lens"])
    if k == "select":
        table, width, total = _table(g, pages)
        mid, half = rand(total, nkv, HD), 1.2 + rand(total, nkv, HD).abs()
        return _State(case, q=rand(n, nh, HD), table=table, width=width, total=total, lens=_i32(z["lens"]),
                      bounds=torch.stack([mid + half, mid - half], 2).to(torch.bfloat16),
                      selected=torch.empty(n, nkv, case["top"], device="cuda", dtype=torch.int32))
    # selected: any `top` pages of each sequence, ascending, -1 behind
    top, width = case["top"], int(pages.max())
    real = torch.arange(width, device="cuda")[None, None, :] < torch.from_numpy(pages).cuda()[:, None, None]
    pick = torch.rand(n, nkv, width, generator=g, device="cuda").masked_fill_(~real, 2.0).argsort(-1)[..., :top]
    pick = torch.where(real.expand(n, nkv, width).gather(-1, pick), pick, width).sort(-1).values
    pick = torch.nn.functional.pad(pick, (0, top - pick.shape[-1]), value=width)
    # large batches: a pool of 65536 pages stands for the whole cache, pages shared at random
    total = min(int(pages.sum()), 1 << 16)
    table = torch.randint(0, total, (n, width), generator=g, device="cuda", dtype=torch.int32)
    if total == int(pages.sum()):
        table, width, total = _table(g, pages)
    return _State(case, q=rand(n, nh, HD), kp=_pool(g, total, nkv, case["cache"]),
                  vp=_pool(g, total, nkv, case["cache"]), table=table, width=width, total=total, lens=_i32(z["lens"]),
                  selected=torch.where(pick < width, pick, -1).to(torch.int32).contiguous(),
                  out=torch.empty(n, nh, HD, device="cuda"))


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
        _held["type"] = {"f32": tm.TMAC_KV_F32, "bf16": tm.TMAC_KV_BF16, "f16": tm.TMAC_KV_F16, "q8": tm.TMAC_KV_Q8_0}
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
        ctx.kv_append_paged(x, row, p(s.q_out), x + 4 * nh * HD, row, x + 4 * (nh + nkv) * HD, row, p(s.kp), p(s.vp),
                            s.total, p(s.table), s.width, p(s.starts), p(s.pos), n, s.t, nh, nkv, HD, MAX_POS, BASE,
                            stream=stream, kv_dtype=dt)
        return _appended(s)
    if k == "bounds":
        ctx.kv_page_bounds(p(s.kp), s.total, p(s.table), s.width, p(s.first), p(s.lens), p(s.bounds), n, nkv, HD,
                           c["new"], stream=stream, kv_dtype=dt)
        return s.bounds
    if k == "select":
        ctx.select_pages(p(s.q), p(s.bounds), s.total, p(s.table), s.width, p(s.lens), p(s.selected), n, nh, nkv, HD,
                         s.width * PAGE, c["top"], 1, 1, stream=stream)
        return s.selected
    if k == "selected":
        ctx.decode_selected(p(s.q), p(s.kp), p(s.vp), s.total, p(s.table), s.width, p(s.lens), p(s.selected), c["top"],
                            p(s.out), n, nh, nkv, HD, stream=stream, kv_dtype=dt)
        return s.out
    ctx.decode_shared(p(s.q), p(s.kp), p(s.vp), s.total, p(s.table), s.width, p(s.lens), p(s.starts), p(s.prefix),
                      c["groups"], p(s.out), n, nh, nkv, HD, c["prefix"], c["tail"], stream=stream, kv_dtype=dt)
    return s.out


def _appended(s):
    """q rotated and both pools; Q8_0 pools as the values they stand for."""
    if s.case["cache"] != "q8":
        return {"q": s.q_out, "k": s.kp, "v": s.vp}
    val = lambda t: t[..., :64].view(torch.int8).unflatten(-1, (2, 32)) * t[..., 64:].view(  # noqa: E731
        torch.float16).unsqueeze(-1)
    return {"q": s.q_out, "k": val(s.kp), "v": val(s.vp)}


# ---------------------------------------------------------------- one pass: the plain forms

def _wide(x):
    """Cache rows [..., 64 values or 68 bytes] in 32 bits, exactly."""
    if x.dtype != torch.uint8:
        return x.float()
    q = x[..., :64].view(torch.int8).float().unflatten(-1, (2, 32))
    return (q * x[..., 64:].contiguous().view(torch.float16).float().unsqueeze(-1)).flatten(-2)


def _angles(pos):
    """cos and sin of the engine's angles: frequency and angle rounded to 32 bits, as in every row that is in a cache
    already; of far positions only the values are computed in 64."""
    e = torch.arange(0, HD, 2, device=pos.device, dtype=torch.float32) / HD
    theta = 1.0 / torch.pow(torch.tensor(BASE, device=pos.device, dtype=torch.float64), e.double()).float()
    a = (pos.float()[:, None] * theta).double()
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
    pos = s.pos[seq] + row - s.starts[seq]
    c, sn = _angles(pos)
    s.q_out.copy_(_rotated(q, c, sn))
    page, at = s.table[seq, pos // PAGE].long(), pos % PAGE
    s.kp[page, at] = _stored(_rotated(k, c, sn), s.kp)
    s.vp[page, at] = _stored(v, s.vp)
    return _appended(s)


def _outward(x, up):
    """Rounded to bf16 toward +inf (up) or -inf."""
    r = x.to(torch.bfloat16)
    off = (r.float() < x) if up else (r.float() > x)
    far = torch.tensor(math.inf if up else -math.inf, device=x.device, dtype=torch.bfloat16)
    return torch.where(off, torch.nextafter(r, far), r).clamp(-BF16_MAX, BF16_MAX)


def _run_bounds(s):
    n, new = s.case["n_seq"], s.case["new"]
    m = (new + PAGE - 2) // PAGE + 1  # pages that `new` rows can touch
    j = (s.first // PAGE)[:, None] + torch.arange(m, device=s.kp.device)
    row = j[..., None] * PAGE + torch.arange(PAGE, device=s.kp.device)
    real = j * PAGE < s.lens[:, None]
    page = torch.gather(s.table, 1, j.clamp(max=s.width - 1).long()).long()[real]
    k = _wide(s.kp[page])
    out = (row >= s.lens[:, None, None])[real][..., None, None]
    hi, lo = k.masked_fill(out, -math.inf).amax(1), k.masked_fill(out, math.inf).amin(1)
    s.bounds[page] = torch.stack([_outward(hi, True), _outward(lo, False)], 2)
    return s.bounds


def _run_select(s):
    n, nkv, top, g = s.case["n_seq"], s.case["nkv"], s.case["top"], s.case["nh"] // s.case["nkv"]
    j = torch.arange(s.width, device=s.q.device)
    pages = ((s.lens + PAGE - 1) // PAGE)[:, None, None]
    b = s.bounds[s.table.long()].double().permute(0, 2, 3, 1, 4)  # [n][nkv][2][page][64]
    q = s.q.view(n, nkv, g, HD).double()
    # 64 bits: the order of scores that differ in the last of 32 decides what is selected
    score = torch.matmul(q.clamp(min=0), b[:, :, 0].transpose(-1, -2).contiguous())
    score = (score + torch.matmul(q.clamp(max=0), b[:, :, 1].transpose(-1, -2).contiguous())).amax(2).float()
    always = ((j < 1) | (j == pages - 1)) & (j < pages)
    score = score.masked_fill(always, math.inf).masked_fill(j >= pages, -math.inf)
    pick = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :top]
    pick = torch.where(pick < pages, pick, s.width).sort(-1).values
    s.selected.fill_(-1)
    s.selected[..., :pick.shape[-1]] = torch.where(pick < s.width, pick, -1)
    return s.selected


def _attend(q, k, v, out):
    """softmax(q k^T / 8) v over the last axis but one of k and v; rows where `out` is true take no part; 0 where none do."""
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()) * 0.125
    x = x.masked_fill(out, -math.inf)
    m = x.amax(-1, keepdim=True).clamp(min=-3e38)
    e = torch.exp(x - m)
    return torch.matmul(e, v) / e.sum(-1, keepdim=True).clamp(min=1e-38)


def _run_selected(s):
    n, nh, nkv, top = s.case["n_seq"], s.case["nh"], s.case["nkv"], s.case["top"]
    page = torch.gather(s.table, 1, s.selected.clamp(min=0).view(n, -1).long()).view(n, nkv, top).long()
    head = torch.arange(nkv, device=page.device)[None, :, None]
    k, v = (_wide(t.transpose(1, 2)[page, head]).reshape(n, nkv, top * PAGE, HD) for t in (s.kp, s.vp))
    row = s.selected[..., None] * PAGE + torch.arange(PAGE, device=page.device)
    out = ((s.selected[..., None] < 0) | (row >= s.lens[:, None, None, None])).view(n, nkv, 1, top * PAGE)
    s.out.copy_(_attend(s.q.view(n, nkv, nh // nkv, HD), k, v, out).view(n, nh, HD))
    return s.out


def _run_shared(s):
    n, nh, nkv = s.case["n_seq"], s.case["nh"], s.case["nkv"]
    g = torch.searchsorted(s.starts, torch.arange(n, device=s.q.device), right=True, out_int32=False) - 1
    row = torch.arange(s.width * PAGE, device=s.q.device)
    at = torch.arange(n, device=s.q.device)[:, None]
    frm = torch.where(row < s.prefix[g][:, None], s.starts[g][:, None].long(), at)  # the sequence whose pages hold it
    page = s.table[frm, row // PAGE].long()
    k, v = (_wide(t[page, row % PAGE]).transpose(1, 2) for t in (s.kp, s.vp))
    out = (row >= s.lens[:, None])[:, None, None, :]
    s.out.copy_(_attend(s.q.view(n, nkv, nh // nkv, HD), k, v, out).reshape(n, nh, HD))
    return s.out


def run(s):
    if own:
        return _run_own(s)
    return {"append": _run_append, "bounds": _run_bounds, "select": _run_select, "selected": _run_selected,
            "shared": _run_shared}[s.case["kind"]](s)


# ---------------------------------------------------------------- the same in 64 bits

def _exact_rows(pool, page, at):
    """float64 values of rows `at` of pool pages `page`."""
    x = pool[page, at]
    if x.dtype != torch.uint8:
        return x.double()
    x = x.cpu().numpy()
    d = np.ascontiguousarray(x[..., 64:]).view(np.float16).astype(np.float64)
    return torch.from_numpy(np.ascontiguousarray(x[..., :64]).view(np.int8) * np.repeat(d, 32, -1)).to(pool.device)


def _softmax_rows(q, k, v):
    """[heads][64] of float64 queries over float64 rows [rows][64]."""
    w = torch.softmax(q @ k.T / 8.0, -1)
    return w @ v


def exact(case, seed):
    s = prepare(case, seed)
    k, n, nh, nkv = case["kind"], case["n_seq"], case["nh"], case["nkv"]
    g, z = nh // nkv, _sizes(case)
    if k == "append":
        pos = np.concatenate([p + np.arange(r) for p, r in zip(z["pos"], z["rows"])])
        seq = np.repeat(np.arange(n), z["rows"])
        theta = np.array([np.float32(1) / np.float32(math.pow(BASE, d / HD)) for d in range(0, HD, 2)], np.float32)
        turn = np.exp(1j * (pos.astype(np.float32)[:, None] * theta).astype(np.float64))  # the definition's angle
        turn = torch.from_numpy(turn).cuda()[:, None, :]
        spin = lambda x: torch.view_as_real(torch.view_as_complex(x.double().unflatten(-1, (32, 2))) * turn).flatten(-2)  # noqa: E731
        x = s.qkv.view(s.t, -1, HD)
        page = s.table[torch.from_numpy(seq).cuda(), torch.from_numpy(pos // PAGE).cuda()].long()
        at = torch.from_numpy(pos % PAGE).cuda()
        pools = []
        for pool, rows in ((s.kp, spin(x[:, nh:nh + nkv])), (s.vp, x[:, nh + nkv:].double())):
            if case["cache"] == "q8":  # what a quantized row holds is no value of its own in 64 bits
                pools.append(None)
                continue
            y = pool.double()
            y[page, at] = rows
            pools.append(y)
        return {"q": spin(x[:, :nh]), "k": pools[0], "v": pools[1]}
    if k == "bounds":  # before the outward rounding to 16 bits
        far = s.bounds.double()
        for i in range(n):
            j = torch.arange(int(z["first"][i]) // PAGE, -(-int(z["lens"][i]) // PAGE), device="cuda")
            page = s.table[i, j].long()
            x = _exact_rows(s.kp, page[:, None], torch.arange(PAGE, device="cuda")[None, :])
            last = int(z["lens"][i]) - (len(j) - 1 + int(j[0])) * PAGE
            far[page, :, 0] = torch.cat([x[:-1].amax(1), x[-1:, :last].amax(1)])
            far[page, :, 1] = torch.cat([x[:-1].amin(1), x[-1:, :last].amin(1)])
        return far
    if k == "select":
        return None  # whole numbers
    out = torch.zeros(n, nh, HD, device="cuda", dtype=torch.float64)
    table = s.table.long()
    for i in range(n):
        length = int(z["lens"][i])
        for h in range(nkv):
            if k == "selected":
                rows = [j * PAGE + r for j in s.selected[i, h].tolist() if j >= 0 for r in range(PAGE)]
                rows = torch.tensor([r for r in rows if r < length], device="cuda", dtype=torch.long)
                page = table[i, rows // PAGE]
            else:
                rows = torch.arange(length, device="cuda")
                grp = int(z["of"][i])
                page = table[i, rows // PAGE]
                p = int(z["prefix"][grp])
                page[:p] = table[int(z["starts"][grp]), rows[:p] // PAGE]
            if rows.numel():
                heads = slice(h * g, (h + 1) * g)
                kk, vv = (_exact_rows(t[:, :, h], page, rows % PAGE) for t in (s.kp, s.vp))
                out[i, heads] = _softmax_rows(s.q[i, heads].double(), kk, vv)
    return out
