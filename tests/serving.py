"""Helpers of the serving tests: page pools on the host, their widened values, and plain
64-bit forms of the serving operators written from their definitions."""
import numpy as np

import oracle
import tmac_attn

PR = tmac_attn.PAGE_ROWS
F32, BF16, F16, Q8 = (tmac_attn.TMAC_KV_F32, tmac_attn.TMAC_KV_BF16, tmac_attn.TMAC_KV_F16, tmac_attn.TMAC_KV_Q8_0)
ALL_DT = [F32, BF16, F16, Q8]
BF16_MAX = np.float32(3.3895313892515355e38)


def store(x, dt):
    """fp32 head rows [..., 64] -> stored head rows [..., 64 values] or [..., 68 bytes]."""
    x = np.ascontiguousarray(x, np.float32)
    if dt == F32:
        return x.copy()
    if dt == F16:
        return x.astype(np.float16).view(np.uint16)
    if dt == BF16:
        u = x.view(np.uint32).astype(np.uint64)
        r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16) & 0xFFFF
        return np.where(np.isnan(x), 0x7FC0, r).astype(np.uint16)
    return oracle.q8_kv_rows(x.reshape(-1, 64)).reshape(x.shape[:-1] + (68,))


def widen(rows, dt):
    """Stored head rows -> fp32 [..., 64], exactly."""
    if dt == F32:
        return np.asarray(rows, np.float32)
    if dt == F16:
        return np.ascontiguousarray(rows).view(np.float16).astype(np.float32)
    if dt == BF16:
        return (rows.astype(np.uint32) << 16).view(np.float32)
    return oracle.q8_kv_widen(np.ascontiguousarray(rows).reshape(-1, 68)).reshape(rows.shape[:-1] + (64,))


def make_pool(seed, n_pages, n_kv, dt, spread=1.0):
    """(stored [n_pages][16][n_kv][64 | 68], widened fp32): N(0, 1) rows of sizes 2^+-spread."""
    x = oracle.normal(seed, (n_pages, PR, n_kv, 64))
    rng = np.random.default_rng(seed)
    x = (x * np.exp2(rng.uniform(-spread, spread, (n_pages, PR, n_kv, 1)))).astype(np.float32)
    s = store(x, dt)
    return s, widen(s, dt)


def tables(rng, lens, extra_pages=0, width=0):
    """Block table over a pool of just the sequences' pages (and a few unused), in random order."""
    need = [-(-int(n) // PR) for n in lens]
    total = sum(need) + extra_pages
    perm = rng.permutation(max(total, 1)).astype(np.int32)
    t = np.zeros((len(lens), max(max(need, default=0), width, 1)), np.int32)
    at = 0
    for s, n in enumerate(need):
        t[s, :n] = perm[at:at + n]
        at += n
    return t, max(total, 1)


def attend64(q, k, v):
    """softmax(q k^T / 8) v in 64 bits; q [G][64], k, v [rows][64]; zeros without rows."""
    if len(k) == 0:
        return np.zeros(q.shape, np.float64)
    x = q.astype(np.float64) @ k.astype(np.float64).T / 8.0
    w = np.exp(x - x.max(-1, keepdims=True))
    return (w @ v.astype(np.float64)) / w.sum(-1, keepdims=True)


def decode64(q, kw, vw, rows_of, n_kv):
    """Attention of every (sequence, kv head) over rows_of(s, h) = (pool pages, rows in them)."""
    n, nh = q.shape[:2]
    G = nh // n_kv
    out = np.zeros((n, nh, 64))
    for s in range(n):
        for h in range(n_kv):
            pg, at = rows_of(s, h)
            out[s, h * G:(h + 1) * G] = attend64(q[s, h * G:(h + 1) * G], kw[pg, at, h], vw[pg, at, h])
    return out


def outward(x, up):
    """fp32 -> the next bf16 at or above (up) or below, finite; as fp32."""
    x = np.asarray(x, np.float32)
    lo16 = (x.view(np.uint32) & 0xFFFF) != 0
    t = x.view(np.uint32) & 0xFFFF0000
    away = lo16 & ((x > 0) if up else (x < 0))
    y = (t + np.where(away, np.uint32(0x10000), np.uint32(0))).astype(np.uint32).view(np.float32)
    return np.clip(y, -BF16_MAX, BF16_MAX)


def bounds_ref(kw, before, table, first, lens, n_kv):
    """bounds [n_pages][n_kv][2][64] as fp32 values, pages outside the ranges as before."""
    b = before.copy()
    for s, n in enumerate(lens):
        f = 0 if first is None else max(int(first[s]), 0)
        if f >= n:
            continue
        for j in range(f // PR, -(-int(n) // PR)):
            rows = kw[table[s, j], :min(PR, int(n) - j * PR)]
            nan = np.isnan(rows).any(0)
            hi = np.where(nan, BF16_MAX, outward(np.fmax.reduce(rows, 0), True))
            lo = np.where(nan, -BF16_MAX, outward(np.fmin.reduce(rows, 0), False))
            b[table[s, j], :, 0], b[table[s, j], :, 1] = hi, lo
    return b


def select_ref(q, b, table, lens, n_kv, top, first, last):
    """selected [n_seq][n_kv][top]: 64-bit sums rounded to fp32, ties to the lower page."""
    n, nh = q.shape[:2]
    G = nh // n_kv
    out = np.full((n, n_kv, top), -1, np.int32)
    for s in range(n):
        m = -(-int(lens[s]) // PR)
        for h in range(n_kv):
            if m <= top:
                out[s, h, :m] = np.arange(m)
                continue
            hi, lo = (b[table[s, :m], h, i].astype(np.float64) for i in (0, 1))
            qq = q[s, h * G:(h + 1) * G].astype(np.float64)
            sc = np.maximum(qq[:, None] * hi, qq[:, None] * lo).sum(-1).max(0).astype(np.float32)
            j = np.arange(m)
            force = (j < first) | (j >= m - last)
            order = np.lexsort((j, -sc.astype(np.float64), ~force))
            out[s, h] = np.sort(order[:top])
    return out


# Shared prefixes that a unit of the prefix kernel walks in several stages (256 rows, fp32 128): name, query heads, kv
# heads, group starts, prefix lengths.
def staged_cases():
    rng = np.random.default_rng(44)
    return [("one group of 96", 14, 2, [0, 96], [12300]),
            ("90 groups of one", 16, 4, list(range(91)), [int(x) for x in rng.integers(500, 901, 90)])]


def stage_rows(dt):
    return 128 if dt == F32 else 256


def runs_of_prefixes(splits, workgroups, most_blocks, starts, nh, nkv):
    """Runs that every prefix is cut into (the kernel's rule), from the arguments of the launch."""
    blocks = min(most_blocks, sum(-(-(b - a) * (nh // nkv) // 64) for a, b in zip(starts, starts[1:])))
    return max(1, min(splits, workgroups // max(1, blocks * nkv)))


def run_rows(prefix, runs):
    """Rows of every run of a prefix, in order."""
    pages = -(-prefix // PR)
    per = max(1, -(-pages // runs)) * PR
    return [(at, min(at + per, prefix)) for at in range(0, prefix, per)]
