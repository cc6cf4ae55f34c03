"""Helpers of the tests of long contexts in a small cache: 4-bit pages on the host, and plain 64-bit forms of the
operators written from their definitions."""
import numpy as np

import oracle
import serving
import tmac_attn
from serving import ALL_DT, F32, PR

Q4 = tmac_attn.TMAC_KV_Q4_PAGES
TYPES = ALL_DT + [Q4]
BLOCK = tmac_attn.Q4_BLOCK_BYTES


def scale4(x):
    """Scales [..., 2] (fp32, 7 significant bits) of head rows [..., 64]."""
    y = np.ascontiguousarray(x, np.float32).reshape(x.shape[:-1] + (2, 32))
    with np.errstate(invalid="ignore", over="ignore"):
        hi, lo = y.max(-1), y.min(-1)  # NaN spreads
        t = np.where(hi > -lo, hi, lo) * np.float32(-0.125)
        u = t.astype(np.float32).view(np.uint32).astype(np.uint64)
        d = (((u + 0xFFFF + ((u >> 17) & 1)) & ~np.uint64(0x1FFFF)) & 0xFFFFFFFF).astype(np.uint32).view(np.float32)
        d = np.where(np.abs(d) < 2.0 ** -14, np.float32(0), np.where(np.abs(d) > 8128, d * np.float32(np.inf), d))
    return np.where(np.isnan(y).any(-1), np.float32(np.nan), d).astype(np.float32)


def codes4(x):
    """(codes uint8 [..., 64], scales fp32 [..., 2])."""
    d = scale4(x)
    y = np.ascontiguousarray(x, np.float32).reshape(x.shape[:-1] + (2, 32))
    with np.errstate(all="ignore"):
        q = np.rint(y / d[..., None]) + np.float32(8)
        q = np.where(np.isnan(q), 0, np.clip(q, 0, 15))
    return np.where(d[..., None] == 0, 8, q).astype(np.uint8).reshape(x.shape), d


def places(key):
    """Of row r, dim d of a block: its byte and whether the high half [16][64], and the half word of its scale [16][2]."""
    r, d = np.arange(16)[:, None], np.arange(64)[None, :]
    b = np.arange(2)[None, :]
    c = d % 8
    if key:
        return 8 * (16 * (d // 16) + r) + 4 * (d // 8 % 2) + c // 4 + 2 * (c % 2), (c // 2 % 2) + 0 * r, 256 + 16 * b + r
    byte = 8 * (16 * (r // 4) + d % 16) + 4 * (d // 32) + np.array([0, 2, 1, 3])[r % 4]
    return byte, (d // 16 % 2) + 0 * r, 256 + 8 * (r // 4) + 4 * b + r % 4


def put4(block, r, x, key):
    """Writes row r (fp32 [64]) into a block (uint8 [576]) in place."""
    byte, high, scale = places(key)
    q, d = codes4(x)
    keep = np.where(high[r] == 1, 0x0F, 0xF0).astype(np.uint8)
    for i in range(64):
        block[byte[r, i]] = (block[byte[r, i]] & keep[i]) | (q[i] << (4 * high[r, i]))
    with np.errstate(over="ignore"):
        block.view(np.float16)[scale[r]] = d


def pack4(x, key):
    """fp32 [n_pages][16][n_kv][64] -> pages uint8 [n_pages][n_kv][576]."""
    byte, high, scale = places(key)
    q, d = codes4(x)
    q, d = q.transpose(0, 2, 1, 3), d.transpose(0, 2, 1, 3)
    out = np.zeros(q.shape[:2] + (BLOCK,), np.uint8)
    for h in (0, 1):
        out[..., byte[high == h]] |= q[..., high == h] << (4 * h)
    out.view(np.float16)[..., scale.reshape(-1)] = d.reshape(d.shape[:2] + (-1,))
    return out


def widen4(pages, key):
    """Pages -> fp32 [n_pages][16][n_kv][64], exactly."""
    byte, high, scale = places(key)
    q = (pages[..., byte] >> (4 * high).astype(np.uint8)) & 15
    d = np.ascontiguousarray(pages).view(np.float16)[..., scale].astype(np.float32)
    with np.errstate(invalid="ignore"):
        x = (q.astype(np.float32) - 8) * np.repeat(d, 32, -1)
    return np.ascontiguousarray(x.transpose(0, 2, 1, 3))


def make_pool(seed, n_pages, n_kv, dt, key, spread=1.0):
    """(stored pool, widened fp32 [n_pages][16][n_kv][64])."""
    if dt != Q4:
        return serving.make_pool(seed, n_pages, n_kv, dt, spread)
    _, x = serving.make_pool(seed, n_pages, n_kv, F32, spread)
    s = pack4(x, key)
    return s, widen4(s, key)


def widen(pool, dt, key):
    return widen4(pool, key) if dt == Q4 else serving.widen(pool, dt)


def rope_axes(x, pos, axis, base):
    """Heads x [n][64], each pair turned by the position on its axis (the oracle's rotation, bit for bit)."""
    out = np.empty_like(x)
    for a in sorted(set(axis)):
        y = oracle.rope_heads(np.ascontiguousarray(x), len(x), 64, int(pos[a]), base).reshape(len(x), 64)
        d = np.flatnonzero(np.repeat(np.asarray(axis) == a, 2))
        out[:, d] = y[:, d]
    return out


def attend64(q, kw, vw, table, lens, n_kv):
    """(out, weights of every row summed over a kv head's query heads, and bounds of the fp32 errors of both).

    A score of 64 products, summed in fp32 from operands that are exact to 2^-22, is off by at most e = (2^-22 + 66 *
    2^-24) sum |q_d k_d| / 8, and one unit of 2^-24 of its own size in log2 units more, where it is kept: e <= 2^-17.7
    sum |q_d k_d| / 8 covers them.  A weight exp(s - m) / l is then off by a factor of 1 + 2 e (its own score and the
    normaliser's) + 2^-20 (exponential, sums of positive terms over up to 2^15 rows in trees, split weights, division)."""
    n, nh = q.shape[:2]
    G = nh // n_kv
    longest = int(max(lens, default=0))
    out, tol = np.zeros((n, nh, 64)), np.zeros((n, nh, 64))
    w_all, w_tol = np.zeros((n, n_kv, longest)), np.zeros((n, n_kv, longest))
    for s in range(n):
        r = np.arange(int(lens[s]))
        if len(r) == 0:
            continue
        page = table[s, r // PR]
        for h in range(n_kv):
            k, v = kw[page, r % PR, h].astype(np.float64), vw[page, r % PR, h].astype(np.float64)
            qq = q[s, h * G:(h + 1) * G].astype(np.float64)
            x = qq @ k.T / 8
            e = 2 * 2.0 ** -17.7 * (np.abs(qq) @ np.abs(k).T / 8).max() + 2.0 ** -20
            w = np.exp(x - x.max(-1, keepdims=True))
            w /= w.sum(-1, keepdims=True)
            out[s, h * G:(h + 1) * G] = w @ v
            tol[s, h * G:(h + 1) * G] = e * (w @ np.abs(v))
            w_all[s, h, :len(r)] = w.sum(0)
            w_tol[s, h, :len(r)] = e * w.sum(0)
    return out, w_all, tol + 1e-30, w_tol + 1e-30


def keep_ref(w, lens, keep, first, last):
    """kept [n][n_kv][keep]."""
    n, n_kv = w.shape[:2]
    out = np.full((n, n_kv, keep), -1, np.int32)
    for s in range(n):
        m = int(lens[s])
        for h in range(n_kv):
            if m <= keep:
                out[s, h, :m] = np.arange(m)
                continue
            x = w[s, h, :m].astype(np.float64)
            x = np.where(np.isnan(x), np.inf, x)
            j = np.arange(m)
            order = np.lexsort((j, -x, ~((j < first) | (j >= m - last))))
            out[s, h] = np.sort(order[:keep])
    return out


def compact_ref(kp, vp, dt, table, lens, kept, to, w, w_out):
    """(k pool, v pool, weights) after the compaction, on copies; stored rows bit for bit."""
    kp, vp = kp.copy(), vp.copy()
    out = None if w is None else np.zeros_like(w_out)
    src = kp.copy(), vp.copy()
    maps = [places(True), places(False)]
    for s, h, j in zip(*np.nonzero(kept >= 0)):
        r = int(kept[s, h, j])
        if r >= lens[s]:
            continue
        page, dst = table[s, r // PR], to[s, j // PR]
        for pool, old, (byte, high, scale) in zip((kp, vp), src, maps):
            if dt == Q4:
                a, b = np.unique(byte[r % PR], return_index=True)[1], byte[j % PR]
                pool[dst, h, b[a]] = old[page, h, byte[r % PR][a]]
                pool.view(np.uint16)[dst, h, scale[j % PR]] = old.view(np.uint16)[page, h, scale[r % PR]]
            else:
                pool[dst, j % PR, h] = old[page, r % PR, h]
        if out is not None:
            out[s, h, j] = w[s, h, r]
    return kp, vp, out
