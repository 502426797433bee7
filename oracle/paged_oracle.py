"""The paged cache, the attention over it and the choice of a token, restated in numpy float64 from their definitions.

Parity unpinned: the reference holds no such operators (it configures a streaming recogniser with look-back at
voice-service/app/services/voice_interface.py:651-653 and leaves the call commented out at :1753-1809)."""
import numpy as np


# ---- e4m3 under power-of-two scales -------------------------------------------------------------------------------------
def e4m3_values():
    """The value of every code 0 .. 255: 4 exponent bits with bias 7, 3 mantissa bits, no infinities, 0x7f and 0xff NaN."""
    v = np.zeros(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = np.ldexp(m / 8.0, -6) if e == 0 else np.ldexp(1 + m / 8.0, e - 7)
        v[c] = (-1.0 if c & 128 else 1.0) * (np.nan if e == 15 and m == 7 else x)
    return v


E4M3 = e4m3_values()


def quantise(x):
    """[..., D] float64 -> codes uint8 [..., D], biased exponents uint8 [...]."""
    x = np.asarray(x, dtype=np.float64)
    top = np.where(np.isfinite(x), np.abs(x), 0.0).max(axis=-1)
    e = np.full(top.shape, -126, dtype=np.int64)
    for k in range(-126, 129):  # the least e with top <= 448 * 2^e
        e = np.where(np.ldexp(448.0, e.astype(np.int32)) < top, k + 1, e)
    e = np.where(top > 0, e, 0)
    y = np.ldexp(x, -e[..., None].astype(np.int32))
    codes = np.zeros(x.shape, dtype=np.uint8)
    grid = E4M3[:127]
    mag = np.minimum(np.abs(np.nan_to_num(y, nan=0.0, posinf=448.0, neginf=-448.0)), 448.0)
    hi = np.clip(np.searchsorted(grid, mag, side="left"), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = mag - grid[lo], grid[hi] - mag
    pick = np.where(dl < dh, lo, np.where(dh < dl, hi, np.where(lo % 2 == 0, lo, hi)))  # ties to the even mantissa
    codes = pick.astype(np.uint8) | (np.signbit(y).astype(np.uint8) << 7)
    codes = np.where(np.isnan(y), codes & 0x80 | 0x7f, codes).astype(np.uint8)
    return codes, (e + 127).astype(np.uint8)


def dequantise(codes, exps):
    return np.ldexp(E4M3[codes], exps[..., None].astype(np.int32) - 127)


# ---- the cache ------------------------------------------------------------------------------------------------------
def page_at(block_table, n_pages, page_size, b, p):
    """Page of position p of sequence b, or -1."""
    i = p // page_size
    if p < 0 or i >= block_table.shape[1]:
        return -1
    page = int(block_table[b, i])
    return page if 0 <= page < n_pages else -1


def new_positions(cu_q, kv_lens):
    """(row, sequence, position) of every packed new row that has a place."""
    for b in range(len(kv_lens)):
        for t in range(int(cu_q[b]), int(cu_q[b + 1])):
            p = int(kv_lens[b]) - int(cu_q[b + 1]) + t
            if p >= 0:
                yield t, b, p


def dense(values, block_table, page_size, b, n):
    """values [pages, heads, page, D] -> ([n, heads, D], there [n])."""
    out = np.zeros((n, values.shape[1], values.shape[3]))
    there = np.zeros(n, dtype=bool)
    for p in range(n):
        page = page_at(block_table, values.shape[0], page_size, b, p)
        if page >= 0:
            out[p], there[p] = values[page, :, p % page_size], True
    return out, there


def visible(pos, n, window, sinks, causal):
    j = np.arange(n)
    see = j <= pos if causal else np.ones(n, dtype=bool)
    if window > 0:
        see = see & ((j > pos - window) | (j < sinks))
    return see if pos >= 0 else np.zeros(n, dtype=bool)


def attend(q, k, v, cu_q, kv_lens, block_table, page_size, window=0, sinks=0, causal=True, scale=None, max_kv=None):
    """q [n, Hq, D], k and v [pages, H, page, D] float64 -> (out [n, Hq, D], per element sum p |v|, per row and head the largest
    scale * sum |q_d k_d|, rows without a sequence marked False).  What is hidden from a row has no part in it."""
    n, hq, d = q.shape
    group = hq // k.shape[1]
    scale = 1.0 / np.sqrt(d) if scale is None else scale
    out, absv, reach = np.zeros(q.shape), np.zeros(q.shape), np.zeros((n, hq))
    owned = np.zeros(n, dtype=bool)
    for b in range(len(kv_lens)):
        t0, t1 = int(cu_q[b]), int(cu_q[b + 1])
        owned[t0:t1] = True
        m = int(kv_lens[b]) if max_kv is None else min(int(kv_lens[b]), max_kv)
        m = max(0, min(m, block_table.shape[1] * page_size))
        kb, there = dense(k, block_table, page_size, b, m)
        vb, _ = dense(v, block_table, page_size, b, m)
        for t in range(t0, t1):
            see = visible(int(kv_lens[b]) - t1 + t, m, window, sinks, causal) & there
            if not see.any():
                continue
            for h in range(hq):
                kh, vh = kb[see, h // group], vb[see, h // group]
                with np.errstate(all="ignore"):
                    s = scale * (kh @ q[t, h])
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    out[t, h] = p @ vh
                    absv[t, h] = p @ np.abs(vh)
                    reach[t, h] = abs(scale) * (np.abs(kh) @ np.abs(q[t, h])).max()
    return out, absv, reach, owned


# ---- choice of a token ---------------------------------------------------------------------------------------------------
def sample_row(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row -> (id, log-probability, distance of the decision from its nearest border relative to the kept weight)."""
    l = np.where(np.isnan(logits), -np.inf, np.asarray(logits, dtype=np.float64))
    if not (l > -np.inf).any():
        return 0, -np.inf, 1.0
    order = np.lexsort((np.arange(l.size), -l))
    top = l[order[0]]
    if not temperature > 0:
        return int(order[0]), 0.0, 1.0
    with np.errstate(invalid="ignore"):
        w = np.where(l == top, 1.0, np.exp((l - top) / temperature))
    n = int((l > -np.inf).sum())
    if 0 < top_k < n:
        n = int(top_k)
    if top_p < 1:
        mass = np.cumsum(w[order[:n]])
        before = np.concatenate([[0.0], mass[:-1]])
        n = max(1, int((before < top_p * mass[-1]).sum()))
    kept = order[:n][w[order[:n]] >= min_p]
    if not kept.size:
        kept = order[:1]
    kept = np.sort(kept)
    mass = np.cumsum(w[kept])
    at = min(max(u, 0.0), 1.0) * mass[-1]
    i = min(int(np.searchsorted(mass, at, side="right")), kept.size - 1)
    return int(kept[i]), float(np.log(w[kept[i]] / mass[-1])), float(np.abs(mass - at).min() / mass[-1])
