"""Plain 64-bit forms of the 8-bit KV cache's operators (numpy, from their
definitions) and makers of ragged calls, shared by the kv8 tests."""
from __future__ import annotations

import numpy as np

PAGE = 16


def pages_for(rows, past):
    return [(p + t + PAGE - 1) // PAGE for t, p in zip(rows, past)]


def make_table(rng, rows, past, n_pages, ld=None):
    """Block table of shuffled pages, unused entries a page number out of range."""
    need = pages_for(rows, past)
    ld = max(max(need), 1) if ld is None else ld
    order = rng.permutation(n_pages)
    table, at = np.full((len(rows), ld), 1 << 30, np.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table


def append(kq, ks, layer, x, row_start, past, table, transposed):
    """Stores rows x [rows][heads][dim] into int8 pages kq / scales ks (in place)."""
    for b in range(len(past)):
        n, p0 = row_start[b + 1] - row_start[b], past[b]
        for pg in range(p0 // PAGE, (p0 + n + PAGE - 1) // PAGE if n else 0):
            page = table[b, pg]
            lo, hi = max(p0 - pg * PAGE, 0), min(p0 + n - pg * PAGE, PAGE)
            first = row_start[b] + pg * PAGE - p0
            for h in range(x.shape[1]):
                blk = kq[page, layer, h].T if transposed else kq[page, layer, h]  # view [16][dim]
                new = x[first + lo:first + hi, h].astype(np.float64)
                was = np.float32(ks[page, layer, h]) if lo else np.float32(0)
                top = np.abs(new).max()
                if not np.isfinite(top) or np.isnan(was):
                    ks[page, layer, h] = np.nan
                    blk[lo:hi] = 0
                    continue
                s = max(np.float32(top / 127.0), was)
                ks[page, layer, h] = s
                if s == 0:
                    blk[lo:hi] = 0
                    continue
                if lo and s != was:
                    blk[:lo] = np.clip(np.rint(blk[:lo].astype(np.float64) * np.float64(was) / np.float64(s)), -127, 127)
                blk[lo:hi] = np.clip(np.rint(new / np.float64(s)), -127, 127)


def values(kq, ks, layer, table_row, n, transposed):
    """Positions 0..n-1 of a sequence: [n][heads][dim] in 64 bits."""
    pg = table_row[: (n + PAGE - 1) // PAGE]
    q = kq[pg, layer].astype(np.float64)
    if transposed:
        q = q.swapaxes(2, 3)
    v = q * ks[pg, layer].astype(np.float64)[:, :, None, None]
    return v.transpose(0, 2, 1, 3).reshape(-1, q.shape[1], q.shape[3])[:n]


def seen(pos, n, window, sinks):
    j = np.arange(n)
    return (j <= pos) & ((window == 0) | (j > pos - window) | (j < sinks))


def attend(k, v, q, past, scale, window=0, sinks=0, vtop=None):
    """One sequence: k, v [n][Hkv][dim], q [T][H][dim] at positions past...  Returns out [T][H][dim]; the summed
    |weight * value| [T][H][dim]; each row's largest scale * sum |q k| (the scores' size); its largest scale * max|q| *
    sum |k|; the sum over pages of 2 * 32 * (the page's largest weight * vtop), vtop [n][Hkv] what a position's block
    can hold at most (a pair's largest is at most the sum of its two pages', twice for either pairing); and the
    number of keys * the largest weight * the largest vtop."""
    T, H, D = q.shape
    G = H // k.shape[1]
    out, mag = np.zeros((T, H, D)), np.zeros((T, H, D))
    size, reach, grain, coarse = np.zeros((4, T, H))
    for i in range(T):
        m = seen(past + i, k.shape[0], window, sinks)
        if not m.any():
            continue
        for h in range(H):
            kk, vv = k[m, h // G], v[m, h // G]
            s = kk @ q[i, h] * scale
            size[i, h] = (np.abs(kk) @ np.abs(q[i, h])).max() * abs(scale)
            reach[i, h] = np.abs(kk).sum(1).max() * np.abs(q[i, h]).max() * abs(scale)
            w = np.exp(s - s.max())
            w /= w.sum()
            out[i, h] = w @ vv
            mag[i, h] = w @ np.abs(vv)
            if vtop is not None:
                x = np.zeros((k.shape[0] + PAGE - 1) // PAGE * PAGE)
                x[: k.shape[0]][m] = w * vtop[m, h // G]
                grain[i, h] = 64 * x.reshape(-1, PAGE).max(1).sum()
                coarse[i, h] = len(w) * w.max() * vtop[m, h // G].max()
    return out, mag, size, reach, grain, coarse
