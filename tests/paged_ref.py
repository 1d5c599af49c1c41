"""Decode attention over a paged cache in 64 bits, with a bound of the error of the kernels' sums."""
import numpy as np
import torch

from norm_rope_ref import EPS_OF, TINY, u


def table_of(rng, lens, page, num_pages, width, shared=()):
    """Distinct pages in random order behind the shared ones; numbers out of range behind a sequence's last page."""
    free = [p for p in rng.permutation(num_pages) if p not in set(shared)]
    t = rng.choice([-1, num_pages, 2 ** 31 - 1, -(2 ** 31)], (len(lens), width))
    at = 0
    for b, n in enumerate(lens):
        m = -(-int(n) // page)
        head = min(m, len(shared))
        t[b, :head] = shared[:head]
        t[b, head:m] = free[at:at + m - head]
        at += m - head
    return t.astype(np.int64)


def want(q, k_pages, v_pages, table, lens, dtype, shared=()):
    """(out, its bound, lse, its bound) of arrays in 64 bits; keys of pages out of range are not there."""
    B, H, D = q.shape
    n_pages, kvH, page, _ = k_pages.shape
    out, err = np.zeros((B, H, D)), np.zeros((B, H, D))
    lse, lse_err = np.full((B, H), -np.inf), np.zeros((B, H))
    for b in range(B):
        n = max(0, min(int(lens[b]), table.shape[1] * page))
        pages = table[b].copy()
        if len(shared) and n >= len(shared) * page:
            pages[:len(shared)] = shared
        j = np.arange(n)
        at = pages[j // page] if n else j
        j, at = j[(at >= 0) & (at < n_pages)], at[(at >= 0) & (at < n_pages)]
        if len(j) == 0:
            continue
        for h in range(H):
            kv = h % kvH
            k, v = k_pages[at, kv, j % page], v_pages[at, kv, j % page]
            s = k @ q[b, h] / D ** 0.5
            size = (np.abs(k) @ np.abs(q[b, h]) / D ** 0.5).max()
            m = s.max()
            p = np.exp(s - m)
            l = p.sum()
            out[b, h] = p @ v / l
            lse[b, h] = m + np.log(l)
            # a score: D products and sums, the scale and the difference to the maximum in 32 bits; the exponential 2 ulp
            score = (D + 4) * u * size + u * np.abs(s - m).max()
            weight = score + 2.0 ** -22
            # sums over keys: an accumulator adds up to half of them, then slices, warps and parts
            chain = (len(j) / 2 + 700) * u
            mag = p @ np.abs(v) / l
            e = (2 * weight + 2 * chain) * mag
            if dtype != torch.float32:  # weights in the cache's type, with a floor of half its smallest step
                e = e + EPS_OF[dtype] * mag + TINY[dtype] * np.abs(v).sum(0) / l
            err[b, h] = e
            lse_err[b, h] = score + 2.0 ** -22 + chain + 4 * u * (abs(m) + abs(lse[b, h]))
    return out, err, lse, lse_err
