"""Rows in 4 bits (numpy): what rows become, in 64 bits, and the bytes of pages that hold them."""
import numpy as np

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
E4M3 = np.array([m / 8 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)][:119])
assert E4M3[-1] == 448 and len(E4M3) == 127


def nearest(x, grid):
    """Index of the number of an ascending grid that is nearest to x, the even one of two equally near."""
    hi = np.clip(np.searchsorted(grid, x), 0, len(grid) - 1)
    lo = np.maximum(hi - 1, 0)
    up, down = grid[hi] - x, x - grid[lo]
    return np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)


def encode(x, factor):
    """(codes, scale bytes) of rows x (..., D)."""
    x = np.asarray(x, dtype=np.float64)
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 16, 16)
    nan = np.isnan(b).any(-1)
    most = np.abs(np.where(nan[..., None], 0, b)).max(-1)
    scales = nearest(np.minimum(most / 6 / factor, 448.0), E4M3)
    step = E4M3[scales] * factor
    with np.errstate(invalid="ignore"):
        r = np.where(step[..., None] > 0, np.abs(b) / np.where(step > 0, step, 1)[..., None], 0)
        codes = nearest(np.minimum(np.nan_to_num(r, nan=0.0), 6.0), E2M1) + 8 * (b < 0)
    codes = np.where(nan[..., None] | (step[..., None] == 0), 0, codes)
    return codes.reshape(x.shape).astype(np.uint8), np.where(nan, 127, scales).astype(np.uint8)


def decode(codes, scales, factor):
    v = E2M1[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    s = np.append(E4M3, np.nan)[scales & 127] * factor
    return (v.reshape(*v.shape[:-1], v.shape[-1] // 16, 16) * s[..., None]).reshape(v.shape)


def turn(row, D):
    return (4 * (row & 1) | (row & 2)) & (D // 32 - 1)


def split_pages(pages, page, D):
    """(codes, scale bytes) of every row of byte pages (n, heads, page * 9 D / 16): (n, heads, page, D) and (..., D / 16)."""
    n, h, _ = pages.shape
    raw = pages[..., :page * D // 2].reshape(n, h, page, D // 32, 16)
    codes = np.empty((n, h, page, D), np.uint8)
    for j in range(page):
        row = raw[:, :, j, [c ^ turn(j, D) for c in range(D // 32)]].reshape(n, h, D // 2)
        codes[:, :, j, 0::2], codes[:, :, j, 1::2] = row & 15, row >> 4
    return codes, pages[..., page * D // 2:].reshape(n, h, page, D // 16)


def join_pages(codes, scales):
    """The bytes of pages of such codes and scales."""
    n, h, page, D = codes.shape
    raw = np.empty((n, h, page, D // 32, 16), np.uint8)
    both = (codes[..., 0::2] | codes[..., 1::2] << 4).reshape(n, h, page, D // 32, 16)
    for j in range(page):
        raw[:, :, j, [c ^ turn(j, D) for c in range(D // 32)]] = both[:, :, j]
    return np.concatenate([raw.reshape(n, h, -1), scales.reshape(n, h, -1)], -1)


def values(pages, page, D, factor):
    return decode(*split_pages(pages, page, D), factor)
