"""Norm and rotation of rows, their gradients and the paged cache's addressing in 64 bits (numpy), with bounds of the error of the
same sums in 32 bits, in units of 2^-24 (``u``)."""
import numpy as np
import torch

u = 2.0 ** -24
EPS_OF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}


def rounded(x, dtype):
    """An array in 64 bits whose values a tensor of ``dtype`` holds."""
    return torch.from_numpy(np.ascontiguousarray(x)).to(dtype).double().numpy()


def pairs(D, rot, interleaved):
    """(partner of every element, its pair, sign of the sine), for the elements that turn."""
    partner, pair, sign = np.arange(D), np.zeros(D, int), np.zeros(D)
    for i in range(rot // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        partner[a], partner[b] = b, a
        pair[a] = pair[b] = i
        sign[a], sign[b] = -1, 1
    return partner, pair, sign


def turn(x, pos, rot, interleaved, freqs, back=False):
    """Rows x (..., D) turned by positions pos (...), and the sum of the magnitudes of each result's terms."""
    D = x.shape[-1]
    partner, pair, sign = pairs(D, rot, interleaved)
    f = np.append(np.asarray(freqs, dtype=np.float64), 0.0)[pair] * (sign != 0)
    a = np.asarray(pos, dtype=np.float64)[..., None] * f
    s = np.sin(a) * sign * (-1 if back else 1)
    # (an element that does not turn has no partner's term, whatever the partner holds)
    other = np.where(sign != 0, x[..., partner], 0.0)
    return x * np.cos(a) + other * s, np.abs(x) + np.abs(other)


def default_freqs(rot, base=10000.0):
    return base ** (-np.arange(0, rot, 2) / max(rot, 1))


def forward(x, w, pos, rot, interleaved, freqs, eps):
    """(y, bound of the error before rounding)."""
    r, xw = 1.0, x
    if w is not None:
        r = 1 / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps)
        xw = x * w
    y, mag = turn(xw, pos, rot, interleaved, freqs)
    # cos and sin: the angle in 32 bits (2^-25 half turns, 1.6 u) and 2 ulp of the function, 4 u together; weight, product and
    # sum 3 u; r: a sum of D squares in chains of 8 and a butterfly 13 u / 2, rsqrt and the product 4 u
    return r * y, (7 + 11) * u * r * mag


def backward(x, w, dy, pos, rot, interleaved, freqs, eps, chain):
    """(dx, its bound, dw, its bound); chain: the most additions that a partial sum of dw went through."""
    g, mag = turn(dy, pos, rot, interleaved, freqs, back=True)
    g_err = 7 * u * mag
    if w is None:
        return g, g_err, None, None
    r = 1 / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps)
    axes = tuple(range(x.ndim - 1))
    dw = (g * x * r).sum(axes)
    dw_err = ((g_err + (13 + chain) * u * mag) * np.abs(x) * r).sum(axes)
    mean = (g * w * x).mean(-1, keepdims=True)
    mean_mag = (mag * np.abs(w * x)).mean(-1, keepdims=True)
    dx = r * (g * w - x * r ** 2 * mean)
    dx_err = r * np.abs(w) * (7 + 16) * u * mag + np.abs(x) * r ** 3 * mean_mag * (7 + 13 + 2 + 3 * 11) * u
    return dx, dx_err, dw, dw_err


def check(got, want, err, dtype, what=""):
    """A result in ``dtype`` against its value and the bound of its error before rounding."""
    got = got.detach().double().cpu().numpy()
    tol = err * (1 + EPS_OF[dtype]) + np.abs(want) * EPS_OF[dtype] + TINY[dtype]
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (what, int(bad.sum()), bad.size, np.abs(got - want)[bad].max(), tol[bad].min())
