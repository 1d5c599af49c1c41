"""Attention over packed sequences in 64 bits, with a bound of the error of the kernel's sums."""
import numpy as np
import torch

from norm_rope_ref import EPS_OF, TINY, check, u


def want(q, k, v, ends, k_ends, causal, dtype):
    """(out, its bound, lse, its bound, rows that are some sequence's) of tensors in 64 bits, (rows, heads, head_dim) each."""
    rows, H, D = q.shape
    kvH = k.shape[1]
    out, err = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full((H, rows), -np.inf, dtype=torch.float64, device=q.device)
    lse_err, mine = torch.zeros_like(lse), torch.zeros(rows, dtype=torch.bool, device=q.device)
    for b in range(len(ends) - 1):
        r, t = slice(int(ends[b]), int(ends[b + 1])), slice(int(k_ends[b]), int(k_ends[b + 1]))
        n, m = r.stop - r.start, t.stop - t.start
        mine[r] = True
        if n == 0 or m == 0:
            continue
        for h in range(H):
            x, y, z = q[r, h], k[t, h % kvH], v[t, h % kvH]
            s = x @ y.T / D ** 0.5
            seen = torch.ones(n, m, dtype=torch.bool, device=q.device)
            if causal:
                seen = torch.arange(m, device=q.device)[None] <= torch.arange(n, device=q.device)[:, None] + (m - n)
            has = seen.any(1)
            s = torch.where(seen, s, -np.inf)
            top = s.amax(1, keepdim=True)
            p = torch.where(seen, torch.exp(s - top), 0.0)
            l = p.sum(1, keepdim=True)
            o = p @ z / l
            # a score: D products and sums, the scale and the difference to the reference in 32 bits (the reference is up to 2^15 off the
            # largest score, in a sum of weights of as much; ln 2^15 = 10.4); the exponential 2 ulp
            size = torch.where(seen, x.abs() @ y.abs().T / D ** 0.5, 0.0).amax(1, keepdim=True)
            far = torch.where(seen, (s - top).abs(), 0.0).amax(1, keepdim=True) + 10.4
            score = (D + 4) * u * size + u * (far + top.abs())
            weight = score + 2.0 ** -22
            chain = (m + 700) * u
            mag = p @ z.abs() / l
            e = (2 * weight + 2 * chain + EPS_OF[dtype]) * mag + TINY[dtype] * seen.double() @ z.abs()
            out[r, h], err[r, h] = torch.where(has[:, None], o, 0.0), torch.where(has[:, None], e, 0.0)
            lse[h, r] = torch.where(has, (top + torch.log(l))[:, 0], -np.inf)
            lse_err[h, r] = torch.where(has, (score + 2.0 ** -22 + chain + 4 * u * (top.abs() + lse[h, r, None].abs() + 11))[:, 0], 0.0)
    return out, err, lse, lse_err, mine


def compare(dtype, q, k, v, ends, k_ends, causal, out, lse, left=7.0):
    """Results against ``want``; rows of no sequence have to be ``left``."""
    o, err, l, l_err, mine = want(*(x.double() for x in (q, k, v)), ends, k_ends, causal, dtype)
    assert (out[~mine] == left).all() and (lse[:, ~mine] == left).all()
    check(out[mine], o[mine].cpu().numpy(), err[mine].cpu().numpy(), dtype, "out")
    l, l_err, got = l[:, mine], l_err[:, mine], lse[:, mine].double()
    there = torch.isfinite(l)
    assert torch.equal(there, torch.isfinite(got)) and (got[~there] == -np.inf).all()
    off = (got - l)[there].abs()
    assert (off <= l_err[there]).all(), off.max()
