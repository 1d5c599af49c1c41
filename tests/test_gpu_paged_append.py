"""Appending to a paged KV cache, K normed and rotated on the way, against the formulas in 64 bits: every row where the table
says and no other row changed."""
import numpy as np
import pytest
import torch

from norm_rope_ref import check, default_freqs, forward, rounded
from ring_attention_b200 import api

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def gpu(x, dtype):
    return torch.from_numpy(np.ascontiguousarray(x)).to(dtype).cuda()


def table_of(rng, lens, page, num_pages, width):
    """Distinct pages in random order; -1 and numbers out of range behind a sequence's last page."""
    free = rng.permutation(num_pages)
    t = rng.choice([-1, num_pages, 2 ** 31 - 1, -(2 ** 31)], (len(lens), width))
    at = 0
    for b, n in enumerate(lens):
        m = -(-n // page)
        t[b, :m] = free[at:at + m]
        at += m
    return t.astype(np.int64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,rot,interleaved,norm", [(32, 32, True, False), (64, 32, False, True), (128, 128, False, True),
                                                    (128, 0, False, False), (256, 256, False, True), (256, 128, True, False)])
@pytest.mark.parametrize("B,H,kvH,T,page", [(1, 1, 1, 1, 16), (5, 12, 4, 1, 32), (3, 6, 2, 37, 16), (2, 8, 8, 300, 128),
                                            (4, 3, 1, 70, 64), (33, 4, 2, 3, 256)])
def test_rows_go_where_the_table_says(dtype, D, rot, interleaved, norm, B, H, kvH, T, page):
    rng = np.random.default_rng(B * T + D)
    before = rng.integers(0, 3 * page, B)
    counts = rng.integers(0, T + 1, B)
    counts[0] = T
    need = [-(-int(n + t) // page) for n, t in zip(before, counts)]
    num_pages = sum(need) + 2
    table = table_of(rng, before + counts, page, num_pages, max(need) + 1)
    k, v, q = (rounded(rng.standard_normal((B, h, T, D)), dtype) for h in (kvH, kvH, H))
    wk, wq = (rounded(1 + 0.3 * rng.standard_normal(D), dtype) if norm else None for _ in range(2))
    old = [rounded(rng.standard_normal((num_pages, kvH, page, D)), dtype) for _ in range(2)]
    pages = [gpu(x, dtype) for x in old]
    q_out = torch.full((B, H, T, D), 5.0, dtype=dtype, device="cuda")
    lens = torch.from_numpy(before.astype(np.int32)).cuda()
    # K token by token in memory, V and Q head by head
    dk = gpu(k.transpose(0, 2, 1, 3), dtype).transpose(1, 2)
    api.paged_append(dk, gpu(v, dtype), *pages, torch.from_numpy(table.astype(np.int32)).cuda(), lens,
                     counts=torch.from_numpy(counts.astype(np.int32)).cuda(),
                     rope=api.Rope.make(rot, interleaved=interleaved) if rot else None,
                     k_weight=gpu(wk, dtype) if norm else None, q_weight=gpu(wq, dtype) if norm else None, q=gpu(q, dtype),
                     q_out=q_out)
    want, err, v_want = old[0].copy(), np.zeros_like(old[0]), old[1].copy()
    fixed = np.ones((num_pages, page), bool)  # rows that must keep their bits
    q_got = q_out.double().cpu().numpy()
    for b in range(B):
        at = before[b] + np.arange(counts[b])
        pg, row = table[b, at // page], at % page
        y, e = forward(k[b, :, :counts[b]], wk, at[None], rot, interleaved, default_freqs(rot), np.float32(1e-6))
        want[pg, :, row], err[pg, :, row] = y.swapaxes(0, 1), np.broadcast_to(e, y.shape).swapaxes(0, 1)
        v_want[pg, :, row] = v[b, :, :counts[b]].swapaxes(0, 1)
        fixed[pg, row] = False
        y, e = forward(q[b, :, :counts[b]], wq, at[None], rot, interleaved, default_freqs(rot), np.float32(1e-6))
        check(q_out[b, :, :counts[b]], y, e, dtype, "q")
        assert (q_got[b, :, counts[b]:] == 5).all()
    check(pages[0], want, err, dtype, "k")
    assert np.array_equal(pages[1].double().cpu().numpy(), v_want)
    kept = pages[0].double().cpu().numpy().swapaxes(1, 2)[fixed]
    assert np.array_equal(kept, old[0].swapaxes(1, 2)[fixed])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_bad_pages_and_lengths_write_nothing(dtype):
    """Numbers out of range, a table that ends, negative lengths and counts: the rows are dropped, the others written."""
    B, kvH, T, D, page, n = 6, 2, 20, 64, 16, 5
    table = torch.tensor([[0, -1], [1, 5], [-(2 ** 31), 2], [3, 2 ** 31 - 1], [4, 4], [4, 4]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([0, 10, 8, 30, -25, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    counts = torch.tensor([20, 20, 20, 20, 20, -3], dtype=torch.int32, device="cuda")
    k = torch.randn(B, kvH, T, D, device="cuda").to(dtype)
    pages = [torch.full((n, kvH, page, D), 9.0, dtype=dtype, device="cuda") for _ in range(2)]
    want = [p.clone() for p in pages]
    for b, rows in ((0, range(16)), (1, range(6)), (2, range(8, 20))):
        for t in rows:
            slot = lens[b].item() + t
            for w in want:
                w[table[b, slot // page], :, slot % page] = k[b, :, t]
    # (sequence 3: its second page is out of range and then the table ends; 4: rows before the first one; 5: no rows)
    api.paged_append(k, k, *pages, table, lens, counts=counts)
    assert torch.equal(pages[0], want[0]) and torch.equal(pages[1], want[1])
    # no pages at all
    none = torch.empty(0, kvH, page, D, dtype=dtype, device="cuda")
    api.paged_append(k, k, none, none, table, lens, counts=counts)
    api.paged_append(k, k, *pages, table[:, :0], lens)
    assert torch.equal(pages[0], want[0]) and torch.equal(pages[1], want[1])


def test_given_positions_and_wide_tables():
    """Positions that are not the rows' places (a context-parallel rank's cache), a table that is a view of a wider one, K in the
    cache's own type with fp32 weights."""
    B, kvH, T, D, page = 2, 2, 9, 64, 16
    rng = np.random.default_rng(3)
    k = rounded(rng.standard_normal((B, kvH, T, D)), torch.bfloat16)
    w = rounded(1 + rng.random(D), torch.float32)
    pos = rng.integers(0, 10 ** 6, (B, T))
    wide = torch.full((B, 7), -1, dtype=torch.int32, device="cuda")
    wide[:, 2] = torch.tensor([1, 0])
    pages = [torch.zeros(2, kvH, page, D, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    lens = torch.tensor([3, 0], dtype=torch.int32, device="cuda")
    api.paged_append(gpu(k, torch.bfloat16), gpu(k, torch.bfloat16), *pages, wide[:, 2:3], lens, rope=api.Rope.make(D),
                     k_weight=gpu(w, torch.float32), positions=torch.from_numpy(pos.astype(np.int32)).cuda())
    y, e = forward(k, w, pos[:, None], D, False, default_freqs(D), np.float32(1e-6))
    check(pages[0][1, :, 3:3 + T], y[0], e[0], torch.bfloat16)
    check(pages[0][0, :, :T], y[1], e[1], torch.bfloat16)
    assert (pages[0][1, :, :3] == 0).all() and (pages[0][:, :, 3 + T:] == 0).all()


def test_offsets_that_pass_32_bits():
    """A cache of more than 2^31 elements: the last page's rows."""
    kvH, page, D = 8, 256, 256
    n = 2 ** 31 // (kvH * page * D) + 3
    pages = [torch.zeros(n, kvH, page, D, device="cuda", dtype=torch.float16) for _ in range(2)]
    assert pages[0].numel() > 2 ** 31
    table = torch.tensor([[n - 1], [0]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([page - 2, 0], dtype=torch.int32, device="cuda")
    k = torch.randn(2, kvH, 2, D, device="cuda").half()
    api.paged_append(k, k, *pages, table, lens)
    for p in pages:
        assert torch.equal(p[n - 1, :, page - 2:], k[0]) and torch.equal(p[0, :, :2], k[1])
        assert p.count_nonzero() == k.count_nonzero()


def test_append_captured_and_replayed():
    B, kvH, D, page = 4, 2, 128, 16
    pages = [torch.zeros(3 * B, kvH, page, D, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    twin = [p.clone() for p in pages]
    table = torch.arange(3 * B, dtype=torch.int32, device="cuda").view(B, 3)
    lens = torch.tensor([0, 15, 16, 40], dtype=torch.int32, device="cuda")
    k, rope = torch.empty(B, kvH, 1, D, device="cuda", dtype=torch.bfloat16), api.Rope.make(D)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        api.paged_append(k, k, *pages, table, lens, rope=rope)
        lens += 1
    lens2 = torch.tensor([0, 15, 16, 40], dtype=torch.int32, device="cuda")
    lens.copy_(lens2)
    for step in range(5):
        k.normal_()
        g.replay()
        api.paged_append(k, k, *twin, table, lens2, rope=rope)
        lens2 += 1
    assert torch.equal(lens, lens2) and all(torch.equal(a, b) for a, b in zip(pages, twin))


def test_append_wrapper_refusals():
    k = torch.zeros(2, 2, 1, 64, device="cuda")
    p = torch.zeros(4, 2, 16, 64, device="cuda")
    t, n = torch.zeros(2, 1, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    for a in ((k, k, p, p[:3], t, n), (k, k, p.transpose(2, 3), p.transpose(2, 3), t, n), (k, k, p, p, t.long(), n),
              (k, k, p, p, t, n[:1]), (k, k, p, p, t[0], n), (k[:1], k[:1], p, p, t, n), (k, k.half(), p, p, t, n),
              (k[..., :32], k[..., :32], p, p, t, n), (k.cpu(), k, p, p, t, n), (k, k, p, p, t.cpu(), n)):
        with pytest.raises(ValueError):
            api.paged_append(*a)
    with pytest.raises(ValueError):
        api.paged_append(k, k, p, p, t, n, q=k)
    with pytest.raises(ValueError):
        api.paged_append(k, k, p, p, t, n, counts=n.float())
    with pytest.raises(api._lib.RingAttentionError):
        api.paged_append(k, k, *[torch.zeros(4, 2, 8, 64, device="cuda")] * 2, t, n)
