"""The paged cache in 4 bits: rows appended are the nearest that the format has, in the bytes that it says; rows read back are
what the bytes stand for; decoding against 64 bits."""
import numpy as np
import pytest
import torch

import four_bit_ref as ref
from norm_rope_ref import check, rounded
from paged_ref import table_of, want
from ring_attention_b200 import api
from ring_attention_b200._lib import RingAttentionError

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]


def gpu(x, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(x))
    return (t.to(dtype) if dtype else t).cuda()


def i32(x):
    return gpu(np.asarray(x).astype(np.int64)).to(torch.int32)


def some_rows(rng, shape, dtype):
    """Rows with what rounding meets: blocks of zeros, blocks large and small beyond the scales' range, elements in the middle between
    two codes, negative zeros."""
    x = rng.standard_normal(shape)
    b = x.reshape(-1, 16)
    kind = rng.integers(0, 8, len(b))
    b[kind == 0] = rng.choice([0.0, -0.0], (int((kind == 0).sum()), 16))
    b[kind == 1] *= 3000.0
    b[kind == 2] *= 2.0 ** -11
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 0.0])
    n = int((kind == 3).sum())
    b[kind == 3] = rng.choice(ties, (n, 16)) * rng.choice([-1, 1], (n, 16)) * ref.E4M3[rng.integers(60, 90, (n, 1))]
    b[kind == 3, 0] = 6 * ref.E4M3[rng.integers(60, 90, n)]
    return rounded(x, dtype)


def same_bytes(got, codes, scales, touched, old, page, D):
    """Pages against the codes and scales that they should hold, rows that no call touched bit for bit as they were."""
    g = ref.split_pages(got, page, D)
    o = ref.split_pages(old, page, D)
    at = np.broadcast_to(touched[:, None, :, None], g[0].shape)
    zero = lambda c: np.where(c == 8, 0, c)  # (the sign of a zero)
    assert np.array_equal(zero(g[0])[at], zero(codes)[at])
    assert np.array_equal(g[0][~at], o[0][~at])
    at = np.broadcast_to(touched[:, None, :, None], g[1].shape)
    assert np.array_equal(g[1][at], scales[at])
    assert np.array_equal(g[1][~at], o[1][~at])


def append_problem(seed, dtype, D, B, kvH, T, page):
    rng = np.random.default_rng(seed)
    before = rng.integers(0, 3 * page, B)
    counts = rng.integers(0, T + 1, B)
    counts[0] = T
    need = [-(-int(n + t) // page) for n, t in zip(before, counts)]
    n = sum(need) + 2
    table = table_of(rng, before + counts, page, n, max(need) + 1)
    old = [rng.integers(0, 256, (n, kvH, page * 9 * D // 16), dtype=np.uint8) for _ in range(2)]
    return rng, before, counts, table, old


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("B,kvH,T,page,scales", [(1, 1, 1, 16, (1.0, 1.0)), (5, 4, 1, 32, (0.25, 8.0)), (3, 2, 37, 16, (1.0, 2.0 ** -20)),
                                                 (2, 8, 300, 128, (4.0, 1.0)), (33, 2, 3, 256, (2.0 ** 10, 0.5)), (4, 1, 70, 64, (1.0, 1.0))])
def test_rows_are_the_nearest_that_the_format_has(dtype, D, B, kvH, T, page, scales):
    rng, before, counts, table, old = append_problem(B * T + D, dtype, D, B, kvH, T, page)
    x = [some_rows(rng, (B, kvH, T, D), dtype) for _ in range(2)]
    pages = [gpu(p) for p in old]
    # K token by token in memory, V head by head and from an address that is no multiple of 16 bytes
    dk = gpu(x[0].transpose(0, 2, 1, 3), dtype).transpose(1, 2)
    dv = torch.empty(x[1].size + 1, dtype=dtype, device="cuda")[1:].view(x[1].shape).copy_(gpu(x[1], dtype))
    api.paged_append_4bit(dk, dv, *pages, i32(table), i32(before), counts=i32(counts), k_scale=scales[0], v_scale=scales[1])
    touched = np.zeros((len(old[0]), page), bool)
    for side in range(2):
        codes, bytes_ = (np.zeros(s, np.uint8) for s in ((len(old[0]), kvH, page, D), (len(old[0]), kvH, page, D // 16)))
        for b in range(B):
            at = before[b] + np.arange(counts[b])
            c, s = ref.encode(x[side][b, :, :counts[b]], scales[side])
            codes[table[b, at // page], :, at % page], bytes_[table[b, at // page], :, at % page] = c.swapaxes(0, 1), s.swapaxes(0, 1)
            touched[table[b, at // page], at % page] = True
        same_bytes(pages[side].cpu().numpy(), codes, bytes_, touched, old[side], page, D)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,rot,interleaved,norm", [(32, 32, False, True), (64, 16, False, False), (64, 64, True, True), (128, 48, False, True),
                                                    (128, 128, False, True), (256, 256, False, False), (256, 240, False, True),
                                                    (128, 0, False, True), (256, 128, True, True)])
@pytest.mark.parametrize("B,H,kvH,T,page", [(3, 6, 2, 37, 16), (17, 4, 4, 1, 32)])
def test_norm_and_rotation_on_the_way(dtype, D, rot, interleaved, norm, B, H, kvH, T, page):
    """As paged_append leaves rows in a cache of 16 bits, rounded from there; the queries bit for bit."""
    rng, before, counts, table, old = append_problem(B + D + rot, dtype, D, B, kvH, T, page)
    k, v, q = (gpu(rng.standard_normal((B, h, T, D)), dtype) for h in (kvH, kvH, H))
    wk, wq = (gpu(1 + 0.3 * rng.standard_normal(D), dtype) if norm else None for _ in range(2))
    rope = api.Rope.make(rot, interleaved=interleaved) if rot else None
    n = len(old[0])
    wide = [torch.zeros(n, kvH, page, D, dtype=dtype, device="cuda") for _ in range(2)]
    q_out = [torch.full((B, H, T, D), 5.0, dtype=dtype, device="cuda") for _ in range(2)]
    args = dict(counts=i32(counts), rope=rope, k_weight=wk, q_weight=wq, q=q)
    api.paged_append(k, v, *wide, i32(table), i32(before), q_out=q_out[0], **args)
    pages = [gpu(p) for p in old]
    api.paged_append_4bit(k, v, *pages, i32(table), i32(before), q_out=q_out[1], v_scale=0.5, **args)
    assert torch.equal(*q_out)
    touched = np.zeros((n, page), bool)
    for b in range(B):
        at = before[b] + np.arange(counts[b])
        touched[table[b, at // page], at % page] = True
    for side, f in ((0, 1.0), (1, 0.5)):
        codes, scales = ref.encode(wide[side].double().cpu().numpy(), f)
        same_bytes(pages[side].cpu().numpy(), codes, scales, touched, old[side], page, D)


@pytest.mark.parametrize("dtype", DTYPES)
def test_what_is_not_finite_stays_in_its_block(dtype):
    D, page = 64, 16
    x = np.random.default_rng(2).standard_normal((1, 1, 5, D))
    x[0, 0, 0, 3] = np.nan
    x[0, 0, 1, 20], x[0, 0, 1, 21] = np.inf, -np.inf
    x[0, 0, 2, 63] = -np.nan
    x[0, 0, 3, :16] = 6e4 if dtype == torch.float16 else 3e38
    pages = [api.pages_4bit(1, 1, page, D) for _ in range(2)]
    k = gpu(x, dtype)
    api.paged_append_4bit(k, k, *pages, i32([[0]]), i32([0]))
    got = ref.values(pages[0].cpu().numpy(), page, D, 1.0)[0, 0]
    assert np.isnan(got[0, :16]).all() and np.isfinite(got[0, 16:]).all() and np.isnan(got[2, 48:]).all() and np.isfinite(got[2, :48]).all()
    assert got[1, 20] == 2688 and got[1, 21] == -2688 and np.isfinite(got[1]).all() and (got[3, :16] == 2688).all()
    out = [torch.zeros(5, 1, D, dtype=dtype, device="cuda") for _ in range(2)]
    api.paged_read_4bit(*pages, i32([[0]]), i32([0, 5]), *out)
    assert np.array_equal(out[0][:, 0].double().cpu().numpy(), got[:5], equal_nan=True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_bad_pages_and_lengths_write_nothing(dtype):
    """Numbers out of range, a table that ends, negative lengths and counts: the rows are dropped, the others written."""
    B, kvH, T, D, page, n = 6, 2, 20, 64, 16, 5
    table = np.array([[0, -1], [1, 5], [-(2 ** 31), 2], [3, 2 ** 31 - 1], [4, 4], [4, 4]])
    lens, counts = np.array([0, 5, 3, 14, -3, 25]), np.array([20, 20, 20, 30, 20, -1])
    lens[4] = -40
    old = np.random.default_rng(3).integers(0, 256, (n, kvH, page * 9 * D // 16), dtype=np.uint8)
    x = rounded(np.random.default_rng(4).standard_normal((B, kvH, T, D)), dtype)
    pages = [gpu(old) for _ in range(2)]
    api.paged_append_4bit(gpu(x, dtype), gpu(x, dtype), *pages, i32(table), i32(lens), counts=i32(counts))
    touched, codes, scales = np.zeros((n, page), bool), np.zeros((n, kvH, page, D), np.uint8), np.zeros((n, kvH, page, D // 16), np.uint8)
    for b in range(B):
        for t in range(min(T, counts[b])):
            j = lens[b] + t
            if 0 <= j < 2 * page and 0 <= table[b, j // page] < n:
                touched[table[b, j // page], j % page] = True
                codes[table[b, j // page], :, j % page], scales[table[b, j // page], :, j % page] = ref.encode(x[b, :, t], 1.0)
    assert touched.any() and not touched[4].any()
    for p in pages:
        same_bytes(p.cpu().numpy(), codes, scales, touched, old, page, D)


# ---- reading back --------------------------------------------------------------------------------


@pytest.mark.parametrize("kind", [torch.float32, torch.float16, torch.bfloat16, (torch.float16, 1.0, 0.125), (torch.bfloat16, 2.0 ** 12, 1.0),
                                  (torch.float16, 2.0 ** -20, 2.0 ** 10)])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("B,kvH,page,lens", [(1, 1, 16, [1]), (5, 3, 16, [0, 33, 1, 0, 64]), (3, 8, 64, [300, 65, 129]),
                                             (40, 2, 128, list(range(0, 200, 5)))])
@pytest.mark.parametrize("strided", [False, True])
def test_rows_read_back(kind, D, B, kvH, page, lens, strided):
    four = isinstance(kind, tuple)
    dtype = kind[0] if four else kind
    rng = np.random.default_rng(B + D)
    lens = np.array(lens)
    start = rng.integers(0, 2 * page, B)
    total = [-(-int(n) // page) for n in lens + start]
    n = sum(total) + 2
    table = table_of(rng, lens + start, page, n, max(total) + 1)
    table[0, 0] = -1  # the first rows of the first sequence are not there
    if four:
        raw = [ref.join_pages(rng.integers(0, 16, (n, kvH, page, D), dtype=np.uint8), rng.integers(0, 127, (n, kvH, page, D // 16), dtype=np.uint8))
               for _ in range(2)]
        rows = [ref.values(p, page, D, f) for p, f in zip(raw, kind[1:])]
        pages = [gpu(p) for p in raw]
    else:
        rows = [rounded(rng.standard_normal((n, kvH, page, D)), dtype) for _ in range(2)]
        pages = [gpu(p, dtype) for p in rows]
    for at in (np.zeros(B, np.int64), start):
        first, behind = 2, 3  # rows of the results that are no sequence's
        ends = first + np.concatenate([[0], np.cumsum(lens)])
        m = int(ends[-1]) + behind
        # strided: K inside wider rows, V from an address that is no multiple of 16 bytes
        outs = [torch.full((m, kvH, D), 7.0, dtype=dtype, device="cuda") for _ in range(2)]
        if strided:
            outs = [torch.full((m, kvH + 2, D), 7.0, dtype=dtype, device="cuda")[:, 1:1 + kvH],
                    torch.full((m * kvH * D + 1,), 7.0, dtype=dtype, device="cuda")[1:].view(m, kvH, D)]
        extra = {} if at is not start else {"start": i32(at)}
        if four:
            api.paged_read_4bit(*pages, i32(table), i32(ends), *outs, k_scale=kind[1], v_scale=kind[2], **extra)
        else:
            api.paged_read(*pages, i32(table), i32(ends), *outs, **extra)
        for got, held in zip(outs, rows):
            expect = np.full((m, kvH, D), 7.0)
            for b in range(B):
                for t in range(lens[b]):
                    j = at[b] + t
                    pg = table[b, j // page]
                    expect[ends[b] + t] = held[pg, :, j % page] if 0 <= pg < n else 0.0
            assert np.array_equal(got.double().cpu().numpy(), rounded(expect, dtype))


def test_reading_outside_the_cache_gives_zeros():
    """Starts before the first row and behind the table, results that the ends do not reach, ends that do not rise."""
    dtype, D, page, kvH = torch.bfloat16, 64, 16, 2
    pages = [torch.ones(3, kvH, page, D, dtype=dtype, device="cuda") for _ in range(2)]
    out = [torch.full((40, kvH, D), 7.0, dtype=dtype, device="cuda") for _ in range(2)]
    api.paged_read(*pages, i32([[0, 1], [2, 3]]), i32([0, 20, 40]), *out, start=i32([-4, 2 ** 31 - 10]))
    for o in out:
        assert (o[:4] == 0).all() and (o[4:20] == 1).all() and (o[20:] == 0).all()
    for bad in ([0, 100, 40], [40, 20, 0], [-5, 2 ** 31 - 1, -(2 ** 31)], [-(2 ** 31), 7, 2 ** 31 - 1]):
        api.paged_read(*pages, i32([[0, 1], [2, 3]]), i32(bad), *out, start=i32([0, 0]))
    empty = [torch.zeros(0, kvH, page, D, dtype=dtype, device="cuda") for _ in range(2)]
    api.paged_read(*empty, i32([[0, 1], [2, 3]]), i32([0, 20, 40]), *out)
    assert all((o == 0).all() for o in out)
    none = torch.zeros(2, 0, dtype=torch.int32, device="cuda")
    out[0].fill_(7)
    api.paged_read(*pages, none, i32([0, 20, 40]), *out)
    assert all((o == 0).all() for o in out)


# ---- decode --------------------------------------------------------------------------------------


def problem(seed, dtype, B, H, kvH, D, page, lens, width=None, bad=False, scale=1.0, factors=(1.0, 1.0)):
    """Queries, byte pages, their values, table. What no sequence has in the pages is bytes of 0xff, whose scales are NaN."""
    rng = np.random.default_rng(seed)
    lens = np.asarray(lens)
    need = [-(-max(0, int(n)) // page) for n in lens]
    n = sum(need) + 2
    table = table_of(rng, np.maximum(lens, 0), page, n, width or max(need) + 1)
    if bad and max(need) > 1:
        b = int(np.argmax(need))
        table[b, rng.integers(0, need[b])] = rng.choice([-1, n, -(2 ** 31)])
    q = rounded(rng.standard_normal((B, H, D)) * scale, dtype)
    raw = []
    for f in factors:
        codes, scales = ref.encode(rng.standard_normal((n, kvH, page, D)) * scale * f, f)
        there = np.zeros((n, page), bool)
        for b in range(B):
            j = np.arange(min(max(0, int(lens[b])), table.shape[1] * page))
            at = table[b, j // page]
            ok = (at >= 0) & (at < n)
            there[at[ok], j[ok] % page] = True
        codes[~np.broadcast_to(there[:, None, :, None], codes.shape)] = 15
        scales[~np.broadcast_to(there[:, None, :, None], scales.shape)] = 255
        raw.append(ref.join_pages(codes, scales))
    return q, raw, [np.nan_to_num(ref.values(p, page, D, f)) for p, f in zip(raw, factors)], table


def compare(dtype, q, values, table, lens, got):
    # (the weights of the sum over V are rounded to fp16, whatever dtype is)
    out, err, lse, lse_err = want(q, *values, table, lens, torch.float16)
    check(got[0], out, err, dtype, "out")
    there = np.isfinite(lse)
    have = got[1].double().cpu().numpy()
    assert np.array_equal(there, np.isfinite(have)) and (have[~there] == -np.inf).all()
    off = np.abs(have[there] - lse[there])
    assert (off <= lse_err[there]).all(), off.max()


def run(dtype, q, raw, table, lens, factors=(1.0, 1.0), **kw):
    dq = gpu(q, dtype)
    out, lse = torch.full_like(dq, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
    api.paged_decode_4bit(dq, gpu(raw[0]), gpu(raw[1]), i32(table), i32(lens), out, lse=lse, k_scale=factors[0], v_scale=factors[1], **kw)
    return out, lse


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("B,H,kvH,page,lens", [
    (1, 1, 1, 16, [1]), (1, 4, 4, 16, [700]), (3, 8, 2, 32, [0, 33, 64]), (4, 12, 3, 64, [65, 1, 0, 127]),
    (2, 5, 2, 128, [129, 300]), (2, 11, 3, 16, [63, 17]), (1, 40, 1, 256, [513]), (2, 20, 1, 16, [16, 15]),
    (5, 8, 8, 32, [-7, 31, 32, 33, 200]), (2, 16, 2, 64, [2000, 3]), (2, 9, 1, 16, [47, 48]), (1, 33, 2, 32, [97])])
def test_decode_against_64_bits(dtype, D, B, H, kvH, page, lens):
    for bad in (False, True):
        q, raw, values, table = problem(B + D, dtype, B, H, kvH, D, page, lens, bad=bad)
        compare(dtype, q, values, table, lens, run(dtype, q, raw, table, lens))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("factors", [(0.25, 8.0), (2.0 ** 6, 2.0 ** -12)])
def test_factors_of_the_scales(dtype, factors):
    lens = [900, 300, 64]
    q, raw, values, table = problem(3, dtype, 3, 8, 2, 64, 16, lens, factors=factors)
    compare(dtype, q, values, table, lens, run(dtype, q, raw, table, lens, factors))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [32, 128])
def test_large_scores_move_the_reference(dtype, D):
    lens = [900, 300, 64]
    q, raw, values, table = problem(3, dtype, 3, 8, 2, D, 16, lens, scale=6.0)
    compare(dtype, q, values, table, lens, run(dtype, q, raw, table, lens))


@pytest.mark.parametrize("size", [2.0 ** -60, 2.0 ** -14, 2.0 ** 20, 2.0 ** 60])
def test_queries_of_any_size(size):
    """bf16 queries far outside fp16's range; K is as far on the other side, as far as its factor goes."""
    lens = [100, 70]
    f = min(max(1 / size, 2.0 ** -30), 2.0 ** 30)
    q, raw, values, table = problem(5, torch.bfloat16, 2, 4, 2, 64, 16, lens, factors=(f, 1.0))
    q = rounded(q * size, torch.bfloat16)
    if abs(np.log2(f * size)) > 20 and size > 1:  # scores so large that one key is all
        out, lse = run(torch.bfloat16, q, raw, table, lens, (f, 1.0))
        for b in range(2):
            j = np.arange(lens[b])
            for h in range(4):
                k, v = (x[table[b, j // 16], h % 2, j % 16] for x in values)
                s = k @ q[b, h]
                assert np.array_equal(out[b, h].double().cpu().numpy(), rounded(v[s.argmax()], torch.bfloat16))
    else:
        compare(torch.bfloat16, q, values, table, lens, run(torch.bfloat16, q, raw, table, lens, (f, 1.0)))


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_sequences(dtype):
    rng = np.random.default_rng(4)
    lens = rng.integers(0, 3, 301) * rng.integers(1, 40, 301)
    lens[[7, 150, 300]] = (777, 1200, 400)
    q, raw, values, table = problem(5, dtype, 301, 4, 2, 32, 16, lens)
    compare(dtype, q, values, table, lens, run(dtype, q, raw, table, lens))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,D", [(2, 64), (16, 128)])
def test_one_long_sequence(dtype, H, D):
    """Its stages lie in the shares of all warps, whose parts the fold sums."""
    lens = [60000]
    q, raw, values, table = problem(8, dtype, 1, H, 1, D, 64, lens)
    compare(dtype, q, values, table, lens, run(dtype, q, raw, table, lens))


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_keys_anywhere(dtype):
    q, raw, values, table = problem(9, dtype, 3, 4, 2, 64, 16, [16, 5, 40])
    for lens, t in (([0, 0, -1], table), ([16, 5, 40], np.full_like(table, -1))):
        out, lse = run(dtype, q, raw, t, lens)
        assert (out == 0).all() and (lse == -np.inf).all()
    none = [np.zeros((0, 2, 16 * 36), np.uint8)] * 2
    out, lse = run(dtype, q, none, table, [16, 5, 40])
    assert (out == 0).all() and (lse == -np.inf).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_lengths_behind_the_table_and_strided_tables(dtype):
    lens = [5 * 16, 3 * 16 - 1]
    q, raw, values, table = problem(10, dtype, 2, 6, 3, 64, 16, lens)
    wide = torch.full((2, 20), -1, dtype=torch.int32, device="cuda")
    wide[:, 3:3 + table.shape[1]] = i32(table)
    t = wide[:, 3:3 + 5]
    dq = gpu(q, dtype)
    out, lse = torch.empty_like(dq), torch.empty(2, 6, device="cuda")
    api.paged_decode_4bit(dq, gpu(raw[0]), gpu(raw[1]), t, i32([2 ** 31 - 1, lens[1]]), out, lse=lse)
    compare(dtype, q, values, table[:, :5], lens, (out, lse))


@pytest.mark.parametrize("dtype", DTYPES)
def test_what_is_not_finite(dtype):
    """NaN in a key or a value of one head of a sequence makes NaN of the rows that read it and of no other."""
    B, H, kvH, D, page, lens = 3, 8, 2, 64, 16, [50, 200, 33]
    q, raw, values, table = problem(11, dtype, B, H, kvH, D, page, lens)
    for side, (b, kv, j) in ((0, (1, 0, 77)), (1, (1, 1, 199)), (0, (2, 1, 32))):
        broken = [r.copy() for r in raw]
        codes, scales = ref.split_pages(broken[side], page, D)
        scales = scales.copy()
        scales[table[b, j // page], kv, j % page, 1] = 127
        broken[side] = ref.join_pages(codes, scales)
        out, lse = (x.double().cpu().numpy() for x in run(dtype, q, broken, table, lens))
        clean = [x.double().cpu().numpy() for x in run(dtype, q, raw, table, lens)]
        for bb in range(B):
            for h in range(H):
                if bb == b and h % kvH == kv:
                    if side == 0:
                        assert np.isnan(out[bb, h]).all() and np.isnan(lse[bb, h])
                    else:
                        assert np.isnan(out[bb, h, 16:32]).all() and np.isfinite(out[bb, h, :16]).all() and np.isfinite(lse[bb, h])
                else:
                    assert np.array_equal(out[bb, h], clean[0][bb, h]) and lse[bb, h] == clean[1][bb, h]
    bad = q.copy()
    bad[0, 3, 7] = np.nan
    out, lse = run(dtype, bad, raw, table, lens)
    assert torch.isnan(out[0, 3]).all() and torch.isnan(lse[0, 3])
    clean = run(dtype, q, raw, table, lens)
    keep = torch.ones(B, H, dtype=torch.bool)
    keep[0, 3] = False
    assert torch.equal(out.cpu()[keep], clean[0].cpu()[keep]) and torch.equal(lse.cpu()[keep], clean[1].cpu()[keep])


def test_offsets_that_pass_32_bits():
    """Pages behind the first 4 GiB of the cache: appended to, decoded and read back."""
    dtype, kvH, page, D = torch.bfloat16, 8, 256, 256
    n = (1 << 32) // (kvH * page * 144) + 40
    pages = [torch.zeros(n, kvH, page * 144, dtype=torch.uint8, device="cuda") for _ in range(2)]
    rng = np.random.default_rng(12)
    table = np.array([[n - 1, 0], [n - 2, n - 30]])
    x = [rounded(rng.standard_normal((2, kvH, 300, D)), dtype) for _ in range(2)]
    api.paged_append_4bit(gpu(x[0], dtype), gpu(x[1], dtype), *pages, i32(table), i32([0, 0]))
    q = rounded(rng.standard_normal((2, 8, D)), dtype)
    out, lse = torch.empty(2, 8, D, dtype=dtype, device="cuda"), torch.empty(2, 8, device="cuda")
    api.paged_decode_4bit(gpu(q, dtype), *pages, i32(table), i32([300, 300]), out, lse=lse)
    held = [ref.decode(*ref.encode(y, 1.0), 1.0) for y in x]
    # the same rows as a cache of four pages
    small, at = [np.zeros((4, kvH, page, D)) for _ in range(2)], np.arange(300)
    t = np.array([[0, 1], [2, 3]])
    for s, h in zip(small, held):
        for b in range(2):
            s[t[b, at // page], :, at % page] = h[b].swapaxes(0, 1)
    compare(dtype, q, small, t, [300, 300], (out, lse))
    back = [torch.empty(600, kvH, D, dtype=dtype, device="cuda") for _ in range(2)]
    api.paged_read_4bit(*pages, i32(table), i32([0, 300, 600]), *back)
    for got, h in zip(back, held):
        assert np.array_equal(got.double().cpu().numpy(), h.transpose(0, 2, 1, 3).reshape(600, kvH, D))


@pytest.mark.parametrize("dtype", DTYPES)
def test_captured_calls_follow_lengths_and_tables(dtype):
    """Append, read and decode in a graph whose lengths, counts and table change between replays."""
    B, H, kvH, D, page = 3, 8, 2, 64, 16
    lens = np.array([150, 47, 0])
    q, raw, _, table = problem(13, dtype, B, H, kvH, D, page, lens + 1, width=20)
    new = [rounded(np.random.default_rng(14).standard_normal((B, kvH, 1, D)), dtype) for _ in range(2)]
    dq, dk, dv, dt, dl, da = gpu(q, dtype), gpu(new[0], dtype), gpu(new[1], dtype), i32(table), i32(lens), i32(lens + 1)
    pages = [gpu(r) for r in raw]
    out, lse = torch.empty_like(dq), torch.empty(B, H, device="cuda")
    back, ends, start = [torch.zeros(B, kvH, D, dtype=dtype, device="cuda") for _ in range(2)], i32([0, 1, 2, 3]), i32(lens)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        api.paged_append_4bit(dk, dv, *pages, dt, dl)
        api.paged_read_4bit(*pages, dt, ends, *back, start=start)
        api.paged_decode_4bit(dq, *pages, dt, da, out, lse=lse)
    for now in (lens, np.array([149, 20, 1]), np.array([0, 47, 0])):
        for t, x in ((dl, now), (da, now + 1), (start, now)):
            t.copy_(i32(x))
        g.replay()
        values = [ref.values(p.cpu().numpy(), page, D, 1.0) for p in pages]
        for got, x in zip(back, new):
            assert np.array_equal(got.double().cpu().numpy(), ref.decode(*ref.encode(x[:, :, 0], 1.0), 1.0))
        compare(dtype, q, [np.nan_to_num(v) for v in values], table, now + 1, (out, lse))


def test_the_same_bits_twice_and_on_two_streams_at_once():
    dtype, lens = torch.bfloat16, [6000, 3001, 5500, 1]
    q, raw, _, table = problem(15, dtype, 4, 16, 4, 128, 64, lens)
    dq, k, v, t, n = gpu(q, dtype), gpu(raw[0]), gpu(raw[1]), i32(table), i32(lens)
    first = torch.empty_like(dq)
    api.paged_decode_4bit(dq, k, v, t, n, first)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.empty_like(dq) for _ in range(8)] for _ in streams]
    for i in range(8):
        for st, o in zip(streams, outs):
            with torch.cuda.stream(st):
                api.paged_decode_4bit(dq, k, v, t, n, o[i])
    torch.cuda.synchronize()
    assert all(torch.equal(first, x) for o in outs for x in o)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fill", [0x00, 0x7F, 0xFF])
def test_caller_workspace_of_just_the_size(dtype, fill):
    """Whatever it holds, and nothing behind it."""
    import ctypes as C
    from ring_attention_b200._lib import PagedKV, lib
    B, H, kvH, D, page, lens = 3, 12, 3, 128, 32, [700, 5, 0]
    q, raw, values, table = problem(16, dtype, B, H, kvH, D, page, lens)
    c = PagedKV(api._DT[dtype], len(raw[0]), kvH, page, D, 1 << 20, 1 << 20, B, table.shape[1], table.shape[1], 1 << 20, 1 << 20)
    need = lib().ra_paged_decode_4bit_workspace_bytes(C.byref(c), H)
    room = torch.full((need + 256,), fill, dtype=torch.uint8, device="cuda")
    compare(dtype, q, values, table, lens, run(dtype, q, raw, table, lens, workspace=room[:need]))
    assert (room[need:] == fill).all()
    with pytest.raises(RingAttentionError):
        run(dtype, q, raw, table, lens, workspace=room[:need - 1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_wait_that_runs_out_is_reported_and_leaves_the_rows(dtype):
    from ring_attention_b200._lib import lib
    lens = [700, 64, 33]
    q, raw, values, table = problem(17, dtype, 3, 8, 2, 64, 16, lens)
    L = lib()
    api.device_status()
    try:
        L.ra_debug_set_wait_limit_ns(20_000_000)
        L.ra_debug_stall_producer_after(1)
        out, lse = run(dtype, q, raw, table, lens)
        torch.cuda.synchronize()
        L.ra_debug_stall_producer_after(-1)
        again = run(dtype, q, raw, table, lens)  # behind the word nothing is written
        torch.cuda.synchronize()
        assert (out == 7).all() and (lse == 7).all() and (again[0] == 7).all() and (again[1] == 7).all()
        assert api.device_status()[0] == 5
    finally:
        L.ra_debug_stall_producer_after(-1)
        L.ra_debug_set_wait_limit_ns(0)
        api.device_status()
    compare(dtype, q, values, table, lens, run(dtype, q, raw, table, lens))


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_and_decode_with_nothing_between_their_launches(dtype):
    """Steps whose decode comes directly behind the append that writes its queries and rows, and the next append directly behind the
    decode that reads them: the same bits as step by step."""
    B, H, kvH, D, page, steps = 6, 8, 2, 128, 32, 40
    rng = np.random.default_rng(19)
    start = np.array([0, 1, 31, 32, 40, 60])
    table = i32(np.arange(B * 4).reshape(B, 4))
    lens = [i32(start + i) for i in range(steps + 1)]
    rope = api.Rope.make(D)
    new = [gpu(rng.standard_normal((steps, B, h, 1, D)), dtype) for h in (H, kvH, kvH)]

    def chain(wait):
        pages = [api.pages_4bit(4 * B, kvH, page, D) for _ in range(2)]
        first = [gpu(rounded(np.random.default_rng(20).standard_normal((B, kvH, 60, D)), dtype)) for _ in range(2)]
        api.paged_append_4bit(first[0].to(dtype), first[1].to(dtype), *pages, table, i32([0] * B), counts=lens[0])
        q, outs = torch.empty(B, H, 1, D, dtype=dtype, device="cuda"), torch.empty(steps, B, H, D, dtype=dtype, device="cuda")
        torch.cuda.synchronize()
        for i in range(steps):
            api.paged_append_4bit(new[1][i], new[2][i], *pages, table, lens[i], rope=rope, q=new[0][i], q_out=q)
            wait()
            api.paged_decode_4bit(q[:, :, 0], *pages, table, lens[i + 1], outs[i])
            wait()
        return outs

    slow = chain(torch.cuda.synchronize)
    for _ in range(3):
        assert torch.equal(slow, chain(lambda: None))


def test_wrapper_refusals():
    dtype, lens = torch.float16, [40]
    q, raw, _, table = problem(21, dtype, 1, 4, 2, 64, 16, lens)
    dq, k, v, t, n = gpu(q, dtype), gpu(raw[0]), gpu(raw[1]), i32(table), i32(lens)
    out = torch.empty_like(dq)
    for bad in (lambda: api.paged_decode_4bit(dq.float(), k, v, t, n, out), lambda: api.paged_decode_4bit(dq, k, v, t, n, out.bfloat16()),
                lambda: api.paged_decode_4bit(dq, k.cpu(), v, t, n, out), lambda: api.paged_decode_4bit(dq, k, v[:1], t, n, out),
                lambda: api.paged_decode_4bit(dq[:, :, :32], k, v, t, n, out), lambda: api.paged_decode_4bit(dq, k, v, t.long(), n, out),
                lambda: api.paged_decode_4bit(dq, k, v, t, n, out, lse=torch.empty(1, 5, device="cuda")),
                lambda: api.paged_decode_4bit(dq.expand(2, -1, -1), k, v, t, n, out)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: api.paged_decode_4bit(dq, k, v, t, n, out, k_scale=3.0), lambda: api.paged_decode_4bit(dq[:, :1].contiguous(), k, v, t, n, out[:, :1].contiguous())):
        with pytest.raises(RingAttentionError):
            bad()
    rows = torch.zeros(1, 2, 3, 64, dtype=dtype, device="cuda")
    for bad in (lambda: api.paged_append_4bit(rows.float(), rows.float(), k, v, t, n), lambda: api.paged_append_4bit(rows, rows.bfloat16(), k, v, t, n),
                lambda: api.paged_append_4bit(rows[:, :1], rows[:, :1], k, v, t, n), lambda: api.paged_append_4bit(rows, rows, k, v, t, n, q=rows)):
        with pytest.raises(ValueError):
            bad()
    to = torch.zeros(40, 2, 64, dtype=dtype, device="cuda")
    for bad in (lambda: api.paged_read_4bit(k, v, t, n, to, to), lambda: api.paged_read_4bit(k, v, t, i32([0, 40]), to.float(), to.float()),
                lambda: api.paged_read_4bit(k, v, t, i32([0, 40]), to, to[:5]), lambda: api.paged_read_4bit(k, v, t, i32([0, 40]), to[:, :1], to[:, :1]),
                lambda: api.paged_read(k, v, t, i32([0, 40]), to, to)):
        with pytest.raises(ValueError):
            bad()


def test_append_wants_four_dimensions():
    rows, pages = torch.zeros(4, 16, 64, dtype=torch.bfloat16, device="cuda"), api.pages_4bit(2, 4, 16, 64)
    with pytest.raises(ValueError):
        api.paged_append_4bit(rows, rows, pages, pages, i32([[0]]), i32([0]))
    with pytest.raises(ValueError):
        api.paged_read_4bit(pages, pages, i32([[0]]), i32([0, 4]), rows[0], rows[0])
    with pytest.raises(ValueError):
        api.paged_decode_4bit(rows[:, :, 0], pages, pages, i32([[0]]), i32([4]), rows[:, :, 0])


def test_scores_one_step_above_the_reference():
    """Scores (in log2) of 2^27 to 2^28, where steps are 16: a key whose score is one step above the reference has all the weight, as a
    weight of 2^16 is beyond fp16. Keys 0 and 16 of a warp's share, read one after the other; every other key's score is 0."""
    D, page = 256, 32
    scale = np.float32(1.4426950408889634) / np.float32(16.0) * np.float32(2.0 ** 20)
    found = []
    for s0 in range(112, 127):
        for t, code in ((1.0, 2), (2.0, 4), (4.0, 6)):
            a, b = 6 * ref.E4M3[s0], 6 * ref.E4M3[s0] + t * 2.0 ** -13
            if np.float32(b) != b:
                continue
            m, s = np.float32(a) * scale, np.float32(b) * scale
            if 2.0 ** 27 <= m and s < 2.0 ** 28 and s - m == 16 and np.float32(m + np.float32(8.0)) == s:
                found.append((s0, code))
    assert found
    for dtype in DTYPES:
        for s0, code in found:
            q = np.zeros((1, 16, D))
            q[..., 0], q[..., 128] = 1.0, 2.0 ** -13
            codes, scales = np.zeros((2, 1, 1, page, D), np.uint8), np.full((2, 1, 1, page, D // 16), 56, np.uint8)  # (56: 1.0)
            scales[0, 0, 0, :, 0] = s0
            codes[0, 0, 0, [0, 16], 0], codes[0, 0, 0, 16, 128], codes[1, 0, 0, 16] = 7, code, 2
            raw = [ref.join_pages(c, s) for c, s in zip(codes, scales)]
            out, lse = run(dtype, q, raw, np.array([[0]]), [32], (2.0 ** 20, 1.0))
            assert (out == 1).all() and torch.isfinite(lse).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("H", [2, 16])
def test_small_weights_count(dtype, D, H):
    """One key takes nearly all of the weight and has a V of zeros, 31 others some 2^-25.6 of its weight each: the result is theirs.
    A weight is off by half of fp16's smallest step where the reference's is 2^7, so by 2^-32 of the reference's."""
    rng, page, f = np.random.default_rng(22), 16, 2.0 ** 10
    q, table, lens = np.ones((1, H, D)), np.array([[1, 0]]), [32]
    k, v = 0.03 * rng.standard_normal((2, 1, page, D)), np.abs(rng.standard_normal((2, 1, page, D))) + 0.5
    k[1, 0, 0], v[1, 0, 0] = 25.6 * np.log(2) / np.sqrt(D), 0.0
    raw = [ref.join_pages(*ref.encode(x * g, g)) for x, g in ((k, 1.0), (v, f))]
    values = [ref.values(p, page, D, g) for p, g in zip(raw, (1.0, f))]
    out, err, lse, lse_err = want(q, *values, table, lens, torch.float32)
    assert (out > 0).all()
    err = err + 2.0 ** -11 * out + 2.0 ** -32 * values[1][:, 0].sum((0, 1))
    assert (err < 0.05 * out).all()
    got = run(dtype, q, raw, table, lens, (1.0, f))
    check(got[0], out, err, dtype, "out")
    assert (np.abs(got[1].double().cpu().numpy() - lse) <= lse_err).all()


@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_the_largest_queries_on_keys_of_zeros(D):
    """Queries and a factor whose product is beyond 32 bits: keys of zeros have scores of 0 all the same, and the key with the largest
    score all the weight."""
    q = np.full((1, 4, D), 2.0 ** 110)
    codes, scales = np.zeros((2, 1, 2, 16, D), np.uint8), np.full((2, 1, 2, 16, D // 16), 56, np.uint8)  # (56: 1.0)
    codes[1] = 2
    raw = [ref.join_pages(c, s) for c, s in zip(codes, scales)]
    out, lse = run(torch.bfloat16, q, raw, np.array([[0]]), [9], (2.0 ** 30, 1.0))
    assert (out == 1).all() and ((lse - np.log(9)).abs() <= 2.0 ** -21).all()
    codes[0, :, :, 5, 0], scales[0, :, :, 5, 0], codes[1, :, :, 5] = 1, 1, 3  # a score of 2^-10, 2^30 and 2^110 over sqrt(D)
    out, lse = run(torch.bfloat16, q, [ref.join_pages(c, s) for c, s in zip(codes, scales)], np.array([[0]]), [9], (2.0 ** 30, 1.0))
    assert (out == 1.5).all()


@pytest.mark.parametrize("D,tokens", [(256, (1 << 28) + 5), (128, (1 << 29) + 5)])
def test_more_threads_than_32_bits_count(D, tokens):
    """As many tokens as wrap a count of their threads; all but the last five lie before the sequence's first row."""
    dtype, page = torch.bfloat16, 16
    row = gpu(np.random.default_rng(23).standard_normal((1, 1, 1, D)), dtype)
    pages = [api.pages_4bit(1, 1, page, D) for _ in range(2)]
    x = row.expand(1, 1, tokens, D)
    api.paged_append_4bit(x, x, *pages, i32([[0]]), i32([5 - tokens]))
    held = ref.decode(*ref.encode(row.double().cpu().numpy()[0, 0, 0], 1.0), 1.0)
    for p in pages:
        got = ref.values(p.cpu().numpy(), page, D, 1.0)[0, 0]
        assert (got[:5] == held).all() and (got[5:] == 0).all()


def test_pages_of_another_head_dim_are_refused():
    """Pages made for rows of 128 elements would hold twice as many of 64 to the byte: refused where pages_4bit made them, and of any
    pages where the call says page_size."""
    dtype, page = torch.bfloat16, 16
    marked = [api.pages_4bit(2, 2, page, 128) for _ in range(2)]
    plain = [p[:] for p in marked]  # (views do not say what they were made for)
    table, lens, ends = i32([[0]]), i32([4]), i32([0, 4])
    for D in (32, 64, 256):
        rows, q, to = (torch.zeros(s, dtype=dtype, device="cuda") for s in ((1, 2, 3, D), (1, 4, D), (4, 2, D)))
        for pages, kw in ((marked, {}), (plain, {"page_size": page}), (marked, {"page_size": page}), ([plain[0], marked[1]], {})):
            for bad in (lambda: api.paged_append_4bit(rows, rows, *pages, table, lens, **kw),
                        lambda: api.paged_decode_4bit(q, *pages, table, lens, torch.empty_like(q), **kw),
                        lambda: api.paged_read_4bit(*pages, table, ends, to, to.clone(), **kw)):
                with pytest.raises(ValueError, match="head_dim|page_size"):
                    bad()
    assert all((p == 0).all() for p in marked)
    rows, q, to = (torch.ones(s, dtype=dtype, device="cuda") for s in ((1, 2, 4, 128), (1, 4, 128), (4, 2, 128)))
    for pages, kw in ((marked, {}), (plain, {"page_size": page}), (plain, {}), (marked, {"page_size": page})):
        api.paged_append_4bit(rows, rows, *pages, table, i32([0]), **kw)
        outs = [torch.zeros_like(to) for _ in range(2)]
        api.paged_read_4bit(*pages, table, ends, *outs, **kw)
        out = torch.zeros_like(q)
        api.paged_decode_4bit(q, *pages, table, lens, out, **kw)
        assert all((x == 6 * 11 / 64).all() for x in (*outs, out))  # (of 1: 1 / 6 is nearest to 11 / 64, 64 / 11 to 6)
        with pytest.raises(ValueError):
            api.paged_read_4bit(*pages, table, ends, *outs, page_size=32)
