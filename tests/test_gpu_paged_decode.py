"""Decode over a paged KV cache against attention in 64 bits: types, head sizes and groups, lengths from none on, pages that end
inside a stage, pages that are not there, what lies behind a sequence's end, shared pages, graphs and streams."""
import numpy as np
import pytest
import torch

from norm_rope_ref import check, default_freqs, forward, rounded
from paged_ref import table_of, want
from ring_attention_b200 import api
from ring_attention_b200._lib import PagedKV

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def gpu(x, dtype):
    return torch.from_numpy(np.ascontiguousarray(x)).to(dtype).cuda()


def i32(x):
    return torch.from_numpy(np.ascontiguousarray(x).astype(np.int32)).cuda()


def problem(seed, dtype, B, H, kvH, D, page, lens, n_shared=0, width=None, bad=False, scale=1.0):
    """Arrays in 64 bits: q, pages (with NaN in all rows that no sequence has), table, shared pages."""
    rng = np.random.default_rng(seed)
    own = [-(-max(0, int(n)) // page) for n in lens]
    num_pages = sum(max(m, 0) for m in own) + n_shared + 2
    shared = rng.permutation(num_pages)[:n_shared]
    table = table_of(rng, np.maximum(lens, 0), page, num_pages, width or max(own + [1]) + 1, shared)
    k, v = (np.full((num_pages, kvH, page, D), np.nan) for _ in range(2))
    for b, n in enumerate(lens):
        j = np.arange(max(0, int(n)))
        for x in (k, v):
            x[table[b, j // page], :, j % page] = rounded(rng.standard_normal((len(j), kvH, D)) * scale, dtype)
    if n_shared:
        for x in (k, v):
            x[shared] = rounded(rng.standard_normal((n_shared, kvH, page, D)) * scale, dtype)
    if bad:  # some pages in the middle are not there
        for b in range(0, B, 2):
            if own[b] > max(2, n_shared):
                table[b, rng.integers(n_shared, own[b])] = rng.choice([-1, num_pages, -(2 ** 31)])
        if n_shared > 1:
            shared = shared.copy()
            shared[rng.integers(0, n_shared)] = num_pages + 5
    q = rounded(rng.standard_normal((B, H, D)) * scale, dtype)
    return q, k, v, table, shared


def run(dtype, q, k, v, table, lens, shared, **kw):
    out = torch.full(q.shape, float("nan"), dtype=dtype, device="cuda")
    lse = torch.full(q.shape[:2], float("nan"), device="cuda")
    api.paged_decode(gpu(q, dtype), gpu(k, dtype), gpu(v, dtype), i32(table), i32(lens), out, lse=lse,
                     shared_pages=i32(shared) if len(shared) else None, **kw)
    return out, lse


def compare(dtype, q, k, v, table, lens, shared, got):
    clean = [np.nan_to_num(x) for x in (k, v)]
    out, err, lse, lse_err = want(q, *clean, table, lens, dtype, shared)
    check(got[0], out, err, dtype, "out")
    there = np.isfinite(lse)
    have = got[1].double().cpu().numpy()
    assert np.array_equal(there, np.isfinite(have)) and (have[~there] == -np.inf).all()
    off = np.abs(have[there] - lse[there])
    assert (off <= lse_err[there]).all(), off.max()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("B,H,kvH,page,lens", [
    (1, 1, 1, 16, [1]), (1, 4, 4, 16, [700]), (3, 8, 2, 32, [0, 33, 64]), (4, 12, 3, 64, [65, 1, 0, 127]),
    (2, 5, 2, 128, [129, 300]), (2, 11, 3, 16, [63, 17]), (1, 40, 1, 256, [513]), (2, 20, 1, 16, [16, 15]),
    (5, 8, 8, 32, [-7, 31, 32, 33, 200]), (2, 16, 2, 64, [2000, 3])])
def test_against_64_bits(dtype, D, B, H, kvH, page, lens):
    for bad in (False, True):
        p = problem(B + D, dtype, B, H, kvH, D, page, np.array(lens), bad=bad)
        compare(dtype, *p[:4], lens, p[4], run(dtype, *p[:4], lens, p[4]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("B,H,kvH,page,n_shared,lens", [
    (2, 4, 2, 16, 3, [50, 61]), (4, 8, 2, 32, 4, [128, 0, 129, 127]), (7, 6, 6, 16, 9, [145, 144, 150, 300, 143, 1, 200]),
    (3, 5, 2, 64, 2, [128, 200, 140]), (20, 12, 3, 128, 2, [257 + 3 * i for i in range(20)]), (33, 16, 2, 256, 1, [256] * 33),
    (2, 40, 1, 16, 40, [700, 660]), (5, 8, 8, 16, 1, [3, 2, 0, 1, 15])])
def test_shared_pages_against_64_bits(dtype, D, B, H, kvH, page, n_shared, lens):
    for bad in (False, True):
        p = problem(B + D, dtype, B, H, kvH, D, page, np.array(lens), n_shared, bad=bad)
        compare(dtype, *p[:4], lens, p[4], run(dtype, *p[:4], lens, p[4]))


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_scores_move_the_reference(dtype):
    """Scores that differ by hundreds, so that the running maximum moves and most weights vanish."""
    p = problem(3, dtype, 3, 8, 2, 64, 16, np.array([900, 300, 64]), 3, scale=6.0)
    compare(dtype, *p[:4], [900, 300, 64], p[4], run(dtype, *p[:4], [900, 300, 64], p[4]))


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_sequences(dtype):
    """More sequences than a block has threads; most of them empty or short, a few long."""
    rng = np.random.default_rng(4)
    lens = rng.integers(0, 3, 301) * rng.integers(1, 40, 301)
    lens[[7, 150, 300]] = (777, 1200, 400)
    p = problem(5, dtype, 301, 4, 2, 32, 16, lens)
    compare(dtype, *p[:4], lens, p[4], run(dtype, *p[:4], lens, p[4]))
    lens[lens > 0] += 32
    p = problem(6, dtype, 301, 4, 2, 32, 16, lens, 2)
    compare(dtype, *p[:4], lens, p[4], run(dtype, *p[:4], lens, p[4]))


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_long_sequence(dtype):
    lens = [60011]
    p = problem(8, dtype, 1, 2, 1, 128, 64, np.array(lens))
    compare(dtype, *p[:4], lens, p[4], run(dtype, *p[:4], lens, p[4]))


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_keys_anywhere(dtype):
    B, H, kvH, D = 3, 4, 2, 64
    q = torch.randn(B, H, D, device="cuda").to(dtype)
    pages = torch.full((2, kvH, 16, D), float("nan"), device="cuda", dtype=dtype)
    for table, lens in ((torch.zeros(B, 0), [5, 5, 5]), (torch.zeros(B, 2), [0, -1, -(2 ** 31)]), (torch.full((B, 2), -1), [9, 32, 40])):
        for shared in (None, i32(np.array([1, 1, 1]))):
            out, lse = torch.full_like(q, 7), torch.full((B, H), 7.0, device="cuda")
            api.paged_decode(q, pages, pages, table.int().cuda(), i32(np.array(lens)), out, lse=lse, shared_pages=shared)
            assert (out == 0).all() and (lse == -float("inf")).all()
    none = torch.empty(0, kvH, 16, D, device="cuda", dtype=dtype)
    out = torch.full_like(q, 7)
    api.paged_decode(q, none, none, torch.zeros(B, 2, dtype=torch.int32, device="cuda"), i32(np.array([3, 3, 3])), out)
    assert (out == 0).all()
    api.paged_decode(q[:0], pages, pages, torch.zeros(0, 2, dtype=torch.int32, device="cuda"), i32(np.array([])), out[:0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_lengths_behind_the_table_and_strided_tables(dtype):
    p = problem(9, dtype, 2, 4, 2, 64, 32, np.array([96, 64]), width=3)
    q, k, v, table, shared = p
    lens = [2 ** 31 - 1, 64]
    wide = torch.full((2, 9), -1, dtype=torch.int32, device="cuda")
    wide[:, 3:6] = i32(table)
    out, lse = torch.empty(q.shape, dtype=dtype, device="cuda"), torch.empty(q.shape[:2], device="cuda")
    api.paged_decode(gpu(q, dtype), gpu(k, dtype), gpu(v, dtype), wide[:, 3:6], i32(np.array(lens)), out, lse=lse)
    compare(dtype, q, k, v, table, [96, 64], shared, (out, lse))


@pytest.mark.parametrize("dtype", DTYPES)
def test_what_is_not_finite(dtype):
    """NaN in a key reaches its sequence's rows of that KV head and no others; a key of -inf has no weight; so with shared pages,
    whose NaN does not reach sequences that do not have them."""
    for n_shared in (0, 2):
        lens = [70, 33, 90, 20]
        q, k, v, table, shared = problem(10, dtype, 4, 4, 2, 64, 16, np.array(lens), n_shared)
        q = np.abs(q) + 0.25
        k[table[2, 80 // 16], 0, 80 % 16] = np.nan
        k[table[0, 40 // 16], 1, 40 % 16] = -np.inf
        if n_shared:
            k[shared[1], 1, 3] = np.nan
        q = rounded(q, dtype)
        out, lse = run(dtype, q, k, v, table, lens, shared)
        nan = out.isnan().any(-1).cpu().numpy()
        hit = np.zeros((4, 4), bool)
        hit[2, 0::2] = True
        if n_shared:
            hit[:3, 1::2] = True  # (the last sequence is shorter than the shared pages; its own row 19 is not that one)
            if table[3, 1] == shared[1]:
                hit[3, 1::2] = True
        assert np.array_equal(nan, hit) and np.array_equal(lse.isnan().cpu().numpy(), hit)
        assert out[torch.from_numpy(~hit).cuda()].isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_offsets_that_pass_32_bits(dtype):
    """A cache of more than 2^31 elements, the last pages of it read."""
    kvH, page, D = 8, 256, 256
    n = 2 ** 31 // (kvH * page * D) + 3
    k, v = (torch.empty(n, kvH, page, D, device="cuda", dtype=dtype) for _ in range(2))
    at = [n - 1, 0, n - 2]
    for x in (k, v):
        x[at] = torch.randn(3, kvH, page, D, device="cuda").to(dtype)
    lens = [600, 300]
    table = np.array([[n - 1, 0, n - 2], [n - 2, n - 1, -1]])
    q = rounded(np.random.default_rng(1).standard_normal((2, 8, D)), dtype)
    out, lse = torch.empty(2, 8, D, dtype=dtype, device="cuda"), torch.empty(2, 8, device="cuda")
    api.paged_decode(gpu(q, dtype), k, v, i32(table), i32(np.array(lens)), out, lse=lse)
    small = {n - 1: 0, 0: 1, n - 2: 2, -1: -1}
    compare(dtype, q, *(x[at].double().cpu().numpy() for x in (k, v)), np.vectorize(small.get)(table), lens, (), (out, lse))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n_shared", [0, 4])
def test_captured_calls_follow_lengths_and_tables(dtype, n_shared):
    B, H, kvH, D, page = 5, 8, 2, 128, 16
    lens = np.array([200, 77, 0, 64, 130])
    q, k, v, table, shared = problem(11, dtype, B, H, kvH, D, page, lens, n_shared)
    dq, dk, dv, dt, dl = gpu(q, dtype), gpu(k, dtype), gpu(v, dtype), i32(table), i32(lens)
    ds = i32(shared) if n_shared else None
    out, lse = torch.empty_like(dq), torch.empty(B, H, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        api.paged_decode(dq, dk, dv, dt, dl, out, lse=lse, shared_pages=ds)
    for now in (lens, np.array([5, 77, 0, 0, 129]), np.array([0, 0, 0, 0, 1]), lens):
        dl.copy_(i32(now))
        g.replay()
        compare(dtype, q, k, v, table, now, shared, (out, lse))
    dt[0] = dt[1]
    table[0] = table[1]
    dl.copy_(i32(np.array([77, 77, 0, 64, 130])))
    g.replay()
    compare(dtype, q, k, v, table, [77, 77, 0, 64, 130], shared, (out, lse))


def test_the_same_bits_twice_and_on_two_streams_at_once():
    dtype = torch.bfloat16
    lens = np.array([4000, 100, 2500, 1])
    p = problem(12, dtype, 4, 16, 4, 128, 64, lens, 1)
    q, k, v = (gpu(x, dtype) for x in p[:3])
    t, n, s = i32(p[3]), i32(lens), i32(p[4])
    first = torch.empty_like(q)
    api.paged_decode(q, k, v, t, n, first, shared_pages=s)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.empty_like(q) for _ in range(8)] for _ in streams]
    for i in range(8):
        for st, o in zip(streams, outs):
            with torch.cuda.stream(st):
                api.paged_decode(q, k, v, t, n, o[i], shared_pages=s)
    torch.cuda.synchronize()
    assert all(torch.equal(first, x) for o in outs for x in o)


@pytest.mark.parametrize("dtype", DTYPES)
def test_caller_workspace_of_just_the_size(dtype):
    lens = np.array([300, 20, 77])
    p = problem(13, dtype, 3, 8, 2, 64, 16, lens, 1)
    pages = gpu(p[1], dtype)
    n, kvH, page, D = pages.shape
    cache = PagedKV(api._DT[dtype], n, kvH, page, D, pages.data_ptr(), pages.data_ptr(), 3, p[3].shape[1], p[3].shape[1], 1, 1)
    need = api.lib().ra_paged_decode_workspace_bytes(cache, 8, 16)
    room = torch.full((need + 256,), 0xFF, dtype=torch.uint8, device="cuda")
    compare(dtype, *p[:4], lens, p[4], run(dtype, *p[:4], lens, p[4], workspace=room[:need]))
    assert (room[need:] == 0xFF).all()
    with pytest.raises(api._lib.RingAttentionError):
        run(dtype, *p[:4], lens, p[4], workspace=room[:need - 16])


@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_rotation_append_and_decode_together(dtype):
    """A prompt's rows and then tokens one by one, as a server runs them: norm and rotation on the way into the cache and to the
    query, decode against it; each step against 64 bits on the rows that the cache holds."""
    B, H, kvH, D, page, T = 3, 6, 2, 64, 16, 40
    rng = np.random.default_rng(14)
    rope, freqs = api.Rope.make(D), default_freqs(D)
    wq, wk = (rounded(1 + 0.2 * rng.standard_normal(D), dtype) for _ in range(2))
    prompt = np.array([40, 17, 1])
    table = rng.permutation(12).reshape(B, 4)
    k_pages, v_pages = (torch.full((12, kvH, page, D), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    dt, lens, counts = i32(table), i32(np.zeros(B)), i32(prompt)
    new = [rounded(rng.standard_normal((B, h, T, D)), dtype) for h in (H, kvH, kvH)]
    q_out = torch.empty(B, H, T, D, dtype=dtype, device="cuda")
    how = dict(rope=rope, q_weight=gpu(wq, dtype), k_weight=gpu(wk, dtype))
    api.paged_append(gpu(new[1], dtype), gpu(new[2], dtype), k_pages, v_pages, dt, lens, counts=counts, q=gpu(new[0], dtype),
                     q_out=q_out, **how)
    lens += counts
    for step in range(4):
        q, k, v = (rounded(rng.standard_normal((B, h, 1, D)), dtype) for h in (H, kvH, kvH))
        q_one, out, lse = (torch.empty(B, H, 1, D, dtype=dtype, device="cuda"), torch.empty(B, H, D, dtype=dtype, device="cuda"),
                           torch.empty(B, H, device="cuda"))
        api.paged_append(gpu(k, dtype), gpu(v, dtype), k_pages, v_pages, dt, lens, q=gpu(q, dtype), q_out=q_one, **how)
        at = prompt + step
        y, e = forward(q, wq, at[:, None, None], D, False, freqs, np.float32(1e-6))
        check(q_one, y, e, dtype)
        for b in range(B):
            y, e = forward(k[b, :, 0], wk, at[b], D, False, freqs, np.float32(1e-6))
            check(k_pages[table[b, at[b] // page], :, at[b] % page], y, e, dtype)
        lens += 1
        api.paged_decode(q_one[:, :, 0], k_pages, v_pages, dt, lens, out, lse=lse)
        compare(dtype, q_one[:, :, 0].double().cpu().numpy(), k_pages.double().cpu().numpy(), v_pages.double().cpu().numpy(),
                table, at + 1, (), (out, lse))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("B,H,kvH,page,n_shared,lens", [
    (7, 12, 6, 16, 430, [6880, 6881, 7000, 0, 6879, 9000, 6900]), (130, 6, 2, 64, 15, [960 + i % 70 for i in range(130)]),
    (40, 15, 3, 32, 66, [2112 + 3 * i - 2112 * (i % 9 == 4) for i in range(40)]), (20, 2, 1, 256, 51, [13056 + 20 * i for i in range(20)]),
    (33, 5, 2, 128, 30, [3840 + i for i in range(33)])])
def test_shared_pages_of_large_batches_against_64_bits(dtype, D, B, H, kvH, page, n_shared, lens):
    """Batches that read the shared pages once for all, which small ones in 16 bits do not."""
    p = problem(B + D, dtype, B, H, kvH, D, page, np.array(lens), n_shared, bad=D in (64, 256))
    compare(dtype, *p[:4], lens, p[4], run(dtype, *p[:4], lens, p[4]))


def test_what_is_not_finite_in_the_pages_of_a_large_batch():
    dtype, lens, n_shared = torch.float16, [20100, 20033, 20090, 19999], 1250
    q, k, v, table, shared = problem(10, dtype, 4, 4, 2, 64, 16, np.array(lens), n_shared)
    q = rounded(np.abs(q) + 0.25, dtype)
    k[table[2, 20080 // 16], 0, 0] = np.nan
    k[shared[7], 1, 3] = np.nan
    table[3, 7] = table[3, 8]  # (the last sequence is shorter than the shared pages: its own table counts)
    out, lse = run(dtype, q, k, v, table, lens, shared)
    hit = np.zeros((4, 4), bool)
    hit[2, 0::2] = True
    hit[:3, 1::2] = True
    assert np.array_equal(out.isnan().any(-1).cpu().numpy(), hit) and np.array_equal(lse.isnan().cpu().numpy(), hit)
    assert out[torch.from_numpy(~hit).cuda()].isfinite().all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,n_shared", [(32, 2500), (64, 1250), (128, 625), (256, 320)])
def test_rows_and_shared_pages_of_nothing_but_nan(dtype, D, n_shared):
    """A query of NaN, of a sequence with no rows but the shared ones and of one with more, gives NaN and not what a row without
    keys gives; so do shared pages whose every key of a KV head is NaN, so that no share of them has a score."""
    P = 16 * n_shared
    lens = [P, P + 33, P + 90, P - 1]
    q, k, v, table, shared = problem(18, dtype, 4, 4, 2, D, 16, np.array(lens), n_shared)
    q[:2, 1] = np.nan
    k[shared, 0] = np.nan
    out, lse = run(dtype, q, k, v, table, lens, shared)
    hit = np.zeros((4, 4), bool)
    hit[:2, 1] = True
    hit[:, 0::2] = True
    assert np.array_equal(out.isnan().any(-1).cpu().numpy(), hit) and np.array_equal(lse.isnan().cpu().numpy(), hit)
    assert out[torch.from_numpy(hit).cuda()].isnan().all()
    assert out[torch.from_numpy(~hit).cuda()].isfinite().all()

def test_captured_calls_of_a_large_batch_follow_lengths():
    dtype, B, H, kvH, D, page = torch.bfloat16, 5, 8, 2, 128, 16
    lens = np.array([7500, 77, 0, 7360, 7700])
    q, k, v, table, shared = problem(11, dtype, B, H, kvH, D, page, lens, 460)
    dq, dk, dv, dt, dl, ds = gpu(q, dtype), gpu(k, dtype), gpu(v, dtype), i32(table), i32(lens), i32(shared)
    out, lse = torch.empty_like(dq), torch.empty(B, H, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        api.paged_decode(dq, dk, dv, dt, dl, out, lse=lse, shared_pages=ds)
    for now in (lens, np.array([7359, 1, 0, 0, 7360]), lens):
        dl.copy_(i32(now))
        g.replay()
        compare(dtype, q, k, v, table, now, shared, (out, lse))


def test_large_batches_on_two_streams_at_once():
    dtype, lens = torch.bfloat16, np.array([6000, 5100, 5500, 1])
    p = problem(12, dtype, 4, 16, 4, 128, 64, lens, 79)
    q, k, v = (gpu(x, dtype) for x in p[:3])
    t, n, s = i32(p[3]), i32(lens), i32(p[4])
    first = torch.empty_like(q)
    api.paged_decode(q, k, v, t, n, first, shared_pages=s)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.empty_like(q) for _ in range(8)] for _ in streams]
    for i in range(8):
        for st, o in zip(streams, outs):
            with torch.cuda.stream(st):
                api.paged_decode(q, k, v, t, n, o[i], shared_pages=s)
    torch.cuda.synchronize()
    assert all(torch.equal(first, x) for o in outs for x in o)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n_shared", [5, 190])
def test_a_chain_of_steps_with_shared_pages(dtype, n_shared):
    """Steps enqueued one behind the other, each of which writes the queries, rows and lengths that the next one reads, with
    nothing waiting between them: the same bits as step by step."""
    B, H, kvH, D, page, steps = 6, 8, 2, 128, 32, 30
    rng = np.random.default_rng(15)
    shared = np.arange(n_shared)
    table = np.concatenate([np.tile(shared, (B, 1)), n_shared + np.arange(B * 3).reshape(B, 3)], 1)
    rope = api.Rope.make(D)
    start = n_shared * page + np.array([0, 1, 31, 32, 40, 60])
    new = [gpu(rng.standard_normal((steps, B, h, 1, D)), dtype) for h in (H, kvH, kvH)]
    pages = [gpu(rng.standard_normal((n_shared + 3 * B, kvH, page, D)), dtype) for _ in range(2)]
    dt, ds = i32(table), i32(shared)

    def chain(wait):
        k_pages, v_pages = (x.clone() for x in pages)
        lens, q = i32(start), torch.empty(B, H, 1, D, dtype=dtype, device="cuda")
        outs = torch.empty(steps, B, H, D, dtype=dtype, device="cuda")
        for i in range(steps):
            api.paged_append(new[1][i], new[2][i], k_pages, v_pages, dt, lens, rope=rope, q=new[0][i], q_out=q)
            lens += 1
            wait()
            api.paged_decode(q[:, :, 0], k_pages, v_pages, dt, lens, outs[i], shared_pages=ds)
            wait()
        return outs

    slow = chain(torch.cuda.synchronize)
    for _ in range(3):
        assert torch.equal(slow, chain(lambda: None))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,n_shared", [(64, 400), (128, 5), (128, 190)])
def test_append_and_decode_with_nothing_between_their_launches(dtype, D, n_shared):
    """Steps whose decode comes directly behind the append that writes its queries and rows, and the next step's append directly
    behind the decode that reads them: the same bits as step by step, enqueued and from a graph. (Lengths of all steps are there
    before the first, so that no launch of the caller's stands between.)"""
    B, H, kvH, page, steps = 6, 8, 2, 32, 40
    rng = np.random.default_rng(19)
    shared = np.arange(n_shared)
    table = np.concatenate([np.tile(shared, (B, 1)), n_shared + np.arange(B * 4).reshape(B, 4)], 1)
    rope = api.Rope.make(D)
    start = n_shared * page + np.array([0, 1, 31, 32, 40, 60])
    lens = [i32(start + i) for i in range(steps + 1)]
    new = [gpu(rng.standard_normal((steps, B, h, 1, D)), dtype) for h in (H, kvH, kvH)]
    pages = [gpu(rng.standard_normal((n_shared + 4 * B, kvH, page, D)), dtype) for _ in range(2)]
    k_pages, v_pages = (x.clone() for x in pages)
    q, outs = torch.empty(B, H, 1, D, dtype=dtype, device="cuda"), torch.empty(steps, B, H, D, dtype=dtype, device="cuda")
    dt, ds = i32(table), i32(shared)

    def begin():
        for x, y in zip((k_pages, v_pages), pages):
            x.copy_(y)
        q.zero_()
        outs.zero_()

    def chain(wait=lambda: None):
        for i in range(steps):
            api.paged_append(new[1][i], new[2][i], k_pages, v_pages, dt, lens[i], rope=rope, q=new[0][i], q_out=q)
            wait()
            api.paged_decode(q[:, :, 0], k_pages, v_pages, dt, lens[i + 1], outs[i], shared_pages=ds)
            wait()

    begin()
    chain(torch.cuda.synchronize)
    slow = outs.clone()
    assert not (slow == 0).all(-1).any()
    for _ in range(5):
        begin()
        chain()
        assert torch.equal(slow, outs)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        chain()
    for _ in range(5):
        begin()
        g.replay()
        assert torch.equal(slow, outs)

@pytest.mark.parametrize("n_shared", [1, 3])
def test_more_sequences_than_the_shared_pages_have_blocks_for(n_shared):
    """A batch whose rows on the shared pages are too many for the tensor-core kernel's list of blocks."""
    B = 5200
    lens = 16 * n_shared + np.arange(B) % 5
    lens[::7] = 15
    p = problem(16, torch.float16, B, 8, 1, 32, 16, lens, n_shared)
    compare(torch.float16, *p[:4], lens, p[4], run(torch.float16, *p[:4], lens, p[4]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,n_shared", [(5200, 1), (1000, 1), (5200, 2)])
def test_one_shared_page_of_many_sequences(dtype, B, n_shared):
    """A page or two that many sequences read once for all: by the tensor-core kernel, and, where it has too few blocks for their
    rows, by the units that the others have."""
    H, kvH, D, page = 8, 1, 128, 16 if B > 1000 else 256
    lens = page * n_shared + np.arange(B) % 5
    lens[::7] = page - 1
    p = problem(20, dtype, B, H, kvH, D, page, lens, n_shared)
    cache = PagedKV(api._DT[dtype], len(p[1]), kvH, page, D, 0x1000, 0x1000, B, p[3].shape[1], p[3].shape[1], 0x1000, 0x1000)
    assert api.lib().ra_debug_paged_route(cache, H, n_shared * page) == (2 if B > 1000 or dtype == torch.float32 else 3)
    compare(dtype, *p[:4], lens, p[4], run(dtype, *p[:4], lens, p[4]))

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n_shared", [0, 40, 960])
def test_a_wait_that_runs_out_is_reported_and_leaves_the_rows(dtype, n_shared):
    lens = [40000, 30000] if n_shared < 960 else [62000, 61500]
    q, k, v, table, shared = problem(17, dtype, 2, 4, 2, 64, 64, np.array(lens), n_shared)
    args = gpu(q, dtype), gpu(k, dtype), gpu(v, dtype), i32(table), i32(lens)
    out, lse = torch.full(q.shape, 7, dtype=dtype, device="cuda"), torch.full(q.shape[:2], 7.0, device="cuda")
    kw = dict(lse=lse, shared_pages=i32(shared) if n_shared else None)
    L = api.lib()
    assert api.device_status()[0] == 0
    L.ra_debug_set_wait_limit_ns(5_000_000)
    L.ra_debug_stall_producer_after(1)  # keys that never come
    try:
        api.paged_decode(*args, out, **kw)
        torch.cuda.synchronize()
    finally:
        L.ra_debug_stall_producer_after(-1)
        L.ra_debug_set_wait_limit_ns(0)
    api.paged_decode(*args, out, **kw)  # behind it nothing is computed until the word is read
    torch.cuda.synchronize()
    assert (out == 7).all() and (lse == 7).all()
    assert api.device_status()[0] == 5 and api.device_status()[0] == 0
    api.paged_decode(*args, out, **kw)
    compare(dtype, q, k, v, table, lens, shared, (out, lse))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n_shared", [0, 3])
@pytest.mark.parametrize("fill", [0x00, 0x01, 0x7F, 0x80, 0xFF])
def test_parts_that_no_warp_has_left(dtype, n_shared, fill):
    """Where no warp computed anything (a status word that was set when they looked, and cleared since), what a workspace happens
    to hold is no list of parts: the rows stay, but for those that have no keys."""
    lens = np.array([700, 48, 0, 300, 17])
    q, k, v, table, shared = problem(21, dtype, 5, 8, 2, 64, 16, lens, n_shared)
    args = gpu(q, dtype), gpu(k, dtype), gpu(v, dtype), i32(table), i32(lens)
    out, lse = torch.full(q.shape, 7, dtype=dtype, device="cuda"), torch.full(q.shape[:2], 7.0, device="cuda")
    kw = dict(lse=lse, shared_pages=i32(shared) if n_shared else None, workspace=torch.full((1 << 23,), fill, dtype=torch.uint8, device="cuda"))
    L = api.lib()
    L.ra_debug_stall_producer_after(0)
    try:
        api.paged_decode(*args, out, **kw)
        torch.cuda.synchronize()
    finally:
        L.ra_debug_stall_producer_after(-1)
    assert api.device_status()[0] == 0
    there = torch.tensor(lens > 0, device="cuda")
    assert (out[there] == 7).all() and (lse[there] == 7).all() and (out[~there] == 0).all() and (lse[~there] == -float("inf")).all()
    api.paged_decode(*args, out, **kw)
    compare(dtype, q, k, v, table, lens, shared, (out, lse))

def test_decode_wrapper_refusals():
    q = torch.zeros(2, 4, 64, device="cuda")
    p, o = torch.zeros(3, 2, 16, 64, device="cuda"), torch.empty_like(q)
    t, n = torch.zeros(2, 1, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    for a, kw in (((q.half(), p, p, t, n, o), {}), ((q[:1], p, p, t, n, o), {}), ((q, p, p, t, n, o.half()), {}),
                  ((q, p, p, t, n, o), {"lse": torch.empty(2, 4, device="cuda").half()}), ((q[0], p, p, t, n, o), {}),
                  ((q, p, p, t, n, o), {"shared_pages": torch.zeros(1, dtype=torch.int64, device="cuda")}),
                  ((q, p, p, t, n, o), {"shared_pages": torch.zeros(1, dtype=torch.int32)}),
                  ((q.transpose(0, 1).contiguous().transpose(0, 1), p, p, t, n, o), {}), ((q.cpu(), p, p, t, n, o), {})):
        with pytest.raises(ValueError):
            api.paged_decode(*a, **kw)
    with pytest.raises(api._lib.RingAttentionError):
        api.paged_decode(q[:, :1].contiguous(), p, p, t, n, o[:, :1].contiguous())  # fewer heads than the cache has
