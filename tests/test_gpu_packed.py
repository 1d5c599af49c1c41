"""Attention over packed sequences of unlike lengths against 64 bits."""
import numpy as np
import pytest
import torch

import four_bit_ref
from packed_ref import compare, want
from ring_attention_b200 import api
from ring_attention_b200._lib import RingAttentionError, lib

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]


def i32(x):
    return torch.as_tensor(np.asarray(x, dtype=np.int64)).to(torch.int32).cuda()


def ends_of(lens, first=0):
    return first + np.concatenate([[0], np.cumsum(np.asarray(lens, dtype=np.int64))]).astype(np.int64)


def some(seed, shape, dtype, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def run(q, k, v, ends, k_ends=None, causal=True):
    out, lse = torch.full_like(q, 7.0, memory_format=torch.contiguous_format), torch.full((q.shape[1], q.shape[0]), 7.0, device="cuda")
    api.packed_attention(q, k, v, i32(ends), out, k_ends=i32(k_ends) if k_ends is not None else None, causal=causal, lse=lse)
    return out, lse


def problem(seed, dtype, H, kvH, D, lens, k_lens=None, scale=1.0, first=0, behind=0, k_first=0, k_behind=0):
    ends = ends_of(lens, first)
    q = some(seed, (int(ends[-1]) + behind, H, D), dtype, scale)
    k_ends = ends if k_lens is None else ends_of(k_lens, k_first)
    n = q.shape[0] if k_lens is None else int(k_ends[-1]) + k_behind
    return q, some(seed + 1, (n, kvH, D), dtype, scale), some(seed + 2, (n, kvH, D), dtype), ends, k_ends


def check(dtype, p, causal=True):
    q, k, v, ends, k_ends = p
    compare(dtype, q, k, v, ends, k_ends, causal, *run(q, k, v, ends, None if k_ends is ends else k_ends, causal))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("H,kvH", [(1, 1), (4, 1), (6, 2), (5, 1), (3, 3), (16, 1)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens", [[1], [128], [129, 1, 0, 64], [300, 17, 255, 256, 257], [0, 0, 33, 0, 31, 32, 0], [520, 7]])
def test_whole_prompts(dtype, D, H, kvH, causal, lens):
    check(dtype, problem(len(lens) + D, dtype, H, kvH, D, lens), causal)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("H,kvH", [(2, 2), (8, 2), (9, 3)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,k_lens", [([5, 64, 1, 33], [700, 64, 300, 40]), ([130, 1], [131, 1000]), ([70, 200, 40], [30, 0, 40]),
                                         ([300, 300, 0, 9], [1, 290, 50, 0]), ([1] * 9, [1, 2, 127, 128, 129, 255, 256, 257, 640])])
def test_chunks_of_prompts(dtype, D, H, kvH, causal, lens, k_lens):
    """More keys than queries, and fewer: rows in front of the first key see none."""
    check(dtype, problem(len(lens) + D, dtype, H, kvH, D, lens, k_lens, k_first=3, k_behind=2), causal)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,kvH,D", [(4, 2, 64), (8, 1, 128), (2, 2, 256)])
@pytest.mark.parametrize("causal", [True, False])
def test_more_sequences_than_a_warp_has_lanes(dtype, H, kvH, D, causal):
    rng = np.random.default_rng(3)
    lens = rng.integers(0, 3, 333) * rng.integers(1, 30, 333)
    lens[[0, 31, 32, 100, 332]] = (400, 129, 257, 64, 300)
    check(dtype, problem(4, dtype, H, kvH, D, lens, first=5, behind=9), causal)
    k_lens = lens + rng.integers(-5, 200, 333).clip(-lens)
    check(dtype, problem(4, dtype, H, kvH, D, lens, k_lens), causal)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_large_scores_move_the_reference(dtype, D):
    check(dtype, problem(6, dtype, 4, 2, D, [900, 300, 64], scale=6.0))
    # later keys are ever larger, so that the reference moves in every tile
    q, k, v, ends, k_ends = problem(7, dtype, 4, 2, D, [700, 513])
    q = q.abs()
    k = (k.abs() * torch.linspace(0.1, 6.0, k.shape[0], device="cuda")[:, None, None]).to(dtype)
    check(dtype, (q, k, v, ends, k_ends))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,kvH,D,causal", [(4, 1, 128, True), (2, 2, 64, True), (2, 1, 256, True), (2, 1, 128, False), (1, 1, 64, False)])
def test_long_sequences(dtype, H, kvH, D, causal):
    check(dtype, problem(8, dtype, H, kvH, D, [5000, 1, 3333, 64]), causal)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,kvH,D", [(40, 1, 64), (64, 2, 128), (34, 2, 32), (20, 1, 256)])
def test_more_heads_than_a_tile_takes(dtype, H, kvH, D):
    check(dtype, problem(41, dtype, H, kvH, D, [150, 3, 40]))
    check(dtype, problem(44, dtype, H, kvH, D, [1, 2, 1, 1], [1, 40, 300, 129]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,kvH,D", [(4, 1, 64), (2, 2, 128), (2, 1, 256), (4, 2, 32)])
@pytest.mark.parametrize("causal", [True, False])
def test_a_long_sequence_among_short_ones(dtype, H, kvH, D, causal):
    """By the average a call of short sequences; one is long, and some have long keys."""
    lens = [1] * 200 + [2500] + [2] * 100
    check(dtype, problem(47, dtype, H, kvH, D, lens), causal)
    k_lens = [1] * 200 + [2600] + [2 + 300 * (i % 50 == 0) for i in range(100)]
    check(dtype, problem(50, dtype, H, kvH, D, lens, k_lens), causal)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_rows_with_strides(dtype, D):
    """Slices of a fused projection, heads before rows, results inside wider ones, a tensor of one row."""
    lens, H, kvH = [200, 33], 6, 2
    ends = ends_of(lens)
    qkv = some(9, (233, H + 2 * kvH, D), dtype)
    q, k, v = qkv[:, :H], qkv[:, H:H + kvH], qkv[:, H + kvH:]
    wide, lse = torch.full((233, H + 2, D + 8), 7.0, dtype=dtype, device="cuda"), torch.full((H, 233), 7.0, device="cuda")
    out = wide[:, 1:1 + H, :D]
    api.packed_attention(q, k, v, i32(ends), out, lse=lse)
    compare(dtype, q, k, v, ends, ends, True, out, lse)
    assert (wide[:, 0] == 7).all() and (wide[:, -1] == 7).all() and (wide[:, :, D:] == 7).all()
    by_head = some(10, (kvH, 233, D), dtype).transpose(0, 1)
    out = torch.full((H, 233, D), 7.0, dtype=dtype, device="cuda").transpose(0, 1)
    api.packed_attention(q, by_head, v, i32(ends), out, lse=lse)
    compare(dtype, q, by_head, v, ends, ends, True, out, lse)
    one = some(11, (1, 1, D), dtype)
    compare(dtype, one, one, one, [0, 1], [0, 1], True, *run(one, one, one, [0, 1]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_other_sequences_do_not_reach_a_sequence(dtype, D, bad):
    """Sequences between others, and rows of none, of nothing but what is not finite: the same bits as between ordinary ones."""
    lens = [130, 40, 1, 129, 7, 100]
    q, k, v, ends, _ = problem(12, dtype, 4, 2, D, lens, first=20, behind=50)
    clean = run(q, k, v, ends)
    q, k, v = (x.clone() for x in (q, k, v))
    good = torch.zeros(q.shape[0], dtype=torch.bool, device="cuda")
    for b in (0, 2, 4):
        good[int(ends[b]):int(ends[b + 1])] = True
    for x in (q, k, v):
        x[~good] = bad
    got = run(q, k, v, ends)
    assert torch.equal(got[0][good], clean[0][good]) and torch.equal(got[1][:, good], clean[1][:, good])
    others = good.clone()
    others[:20] = others[int(ends[-1]):] = True
    assert torch.isnan(got[0][~others]).all() and torch.isnan(got[1][:, ~others]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_what_is_not_finite_in_a_row(dtype, D):
    """A query or a key of NaN: the rows that read it, and no other."""
    q, k, v, ends, _ = problem(13, dtype, 4, 2, D, [300, 60])
    clean = run(q, k, v, ends)
    q2 = q.clone()
    q2[70, 1, 3] = float("nan")
    out, lse = run(q2, k, v, ends)
    keep = torch.ones(360, 4, dtype=torch.bool, device="cuda")
    keep[70, 1] = False
    assert torch.equal(out[keep], clean[0][keep]) and torch.isnan(out[70, 1]).all() and torch.isnan(lse[1, 70])
    k2 = k.clone()
    k2[200, 1, 5] = float("nan")
    out, lse = run(q, k2, v, ends)
    keep[70, 1] = True
    keep[200:300, 1::2] = False
    assert torch.equal(out[keep], clean[0][keep]) and torch.isnan(out[~keep]).all() and torch.equal(lse.T[keep], clean[1].T[keep])


def test_nothing_to_do():
    dtype, D = torch.bfloat16, 64
    q, kv = some(14, (9, 4, D), dtype), some(15, (0, 2, D), dtype)
    out, lse = run(q, kv, kv, [0, 4, 9], [0, 0, 0])  # no keys at all
    assert (out == 0).all() and (lse == -np.inf).all()
    out, lse = run(q, kv, kv, [0, 4, 9], [0, 3, 8])  # ends behind the keys that there are
    assert (out == 0).all() and (lse == -np.inf).all()
    out, lse = run(q, q[:, :2], q[:, :2], [0])  # no sequences
    assert (out == 7).all() and (lse == 7).all()
    out, lse = run(q, q[:, :2], q[:, :2], [4, 4, 4])
    assert (out == 7).all() and (lse == 7).all()
    none = some(16, (0, 4, D), dtype)
    api.packed_attention(none, none[:, :2], none[:, :2], i32([0, 0]), torch.empty_like(none))


@pytest.mark.parametrize("D", [64, 128, 256])
def test_ends_that_do_not_rise_stay_inside(D):
    """Whatever the ends hold, nothing outside the results is written and the call ends."""
    dtype, H = torch.float16, 4
    q, k, v = some(17, (200, H, D), dtype), some(18, (300, 2, D), dtype), some(19, (300, 2, D), dtype)
    room = torch.full((400, H, D), 7.0, dtype=dtype, device="cuda")
    big = 2 ** 31 - 1
    for ends, k_ends in (([0, 500, 100], [0, 100, 900]), ([-7, 40, -3], [5, -9, big]), ([150, 20, 200], [299, 0, 300]),
                         ([-big - 1, big, -big - 1], [-big - 1, big, big]), ([0, 200, big], [300, 0, 0])):
        api.packed_attention(q, k, v, i32(ends), room[100:300], k_ends=i32(k_ends))
        torch.cuda.synchronize()
        assert (room[:100] == 7).all() and (room[300:] == 7).all()
    assert api.device_status()[0] == 0


def test_offsets_that_pass_32_bits():
    """Sequences at the end of tensors of more than 2^32 elements; a query head's results behind 2^31 others."""
    dtype, H, kvH, D = torch.bfloat16, 64, 64, 128
    rows = (1 << 32) // (H * D) + 1000
    first = rows - 517
    q, k, v, out = (torch.zeros(rows, H, D, dtype=dtype, device="cuda") for _ in range(4))
    for i, x in enumerate((q, k, v)):
        x[first:] = some(20 + i, (517, H, D), dtype)
    ends = [0, 0, first + 0, first + 300, rows - 1]
    ends[1] = ends[2]  # one long sequence of zeros would be all the work: it has no rows
    ends[0] = ends[1]
    lse = torch.zeros(H, rows, device="cuda")
    api.packed_attention(q, k, v, i32(ends), out, lse=lse)
    at = [e - first for e in ends]
    out[rows - 1] = 7
    lse[:, rows - 1] = 7
    compare(dtype, q[first:], k[first:], v[first:], at, at, True, out[first:], lse[:, first:])
    assert (out[:first] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_captured_calls_follow_the_ends(dtype, D):
    H, kvH, rows, keys = 4, 2, 400, 900
    q, k, v = some(23, (rows, H, D), dtype), some(24, (keys, kvH, D), dtype), some(25, (keys, kvH, D), dtype)
    ends, k_ends = i32([0, 0, 0, 0]), i32([0, 0, 0, 0])
    out, lse = torch.zeros_like(q), torch.zeros(H, rows, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        api.packed_attention(q, k, v, ends, out, k_ends=k_ends, lse=lse)
    for e, ke in (([0, 100, 101, 400], [0, 100, 500, 900]), ([3, 3, 200, 390], [0, 10, 300, 490]), ([0, 400, 400, 400], [0, 900, 900, 900])):
        ends.copy_(i32(e))
        k_ends.copy_(i32(ke))
        out.fill_(7)
        lse.fill_(7)
        g.replay()
        compare(dtype, q, k, v, e, ke, True, out, lse)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_the_same_bits_twice_and_on_two_streams_at_once(D):
    dtype = torch.bfloat16
    q, k, v, ends, _ = problem(26, dtype, 8, 2, D, [2000, 300, 1, 777])
    e = i32(ends)
    first = torch.full_like(q, 7.0)
    api.packed_attention(q, k, v, e, first)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.full_like(q, 7.0) for _ in range(6)] for _ in streams]
    for i in range(6):
        for st, o in zip(streams, outs):
            with torch.cuda.stream(st):
                api.packed_attention(q, k, v, e, o[i])
    torch.cuda.synchronize()
    assert all(torch.equal(first, x) for o in outs for x in o)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_one_sequence_is_what_the_step_kernel_computes(dtype, D):
    H, kvH, n = 4, 2, 700
    q, k, v, ends, _ = problem(27, dtype, H, kvH, D, [n])
    out, lse = run(q, k, v, ends)
    s = api.AttentionShape(1, H, n, n, D, kvH)
    o, m, l = torch.empty(1, H, n, D, device="cuda"), torch.empty(1, H, n, device="cuda"), torch.empty(1, H, n, device="cuda")
    at = api.SegMap.make([0], n)
    api.attention_step_ex(*(x.transpose(0, 1).contiguous()[None] for x in (q, k, v)), o, m, l, s, at, at, causal=True, fresh=True, finalize=True)
    # both are the same sums of rounded weights in another order: each within half a step of dtype on the weights and a few of fp32's
    tol = {torch.float16: 2.0 ** -9, torch.bfloat16: 2.0 ** -6}[dtype]
    assert ((out.transpose(0, 1).float() - o[0]).abs() <= tol * (1 + o[0].abs())).all()
    assert ((lse - api.attention_lse(m, l)[0]).abs() <= 2.0 ** -17 * (1 + lse.abs())).all()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("items", [0, 1, 3])
def test_a_wait_that_runs_out_is_reported_and_leaves_the_rows(D, items):
    dtype = torch.bfloat16
    q, k, v, ends, k_ends = problem(28, dtype, 4, 2, D, [700, 300])
    L = lib()
    api.device_status()
    try:
        L.ra_debug_set_wait_limit_ns(20_000_000)
        L.ra_debug_stall_producer_after(items)
        out, lse = run(q, k, v, ends)
        torch.cuda.synchronize()
        L.ra_debug_stall_producer_after(-1)
        again = run(q, k, v, ends)  # behind the word nothing is written
        torch.cuda.synchronize()
        assert (again[0] == 7).all() and (again[1] == 7).all()
        assert api.device_status()[0] == 5
    finally:
        L.ra_debug_stall_producer_after(-1)
        L.ra_debug_set_wait_limit_ns(0)
        api.device_status()
    # blocks of one key tile are done with two items of the ring; every other row is as it was
    clean = run(q, k, v, ends)
    left = (out == 7).all(-1)
    assert torch.equal(out[~left], clean[0][~left]) and torch.equal(lse.T[~left], clean[1].T[~left]) and (lse.T[left] == 7).all()
    assert left.all() if items < 2 else left.any()
    check(dtype, (q, k, v, ends, k_ends))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_prompts_chunks_and_tokens_out_of_a_cache_in_4_bits(dtype, D):
    """A server's way: prompts by packed attention and into the cache, their next chunks behind the rows read back, then tokens. Every
    result is that of the 64-bit formula on what the cache holds."""
    H, kvH, page, B = 8, 2, 16, 3
    lens, more = np.array([70, 5, 129]), np.array([40, 130, 1])
    table = i32(np.arange(B * 20).reshape(B, 20))
    pages = [api.pages_4bit(B * 20, kvH, page, D) for _ in range(2)]
    q, k, v, ends, _ = problem(29, dtype, H, kvH, D, lens)
    out, lse = run(q, k, v, ends)
    compare(dtype, q, k, v, ends, ends, True, out, lse)

    def padded(x, n):  # packed rows as (batch, heads, rows, head_dim)
        y = torch.zeros(B, x.shape[1], int(max(n)), D, dtype=dtype, device="cuda")
        for b, e in enumerate(ends_of(n)[:-1]):
            y[b, :, :n[b]] = x[int(e):int(e) + int(n[b])].transpose(0, 1)
        return y

    api.paged_append_4bit(padded(k, lens), padded(v, lens), *pages, table, i32([0] * B), counts=i32(lens))
    q, k, v, ends, _ = problem(32, dtype, H, kvH, D, more)
    api.paged_append_4bit(padded(k, more), padded(v, more), *pages, table, i32(lens), counts=i32(more))
    both = lens + more
    k_ends = ends_of(both)
    rows = [torch.empty(int(k_ends[-1]), kvH, D, dtype=dtype, device="cuda") for _ in range(2)]
    api.paged_read_4bit(*pages, table, i32(k_ends), *rows)
    for held, x in zip(rows, (k, v)):  # the chunk's rows are the nearest to what was appended
        for b in range(B):
            codes = four_bit_ref.encode(x[int(ends[b]):int(ends[b + 1])].double().cpu().numpy(), 1.0)
            got = held[int(k_ends[b]) + int(lens[b]):int(k_ends[b + 1])].double().cpu().numpy()
            assert np.array_equal(got, four_bit_ref.decode(*codes, 1.0))
    compare(dtype, q, *rows, ends, k_ends, True, *run(q, *rows, ends, k_ends))
    token = some(35, (B, H, D), dtype)
    o, l = torch.empty_like(token), torch.empty(B, H, device="cuda")
    api.paged_decode_4bit(token, *pages, table, i32(both), o, lse=l)
    compare(dtype, token, *rows, np.arange(B + 1), k_ends, True, o, l.T)
    # and a token is a chunk of one row
    compare(dtype, token, *rows, np.arange(B + 1), k_ends, True, *run(token, *rows, np.arange(B + 1), k_ends))


def test_rows_read_from_a_cache_in_16_bits():
    """Chunks of prompts behind what paged_read brings of a cache that paged_append filled, norms and rotation on the way."""
    dtype, H, kvH, D, page, B = torch.bfloat16, 4, 2, 64, 32, 2
    k, v, q = (some(36 + i, (B, h, 150, D), dtype) for i, h in enumerate((kvH, kvH, H)))
    pages = [torch.zeros(B * 6, kvH, page, D, dtype=dtype, device="cuda") for _ in range(2)]
    table, q_out = i32(np.arange(B * 6).reshape(B, 6)), torch.empty_like(q)
    api.paged_append(k, v, *pages, table, i32([0] * B), rope=api.Rope.make(D), q=q, q_out=q_out)
    rows = [torch.empty(B * 150, kvH, D, dtype=dtype, device="cuda") for _ in range(2)]
    api.paged_read(*pages, table, i32([0, 150, 300]), *rows)
    assert torch.equal(rows[1], v.transpose(1, 2).reshape(300, kvH, D))
    chunk = q_out[:, :, 100:].transpose(1, 2).reshape(100, H, D)
    compare(dtype, chunk, *rows, [0, 50, 100], [0, 150, 300], True, *run(chunk, *rows, [0, 50, 100], [0, 150, 300]))


def test_wrapper_refusals():
    q, k, v, ends, _ = problem(39, torch.float16, 4, 2, 64, [20, 5])
    e, out = i32(ends), torch.empty_like(q)
    for bad in (lambda: api.packed_attention(q.float(), k.float(), v.float(), e, out.float()), lambda: api.packed_attention(q, k.bfloat16(), v, e, out),
                lambda: api.packed_attention(q, k, v[:5], e, out), lambda: api.packed_attention(q, k, v, e.long(), out),
                lambda: api.packed_attention(q, k, v, e, out[:5]), lambda: api.packed_attention(q, k[..., :32], v, e, out),
                lambda: api.packed_attention(q[0], k, v, e, out), lambda: api.packed_attention(q, k, v, e[:0], out),
                lambda: api.packed_attention(q, k, v, e, out, k_ends=e[:2]), lambda: api.packed_attention(q.cpu(), k, v, e, out),
                lambda: api.packed_attention(q, k, v, e, out, lse=torch.empty(25, 4, device="cuda")),
                lambda: api.packed_attention(q, k, v, e, out[:, :1].expand(-1, 4, -1)),
                lambda: api.packed_attention(q, k, v, e, torch.empty(25, 64, 4, dtype=q.dtype, device="cuda").transpose(1, 2))):
        with pytest.raises(ValueError):
            bad()
    three = some(40, (25, 3, 64), torch.float16)
    for bad in (lambda: api.packed_attention(q, three, three, e, out), lambda: api.packed_attention(q, k[:, :1].expand(-1, 2, -1), v, e, out),
                lambda: api.packed_attention(torch.empty(25, 4, 68, dtype=q.dtype, device="cuda")[..., :64], k, v, e, out)):
        with pytest.raises(RingAttentionError):
            bad()


def test_many_places_without_a_sequence():
    """One prompt and 32767 places that have none: no wait comes near a limit of 50 ms while blocks go through what there is not."""
    dtype, H, D, n, B = torch.bfloat16, 8, 64, 300, 32768
    q, k, v, _, _ = problem(53, dtype, H, H, D, [n])
    ends = np.full(B + 1, n)
    ends[0] = 0
    L = lib()
    api.device_status()
    try:
        L.ra_debug_set_wait_limit_ns(50_000_000)
        out, lse = run(q, k, v, ends)
        torch.cuda.synchronize()
        assert api.device_status()[0] == 0
    finally:
        L.ra_debug_set_wait_limit_ns(0)
        api.device_status()
    compare(dtype, q, k, v, [0, n], [0, n], True, out, lse)


@pytest.mark.parametrize("H", [1, 8])
def test_as_many_places_as_a_call_takes(H):
    """2^22 places, of which the first and the last have a prompt: no wait runs out."""
    dtype, D, B = torch.bfloat16, 64, 1 << 22
    q, k, v, _, _ = problem(56, dtype, H, H, D, [300, 70])
    ends = torch.full((B + 1,), 300, dtype=torch.int32, device="cuda")
    ends[0], ends[B] = 0, 370
    out, lse = torch.full_like(q, 7.0), torch.full((H, 370), 7.0, device="cuda")
    api.device_status()
    api.packed_attention(q, k, v, ends, out, lse=lse)
    torch.cuda.synchronize()
    assert api.device_status()[0] == 0
    compare(dtype, q, k, v, [0, 300, 370], [0, 300, 370], True, out, lse)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,kvH,D", [(2, 2, 32), (2, 2, 64), (8, 2, 64), (2, 2, 128), (4, 1, 128), (2, 2, 256)])
@pytest.mark.parametrize("before", [0, 1, 64, 127])
def test_how_far_a_value_that_is_not_finite_reaches(dtype, H, kvH, D, before):
    """Queries that see it, and none that is 255 keys or more before it."""
    n, at = 900, 700
    q, k, v, ends, k_ends = problem(59, dtype, H, kvH, D, [n], [n + before])
    clean = run(q, k, v, ends, k_ends)
    v = v.clone()
    v[at, 0, 3] = float("inf")
    out, lse = run(q, k, v, ends, k_ends)
    assert torch.equal(lse, clean[1])
    assert kvH == 1 or torch.equal(out[:, 1::kvH], clean[0][:, 1::kvH])
    first = at - before  # the first query that sees it
    assert not torch.isfinite(out[first:, ::kvH, 3]).any()
    keep = torch.arange(D, device="cuda") != 3
    assert torch.equal(out[..., keep], clean[0][..., keep])
    assert torch.equal(out[:first - 254], clean[0][:first - 254])
