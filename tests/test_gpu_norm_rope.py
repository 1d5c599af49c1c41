"""Norms of queries and keys with the position rotation, forward and backward, against the formulas in 64 bits: types, head
sizes, pairings, layouts of a ring's shards, strides and alignment, rows that nothing may touch."""
import numpy as np
import pytest
import torch

from norm_rope_ref import backward, check, default_freqs, forward, rounded
from ring_attention_b200 import api
from ring_attention_b200._lib import lib

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def inputs(seed, B, heads, S, D, dtype, scale=1.7):
    return rounded(np.random.default_rng(seed).standard_normal((B, heads, S, D)) * scale, dtype)


def weight(seed, D, dtype):
    return rounded(1 + 0.3 * np.random.default_rng(seed).standard_normal(D), dtype)


def gpu(x, dtype):
    return torch.from_numpy(np.ascontiguousarray(x)).to(dtype).cuda()


def token_major(x, dtype):
    """The same values as a projection leaves them: (batch, seq, heads, head_dim) in memory."""
    return gpu(x.transpose(0, 2, 1, 3), dtype).transpose(1, 2)


def chain_of(B, S, heads):
    """The most additions that a term of a weight's gradient goes through: a lane's walk over tokens and heads, a warp's rows,
    eight warps, the blocks' list in eight slices."""
    blocks = lib().ra_qk_norm_rope_backward_workspace_bytes(32) // (2 * 32 * 4)
    return -(-B * S // (8 * blocks)) * heads + 3 + 8 + -(-blocks // 8) + 8


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,rot,interleaved,norm", [(32, 32, False, True), (32, 16, True, True), (64, 64, False, False),
                                                    (64, 32, False, True), (128, 128, False, True), (128, 96, False, True),
                                                    (128, 48, True, False), (256, 256, False, True), (256, 128, True, True),
                                                    (256, 16, False, True), (128, 0, False, True)])
@pytest.mark.parametrize("B,H,kvH,S", [(1, 1, 1, 1), (2, 3, 1, 5), (3, 12, 4, 67), (1, 9, 9, 33), (64, 32, 8, 1)])
def test_forward_and_backward(dtype, D, rot, interleaved, norm, B, H, kvH, S):
    rope = api.Rope.make(rot, base=500000.0, interleaved=interleaved) if rot else None
    freqs = default_freqs(rot, 500000.0)
    q, k = inputs(1, B, H, S, D, dtype), inputs(2, B, kvH, S, D, dtype, 0.6)
    wq, wk = (weight(3, D, dtype), weight(4, D, dtype)) if norm else (None, None)
    pos = np.broadcast_to(np.arange(S) + 40000, (B, 1, S))
    seg = api.SegMap.make([40000], S)
    how = dict(q_weight=gpu(wq, dtype) if norm else None, k_weight=gpu(wk, dtype) if norm else None, eps=1e-5, rope=rope, segmap=seg)
    dq, dk = gpu(q, dtype), token_major(k, dtype)
    q_out, k_out = torch.full_like(dq, float("nan")), torch.full((B, kvH, S, D), float("nan"), dtype=dtype, device="cuda")
    api.qk_norm_rope(dq, dk, q_out, k_out, **how)
    for got, x, w in ((q_out, q, wq), (k_out, k, wk)):
        check(got, *forward(x, w, pos, rot, interleaved, freqs, np.float32(1e-5)), dtype, "forward")
    # backward
    gq, gk = inputs(5, B, H, S, D, dtype), inputs(6, B, kvH, S, D, dtype)
    rq, rk = torch.full_like(q_out, float("nan")), torch.full_like(k_out, float("nan"))
    dwq, dwk = (torch.full((D,), float("nan"), device="cuda") if norm else None for _ in range(2))
    api.qk_norm_rope_backward(dq, dk, token_major(gq, dtype), gpu(gk, dtype), rq, rk, dq_weight=dwq, dk_weight=dwk, **how)
    for got, dw, x, w, g, h in ((rq, dwq, q, wq, gq, H), (rk, dwk, k, wk, gk, kvH)):
        dx, dx_err, want, err = backward(x, w, g, pos, rot, interleaved, freqs, np.float32(1e-5), chain_of(B, S, h))
        check(got, dx, dx_err, dtype, "dx")
        if norm:
            check(dw, want, err, torch.float32, "dw")


@pytest.mark.parametrize("dtype,D,rot,interleaved,S,w_dtype", [
    (torch.bfloat16, 128, 128, False, 2001, torch.bfloat16), (torch.float32, 128, 96, False, 2001, torch.float32),
    (torch.float16, 32, 32, True, 6667, torch.float32), (torch.bfloat16, 64, 32, True, 3335, torch.float32),
    (torch.bfloat16, 256, 256, False, 1003, torch.float32), (torch.float32, 256, 64, True, 1003, torch.float32)])
def test_walks_over_many_tokens_and_heads(dtype, D, rot, interleaved, S, w_dtype):
    """So many tokens that a warp takes more heads than it has on their way at once, and in the backward pass several units one
    after the other; 13 and 4 heads are no multiple of what it takes, so that some have heads of both sides; the last
    warp has lanes without a token."""
    B, H, kvH = 3, 13, 4
    rope, freqs = api.Rope.make(rot, interleaved=interleaved), default_freqs(rot)
    q, k = inputs(1, B, H, S, D, dtype), inputs(2, B, kvH, S, D, dtype, 0.6)
    wq, wk = weight(3, D, w_dtype), weight(4, D, w_dtype)
    pos = np.broadcast_to(np.arange(S) * 3 + 7, (B, 1, S))
    how = dict(q_weight=gpu(wq, w_dtype), k_weight=gpu(wk, w_dtype), eps=1e-5, rope=rope, segmap=api.SegMap.make([7], S), pos_stride=3)
    dq, dk = token_major(q, dtype), gpu(k, dtype)
    q_out, k_out = (torch.full((B, h, S, D), float("nan"), dtype=dtype, device="cuda") for h in (H, kvH))
    api.qk_norm_rope(dq, dk, q_out, k_out, **how)
    for got, x, w in ((q_out, q, wq), (k_out, k, wk)):
        check(got, *forward(x, w, pos, rot, interleaved, freqs, np.float32(1e-5)), dtype, "forward")
    gq, gk = inputs(5, B, H, S, D, dtype), inputs(6, B, kvH, S, D, dtype)
    rq, rk = torch.full_like(q_out, float("nan")), torch.full_like(k_out, float("nan"))
    dwq, dwk = (torch.full((D,), float("nan"), device="cuda") for _ in range(2))
    api.qk_norm_rope_backward(dq, dk, gpu(gq, dtype), token_major(gk, dtype), rq, rk, dq_weight=dwq, dk_weight=dwk, **how)
    for got, dw, x, w, g, h in ((rq, dwq, q, wq, gq, H), (rk, dwk, k, wk, gk, kvH)):
        dx, dx_err, want, err = backward(x, w, g, pos, rot, interleaved, freqs, np.float32(1e-5), chain_of(B, S, h))
        check(got, dx, dx_err, dtype, "dx")
        check(dw, want, err, torch.float32, "dw")

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout,cp,n_splits", [(0, 2, 2), (1, 2, 2), (1, 4, 4), (2, 4, 2)])
def test_positions_of_a_rings_shards(dtype, layout, cp, n_splits):
    """Every rank's shard, with the maps that its ring steps take, gives the rows of the whole sequence."""
    H, kvH, D, seq = 4, 2, 64, 208
    q, k = inputs(1, 1, H, seq, D, dtype), inputs(2, 1, kvH, seq, D, dtype)
    rope, freqs = api.Rope.make(D), default_freqs(D)
    for rank in range(cp):
        part = api.RingPartition(cp, rank, seq, layout, n_splits)
        qmap, _, stride = part.step_maps(0)
        at = part.local_positions().numpy()
        dq, dk = gpu(q[:, :, at], dtype), gpu(k[:, :, at], dtype)
        api.qk_norm_rope(dq, dk, dq, dk, rope=rope, segmap=qmap, pos_stride=stride)  # in place
        for got, x in ((dq, q), (dk, k)):
            check(got, *forward(x[:, :, at], None, at[None, None], D, False, freqs, 0), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_positions_from_a_tensor(dtype, interleaved):
    B, H, S, D = 3, 5, 7, 128
    x = inputs(1, B, H, S, D, dtype)
    pos = np.random.default_rng(2).integers(-(2 ** 31), 2 ** 31, (B, S))
    pos[0, :3] = (2 ** 31 - 1, -(2 ** 31), 0)
    rope = api.Rope.make(D, interleaved=interleaved)
    # in the frequencies that the table holds: at these positions those of the formula are off by more than a step
    freqs = np.array([rope.turns[i] for i in range(D // 2)], dtype=np.longdouble) / np.longdouble(2.0) ** 64
    turns = (pos[..., None].astype(np.longdouble) * freqs) % 1
    table = torch.full((B, S + 3), 0, dtype=torch.int32, device="cuda")
    table[:, :S] = torch.from_numpy(pos.astype(np.int32))
    q = gpu(x, dtype)
    out = torch.empty_like(q)
    api.qk_norm_rope(q, None, out, None, rope=rope, positions=table[:, :S])
    want = np.zeros_like(x)
    err = np.zeros_like(x)
    for b in range(B):
        for s in range(S):
            # one turn of 2 pi t: the angle as a position 1 with that frequency
            y, e = forward(x[b, :, s], None, 1, D, interleaved, (turns[b, s] * 2 * np.longdouble(np.pi)).astype(np.float64), 0)
            want[b, :, s], err[b, :, s] = y, e
    check(out, want, err, dtype)
    one = torch.empty_like(q)
    api.qk_norm_rope(q, None, one, None, rope=rope, positions=table[1, :S].contiguous())  # the same for every sequence
    assert torch.equal(one[1], out[1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,off", [(32, 1), (64, 3), (128, 1), (256, 1)])
def test_rows_that_are_not_aligned(dtype, D, off):
    """Views that begin at odd elements and rows an odd number of elements apart; what lies between the rows stays."""
    B, H, kvH, S = 2, 3, 2, 9
    q, k = inputs(1, B, H, S, D, dtype), inputs(2, B, kvH, S, D, dtype)
    w = weight(3, D, dtype)
    rope, freqs = api.Rope.make(D), default_freqs(D)

    def odd(x):
        flat = torch.full((x.shape[0] * x.shape[1] * x.shape[2] * (D + off) + off,), 7.0, dtype=dtype, device="cuda")
        v = flat[off:].view(x.shape[0], x.shape[1], x.shape[2], D + off)[..., :D]
        v.copy_(gpu(x, dtype))
        return flat, v

    (_, dq), (_, dk) = odd(q), odd(k)
    (fq, oq), (_, ok) = odd(q * 0), odd(k * 0)
    api.qk_norm_rope(dq, dk, oq, ok, q_weight=gpu(w, dtype), k_weight=gpu(w, dtype), rope=rope)
    pos = np.arange(S)
    for got, x in ((oq, q), (ok, k)):
        check(got, *forward(x, w, pos, D, False, freqs, np.float32(1e-6)), dtype)
    gaps = fq[off:].view(B, H, S, D + off)[..., D:]
    assert (gaps == 7).all() and (fq[:off] == 7).all()
    gq, gk = odd(inputs(5, B, H, S, D, dtype)), odd(inputs(6, B, kvH, S, D, dtype))
    rq, rk = odd(q * 0)[1], odd(k * 0)[1]
    dwq, dwk = torch.empty(D, device="cuda"), torch.empty(D, device="cuda")
    api.qk_norm_rope_backward(dq, dk, gq[1], gk[1], rq, rk, dq_weight=dwq, dk_weight=dwk, q_weight=gpu(w, dtype),
                              k_weight=gpu(w, dtype), rope=rope)
    for got, dw, x, g in ((rq, dwq, q, gq[1]), (rk, dwk, k, gk[1])):
        dx, e, want, err = backward(x, w, g.double().cpu().numpy(), pos, D, False, freqs, np.float32(1e-6),
                                    chain_of(B, S, x.shape[1]))
        check(got, dx, e, dtype)
        check(dw, want, err, torch.float32)


def test_broadcast_rows_and_one_side_alone():
    """Keys that all batches share (a stride of zero) come out once a batch; with one side absent the other is the same."""
    B, H, S, D = 3, 4, 11, 64
    q, k = torch.randn(B, H, S, D, device="cuda"), torch.randn(1, 2, S, D, device="cuda").expand(B, -1, -1, -1)
    w = 1 + torch.rand(D, device="cuda")
    rope = api.Rope.make(D)
    qo, ko = torch.empty_like(q), torch.empty(B, 2, S, D, device="cuda")
    api.qk_norm_rope(q, k, qo, ko, q_weight=w, k_weight=w, rope=rope)
    assert torch.equal(ko[0], ko[1]) and torch.equal(ko[0], ko[2])
    for a, b, n in ((q, qo, "q"), (k, ko, "k")):
        alone = torch.empty_like(b)
        args = (a, None, alone, None) if n == "q" else (None, a, None, alone)
        api.qk_norm_rope(*args, **{n + "_weight": w}, rope=rope)
        assert torch.equal(alone, b)
    dy = torch.randn_like(ko)
    dk, dw = torch.empty_like(dy), torch.empty(D, device="cuda")
    api.qk_norm_rope_backward(None, k, None, dy, None, dk, dk_weight=dw, k_weight=w, rope=rope)
    x = k.double().cpu().numpy()
    dx, e, want, err = backward(x, w.double().cpu().numpy(), dy.double().cpu().numpy(), np.arange(S), D, False, default_freqs(D),
                                np.float32(1e-6), chain_of(B, S, 2))
    check(dk, dx, e, torch.float32)
    check(dw, want, err, torch.float32)


def test_gradients_of_one_side_with_the_rows_of_both():
    """One of q and k needs no gradient: its rows and weight go in as in the forward call and change nothing."""
    B, H, kvH, S, D = 2, 6, 2, 9, 64
    q, k = torch.randn(B, H, S, D, device="cuda"), torch.randn(B, kvH, S, D, device="cuda")
    w, rope = {n + "_weight": 1 + torch.rand(D, device="cuda") for n in "qk"}, api.Rope.make(D)
    for x, n in ((q, "q"), (k, "k")):
        dy = torch.randn_like(x)
        got = []
        for both in (False, True):
            dx, dw = torch.empty_like(x), torch.empty(D, device="cuda")
            rows = (q, k) if both else (q, None) if n == "q" else (None, k)
            args = (dy, None, dx, None) if n == "q" else (None, dy, None, dx)
            how = w if both else {n + "_weight": w[n + "_weight"]}
            api.qk_norm_rope_backward(*rows, *args, **{f"d{n}_weight": dw}, **how, rope=rope)
            got.append((dx, dw))
        assert all(torch.equal(a, b) for a, b in zip(*got))
    with pytest.raises(ValueError):
        api.qk_norm_rope_backward(q, k, None, None, None, None, **w, rope=rope)

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_fp32_weights_of_16_bit_rows(dtype):
    B, H, S, D = 2, 4, 6, 128
    x, w = inputs(1, B, H, S, D, dtype), weight(2, D, torch.float32)
    q = gpu(x, dtype)
    out = torch.empty_like(q)
    api.qk_norm_rope(q, None, out, None, q_weight=gpu(w, torch.float32))
    check(out, *forward(x, w, np.zeros(S), 0, False, [], np.float32(1e-6)), dtype)


def test_rows_of_zeros_and_what_is_not_finite():
    D = 64
    x = torch.zeros(1, 1, 4, D, device="cuda")
    x[0, 0, 1] = float("inf")
    x[0, 0, 2, 5] = float("nan")
    x[0, 0, 3, 40] = float("inf")  # behind the elements that turn
    out, rope = torch.empty_like(x), api.Rope.make(32)
    api.qk_norm_rope(x, None, out, None, q_weight=torch.ones(D, device="cuda"), rope=rope)
    assert (out[0, 0, 0] == 0).all() and out[0, 0, 1].isnan().all() and out[0, 0, 2].isnan().all()
    api.qk_norm_rope(x, None, out, None, rope=rope)  # without a norm: only the pairs that hold it
    assert out[0, 0, 3, 40].isposinf() and (out[0, 0, 3, :40] == 0).all() and (out[0, 0, 3, 41:] == 0).all()
    assert out[0, 0, 2].isnan().nonzero().flatten().tolist() == [5, 21]
    dx, dw = torch.empty_like(x), torch.empty(D, device="cuda")
    api.qk_norm_rope_backward(x[:, :, :1], None, torch.ones_like(x[:, :, :1]), None, dx[:, :, :1], None, dq_weight=dw,
                              q_weight=torch.ones(D, device="cuda"), rope=rope)
    assert dx[0, 0, 0].isfinite().all() and (dw == 0).all()


def test_no_rows():
    D = 128
    e = torch.empty(2, 4, 0, D, device="cuda", dtype=torch.float16)
    api.qk_norm_rope(e, e, e, e, rope=api.Rope.make(D))
    dw, w = torch.full((D,), 5.0, device="cuda"), torch.ones(D, device="cuda", dtype=torch.float16)
    api.qk_norm_rope_backward(e, e, e, e, e, e, dq_weight=dw, q_weight=w, k_weight=w)
    assert (dw == 0).all()


def test_backward_gives_the_same_bits_and_follows_differences():
    """The gradient of a loss in the kernels' own forward pass: its difference along a direction, in fp32 with steps that the
    rounding of the loss (2^-24 of the sum of its terms' magnitudes, over the step) allows."""
    B, H, S, D = 2, 3, 50, 64
    gen = torch.Generator(device="cuda").manual_seed(3)
    x, dy, a = (torch.randn(B, H, S, D, device="cuda", generator=gen) for _ in range(3))
    w, aw = (torch.randn(D, device="cuda", generator=gen) for _ in range(2))
    rope = api.Rope.make(D)
    dx, dw, again = torch.empty_like(x), torch.empty(D, device="cuda"), torch.empty(D, device="cuda")
    for out in (dw, again):
        api.qk_norm_rope_backward(x, None, dy, None, dx, None, dq_weight=out, q_weight=w, rope=rope)
    assert torch.equal(dw, again)

    def value(x, w):
        y = torch.empty_like(x)
        api.qk_norm_rope(x, None, y, None, q_weight=w, rope=rope)
        return (y.double() * dy.double()).sum().item(), (y.double() * dy.double()).abs().sum().item()

    h = 2.0 ** -8
    up, size = value(x + h * a, w + h * aw)
    down, _ = value(x - h * a, w - h * aw)
    want = (dx.double() * a.double()).sum().item() + (dw.double() * aw.double()).sum().item()
    # inputs x +- h a are rounded (2^-24 of a loss's terms), results to 18 u of theirs; the third derivative of x / rms along a
    # direction of unit elements is below 8 times the loss's terms in sum of magnitudes
    tol = 2 * 20 * 2.0 ** -24 * size / (2 * h) + 8 * size * h * h
    assert abs((up - down) / (2 * h) - want) <= tol


def test_captured_and_replayed_on_another_stream():
    B, H, S, D = 2, 6, 33, 128
    q, k = (torch.randn(B, h, S, D, device="cuda").bfloat16() for h in (H, 2))
    w, rope = torch.rand(D, device="cuda").bfloat16() + 0.5, api.Rope.make(D)
    qo, ko, dq, dk = (torch.empty_like(t) for t in (q, k, q, k))
    dw = torch.empty(D, device="cuda")

    def both():
        api.qk_norm_rope(q, k, qo, ko, q_weight=w, k_weight=w, rope=rope)
        api.qk_norm_rope_backward(q, k, qo, ko, dq, dk, dq_weight=dw, q_weight=w, k_weight=w, rope=rope)

    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=side):
        both()
    for seed in (1, 2):
        q.copy_(torch.randn(B, H, S, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)))
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (qo, ko, dq, dk, dw)]
        both()
        assert all(torch.equal(x, y) for x, y in zip(got, (qo, ko, dq, dk, dw)))


def test_wrapper_refusals():
    q = torch.zeros(1, 2, 3, 64, device="cuda")
    o = torch.empty_like(q)
    for call in (lambda: api.qk_norm_rope(q, None, None, None), lambda: api.qk_norm_rope(None, None, None, None),
                 lambda: api.qk_norm_rope(q, None, o.half(), None), lambda: api.qk_norm_rope(q, None, o[:, :, :2], None),
                 lambda: api.qk_norm_rope(q, None, o.cpu(), None), lambda: api.qk_norm_rope(q.double(), None, o.double(), None),
                 lambda: api.qk_norm_rope(q, None, o[:, :, :1].expand(-1, -1, 3, -1), None),
                 lambda: api.qk_norm_rope(q.transpose(2, 3), None, o.transpose(2, 3), None),
                 lambda: api.qk_norm_rope(q, None, o, None, q_weight=torch.ones(64, device="cuda").half()),
                 lambda: api.qk_norm_rope(q, None, o, None, q_weight=torch.ones(32, device="cuda")),
                 lambda: api.qk_norm_rope(q, None, o, None, rope=api.Rope.make(64), positions=torch.zeros(1, 3, device="cuda")),
                 lambda: api.qk_norm_rope(q, None, o, None, rope=api.Rope.make(64),
                                          positions=torch.zeros(1, 2, dtype=torch.int32, device="cuda")),
                 lambda: api.qk_norm_rope_backward(q, None, q, None, None, None),
                 lambda: api.qk_norm_rope_backward(q, None, q, None, o, None, q_weight=torch.ones(64, device="cuda"),
                                                   dq_weight=torch.ones(64, device="cuda").half())):
        with pytest.raises(ValueError):
            call()
