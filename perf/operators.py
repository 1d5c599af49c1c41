"""The operators around attention that serving and training with this library calls, case by case: norms of queries and keys
with the position rotation (forward and backward), appending to a paged KV cache, decoding against one, and decoding a batch
whose sequences share a long prefix.

``own`` false computes the plain form in torch, true calls the library. Lengths of a batch are fixed by the case, and which
sequence has which is drawn from the seed, so that ``work`` can count them.
"""
import functools
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
EPS = 1e-6


# ---- cases ---------------------------------------------------------------------------------------


def rows_case(kind, dtype, batch, heads, kv_heads, seq, head_dim, rot_dim, norm=True, interleaved=False, base=10000.0, cp=1,
              rank=0, layout="contiguous", token_major=False, name=None):
    c = {"kind": kind, "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads, "seq": seq, "head_dim": head_dim,
         "rot_dim": rot_dim, "norm": norm, "interleaved": interleaved, "base": base, "cp": cp, "rank": rank,
         "layout": layout, "token_major": token_major}
    return {"name": name, **c} if name else c


def append_case(dtype, batch, heads, kv_heads, most_before, tokens, head_dim, rot_dim, page_size, norm=True,
                interleaved=False, base=10000.0, name=None):
    c = {"kind": "append", "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads, "most_before": most_before,
         "tokens": tokens, "head_dim": head_dim, "rot_dim": rot_dim, "page_size": page_size, "norm": norm,
         "interleaved": interleaved, "base": base}
    return {"name": name, **c} if name else c


def decode_case(kind, dtype, batch, heads, kv_heads, most, head_dim, page_size, ragged=0.5, pad=0, shared=0, name=None):
    c = {"kind": kind, "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads, "most": most,
         "head_dim": head_dim, "page_size": page_size, "ragged": ragged, "pad": pad, "shared": shared}
    return {"name": name, **c} if name else c


def listed():
    return [
        # the new tokens of a small batch, straight from a fused projection: latency
        rows_case("norm_rope", "bf16", 16, 32, 8, 1, 128, 128, token_major=True, name="norm_rope_tokens"),
        # one rank of four of a long striped prompt, before its ring pass
        rows_case("norm_rope", "bf16", 1, 32, 8, 32768, 128, 128, base=500000.0, cp=4, rank=1, layout="striped",
                  token_major=True, name="norm_rope_prompt"),
        # a training step's backward of a small ragged batch, fp32, half of each head rotated, neighbours paired
        rows_case("norm_rope_backward", "fp32", 2, 12, 4, 1531, 64, 32, interleaved=True, name="norm_rope_bwd_ragged"),
        # the same of a long context under the zig-zag layout
        rows_case("norm_rope_backward", "bf16", 1, 16, 16, 32768, 128, 128, base=500000.0, cp=2, rank=1, layout="zigzag",
                  name="norm_rope_bwd_long"),
        # a decode step's new rows of every sequence into the cache
        append_case("bf16", 64, 32, 8, 100, 1, 128, 128, 16, name="append_tokens"),
        # chunks of four prompts, of unlike lengths
        append_case("fp16", 4, 32, 8, 500, 4099, 128, 128, 64, norm=False, name="append_chunks"),
        # a small batch on chat-sized contexts, two padded places of a fixed batch among them
        decode_case("decode", "bf16", 7, 24, 6, 1531, 64, 16, pad=2, name="decode_short"),
        # fp32 cache, few sequences, a head of its own for every query head
        decode_case("decode", "fp32", 3, 8, 8, 16384, 128, 32, name="decode_fp32"),
        # long contexts: the benchmark's decode workload out of pages and with unlike lengths
        decode_case("decode", "fp16", 4, 32, 8, 262144, 128, 64, name="decode_long"),
        # a few requests behind a short common prompt
        decode_case("shared", "fp16", 8, 24, 6, 2300, 64, 16, ragged=0.1, shared=2048, name="shared_short"),
        # requests behind a long common document
        decode_case("shared", "bf16", 32, 32, 8, 33333, 128, 64, ragged=0.015, shared=32768, name="shared_long"),
        # a full batch behind a long system prompt
        decode_case("shared", "bf16", 256, 32, 8, 17000, 128, 16, ragged=0.03, shared=16384, name="shared_wide"),
    ]


def _spread(rng, lo, hi):
    """A whole number, even over the logarithm of the range."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng, most):
    kv = rng.choice([k for k in (1, 2, 3, 4, 6, 8, 16) if k <= most])
    group = rng.choice([g for g in (1, 2, 3, 4, 6, 8, 16) if g * kv <= most])
    return kv * group, kv


def draw(rng):
    while True:
        kind = rng.choice(["norm_rope", "norm_rope_backward", "append", "decode", "decode", "shared", "shared"])
        dtype = rng.choice(["bf16", "fp16", "bf16", "fp16", "fp32"])
        D = rng.choice([32, 64, 128, 128, 256])
        heads, kv_heads = _heads(rng, 64)
        rot = rng.choice([D, D, D // 2])
        page = rng.choice([16, 16, 32, 64, 128, 256])
        if kind in ("norm_rope", "norm_rope_backward"):
            batch, seq = _spread(rng, 1, 64), _spread(rng, 1, 65536)
            layout = rng.choice(["contiguous", "zigzag", "striped"])
            if layout == "zigzag":
                seq += seq % 2
            cp = rng.choice([1, 2, 4, 8])
            c = rows_case(kind, dtype, batch, heads, kv_heads, seq, D, rot, rng.random() < 0.7, rng.random() < 0.3,
                          rng.choice([10000.0, 500000.0]), cp, rng.randrange(cp), layout, rng.random() < 0.5)
            if batch * seq * (heads + kv_heads) * D <= 32768 * 32 * 128:
                return c
        elif kind == "append":
            batch, tokens = _spread(rng, 1, 256), rng.choice([1, _spread(rng, 1, 8192)])
            before = _spread(rng, 1, 2000)
            c = append_case(dtype, batch, heads, kv_heads, before, tokens, D, rot, page, rng.random() < 0.5, rng.random() < 0.3,
                            rng.choice([10000.0, 500000.0]))
            if batch * (tokens + before + page) * (heads + kv_heads) * D <= 4 * 4700 * 40 * 128:
                return c
        elif kind == "decode":
            batch, most = _spread(rng, 1, 256), _spread(rng, 1, 262144)
            c = decode_case(kind, dtype, batch, heads, kv_heads, most, D, page, rng.choice([0.0, 0.5, 0.9]),
                            rng.choice([0, 0, batch // 4]))
            if batch * (most + page) * heads * D * (16 if dtype == "fp32" else 8) <= 262144 * 32 * 128 * 4:
                return c
        else:
            batch, shared = _spread(rng, 2, 256), page * _spread(rng, 1, 65536 // page)
            tail = _spread(rng, 1, 1000)
            c = decode_case(kind, dtype, batch, heads, kv_heads, shared + tail, D, page, min(0.9, tail / (shared + tail)),
                            rng.choice([0, 0, batch // 4]), shared)
            if batch * heads * (shared + 4 * tail) * D * (8 if dtype == "fp32" else 2) <= 256 * 32 * 16384 * 128:
                return c


# ---- inputs --------------------------------------------------------------------------------------


def _lengths(c):
    """The lengths of a decode batch, longest first, padded places (no keys) last."""
    n = c["batch"] - c["pad"]
    low = 0.6180339887498949
    return [max(1, int(c["most"] * (1.0 - c["ragged"] * ((i * low) % 1.0)))) for i in range(n)] + [0] * c["pad"]


def _before(c):
    """(tokens cached, tokens that come) of every sequence of an append."""
    low = 0.6180339887498949
    return [(int(c["most_before"] * ((i * low) % 1.0)), max(1, int(c["tokens"] * (1.0 - 0.5 * ((i * low * low) % 1.0)))))
            for i in range(c["batch"])]


def _pages_of(lengths, page):
    return [-(-n // page) for n in lengths]


def _table(g, counts, num_pages, width):
    """Page numbers in random order, -1 behind a sequence's last page."""
    free = torch.randperm(num_pages, generator=g, device="cuda")
    table = torch.full((len(counts), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = free[at:at + n].int()
        at += n
    return table


def _strided(g, c, heads, seq):
    """Rows of every head, (batch, heads, seq, head_dim): contiguous, or as a projection leaves them, token by token."""
    B, D, dt = c["batch"], c["head_dim"], DTYPES[c["dtype"]]
    if c.get("token_major", True):
        return torch.randn((B, seq, heads, D), generator=g, device="cuda", dtype=dt).transpose(1, 2)
    return torch.randn((B, heads, seq, D), generator=g, device="cuda", dtype=dt)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, H, kvH, D, dt = c["batch"], c["heads"], c["kv_heads"], c["head_dim"], DTYPES[c["dtype"]]
    s = {"c": c}
    if c.get("norm"):
        for n in ("q", "k"):
            s["w" + n] = (1 + 0.3 * torch.randn(D, generator=g, device="cuda")).to(dt)
    if c["kind"] in ("norm_rope", "norm_rope_backward"):
        S = c["seq"]
        # a projection's outputs are not of unit size
        s["q"], s["k"] = _strided(g, c, H, S).mul_(1.7), _strided(g, c, kvH, S).mul_(0.6)
        s["q_out"], s["k_out"] = (torch.zeros((B, h, S, D), device="cuda", dtype=dt) for h in (H, kvH))
        if c["kind"] == "norm_rope_backward":
            s["dq_out"], s["dk_out"] = (torch.randn((B, h, S, D), generator=g, device="cuda", dtype=dt) for h in (H, kvH))
            s["dwq"], s["dwk"] = (torch.zeros(D, device="cuda") for _ in range(2))
        return s
    page = c["page_size"]
    if c["kind"] == "append":
        T = c["tokens"]
        both = [_before(c)[i] for i in torch.randperm(B, generator=g, device="cuda").tolist()]
        counts = _pages_of([n + t for n, t in both], page)
        num_pages = sum(counts) + 3
        s["lens"] = torch.tensor([n for n, _ in both], dtype=torch.int32, device="cuda")
        s["counts"] = torch.tensor([t for _, t in both], dtype=torch.int32, device="cuda")
        s["table"] = _table(g, counts, num_pages, max(counts) + 1)
        s["q"], s["k"], s["v"] = (_strided(g, c, h, T) for h in (H, kvH, kvH))
        s["q_out"] = torch.zeros((B, H, T, D), device="cuda", dtype=dt)
    else:
        lens = [_lengths(c)[i] for i in torch.randperm(B, generator=g, device="cuda").tolist()]
        first = c["shared"] // page
        counts = _pages_of([max(0, n - c["shared"]) for n in lens], page)
        num_pages = sum(counts) + first + 3
        table = _table(g, [first] + counts, num_pages, max(1, max(counts), first))
        s["shared_pages"] = table[0, :first].contiguous()
        s["table"] = torch.full((B, first + max(1, max(counts))), -1, dtype=torch.int32, device="cuda")
        s["table"][:, first:] = table[1:, :max(1, max(counts))]
        there = torch.tensor([n > 0 for n in lens], device="cuda")
        s["table"][:, :first] = torch.where(there[:, None], s["shared_pages"][None], -1)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["q"] = torch.randn((B, H, D), generator=g, device="cuda", dtype=dt)
        s["out"] = torch.zeros((B, H, D), device="cuda", dtype=dt)
        s["lse"] = torch.zeros((B, H), device="cuda")
    for n in ("k_pages", "v_pages"):
        s[n] = torch.randn((num_pages, kvH, page, D), generator=g, device="cuda", dtype=dt)
    return s


def _segments(c):
    """(first position of each segment, rows of a segment, step between rows) of a rank's shard."""
    cp, r, S = c["cp"], c["rank"], c["seq"]
    if c["layout"] == "striped":
        return [r], S, cp
    if c["layout"] == "zigzag":
        return [r * (S // 2), (2 * cp - 1 - r) * (S // 2)], S // 2, 1
    return [r * S], S, 1


# ---- plain form ----------------------------------------------------------------------------------


def _row_positions(c):
    bases, n, step = _segments(c)
    return (torch.tensor(bases, device="cuda")[:, None] + torch.arange(n, device="cuda")[None] * step).reshape(-1)


def _cos_sin(c, positions):
    """cos and sin of every position's angles, (..., rot_dim / 2); the angles in 64 bits."""
    R = c["rot_dim"]
    freqs = c["base"] ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R)
    a = positions.double()[..., None] * freqs
    return a.cos().float(), a.sin().float()


def _rotate(c, x, cos, sin):
    R = c["rot_dim"]
    if c["interleaved"]:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return turned if R == x.shape[-1] else torch.cat((turned, x[..., R:]), -1)


def _norm_rotate(c, x, w, cos, sin):
    y = x.float()
    if w is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w.float()
    return _rotate(c, y, cos, sin)


def _norm_rotate_backward(c, x, w, dy, cos, sin):
    g = _rotate(c, dy.float(), cos, -sin)
    if w is None:
        return g, None
    x = x.float()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    n = x * r
    dw = (g * n).sum((0, 1, 2), dtype=torch.float64).float()
    g = g * w.float()
    return r * (g - n * (g * n).mean(-1, keepdim=True)), dw


def _plain_rows(s):
    c = s["c"]
    cos, sin = _cos_sin(c, _row_positions(c))
    if c["kind"] == "norm_rope":
        return {n: _norm_rotate(c, s[n], s.get("w" + n), cos, sin).to(s[n].dtype) for n in ("q", "k")}
    dq, dwq = _norm_rotate_backward(c, s["q"], s.get("wq"), s["dq_out"], cos, sin)
    dk, dwk = _norm_rotate_backward(c, s["k"], s.get("wk"), s["dk_out"], cos, sin)
    return {"dq": dq.to(s["q"].dtype), "dk": dk.to(s["k"].dtype), "dwq": dwq, "dwk": dwk}


def _plain_append(s):
    c = s["c"]
    B, T, page = c["batch"], c["tokens"], c["page_size"]
    t = torch.arange(T, device="cuda")[None].expand(B, T)
    valid = t < s["counts"][:, None]
    slots = s["lens"][:, None] + t
    cos, sin = (x[:, None] for x in _cos_sin(c, slots))
    k = _norm_rotate(c, s["k"], s.get("wk"), cos, sin).to(s["k"].dtype)
    q = _norm_rotate(c, s["q"], s.get("wq"), cos, sin).to(s["q"].dtype)
    q = torch.where(valid[:, None, :, None], q, torch.zeros((), dtype=q.dtype, device="cuda"))
    # a row that does not come stands for its sequence's last one, which is then written twice
    last = torch.minimum(t, s["counts"][:, None].long() - 1)
    slots = s["lens"][:, None] + last
    pages = s["table"].gather(1, slots // page).long()
    at = last[:, None, :, None].expand(B, c["kv_heads"], T, c["head_dim"])
    s["k_pages"][pages, :, slots % page] = k.gather(2, at).transpose(1, 2)
    s["v_pages"][pages, :, slots % page] = s["v"].gather(2, at).transpose(1, 2)
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"], "q": q}


def _gather(pages, table):
    """(batch, kv heads, keys, head_dim) of the pages that a table names."""
    x = pages[table.clamp_min(0).long()].float()  # (batch, pages, kv heads, page, head_dim)
    return x.transpose(1, 2).flatten(2, 3)


def _plain_decode(s):
    c = s["c"]
    B, H, kvH, D, P = c["batch"], c["heads"], c["kv_heads"], c["head_dim"], c["shared"]
    q = s["q"].float().view(B, H // kvH, kvH, D).transpose(1, 2) / math.sqrt(D)  # query head h reads KV head h % kvH
    own_pages = s["table"][:, P // c["page_size"]:]
    k, v = _gather(s["k_pages"], own_pages), _gather(s["v_pages"], own_pages)
    keys = P + torch.arange(k.shape[2], device="cuda")
    scores = (q @ k.transpose(-1, -2)).masked_fill(keys >= s["lens"][:, None, None, None], -math.inf)
    if P:
        # all sequences' rows against the prefix at once
        k0, v0 = (_gather(s[n], s["shared_pages"][None])[0] for n in ("k_pages", "v_pages"))
        rows = q.permute(1, 0, 2, 3).reshape(kvH, -1, D)
        first = (rows @ k0.transpose(-1, -2)).view(kvH, B, H // kvH, P).transpose(0, 1)
        first = first.masked_fill(torch.arange(P, device="cuda") >= s["lens"][:, None, None, None], -math.inf)
        scores = torch.cat((first, scores), -1)
    m = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(m == -math.inf, 0.0, m))
    l = p.sum(-1, keepdim=True)
    out = p[..., P:] @ v
    if P:
        out = out + (p[..., :P].transpose(0, 1).reshape(kvH, -1, P) @ v0).view(kvH, B, H // kvH, D).transpose(0, 1)
    out = torch.where(l > 0, out / l, 0.0)
    lse = torch.where(l > 0, m + torch.log(l), -math.inf)[..., 0]
    return {"out": out.transpose(1, 2).reshape(B, H, D).to(s["q"].dtype), "lse": lse.transpose(1, 2).reshape(B, H)}


# ---- the library ---------------------------------------------------------------------------------


@functools.lru_cache(maxsize=None)
def _rope(rot_dim, base, interleaved):
    from ring_attention_b200 import api
    return api.Rope.make(rot_dim, base=base, interleaved=interleaved)


@functools.lru_cache(maxsize=None)
def _segmap(bases, rows):
    from ring_attention_b200 import api
    return api.SegMap.make(bases, rows)


def _own(s):
    from ring_attention_b200 import api
    c = s["c"]
    if c["kind"] in ("decode", "shared"):
        api.paged_decode(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["out"], lse=s["lse"],
                         shared_pages=s["shared_pages"] if c["shared"] else None)
        return {"out": s["out"], "lse": s["lse"]}
    rope = _rope(c["rot_dim"], c["base"], c["interleaved"])
    wq, wk = s.get("wq"), s.get("wk")
    if c["kind"] == "append":
        api.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"], counts=s["counts"], rope=rope,
                         k_weight=wk, q=s["q"], q_out=s["q_out"], q_weight=wq, eps=EPS)
        return {"k_pages": s["k_pages"], "v_pages": s["v_pages"], "q": s["q_out"]}
    bases, rows, step = _segments(c)
    segmap = _segmap(tuple(bases), rows)
    if c["kind"] == "norm_rope":
        api.qk_norm_rope(s["q"], s["k"], s["q_out"], s["k_out"], q_weight=wq, k_weight=wk, eps=EPS, rope=rope, segmap=segmap,
                         pos_stride=step)
        return {"q": s["q_out"], "k": s["k_out"]}
    api.qk_norm_rope_backward(s["q"], s["k"], s["dq_out"], s["dk_out"], s["q_out"], s["k_out"],
                              dq_weight=s["dwq"] if wq is not None else None, dk_weight=s["dwk"] if wk is not None else None,
                              q_weight=wq, k_weight=wk, eps=EPS, rope=rope, segmap=segmap, pos_stride=step)
    return {"dq": s["q_out"], "dk": s["k_out"], "dwq": s["dwq"] if wq is not None else None,
            "dwk": s["dwk"] if wk is not None else None}


def run(state):
    if own:
        return _own(state)
    kind = state["c"]["kind"]
    if kind == "append":
        return _plain_append(state)
    if kind in ("decode", "shared"):
        return _plain_decode(state)
    return _plain_rows(state)


# ---- work ----------------------------------------------------------------------------------------


def work(case):
    c = case
    B, H, kvH, D, es = c["batch"], c["heads"], c["kv_heads"], c["head_dim"], BYTES[c["dtype"]]
    if c["kind"] in ("norm_rope", "norm_rope_backward"):
        n = B * (H + kvH) * c["seq"] * D
        back = c["kind"] == "norm_rope_backward"
        # without a norm the gradient is the rotation of the gradient alone
        return {"bytes": (3 if back and c["norm"] else 2) * es * n, "flops": n * (3 + 4 * c["norm"]) * (2 if back else 1)}
    if c["kind"] == "append":
        n = sum(t for _, t in _before(c))
        return {"bytes": 2 * es * n * (2 * kvH + H) * D, "flops": n * (H + kvH) * D * (3 + 4 * c["norm"])}
    lens, P = _lengths(c), c["shared"]
    tails = sum(max(0, n - P) for n in lens)
    return {"bytes": 2 * es * kvH * D * (P + tails) + (2 * es * D + 4) * B * H, "flops": 4 * H * D * sum(lens)}


# ---- the definition in 64 bits -------------------------------------------------------------------


def _turned64(c, y, positions):
    """The rotation as a product of complex numbers."""
    R = c["rot_dim"]
    pairs = torch.arange(R // 2, dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       positions.double().unsqueeze(-1) / torch.pow(torch.tensor(c["base"], dtype=torch.float64, device="cuda"), 2 * pairs / R))
    i = torch.arange(R // 2, device="cuda")
    first, second = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + R // 2)
    z = torch.complex(y.index_select(-1, first), y.index_select(-1, second)) * turn
    return y.index_copy(-1, first, z.real).index_copy(-1, second, z.imag)


def _rows64(c, x, w, positions):
    if w is not None:
        x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * w
    return _turned64(c, x, positions)


def _positions64(c):
    bases, n, step = _segments(c)
    return torch.tensor([b + i * step for b in bases for i in range(n)], dtype=torch.float64, device="cuda")


def exact(case, seed):
    c, s = case, prepare(case, seed)
    weights = {n: s["w" + n].double() if c.get("norm") else None for n in ("q", "k")}
    if c["kind"] == "norm_rope":
        at = _positions64(c)
        return {n: _rows64(c, s[n].double(), weights[n], at) for n in ("q", "k")}
    if c["kind"] == "norm_rope_backward":
        at, got = _positions64(c), {}
        for n in ("q", "k"):
            leaves = [s[n].double().contiguous().requires_grad_()]
            if weights[n] is not None:
                leaves.append(weights[n].requires_grad_())
            grads = torch.autograd.grad(_rows64(c, leaves[0], weights[n], at), leaves, s["d%s_out" % n].double())
            got["d" + n], got["dw" + n] = grads[0], grads[1] if len(grads) > 1 else None
        return got
    B, H, kvH, D, page = c["batch"], c["heads"], c["kv_heads"], c["head_dim"], c["page_size"]
    if c["kind"] == "append":
        q_out = torch.zeros_like(s["q"], dtype=torch.float64)
        pages = {n: s[n + "_pages"].double() for n in ("k", "v")}
        for b, (n, m) in enumerate(zip(s["lens"].tolist(), s["counts"].tolist())):
            at = torch.arange(n, n + m, device="cuda")
            q_out[b, :, :m] = _rows64(c, s["q"][b, :, :m].double(), weights["q"], at)
            rows = {"k": _rows64(c, s["k"][b, :, :m].double(), weights["k"], at), "v": s["v"][b, :, :m].double()}
            where = s["table"][b].long()[at // page]
            for x in ("k", "v"):
                pages[x][where, :, at % page] = rows[x].transpose(0, 1)
        return {"k_pages": pages["k"], "v_pages": pages["v"], "q": q_out.contiguous()}
    out = torch.zeros((B, H, D), dtype=torch.float64, device="cuda")
    lse = torch.full((B, H), -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lens"].tolist()):
        where = s["table"][b, :-(-n // page)].long()
        for kv in range(kvH if n else 0):
            k, v = (s[x][where, kv].reshape(-1, D)[:n].double() for x in ("k_pages", "v_pages"))
            scores = s["q"][b, kv::kvH].double() @ k.T / D ** 0.5
            lse[b, kv::kvH] = torch.logsumexp(scores, -1)
            out[b, kv::kvH] = torch.softmax(scores, -1) @ v
    return {"out": out, "lse": lse}
