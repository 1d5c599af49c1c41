"""What serving prompts out of a paged cache in 4 bits calls beside decoding, case by case: attention over packed prompts of
unlike lengths, whole or as chunks behind cached rows, appending to a cache in 4 bits, reading rows of sequences back out of a
paged cache, and decoding against one in 4 bits.

``own`` false computes the plain form in torch, true calls the library. Lengths of a batch are fixed by the case, and which
sequence has which is drawn from the seed, so that ``work`` can count them.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
GOLDEN = 0.6180339887498949


# ---- cases ---------------------------------------------------------------------------------------


def packed_case(dtype, heads, kv_heads, head_dim, batch, most, ragged, before=0, causal=True, fused=True, pad=0, name=None):
    c = {"kind": "packed", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "batch": batch,
         "most": most, "ragged": ragged, "before": before, "causal": causal, "fused": fused, "pad": pad}
    return {"name": name, **c} if name else c


def append_case(dtype, batch, kv_heads, most_before, tokens, head_dim, page_size, scale=1.0, name=None):
    c = {"kind": "append", "dtype": dtype, "batch": batch, "kv_heads": kv_heads, "most_before": most_before, "tokens": tokens,
         "head_dim": head_dim, "page_size": page_size, "scale": scale}
    return {"name": name, **c} if name else c


def read_case(dtype, batch, kv_heads, most, head_dim, page_size, ragged, bits, name=None):
    c = {"kind": "read", "dtype": dtype, "batch": batch, "kv_heads": kv_heads, "most": most, "head_dim": head_dim,
         "page_size": page_size, "ragged": ragged, "bits": bits}
    return {"name": name, **c} if name else c


def decode_case(dtype, batch, heads, kv_heads, most, head_dim, page_size, ragged=0.5, pad=0, scale=1.0, name=None):
    c = {"kind": "decode", "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads, "most": most,
         "head_dim": head_dim, "page_size": page_size, "ragged": ragged, "pad": pad, "scale": scale}
    return {"name": name, **c} if name else c


def listed():
    return [
        # the prompts of a chat server's step, short ones of unlike lengths, from a fused projection: latency
        packed_case("bf16", 24, 6, 64, 13, 200, 0.9, pad=3, name="packed_chat"),
        # a full step of prompts, from a sentence to a document
        packed_case("bf16", 32, 8, 128, 16, 4099, 0.97, name="packed_mixed"),
        # two long documents, a head of its own for every query head, the benchmark's heads
        packed_case("fp16", 8, 8, 64, 2, 32768, 0.5, fused=False, name="packed_long"),
        # the next chunks of four prompts behind what is cached of them
        packed_case("bf16", 32, 8, 128, 4, 1531, 0.5, before=16384, fused=False, name="packed_chunks"),
        # a decode step's new rows of every sequence into the cache
        append_case("bf16", 64, 8, 100, 1, 128, 16, name="append4_tokens"),
        # chunks of four prompts, of unlike lengths, V's values being small
        append_case("fp16", 4, 8, 500, 4099, 128, 64, scale=0.25, name="append4_chunks"),
        # a few short sequences read back
        read_case("bf16", 3, 6, 1531, 64, 16, 0.5, 16, name="read_short"),
        # what is cached of long prompts, for the attention of their next chunks
        read_case("bf16", 4, 8, 32768, 128, 64, 0.5, 4, name="read4_long"),
        # a small batch on chat-sized contexts, two padded places of a fixed batch among them
        decode_case("bf16", 7, 24, 6, 1531, 64, 16, pad=2, name="decode4_short"),
        # a full batch on middling contexts
        decode_case("bf16", 64, 32, 8, 8191, 128, 16, scale=0.5, name="decode4_batch"),
        # wide heads, many query heads to a KV head
        decode_case("fp16", 5, 32, 2, 33333, 256, 32, name="decode4_wide"),
        # long contexts: the benchmark's decode workload out of pages in 4 bits and with unlike lengths
        decode_case("fp16", 4, 32, 8, 262144, 128, 64, name="decode4_long"),
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
        kind = rng.choice(["packed", "packed", "append", "read", "decode", "decode"])
        dtype = rng.choice(["bf16", "fp16"])
        D = rng.choice([32, 64, 128, 128, 256])
        heads, kv_heads = _heads(rng, 64)
        page = rng.choice([16, 16, 32, 64, 128, 256])
        if kind == "packed":
            batch, most = _spread(rng, 1, 128), _spread(rng, 1, 32768)
            c = packed_case(dtype, heads, kv_heads, D, batch, most, rng.choice([0.0, 0.5, 0.97]),
                            rng.choice([0, 0, _spread(rng, 1, 32768)]), rng.random() < 0.85, rng.random() < 0.5, rng.choice([0, 0, 5]))
            rows = c["pad"] + sum(n for n, _ in _prompts(c))
            keys = sum(n for _, n in _prompts(c))
            # (the plain form works out every pair, and in fp32)
            pairs = heads * sum(n * m for n, m in _prompts(c))
            if pairs * max(D, 64) <= 8 * 64 * 32768 ** 2 * 1.25 and (rows * heads + keys * kv_heads) * D <= 1 << 28:
                return c
        elif kind == "append":
            batch, tokens = _spread(rng, 1, 256), rng.choice([1, _spread(rng, 1, 8192)])
            before = _spread(rng, 1, 2000)
            c = append_case(dtype, batch, kv_heads, before, tokens, D, page, rng.choice([1.0, 1.0, 0.25, 8.0]))
            if batch * (tokens + before + page) * kv_heads * D <= 4 * 4700 * 8 * 128:
                return c
        elif kind == "read":
            bits = rng.choice([4, 4, 16, 32])
            batch, most = _spread(rng, 1, 64), _spread(rng, 1, 65536)
            c = read_case("fp32" if bits == 32 else dtype, batch, kv_heads, most, D, page, rng.choice([0.0, 0.5, 0.9]), bits)
            if batch * (most + page) * kv_heads * D * (2 if bits == 32 else 1) <= 4 * 32768 * 8 * 128:
                return c
        else:
            batch, most = _spread(rng, 1, 256), _spread(rng, 1, 262144)
            c = decode_case(dtype, batch, heads, kv_heads, most, D, page, rng.choice([0.0, 0.5, 0.9]),
                            rng.choice([0, 0, batch // 4]), rng.choice([1.0, 1.0, 0.25]))
            if batch * (most + page) * heads * D <= 262144 * 32 * 128 * 4 and batch * (most + page) * kv_heads * D <= 262144 * 8 * 128 * 4:
                return c


# ---- inputs --------------------------------------------------------------------------------------


def _prompts(c):
    """(query rows, keys) of every packed sequence."""
    rows = [max(1, int(c["most"] * (1.0 - c["ragged"] * ((i * GOLDEN) % 1.0)))) for i in range(c["batch"])]
    return [(n, n + int(c["before"] * ((0.9 + i * GOLDEN) % 1.0))) for i, n in enumerate(rows)]


def _lengths(c):
    """The lengths of a decode batch or of what is read, longest first, padded places (no keys) last."""
    n = c["batch"] - c.get("pad", 0)
    return [max(1, int(c["most"] * (1.0 - c["ragged"] * ((i * GOLDEN) % 1.0)))) for i in range(n)] + [0] * c.get("pad", 0)


def _before(c):
    """(tokens cached, tokens that come) of every sequence of an append."""
    return [(int(c["most_before"] * ((i * GOLDEN) % 1.0)), max(1, int(c["tokens"] * (1.0 - 0.5 * ((i * GOLDEN * GOLDEN) % 1.0)))))
            for i in range(c["batch"])]


def _ends(counts):
    """Where each of the rows of sequences one after the other begins, and where the last one ends."""
    ends = [0]
    for n in counts:
        ends.append(ends[-1] + n)
    return torch.tensor(ends, dtype=torch.int32, device="cuda")


def _table(g, counts, num_pages, width):
    """Page numbers in random order, -1 behind a sequence's last page."""
    free = torch.randperm(num_pages, generator=g, device="cuda")
    table = torch.full((len(counts), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = free[at:at + n].int()
        at += n
    return table


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, kvH, D, dt = c["batch"], c["kv_heads"], c["head_dim"], DTYPES[c["dtype"]]
    s = {"c": c}
    order = torch.randperm(B, generator=g, device="cuda").tolist()
    if c["kind"] == "packed":
        H = c["heads"]
        s["prompts"] = [_prompts(c)[i] for i in order]
        rows, keys = c["pad"] + sum(n for n, _ in s["prompts"]), sum(n for _, n in s["prompts"])
        if c["fused"] and not c["before"]:
            qkv = torch.randn((rows, H + 2 * kvH, D), generator=g, device="cuda", dtype=dt)
            s["q"], s["k"], s["v"] = qkv[:, :H], qkv[:, H:H + kvH], qkv[:, H + kvH:]
        else:
            s["q"] = torch.randn((rows, H, D), generator=g, device="cuda", dtype=dt)
            s["k"], s["v"] = (torch.randn((keys, kvH, D), generator=g, device="cuda", dtype=dt) for _ in range(2))
        s["ends"] = _ends([n for n, _ in s["prompts"]])
        s["k_ends"] = _ends([n for _, n in s["prompts"]]) if c["before"] else None
        s["out"] = torch.zeros((rows, H, D), device="cuda", dtype=dt)
        s["lse"] = torch.zeros((H, rows), device="cuda")
        return s
    page = c["page_size"]
    if c["kind"] == "append":
        both = [_before(c)[i] for i in order]
        counts = [-(-(n + t) // page) for n, t in both]
        rows = sum(t for _, t in both)
        s["lens"] = torch.tensor([n for n, _ in both], dtype=torch.int32, device="cuda")
        s["counts"] = torch.tensor([t for _, t in both], dtype=torch.int32, device="cuda")
        s["ends"] = _ends([t for _, t in both])
        T = c["tokens"]
        # as a projection leaves them, token by token
        s["k"], s["v"] = (torch.randn((B, T, kvH, D), generator=g, device="cuda", dtype=dt).mul_(f).transpose(1, 2)
                          for f in (1.3, c["scale"]))
        s["k_out"], s["v_out"] = (torch.zeros((rows, kvH, D), device="cuda", dtype=dt) for _ in range(2))
    else:
        lens = [_lengths(c)[i] for i in order]
        counts = [-(-n // page) for n in lens]
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        if c["kind"] == "read":
            s["ends"] = _ends(lens)
            s["k_out"], s["v_out"] = (torch.zeros((sum(lens), kvH, D), device="cuda", dtype=dt) for _ in range(2))
        else:
            s["q"] = torch.randn((B, c["heads"], D), generator=g, device="cuda", dtype=dt)
            s["out"] = torch.zeros((B, c["heads"], D), device="cuda", dtype=dt)
            s["lse"] = torch.zeros((B, c["heads"]), device="cuda")
    num_pages = sum(counts) + 3
    s["table"] = _table(g, counts, num_pages, max(1, max(counts)) + 1)
    if c.get("bits", 4) != 4:
        s["k_pages"], s["v_pages"] = (torch.randn((num_pages, kvH, page, D), generator=g, device="cuda", dtype=dt) for _ in range(2))
        return s
    s["factors"] = (1.0, c.get("scale", 1.0))
    for n, f in zip(("k_pages", "v_pages"), s["factors"]):
        s[n] = torch.empty((num_pages, kvH, page * 9 * D // 16), dtype=torch.uint8, device="cuda")
        step = max(1, (1 << 27) // (kvH * page * D))
        for i in range(0, num_pages, step):
            x = torch.randn((min(step, num_pages - i), kvH, page, D), generator=g, device="cuda") * (f if n == "v_pages" else 1.0)
            s[n][i:i + step] = _to_page(*_to_4bit(x, f))
    return s


# ---- plain form ----------------------------------------------------------------------------------

# the values of codes 0 to 7; 8 is the sign
CODES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _to_4bit(x, factor):
    """(codes, scales) of rows: 16 elements share a scale in e4m3, a sixteenth of a row's codes."""
    x = x.float().unflatten(-1, (-1, 16))
    scales = (x.abs().amax(-1) / (6.0 * factor)).clamp(max=448.0).to(torch.float8_e4m3fn)
    step = scales.float()[..., None] * factor
    a = x.abs()
    # borders of the codes times a scale are exact; those between an odd and the next even code belong to the latter
    code = (a > 0.25 * step).to(torch.uint8)
    for border, up in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (a >= border * step) if up else (a > border * step)
    code = torch.where(step > 0, code + 8 * (x < 0).to(torch.uint8), torch.zeros((), dtype=torch.uint8, device="cuda"))
    return code.flatten(-2), scales


def _place(page, D):
    """Where byte i of the codes of row j is among the codes of its page: pieces of 16 bytes change places with the row."""
    j, i = torch.arange(page, device="cuda")[:, None], torch.arange(D // 2, device="cuda")[None]
    turn = ((j & 1) * 4 | (j & 2)) & (D // 32 - 1)
    return j * (D // 2) + (i // 16 ^ turn) * 16 + i % 16


def _to_page(codes, scales):
    """The bytes of whole pages, (..., page, D) codes: two codes a byte, then the scales."""
    page, D = codes.shape[-2:]
    packed = (codes[..., 0::2] | codes[..., 1::2] << 4).flatten(-2)
    placed = torch.empty_like(packed)
    placed[..., _place(page, D).flatten()] = packed
    return torch.cat((placed, scales.view(torch.uint8).flatten(-2)), -1)


def _values(pages, page, D, factor):
    """The rows of whole pages, (..., page, D), in fp32."""
    codes = pages[..., _place(page, D)]
    scales = pages[..., page * D // 2:].contiguous().view(torch.float8_e4m3fn).unflatten(-1, (page, D // 16)).float()
    lut = torch.tensor(CODES + tuple(-v for v in CODES), device="cuda")
    both = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    return (lut[both.int()].unflatten(-1, (-1, 16)) * scales[..., None]).flatten(-2) * factor


def _plain_packed(s):
    c = s["c"]
    H, kvH, D = c["heads"], c["kv_heads"], c["head_dim"]
    out, lse = torch.zeros_like(s["out"]), torch.zeros_like(s["lse"])
    q0 = k0 = 0
    for n, m in s["prompts"]:
        # query head h reads KV head h % kvH
        q = s["q"][q0:q0 + n].float().view(n, H // kvH, kvH, D).permute(2, 1, 0, 3) / math.sqrt(D)
        k, v = (s[x][k0:k0 + m].float().transpose(0, 1) for x in ("k", "v"))
        hidden = torch.arange(m, device="cuda") > torch.arange(n, device="cuda")[:, None] + (m - n) if c["causal"] else None
        step = max(1, (1 << 30) // (n * m * (H // kvH)))
        for h in range(0, kvH, step):
            scores = q[h:h + step].flatten(1, 2) @ k[h:h + step].transpose(1, 2)  # (heads, group * n, m)
            if hidden is not None:
                scores.unflatten(1, (-1, n)).masked_fill_(hidden, -math.inf)
            top = scores.amax(-1, keepdim=True)
            p = scores.sub_(top).exp_()
            l = p.sum(-1, keepdim=True)
            o = (p @ v[h:h + step]) / l
            hs = o.shape[0]
            out[q0:q0 + n].unflatten(1, (H // kvH, kvH))[:, :, h:h + step] = o.view(hs, H // kvH, n, D).permute(2, 1, 0, 3).to(out.dtype)
            lse.unflatten(0, (H // kvH, kvH))[:, h:h + step, q0:q0 + n] = (top + l.log()).view(hs, H // kvH, n).transpose(0, 1)
        q0, k0 = q0 + n, k0 + m
    return {"out": out, "lse": lse}


def _plain_append(s):
    c = s["c"]
    B, T, page, D = c["batch"], c["tokens"], c["page_size"], c["head_dim"]
    t = torch.arange(T, device="cuda")[None].expand(B, T)
    b, t = (t < s["counts"][:, None]).nonzero(as_tuple=True)
    slots = s["lens"].long()[b] + t
    pages, rows = s["table"][b, slots // page].long(), slots % page
    got = {}
    for n, f in zip(("k", "v"), s["factors"]):
        x = s[n][b, :, t]  # (rows, heads, D)
        codes, scales = _to_4bit(x, f)
        to = s[n + "_pages"]
        to[pages[:, None], :, _place(page, D)[rows]] = (codes[..., 0::2] | codes[..., 1::2] << 4).transpose(1, 2)
        at = page * D // 2 + rows[:, None] * (D // 16) + torch.arange(D // 16, device="cuda")
        to[pages[:, None], :, at] = scales.view(torch.uint8).transpose(1, 2)
        lut = torch.tensor(CODES + tuple(-v for v in CODES), device="cuda")
        got[n] = (lut[codes.int()].unflatten(-1, (-1, 16)) * (scales.float()[..., None] * f)).flatten(-2).to(x.dtype)
    return got


def _plain_read(s):
    c = s["c"]
    page, D = c["page_size"], c["head_dim"]
    got = {}
    for i, n in enumerate(("k", "v")):
        parts = []
        for b, length in enumerate(_host_lengths(s)):
            pages = s[n + "_pages"][s["table"][b, :-(-length // page)].long()]  # (pages, heads, ...)
            x = pages if c["bits"] != 4 else _values(pages, page, D, s["factors"][i])
            parts.append(x.transpose(1, 2).flatten(0, 1)[:length].to(s[n + "_out"].dtype))
        got[n] = torch.cat(parts)
    return got


def _host_lengths(s):
    """The lengths of the sequences, which the program that cached them knows."""
    if "host" not in s:
        s["host"] = s["lens"].tolist()
    return s["host"]


def _plain_decode(s):
    c = s["c"]
    H, kvH, D, page = c["heads"], c["kv_heads"], c["head_dim"], c["page_size"]
    out, lse = torch.zeros_like(s["out"]), torch.full_like(s["lse"], -math.inf)
    for b, length in enumerate(_host_lengths(s)):
        if length == 0:
            continue
        where = s["table"][b, :-(-length // page)].long()
        k, v = (_values(s[n][where], page, D, f).transpose(0, 1).flatten(1, 2)[:, :length]
                for n, f in zip(("k_pages", "v_pages"), s["factors"]))
        q = s["q"][b].float().view(H // kvH, kvH, D).transpose(0, 1) / math.sqrt(D)
        scores = q @ k.transpose(1, 2)
        top = scores.amax(-1, keepdim=True)
        p = torch.exp(scores - top)
        l = p.sum(-1, keepdim=True)
        out[b] = ((p @ v) / l).transpose(0, 1).reshape(H, D).to(out.dtype)
        lse[b] = (top + l.log())[..., 0].transpose(0, 1).reshape(H)
    return {"out": out, "lse": lse}


# ---- the library ---------------------------------------------------------------------------------


def _own(s):
    from ring_attention_b200 import api
    c = s["c"]
    if c["kind"] == "packed":
        api.packed_attention(s["q"], s["k"], s["v"], s["ends"], s["out"], k_ends=s["k_ends"], causal=c["causal"], lse=s["lse"])
        return {"out": s["out"], "lse": s["lse"]}
    if c["kind"] == "read" and c["bits"] != 4:
        api.paged_read(s["k_pages"], s["v_pages"], s["table"], s["ends"], s["k_out"], s["v_out"])
        return {"k": s["k_out"], "v": s["v_out"]}
    kf, vf = s["factors"]
    if c["kind"] == "decode":
        api.paged_decode_4bit(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["out"], lse=s["lse"],
                              k_scale=kf, v_scale=vf)
        return {"out": s["out"], "lse": s["lse"]}
    if c["kind"] == "append":
        api.paged_append_4bit(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"], counts=s["counts"],
                              k_scale=kf, v_scale=vf)
        # the rows as the cache has them now
        api.paged_read_4bit(s["k_pages"], s["v_pages"], s["table"], s["ends"], s["k_out"], s["v_out"], start=s["lens"],
                            k_scale=kf, v_scale=vf)
    else:
        api.paged_read_4bit(s["k_pages"], s["v_pages"], s["table"], s["ends"], s["k_out"], s["v_out"], k_scale=kf, v_scale=vf)
    return {"k": s["k_out"], "v": s["v_out"]}


def run(state):
    if own:
        return _own(state)
    return {"packed": _plain_packed, "append": _plain_append, "read": _plain_read, "decode": _plain_decode}[state["c"]["kind"]](state)


# ---- work ----------------------------------------------------------------------------------------


def work(case):
    c = case
    kvH, D, es = c["kv_heads"], c["head_dim"], BYTES[c["dtype"]]
    four = 9 / 16  # bytes of an element in 4 bits
    if c["kind"] == "packed":
        H, both = c["heads"], _prompts(c)
        rows, keys = sum(n for n, _ in both), sum(m for _, m in both)
        pairs = sum(n * m - (n * (n - 1) // 2 if c["causal"] else 0) for n, m in both)
        return {"bytes": 2 * es * D * (rows * H + keys * kvH) + 4 * H * rows, "flops": 4 * H * D * pairs}
    if c["kind"] == "append":
        n = 2 * kvH * D * sum(t for _, t in _before(c))
        return {"bytes": int(n * (2 * es + four)), "flops": 8 * n}
    n = 2 * kvH * D * sum(_lengths(c))
    if c["kind"] == "read":
        return {"bytes": int(n * (es + (four if c["bits"] == 4 else es))), "flops": 2 * n if c["bits"] == 4 else 0}
    return {"bytes": int(n * four) + (2 * es * D + 4) * c["batch"] * c["heads"], "flops": 4 * c["heads"] * D * sum(_lengths(c))}


# ---- the definition in 64 bits -------------------------------------------------------------------


def _grid64(bits, low, top):
    """All magnitudes of a small float format: `bits` of fraction, exponents from `low` (of the numbers below 2^low, too) up to
    the largest number `top`."""
    steps = 1 << bits
    below = [i / steps * 2.0 ** low for i in range(steps)]
    above = [(1 + i / steps) * 2.0 ** e for e in range(low, 40) for i in range(steps)]
    return torch.tensor([v for v in below + above if v <= top], dtype=torch.float64, device="cuda")


def _nearest64(x, grid):
    """Index of the number nearest to each x >= 0, the even one of two that are equally near."""
    hi = torch.searchsorted(grid, x.contiguous()).clamp(max=len(grid) - 1)
    lo = (hi - 1).clamp(min=0)
    up, down = grid[hi] - x, x - grid[lo]
    return torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)


def _rounded64(x, factor):
    """What rows are in the cache's 4 bits."""
    e2m1, e4m3 = _grid64(1, 0, 6.0), _grid64(3, -6, 448.0)
    x = x.double().unflatten(-1, (-1, 16))
    scale = e4m3[_nearest64(x.abs().amax(-1) / 6 / factor, e4m3)][..., None] * factor
    r = torch.where(scale > 0, x.abs() / torch.where(scale > 0, scale, 1.0), 0.0)
    return (e2m1[_nearest64(r, e2m1)] * scale * torch.sign(x)).flatten(-2)


def _cached64(pages, c, factor):
    """The rows of whole pages in 4 bits, (pages, heads, page, D), by the bytes."""
    page, D = c["page_size"], c["head_dim"]
    e2m1, e4m3 = _grid64(1, 0, 6.0), _grid64(3, -6, 448.0)
    codes, scales = pages[..., :page * D // 2].unflatten(-1, (-1, 16)), pages[..., page * D // 2:].unflatten(-1, (page, D // 16))
    pieces = D // 32
    order = [j * pieces + (p ^ (4 * (j % 2) + 2 * (j // 2 % 2)) % pieces) for j in range(page) for p in range(pieces)]
    byte = codes[..., torch.tensor(order, device="cuda"), :].flatten(-2).unflatten(-1, (page, D // 2))
    code = torch.stack((byte % 16, byte // 16), -1).flatten(-2).long()
    x = e2m1[code % 8] * torch.where(code >= 8, -1.0, 1.0)
    return (x.unflatten(-1, (-1, 16)) * (e4m3[scales.long()] * factor)[..., None]).flatten(-2)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    D = c["head_dim"]
    if c["kind"] == "packed":
        H, kvH = c["heads"], c["kv_heads"]
        out, lse = torch.zeros_like(s["out"], dtype=torch.float64), torch.zeros_like(s["lse"], dtype=torch.float64)
        q0 = k0 = 0
        for n, m in s["prompts"]:
            for h in range(H):
                k, v = (s[x][k0:k0 + m, h % kvH].double() for x in ("k", "v"))
                step = max(1, (1 << 28) // m)
                for i in range(0, n, step):
                    rows = torch.arange(i, min(i + step, n), device="cuda")
                    scores = s["q"][q0 + rows, h].double() @ k.T / D ** 0.5
                    if c["causal"]:
                        seen = torch.arange(m, device="cuda")[None] - (m - n) <= rows[:, None]
                        scores = torch.where(seen, scores, -math.inf)
                    lse[h, q0 + rows] = torch.logsumexp(scores, -1)
                    out[q0 + rows, h] = torch.softmax(scores, -1) @ v
            q0, k0 = q0 + n, k0 + m
        return {"out": out, "lse": lse}
    if c["kind"] == "append":
        return {n: torch.cat([_rounded64(s[n][b, :, :t].transpose(0, 1), f) for b, t in enumerate(s["counts"].tolist())])
                for n, f in zip(("k", "v"), s["factors"])}
    page, lens = c["page_size"], s["lens"].tolist()

    def rows_of(n, b, heads=slice(None)):
        pages = s[n + "_pages"][s["table"][b, :-(-lens[b] // page)].long(), heads]
        if c.get("bits", 4) == 4:
            pages = _cached64(pages, c, s["factors"][n == "v"])
        return pages.double().movedim(0, -3).flatten(-3, -2)[..., :lens[b], :]

    if c["kind"] == "read":
        return {n: torch.cat([rows_of(n, b).transpose(0, 1) for b in range(c["batch"])]) for n in ("k", "v")}
    B, H, kvH = c["batch"], c["heads"], c["kv_heads"]
    out = torch.zeros((B, H, D), dtype=torch.float64, device="cuda")
    lse = torch.full((B, H), -math.inf, dtype=torch.float64, device="cuda")
    for b in range(B):
        for kv in range(kvH if lens[b] else 0):
            k, v = (rows_of(n, b, kv) for n in ("k", "v"))
            scores = s["q"][b, kv::kvH].double() @ k.T / D ** 0.5
            lse[b, kv::kvH] = torch.logsumexp(scores, -1)
            out[b, kv::kvH] = torch.softmax(scores, -1) @ v
    return {"out": out, "lse": lse}
