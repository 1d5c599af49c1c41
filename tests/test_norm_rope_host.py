"""Norm, rotation and paged append without a GPU: the rotation's table, the cache's addressing, and what is refused before any
CUDA call."""
import ctypes as C
import math
import os
import subprocess

import numpy as np
import pytest

from ring_attention_b200 import _lib
from ring_attention_b200._lib import (NormRope, PagedKV, RingAttentionError, Rope, Rows, SegMap, Shape, check, lib)

DTYPES = (_lib.RA_F32, _lib.RA_F16, _lib.RA_BF16)


@pytest.mark.parametrize("rot,base,scale", [(16, 10000.0, 1.0), (64, 10000.0, 0.125), (128, 500000.0, 1.0), (256, 1e6, 4.0)])
def test_turns_are_the_frequencies_in_parts_of_a_turn(rot, base, scale):
    r = Rope.make(rot, base=base, scale=scale)
    assert (r.rot_dim, r.interleaved) == (rot, 0)
    for i in range(rot // 2):
        part = base ** (-2 * i / rot) * scale / (2 * math.pi) % 1.0
        assert abs(r.turns[i] / 2.0 ** 64 - part) <= 2.0 ** -52
    same = Rope.from_freqs([base ** (-2 * i / rot) * scale for i in range(rot // 2)], interleaved=True)
    assert same.interleaved == 1
    assert all(abs(same.turns[i] - r.turns[i]) <= 2.0 ** 12 for i in range(rot // 2))


def test_far_positions_keep_their_place_in_the_turn():
    # position * turns modulo 2^64, as the kernels take it, at the last position that an int32 holds
    r, pos = Rope.make(64), 2 ** 31 - 1
    for i in range(32):
        # 10000^(-2 i / 64) in 64 bits is off by 2^-53 of itself, times the position
        want = pos * (10000.0 ** (-2 * i / 64)) / (2 * math.pi)
        got = (pos * r.turns[i] % 2 ** 64) / 2.0 ** 64
        off = abs(got - want % 1.0)
        assert min(off, 1 - off) <= 2.0 ** -20


def test_negative_frequencies_turn_the_other_way():
    r = Rope.from_freqs([0.5] * 8 + [-0.5] * 8)
    assert (r.turns[0] + r.turns[8]) % 2 ** 64 == 0


@pytest.mark.parametrize("call", [lambda: Rope.make(0), lambda: Rope.make(24), lambda: Rope.make(272), lambda: Rope.make(-16),
                                  lambda: Rope.make(32, base=0.0), lambda: Rope.make(32, base=math.inf),
                                  lambda: Rope.make(32, scale=math.nan), lambda: Rope.from_freqs([1.0] * 7),
                                  lambda: Rope.from_freqs([]), lambda: Rope.from_freqs([math.inf] * 8)])
def test_bad_rotations_are_refused(call):
    with pytest.raises(RingAttentionError) as e:
        call()
    assert e.value.code == 1
    with pytest.raises(ValueError):
        Rope.from_freqs([1.0] * 129)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_places_in_the_cache(page):
    table = [3, 0, -1, 7, 6, 5]
    t = (C.c_int * len(table))(*table)
    for slot in list(range(0, 6 * page, 7)) + [page - 1, page, 6 * page - 1]:
        at = table[slot // page]
        want = (at * 5) * page + slot % page if 0 <= at < 7 else -1  # 7 pages: numbers -1 and 7 are none
        assert lib().ra_debug_paged_row(t, 6, 7, page, 5, slot) == want
    for slot in (-1, -(2 ** 31), 6 * page, 2 ** 31, 2 ** 40):
        assert lib().ra_debug_paged_row(t, 6, 7, page, 5, slot) == -1
    # a cache of more rows than 32 bits count
    big = (C.c_int * 1)(2 ** 31 - 2)
    assert lib().ra_debug_paged_row(big, 1, 2 ** 31 - 1, page, 128, 9) == (2 ** 31 - 2) * 128 * page + 9


P = 4096  # never read: every call here is refused, or has nothing to do


def rows(p=P):
    return Rows(p, 1024, 128, 128)


def how(**k):
    return NormRope(eps=1e-6, pos_stride=1, **k)


def refused(rc, code, word):
    assert rc == code and word in lib().ra_last_error().decode()


def test_norm_rope_refusals():
    L = lib()
    sh = Shape(2, 4, 8, 8, 64, 2)
    rope, seg = Rope.make(64), SegMap.make([0], 8)

    def call(dtype=1, q=rows(), k=rows(), qo=rows(), ko=rows(), s=sh, h=how()):
        return L.ra_qk_norm_rope(dtype, q, k, qo, ko, s, h, None)

    refused(call(dtype=3), 1, "dtype")
    refused(call(s=None), 1, "null")
    refused(call(h=None), 1, "null")
    refused(call(qo=None), 1, "without")
    refused(call(k=None), 1, "without")
    refused(call(q=rows(None)), 1, "null")
    refused(call(s=Shape(2, 4, 8, 8, 48, 2)), 3, "head_dim=48")
    refused(call(s=Shape(2, 4, 8, 9, 64, 2)), 1, "same tokens")
    refused(call(s=Shape(-1, 4, 8, 8, 64, 2)), 1, "shape")
    refused(call(s=Shape(2, 0, 8, 8, 64, 2)), 1, "heads")
    refused(call(h=NormRope(eps=math.nan)), 1, "eps")
    refused(call(h=NormRope(eps=-1.0)), 1, "eps")
    refused(call(h=how(q_weight=P, weight_dtype=2)), 1, "weights")
    refused(call(h=how(rope=C.pointer(rope))), 1, "segment map")
    refused(call(h=how(rope=C.pointer(Rope.make(128)), segmap=C.pointer(seg))), 1, "rot_dim=128")
    refused(call(h=how(rope=C.pointer(rope), segmap=C.pointer(SegMap.make([0, 8], 8)))), 1, "n_seg")
    refused(call(h=NormRope(rope=C.pointer(rope), segmap=C.pointer(seg), pos_stride=0)), 1, "pos_stride")
    bad = SegMap.make([0], 8)
    bad.n_seg = 17
    refused(call(h=how(rope=C.pointer(rope), segmap=C.pointer(bad))), 1, "n_seg")
    # what is not aligned to its elements
    refused(call(q=rows(P + 1)), 1, "aligned")
    refused(call(ko=rows(P + 1)), 1, "aligned")
    refused(call(dtype=0, k=rows(P + 2)), 1, "aligned")
    refused(call(h=how(q_weight=P + 2, weight_dtype=0)), 1, "aligned")
    refused(call(h=how(k_weight=P + 1, weight_dtype=1)), 1, "aligned")
    refused(call(h=how(rope=C.pointer(rope), positions=P + 2)), 1, "aligned")
    # nothing to do
    assert call(s=Shape(0, 4, 8, 8, 64, 2)) == 0
    assert call(q=rows(None), qo=rows(None), s=Shape(2, 4, 0, 0, 64, 2)) == 0
    assert call(q=None, k=None, qo=None, ko=None) == 0


def test_norm_rope_backward_refusals():
    L = lib()
    need = L.ra_qk_norm_rope_backward_workspace_bytes(64)
    assert need > 0 and L.ra_qk_norm_rope_backward_workspace_bytes(-1) == 0

    def call(q=rows(), k=rows(), dyq=rows(), dyk=rows(), dq=rows(), dk=rows(), dwq=None, dwk=None, s=Shape(2, 4, 8, 8, 64, 2),
             h=how(), ws=None, n=0, dtype=1):
        return L.ra_qk_norm_rope_backward(dtype, q, k, dyq, dyk, dq, dk, dwq, dwk, s, h, ws, n, None)

    w = how(q_weight=P, k_weight=P, weight_dtype=1)
    refused(call(dtype=-1), 1, "dtype")
    refused(call(dq=None), 1, "gradient")
    refused(call(dyk=None), 1, "gradient")
    refused(call(dwq=P), 1, "weight that there is not")
    refused(call(q=None, h=w), 1, "needs the rows")
    refused(call(k=rows(None), h=w), 1, "null")
    refused(call(h=w, dwq=P), 6, "workspace")
    refused(call(h=w, dwk=P, ws=P, n=need - 1), 6, "workspace")
    refused(call(q=None, dyq=None, dq=None, h=w, dwq=P, ws=P, n=need), 1, "weight that there is not")
    refused(call(h=w, dwk=P, ws=P + 4, n=need), 6, "aligned")
    refused(call(h=w, dwk=P + 2, ws=P, n=need), 1, "aligned")
    refused(call(h=w, q=rows(P + 1)), 1, "aligned")
    refused(call(dq=rows(P + 1)), 1, "aligned")
    refused(call(dtype=0, dyk=rows(P + 2)), 1, "aligned")
    assert call(s=Shape(2, 4, 0, 0, 64, 2)) == 0


def paged(**k):
    c = PagedKV(1, 10, 2, 16, 64, P, P, 3, 4, 4, P, P)
    for n, v in k.items():
        setattr(c, n, v)
    return c


def test_append_refusals():
    L = lib()

    def call(c=paged(), k=rows(), v=rows(), n=1, q=None, qo=None, heads=0, h=None):
        return L.ra_paged_append(c, k, v, n, None, q, qo, heads, h, None)

    refused(call(c=None), 1, "null")
    refused(call(k=None), 1, "null")
    refused(call(v=rows(None)), 1, "null")
    refused(call(c=paged(dtype=7)), 1, "dtype")
    refused(call(c=paged(head_dim=96)), 3, "head_dim=96")
    for page in (0, 1, 8, 48, 512, -16):
        refused(call(c=paged(page_size=page)), 3, "page_size")
    refused(call(c=paged(kv_heads=0)), 1, "bad cache")
    refused(call(c=paged(num_pages=-1)), 1, "bad cache")
    refused(call(c=paged(max_pages=-1)), 1, "bad cache")
    refused(call(c=paged(k=None)), 1, "null")
    refused(call(c=paged(v=P + 8)), 1, "aligned")
    refused(call(c=paged(lens=None)), 1, "null")
    refused(call(c=paged(page_table=None)), 1, "null")
    refused(call(c=paged(table_stride=-4)), 1, "stride")
    refused(call(n=-1), 1, "shape")
    refused(call(q=rows()), 1, "queries")
    refused(call(q=rows(), qo=rows(), heads=0), 1, "queries")
    refused(call(h=how(rope=C.pointer(Rope.make(128)))), 1, "rot_dim")
    refused(call(k=rows(P + 1)), 1, "aligned")
    refused(call(c=paged(dtype=0), v=rows(P + 2)), 1, "aligned")
    refused(call(q=rows(), qo=rows(P + 1), heads=2), 1, "aligned")
    refused(call(c=paged(lens=P + 2)), 1, "aligned")
    refused(call(c=paged(page_table=P + 1)), 1, "aligned")
    refused(L.ra_paged_append(paged(), rows(), rows(), 1, P + 2, None, None, 0, None, None), 1, "aligned")
    assert call(n=0) == 0 and call(c=paged(batch=0)) == 0


def test_decode_refusals():
    L = lib()
    need = L.ra_paged_decode_workspace_bytes(paged(), 4, 0)
    # (a small 16-bit batch has no parts of the shared pages, a large one has)
    assert need > 0 and L.ra_paged_decode_workspace_bytes(paged(), 4, 32) == need < L.ra_paged_decode_workspace_bytes(paged(), 4, 1 << 20)
    assert L.ra_paged_decode_workspace_bytes(paged(dtype=0), 4, 32) > L.ra_paged_decode_workspace_bytes(paged(dtype=0), 4, 0)
    assert L.ra_paged_decode_workspace_bytes(None, 4, 0) == 0 and L.ra_paged_decode_workspace_bytes(paged(page_size=7), 4, 0) == 0

    def call(c=paged(), q=P, heads=4, pages=None, n=0, out=P, ws=P, room=1 << 40):
        return L.ra_paged_decode(c, q, heads, pages, n, out, None, ws, room, None)

    refused(call(c=None), 1, "null")
    refused(call(q=None), 1, "null")
    refused(call(out=None), 1, "null")
    refused(call(q=P + 8), 1, "aligned")
    refused(call(out=P + 4), 1, "aligned")
    refused(call(c=paged(dtype=3)), 1, "dtype")
    refused(call(c=paged(head_dim=80)), 3, "head_dim=80")
    refused(call(c=paged(page_size=24)), 3, "page_size")
    refused(call(c=paged(v=None)), 1, "null")
    refused(call(c=paged(lens=None)), 1, "null")
    refused(call(heads=1), 1, "heads")
    refused(call(heads=4097), 1, "heads")
    refused(call(c=paged(batch=1 << 23)), 1, "rows")
    refused(call(pages=P + 2, n=16), 1, "aligned")
    refused(L.ra_paged_decode(paged(), P, 4, None, 0, P, P + 2, P, 1 << 40, None), 1, "aligned")
    refused(call(pages=P, n=(1 << 30) + 16), 1, "2^30")
    assert L.ra_paged_decode_workspace_bytes(paged(), 4, 2 ** 31 - 16) == 0
    refused(call(n=16), 1, "shared")
    refused(call(pages=P, n=17), 1, "whole")
    refused(call(pages=P, n=-16), 1, "whole")
    refused(call(ws=None), 6, "workspace")
    refused(call(ws=P + 8), 6, "workspace")
    refused(call(room=need - 1), 6, "workspace")
    refused(call(c=paged(max_pages=2 ** 31 - 1, batch=4000)), 1, "too many keys")
    assert call(c=paged(batch=0)) == 0


@pytest.mark.parametrize("route,dtype,B,H,kvH,D,page,n_shared", [
    (0, 1, 4, 4, 2, 64, 16, 0), (0, 0, 4, 4, 2, 64, 16, 0),
    # each sequence for itself: 16 bits and little to read over again
    (1, 1, 7, 6, 6, 32, 16, 9), (1, 2, 33, 16, 2, 256, 256, 1), (1, 1, 8, 24, 6, 64, 16, 128), (1, 1, 5200, 8, 1, 32, 16, 1),
    # fp32; heads that are no multiple of the cache's; rows of more query blocks than the tensor-core kernel's list has
    (2, 0, 7, 6, 6, 32, 16, 9), (2, 0, 256, 32, 8, 128, 16, 1024), (2, 1, 33, 5, 2, 128, 128, 30), (2, 1, 5200, 8, 1, 32, 16, 3),
    (2, 1, 5200, 8, 1, 128, 16, 1), (2, 2, 5200, 8, 1, 128, 16, 1),
    # one page and many, on the tensor core
    (3, 1, 1000, 8, 1, 128, 256, 1), (3, 2, 32, 32, 8, 128, 64, 512), (3, 2, 256, 32, 8, 128, 16, 1024), (3, 1, 4, 4, 2, 64, 16, 1250),
    (3, 2, 6, 8, 2, 128, 32, 190), (3, 1, 5, 8, 2, 128, 16, 460), (3, 2, 4, 16, 4, 128, 64, 79)])
def test_which_way_shared_pages_are_read(route, dtype, B, H, kvH, D, page, n_shared):
    """The ways that the GPU tests mean to take, so that another threshold does not take them elsewhere unseen."""
    c = PagedKV(dtype, 10, kvH, page, D, P, P, B, 4, 4, P, P)
    assert lib().ra_debug_paged_route(c, H, n_shared * page) == route
    assert lib().ra_debug_paged_route(c, H, n_shared * page + 1) == -1 and lib().ra_debug_paged_route(None, H, 0) == -1
    c.num_pages = 0
    assert lib().ra_debug_paged_route(c, H, n_shared * page) == 0


def test_structures_are_those_of_the_header(tmp_path):
    """Sizes and offsets of the fields as a C compiler lays them out."""
    names = {"ra_rope": Rope, "ra_rows": Rows, "ra_norm_rope": NormRope, "ra_paged_kv": PagedKV}
    lines = [f'printf("%zu\\n", sizeof({n}));' for n in names]
    lines += [f'printf("%zu\\n", offsetof({n}, {f[0]}));' for n, s in names.items() for f in s._fields_]
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "ring_attention_b200.h"\nint main(void) {' + "\n".join(lines) +
                   "return 0; }")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "sizes")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "sizes")], capture_output=True, check=True).stdout.split()]
    want = [C.sizeof(s) for s in names.values()] + [getattr(s, f[0]).offset for s in names.values() for f in s._fields_]
    assert got == want
    # and the packed forms of the same
    c = PagedKV(1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12)
    assert _lib.PACK_PAGED_KV(1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12) == bytes(c)
    assert _lib.PACK_ROWS(1, 2, 3, 4) == bytes(Rows(1, 2, 3, 4)) and _lib.PACK_SHAPE(*range(6)) == bytes(Shape(*range(6)))
    h = NormRope(1, 2, 3, 0.5, None, None, 4, 5, 6)
    assert _lib.PACK_NORM_ROPE(1, 2, 3, 0.5, 0, 0, 4, 5, 6) == bytes(h)


@pytest.mark.parametrize("interleaved", [False, True])
def test_reference_gradient_is_that_of_differences(interleaved):
    """The oracle's own backward pass against differences of its forward pass, in 64 bits."""
    from norm_rope_ref import backward, default_freqs, forward
    rng = np.random.default_rng(1)
    x, dy, w = rng.standard_normal((3, 32)), rng.standard_normal((3, 32)), 1 + 0.3 * rng.standard_normal(32)
    pos, f = np.array([0, 7, 100003]), default_freqs(16)
    dx, _, dw, _ = backward(x, w, dy, pos, 16, interleaved, f, 1e-6, 0)
    h = 2.0 ** -17  # differences: h^2 of the third derivative, 2^-53 / h of the value

    def loss(x, w):
        return (forward(x, w, pos, 16, interleaved, f, 1e-6)[0] * dy).sum()

    for _ in range(5):
        a, b = rng.standard_normal(x.shape), rng.standard_normal(w.shape)
        got = (loss(x + h * a, w + h * b) - loss(x - h * a, w - h * b)) / (2 * h)
        assert abs(got - ((dx * a).sum() + (dw * b).sum())) <= 1e-7 * (np.abs(dx * a).sum() + np.abs(dw * b).sum())
