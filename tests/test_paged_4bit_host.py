"""The cache in 4 bits and reading rows back without a GPU: the reference's own pages, and what is refused before any CUDA call."""
import ctypes as C

import numpy as np
import pytest
import torch

import four_bit_ref as ref
from ring_attention_b200 import _lib, api
from ring_attention_b200._lib import NormRope, PagedKV, Rows, lib

P = 1 << 20


def rows(p=P):
    return C.byref(Rows(p, 0, 0, 0))


def refused(rc, code, word):
    assert rc == code and word in lib().ra_last_error().decode(), (rc, lib().ra_last_error())


def paged(**k):
    a = dict(dtype=_lib.RA_BF16, num_pages=10, kv_heads=2, page_size=16, head_dim=64, k=P, v=P, batch=3, max_pages=4, table_stride=4,
             page_table=P, lens=P)
    a.update(k)
    return C.byref(PagedKV(*(a[f[0]] for f in PagedKV._fields_)))


CACHES = [(dict(dtype=_lib.RA_F32), 1, "fp16 or bf16"), (dict(dtype=7), 1, "dtype"), (dict(head_dim=80), 3, "head_dim=80"),
          (dict(page_size=24), 3, "page_size"), (dict(kv_heads=0), 1, "bad cache"), (dict(k=None), 1, "null"),
          (dict(v=P + 8), 1, "aligned"), (dict(table_stride=-1), 1, "stride"), (dict(page_table=P + 2), 1, "aligned")]
SCALES = [(0.0, 1.0), (1.0, 3.0), (-1.0, 1.0), (2.0 ** 31, 1.0), (1.0, 2.0 ** -31), (float("nan"), 1.0), (float("inf"), 1.0)]


def test_append_refusals():
    L = lib()

    def call(c=None, ks=1.0, vs=1.0, k=rows(), v=rows(), t=5, counts=None, q=None, q_out=None, heads=0, how=None):
        return L.ra_paged_append_4bit(c if c is not None else paged(), ks, vs, k, v, t, counts, q, q_out, heads, how, None)

    for change, code, word in CACHES:
        refused(call(paged(**change)), code, word)
    for ks, vs in SCALES:
        refused(call(ks=ks, vs=vs), 1, "powers of two")
    refused(call(k=None), 1, "null")
    refused(call(v=rows(None)), 1, "null")
    refused(call(k=rows(P + 1)), 1, "aligned")
    refused(call(counts=P + 2), 1, "aligned")
    refused(call(q=rows()), 1, "queries")
    refused(call(q=rows(), q_out=rows(), heads=0), 1, "queries")
    refused(call(t=-1), 1, "shape")
    refused(call(paged(lens=None)), 1, "null")
    refused(call(how=C.byref(NormRope(P, P, 2, -1.0))), 1, "eps")
    assert call(paged(batch=0)) == 0 and call(t=0) == 0


def test_decode_refusals():
    L = lib()
    need = L.ra_paged_decode_4bit_workspace_bytes(paged(), 4)
    assert need > 0 and L.ra_paged_decode_4bit_workspace_bytes(None, 4) == 0
    assert L.ra_paged_decode_4bit_workspace_bytes(paged(page_size=7), 4) == 0

    def call(c=None, ks=1.0, vs=1.0, q=P, heads=4, out=P, lse=None, ws=P, room=1 << 40):
        return L.ra_paged_decode_4bit(c if c is not None else paged(), ks, vs, q, heads, out, lse, ws, room, None)

    for change, code, word in CACHES:
        refused(call(paged(**change)), code, word)
    for ks, vs in SCALES:
        refused(call(ks=ks, vs=vs), 1, "powers of two")
    refused(L.ra_paged_decode_4bit(None, 1.0, 1.0, P, 4, P, None, P, 1 << 40, None), 1, "null")
    refused(call(q=None), 1, "null")
    refused(call(out=None), 1, "null")
    refused(call(q=P + 8), 1, "aligned")
    refused(call(out=P + 4), 1, "aligned")
    refused(call(lse=P + 2), 1, "aligned")
    refused(call(heads=1), 1, "heads")
    refused(call(heads=4097), 1, "heads")
    refused(call(paged(batch=1 << 23)), 1, "rows")
    refused(call(paged(num_pages=1 << 30)), 1, "pages")
    refused(call(ws=None), 6, "workspace")
    refused(call(ws=P + 8), 6, "workspace")
    refused(call(room=need - 1), 6, "workspace")
    refused(call(paged(max_pages=2 ** 31 - 1, batch=6000)), 1, "too many keys")
    assert call(paged(batch=0)) == 0


@pytest.mark.parametrize("four", [False, True])
def test_read_refusals(four):
    L = lib()

    def call(c=None, ks=1.0, vs=1.0, ends=P, start=None, k=rows(), v=rows(), n=5):
        c = c if c is not None else paged(lens=None)
        if four:
            return L.ra_paged_read_4bit(c, ks, vs, ends, start, k, v, n, None)
        return L.ra_paged_read(c, ends, start, k, v, n, None)

    for change, code, word in CACHES:
        if not four and "dtype" in change:
            continue
        refused(call(paged(**change)), code, word)
    if four:
        for ks, vs in SCALES:
            refused(call(ks=ks, vs=vs), 1, "powers of two")
    else:
        refused(call(paged(dtype=7)), 1, "dtype")
    refused(call(ends=None), 1, "null")
    refused(call(ends=P + 2), 1, "aligned")
    refused(call(start=P + 2), 1, "aligned")
    refused(call(k=None), 1, "null")
    refused(call(v=rows(None)), 1, "null")
    refused(call(k=rows(P + 1)), 1, "aligned")
    refused(call(n=-1), 1, "shape")
    assert call(n=0) == 0 and call(paged(batch=0)) == 0


@pytest.mark.parametrize("D,page", [(32, 16), (64, 32), (128, 16), (256, 16)])
def test_reference_pages(D, page):
    rng = np.random.default_rng(D)
    codes, scales = rng.integers(0, 16, (3, 2, page, D), dtype=np.uint8), rng.integers(0, 127, (3, 2, page, D // 16), dtype=np.uint8)
    pages = ref.join_pages(codes, scales)
    assert pages.shape == tuple(api.pages_4bit(3, 2, page, D, device="cpu").shape)
    back = ref.split_pages(pages, page, D)
    assert np.array_equal(back[0], codes) and np.array_equal(back[1], scales)
    # the codes of a row are the row's again once they are written by value
    x = ref.decode(codes, scales, 0.5)
    again = ref.decode(*ref.encode(x, 0.5), 0.5)
    off = np.abs(again - x).reshape(3, 2, page, -1, 16)
    # (where a block's largest code is below 6 its new scale is another one)
    full = codes.reshape(off.shape)[..., :] % 8 == 7
    assert (off.max(-1)[full.any(-1)] == 0).all()


def test_reference_scales_are_torchs():
    x = np.concatenate([np.random.default_rng(1).standard_normal(4000) * 50, ref.E4M3, (ref.E4M3[1:] + ref.E4M3[:-1]) / 2])
    want = torch.from_numpy(np.abs(x)).to(torch.float32).clamp(max=448).to(torch.float8_e4m3fn).double().numpy()
    got = ref.E4M3[ref.nearest(np.minimum(np.abs(x.astype(np.float32)).astype(np.float64), 448), ref.E4M3)]
    assert np.array_equal(got, want)


def test_wrapper_refusals():
    """What the Python functions refuse by themselves, on tensors of the CPU (their device is asked for first on a GPU alone)."""
    with pytest.raises(ValueError):
        api._paged_4bit(torch.zeros(3, 2, 100, dtype=torch.uint8), torch.zeros(3, 2, 100, dtype=torch.uint8), torch.zeros(1, 1, dtype=torch.int32),
                        torch.zeros(1, dtype=torch.int32), 64, torch.float16)
    pages = api.pages_4bit(3, 2, 16, 64, device="cpu")
    table, lens = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    assert api._paged_4bit(pages, pages, table, lens, 64, torch.float16)[1:] == (2, 1)
    for bad in (pages.float(), pages[:, :, ::2], pages[0], pages[:2]):
        with pytest.raises(ValueError):
            api._paged_4bit(pages, bad, table, lens, 64, torch.float16)
    for dtype in (torch.float32, torch.uint8):
        with pytest.raises(ValueError):
            api._paged_4bit(pages, pages, table, lens, 64, dtype)
    for bad in (table.long(), table[0]):
        with pytest.raises(ValueError):
            api._paged_4bit(pages, pages, bad, lens, 64, torch.float16)
    with pytest.raises(ValueError):
        api._packed_rows(torch.zeros(4, 2, 64).expand(4, 2, 64)[:, :1].expand(4, 2, 64), (4, 2, 64), torch.float32, True)
    with pytest.raises(ValueError):
        api._packed_rows(torch.zeros(4, 64, 2).transpose(1, 2), (4, 2, 64), torch.float32)


def test_pages_say_what_they_were_made_for():
    pages = api.pages_4bit(3, 2, 16, 128, device="cpu")
    table, lens = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    assert api._paged_4bit(pages, pages, table, lens, 128, torch.float16)[1:] == (2, 1)
    for D in (32, 64, 256):
        with pytest.raises(ValueError):
            api._paged_4bit(pages, pages, table, lens, D, torch.float16)
        with pytest.raises(ValueError):
            api._paged_4bit(pages[:], pages[:], table, lens, D, torch.float16, page_size=16)
    assert api._paged_4bit(pages[:], pages[:], table, lens, 128, torch.float16, page_size=16)[1:] == (2, 1)


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.cpu_only
def test_rows_read_back_share_no_memory(four):
    L = lib()

    def call(row, head, n=5, other=False, **c):
        cache, one, two = paged(lens=None, **c), C.byref(Rows(P, 0, head, row)), C.byref(Rows(P, 0, 64, 128))
        args = (P, None, two, one) if other else (P, None, one, two)
        return L.ra_paged_read_4bit(cache, 1.0, 1.0, *args, n, None) if four else L.ra_paged_read(cache, *args, n, None)

    for row, head in ((0, 64), (128, 0), (64, 64), (127, 64), (-100, 64), (128, 256), (192, -192), (32, 6400)):
        for other in (False, True):
            refused(call(row, head, other=other), 1, "overlap")
    for row, head, more in ((128, 64, {}), (-128, 64, {}), (64, 320, {}), (128, 192, {}), (0, 64, dict(n=1)), (64, 0, dict(kv_heads=1))):
        assert call(row, head, **more) in (0, 2), L.ra_last_error()
