"""Attention over packed sequences without a GPU: what is refused before any CUDA call."""
import ctypes as C

import pytest

from ring_attention_b200 import _lib
from ring_attention_b200._lib import Rows, Shape, lib

P = 1 << 20


def rows(p=P, row=256, head=64):
    return C.byref(Rows(p, 0, head, row))


def refused(rc, code, word):
    assert rc == code and word in lib().ra_last_error().decode(), (rc, lib().ra_last_error())


def call(dtype=_lib.RA_BF16, q=rows(), k=rows(), v=rows(), out=rows(), lse=P, shape=None, ends=P, k_ends=None, **s):
    a = dict(batch=3, heads=4, seq_q=100, seq_k=100, head_dim=64, kv_heads=2)
    a.update(s)
    return lib().ra_packed_attention(dtype, q, k, v, out, lse, C.byref(Shape(*(a[f[0]] for f in Shape._fields_))) if shape is None else shape,
                                     ends, k_ends, 1, None)


def test_refusals():
    for name in ("q", "k", "v", "out"):
        refused(call(**{name: None}), 1, "null")
        refused(call(**{name: rows(None)}), 1, "null")
        refused(call(**{name: rows(P + 8)}), 1, "16 bytes")
        refused(call(**{name: rows(row=68)}), 1, "16 bytes")
        refused(call(**{name: rows(head=36)}), 1, "16 bytes")
        # rows or heads that share memory
        refused(call(**{name: rows(row=0)}), 1, "overlap")
        refused(call(**{name: rows(row=-256)}), 1, "overlap")
        refused(call(**{name: rows(head=32)}), 1, "overlap")
        refused(call(**{name: rows(row=1 << 33)}), 1, "overlap")
    refused(call(dtype=_lib.RA_F32), 1, "fp16 or bf16")
    refused(call(dtype=9), 1, "fp16 or bf16")
    refused(call(head_dim=80), 3, "head_dim=80")
    refused(call(head_dim=0), 3, "head_dim=0")
    refused(call(heads=5), 1, "multiple")
    refused(call(heads=0), 1, "multiple")
    refused(call(heads=1), 1, "multiple")
    refused(call(heads=1 << 17), 1, "multiple")
    refused(call(kv_heads=-1, heads=-4), 1, "multiple")
    refused(call(batch=-1), 1, "shape")
    refused(call(seq_q=-1), 1, "shape")
    refused(call(seq_k=-1), 1, "shape")
    refused(call(seq_q=(1 << 30) + 1), 1, "too many")
    refused(call(ends=None), 1, "null")
    refused(call(ends=P + 2), 1, "aligned")
    refused(call(k_ends=P + 2), 1, "aligned")
    refused(call(lse=P + 2), 1, "aligned")
    refused(lib().ra_packed_attention(2, rows(), rows(), rows(), rows(), None, None, P, None, 1, None), 1, "null")
    assert call(batch=0) == 0 and call(seq_q=0, q=rows(None)) == 0


@pytest.mark.parametrize("name", ["q", "k", "v", "out"])
def test_strides_of_one_row_or_head_do_not_count(name):
    """(the call goes on to the device, which is not there: not a refusal of its arguments)"""
    rc = call(**{name: rows(row=3, head=5)}, seq_q=1, seq_k=1, heads=1, kv_heads=1)
    assert rc in (0, 2), lib().ra_last_error()


@pytest.mark.cpu_only
def test_rows_of_a_result_share_no_memory():
    """Head h + 1 of a row may not be head h of the next; interleaved rows that only look so are none of that."""
    D = 64
    for row, head in ((64, 64), (128, 64), (64, 128), (192, 64), (200, 72), (128, 128), (128, 136)):
        refused(call(out=rows(row=row, head=head)), 1, "overlap")
    # heads side by side, rows side by side, rows with room, and two heads whose rows lie between one another's
    for row, head, more in ((256, 64, {}), (64, 6400, {}), (264, 64, {}), (128, 64, dict(heads=2)), (128, 192, dict(heads=2)),
                            (128, 64 * 201, dict(heads=2)), (64, 64, dict(seq_q=1)), (64, 64, dict(heads=1, kv_heads=1))):
        rc = call(out=rows(row=row, head=head), **more)
        assert rc in (0, 2), lib().ra_last_error()
    # (rows that are only read may lie as they like)
    for name in ("q", "k", "v"):
        assert call(**{name: rows(row=64, head=64)}) in (0, 2), lib().ra_last_error()


def test_more_places_than_waits_have_time_for():
    """(batch 0 comes before it: nothing to do)"""
    refused(call(batch=(1 << 22) + 1, heads=1, kv_heads=1), 1, "too many")
    refused(call(batch=1 << 22, heads=9, kv_heads=1), 1, "too many")
    refused(call(batch=1 << 30, heads=1, kv_heads=1), 1, "too many")
    refused(call(batch=1 << 20, heads=33, kv_heads=33), 1, "too many")
