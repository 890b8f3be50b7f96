"""The decode kernel counts slices of its work in 32 bits: which calls that refuses, before any CUDA call."""
from __future__ import annotations

import ctypes as C

import pytest

import odf_b200 as odf
from test_paged_cpu import _decode

TOP = 2 ** 31 - 1


def _work(keys, batch, heads_kv, group, row_bytes):
    slices = -(-keys // (16 if row_bytes >= 256 else 32))
    return (slices + 12) * batch * heads_kv * -(-group // (8 if group <= 8 else 16))


@pytest.mark.parametrize("head_dim,kv,group", [(128, odf.ODF_DTYPE_BF16, 1), (128, odf.ODF_DTYPE_BF16, 8),
                                               (128, odf.ODF_DTYPE_BF16, 9), (64, odf.ODF_DTYPE_BF16, 33),
                                               (128, odf.ODF_DTYPE_E4M3, 1), (64, odf.ODF_DTYPE_E4M3, 20)])
@pytest.mark.parametrize("pages,window,sinks", [(1, 0, 0), (4096, 0, 0), (4096, 100, 0), (4096, 100, 30), (50, 10 ** 12, 5)])
def test_work_past_32_bits_is_refused(head_dim, kv, group, pages, window, sinks):
    """The largest batch that the formula allows gets past this check (to the missing workspace), one more does not."""
    lib = odf.load_library()
    heads_kv, page = 64, 16
    room = pages * page
    keys = min(room, window + sinks) if window else room
    row = head_dim * (2 if kv == odf.ODF_DTYPE_BF16 else 1)
    per = _work(keys, 1, heads_kv, group, row)
    most = min(TOP // per, 0x7fffff, TOP // (heads_kv * group))
    params = {"heads_q": heads_kv * group, "cache.heads_kv": heads_kv, "cache.head_dim": head_dim, "cache.kv_dtype": kv,
              "cache.page_size": page, "cache.max_pages": pages, "window": window, "sinks": sinks, "workspace": None}
    p = _decode(**params, batch=most)
    assert lib.odf_paged_decode_sm100(C.byref(p), None) == odf.ODF_ERR_INVALID_ARG and "workspace" in odf.last_error()
    p = _decode(**params, batch=most + 1)
    assert lib.odf_paged_decode_sm100(C.byref(p), None) == odf.ODF_ERR_UNSUPPORTED
    if most == TOP // per:
        assert "32 bits" in odf.last_error()


def test_the_headers_example():
    """One page each for 8388607 sequences of 64 kv-heads: few slices, but every item counts twelve more."""
    p = _decode(**{"batch": 8388607, "heads_q": 64, "cache.heads_kv": 64, "cache.head_dim": 128, "cache.max_pages": 1})
    assert odf.load_library().odf_paged_decode_sm100(C.byref(p), None) == odf.ODF_ERR_UNSUPPORTED
    assert "32 bits" in odf.last_error()
