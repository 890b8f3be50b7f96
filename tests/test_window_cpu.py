"""Refusals of the sliding-window entry (before any CUDA call) and its workspace room."""
from __future__ import annotations

import ctypes as C

import pytest

import odf_b200 as odf
from test_capi_cpu import _params

INV, UNS = odf.ODF_ERR_INVALID_ARG, odf.ODF_ERR_UNSUPPORTED


@pytest.mark.parametrize("over,win,code", [
    ({}, (0, 0, 0), INV), ({}, (-1, 0, 0), INV), ({}, (8, -1, 0), INV), ({}, (8, 0, -1), INV),
    ({}, (8, 0, 2 ** 31), UNS), ({}, (8, 0, 2 ** 31 - 200), UNS), ({"q": None}, (8, 0, 0), INV),
    ({"head_dim": 96}, (8, 0, 0), UNS), ({"heads_kv": 3}, (8, 0, 0), INV), ({"workspace": 4100}, (8, 0, 0), INV),
    ({"block_mask": 4096, "mask_qbs": 1, "mask_kbs": 1, "mask_qblocks": 1, "mask_kblocks": 1}, (8, 0, 0), UNS),
    ({"bias_kind": odf.ODF_BIAS_SAME_SHAPE, "bias": 4096}, (8, 0, 0), UNS), ({"tile_visits": 4096}, (8, 0, 0), UNS),
    ({"seqlen_k": 65535 * 128}, (8, 0, 0), UNS),
])
def test_window_refuses(over, win, code):
    lib = odf.load_library()
    assert lib.odf_flash_fwd_window_sm100(C.byref(_params(**over)), C.byref(odf.Window(*win)), None) == code
    assert odf.last_error()


def test_window_null():
    lib = odf.load_library()
    assert lib.odf_flash_fwd_window_sm100(None, C.byref(odf.Window(8, 0, 0)), None) == INV
    assert lib.odf_flash_fwd_window_sm100(C.byref(_params()), None, None) == INV
    assert lib.odf_fwd_window_workspace_size(C.byref(_params()), None) == 0


def test_window_workspace_room():
    """Room for splits goes by the keys that a window visits, not by all of them."""
    lib = odf.load_library()

    def room(window, sinks=0, **over):
        p = _params(heads_q=4, heads_kv=4, seqlen_q=64, seqlen_k=32768, head_dim=128, value_dim=128, **over)
        return lib.odf_fwd_window_workspace_size(C.byref(p), C.byref(odf.Window(window, sinks, 0)))

    assert room(128) == 256  # three tiles: too few to split
    assert 256 < room(4096) < room(32768)
    assert room(2048, sinks=4) >= room(2048)
    assert room(32768, batch=64) == 256  # enough items without


def test_window_binding_checks():
    import torch

    bf = torch.bfloat16
    q = torch.zeros((1, 2, 8, 64), dtype=bf)
    with pytest.raises(ValueError, match="CUDA"):
        odf.flash_fwd_window(q, q, q, window=4)
    with pytest.raises(ValueError, match="bfloat16"):
        odf.flash_fwd_window(q.float(), q, q, window=4)
    with pytest.raises(ValueError, match="shape"):
        odf.flash_fwd_window(q, q, q[:, :1], window=4)
