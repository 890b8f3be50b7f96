"""Strides that the binding hands to the C side, where all zero means contiguous: a tensor whose every leading
dimension is broadcast has those strides without being contiguous, and must not get through as one."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

import odf_b200 as odf


@pytest.mark.parametrize("sizes", [(4, 8), (2, 1, 5), (4, 8, 16), (1, 1, 7), (2, 4, 8, 16)])
def test_broadcast_tensors_are_refused(sizes):
    x = torch.zeros(128, dtype=torch.bfloat16).expand(*sizes, 128)
    with pytest.raises(ValueError, match="broadcast"):
        odf._strides(x, "q")


def test_partly_broadcast_tensors_are_refused():
    x = torch.zeros((4, 1, 16, 64), dtype=torch.bfloat16).expand(4, 3, 16, 64)
    with pytest.raises(ValueError, match="k is broadcast in dimension 1"):
        odf._strides(x, "k")


def test_strides_of_usual_tensors_stand():
    x = torch.zeros((2, 16, 3, 64), dtype=torch.bfloat16)
    assert tuple(odf._strides(x, "x")) == (0, 0, 0)  # contiguous
    assert odf._strides(x.transpose(1, 2), "x") == [16 * 3 * 64, 64, 3 * 64]
    assert odf._strides(x[:, ::2], "x") == [16 * 3 * 64, 2 * 3 * 64, 64]
    one = torch.zeros((1, 3, 1, 128), dtype=torch.bfloat16)[..., :64]  # dimensions of one element have no stride
    assert odf._strides(one, "x") == [3 * 64, 128, 64]
    layers = torch.zeros((2, 5, 3, 16, 96), dtype=torch.bfloat16)[..., :64]
    assert odf._strides(layers, "x") == [3 * 16 * 96, 16 * 96, 96]


def _fill(q, k, v, o, bias=None):
    return odf.fill_params(q, k, v, o, None, causal=False, scale=0.125, block_mask=None, mask_block=(128, 128), alibi=False,
                           alibi_slopes_host=None, softcap=0.0, workspace=None, visits=None, bias=bias)[0]


@pytest.mark.parametrize("which", range(4))
def test_forward_refuses_broadcast_tensors(which):
    ts = [torch.zeros((2, 4, 8, 64), dtype=torch.bfloat16) for _ in range(4)]
    _fill(*ts)
    ts[which] = torch.zeros(64, dtype=torch.bfloat16).expand(2, 4, 8, 64)
    with pytest.raises(ValueError, match="broadcast"):
        _fill(*ts)


def test_forward_takes_one_row():
    ts = [torch.zeros(64, dtype=torch.bfloat16).expand(1, 1, 1, 64) for _ in range(4)]
    _fill(*ts)


@pytest.mark.parametrize("M,N", [(8, 24), (1, 24), (8, 1), (1, 1)])
def test_forward_bias_of_one_value(M, N):
    """Strides that stay inside what holds the value: 0 over rows, 1 over a row of N copies."""
    q, o = (torch.zeros((2, 4, M, 64), dtype=torch.bfloat16) for _ in range(2))
    k, v = (torch.zeros((2, 4, N, 64), dtype=torch.bfloat16) for _ in range(2))
    for bias in (torch.tensor(2.5), torch.full((1, 1, 1, 1), 2.5), torch.tensor([2.5]).expand(2, 4, M, N)):
        p, keep = odf.fill_params(q, k, v, o, None, causal=False, scale=0.125, block_mask=None, mask_block=(128, 128),
                                  alibi=False, alibi_slopes_host=None, softcap=0.0, workspace=None, visits=None, bias=bias)
        strides = list(p.bias_strides)
        assert any(strides) and all(s == 0 or n == 1 for s, n in zip(strides[:3], (2, 4, M)))
        held = (C.c_float * (1 + (N - 1) * strides[3])).from_address(p.bias)
        assert list(held) == [2.5] * len(held) and (N == 1 or strides[3] <= 1)
        del keep


def test_forward_bias_strides_stand():
    q, k, v, o = (torch.zeros((2, 4, 8, 64), dtype=torch.bfloat16) for _ in range(4))
    for shape, strides in (((1, 1, 1, 8), [0, 0, 0, 1]), ((2, 1, 1, 1), [1, 0, 0, 0]), ((1, 4, 8, 8), [0, 64, 8, 1])):
        bias = torch.zeros(shape)
        p = _fill(q, k, v, o, bias)
        assert list(p.bias_strides) == strides and p.bias == bias.data_ptr()
