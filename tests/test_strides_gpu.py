"""A bias of one value for every score on the GPU (its strides are all zero, which the C side takes for contiguous)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import odf_b200 as odf

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N", [1, 300])
def test_bias_of_one_value(N):
    """The same bits as with the value written out, on the device and on the host entry."""
    q = torch.randn((2, 3, 200, 64), device="cuda").to(torch.bfloat16)
    k, v = (torch.randn((2, 3, N, 64), device="cuda").to(torch.bfloat16) for _ in range(2))
    want, want_l = odf.flash_fwd(q, k, v, bias=torch.full((2, 3, 200, N), 1.5, device="cuda"), softcap=4.0)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for bias in (torch.tensor(1.5, device="cuda"), torch.full((1, 1, 1, 1), 1.5, device="cuda")):
        for stream in (None, side.cuda_stream):
            o, lse = odf.flash_fwd(q, k, v, bias=bias, softcap=4.0, stream=stream)
            torch.cuda.synchronize()
            assert torch.equal(o, want) and torch.equal(lse, want_l)
    lse = np.empty((2, 3, 200), np.float32)
    o, _ = odf.flash_fwd_host(*(x.float().cpu().numpy() for x in (q, k, v)), bias=np.float32(1.5), softcap=4.0, lse_out=lse)
    assert np.array_equal(o, want.cpu().numpy()) and np.array_equal(lse, want_l.cpu().numpy())
