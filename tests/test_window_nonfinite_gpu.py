"""Rows of a sliding-window call that see a key with a NaN have NaN as output and LSE, as in the formula; LSE -inf is
kept for rows that see nothing, so that whoever joins partial results by LSE does not take the one for the other."""
from __future__ import annotations

import math

import pytest
import torch

import odf_b200 as odf
import paged_ref as ref

pytestmark = pytest.mark.gpu

# M, N, window, sinks, q_offset, heads, keys: whole rows, few rows split over the keys, rows that see one key only
CASES = [(700, 700, 200, 3, 0, 2, [300]), (700, 700, 200, 3, 0, 2, [1]), (300, 300, 1, 0, 0, 2, [40, 41, 200]),
         (100, 8192, 4000, 4, 8092, 8, [6000]), (100, 8192, 4000, 4, 8092, 8, [2]), (1, 4096, 4096, 0, 4095, 4, [0]),
         (2, 4096, 4096, 0, 4094, 4, list(range(4096))), (40, 6000, 6000, 0, 5960, 1, list(range(0, 6000, 97)))]


@pytest.mark.parametrize("mod", [{}, {"softcap": 20.0}], ids=["plain", "softcap"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "_".join(str(x) for x in c[:6]) + f"_{len(c[6])}")
def test_lse_of_rows_that_see_a_nonfinite_key(case, bad, D, mod):
    M, N, window, sinks, off, H, keys = case
    g = torch.Generator(device="cuda").manual_seed(N + D)
    q, k, v = (torch.randn((1, H, n, D), generator=g, device="cuda").to(torch.bfloat16) for n in (M, N, N))
    want, want_l = odf.flash_fwd_window(q, k, v, window=window, sinks=sinks, q_offset=off, **mod)
    sees = ref.visible(off + torch.arange(M, device="cuda"), torch.arange(N, device="cuda"), N, window, sinks)[:, keys].any(1)
    assert sees.any()
    k[:, :, keys] = bad
    if bad == math.inf:  # a score of NaN as well: infinities of both signs meet
        q[..., 0], q[..., 1] = q[..., 0].abs() + 0.1, -q[..., 1].abs() - 0.1
        q0 = q.clone()
        k1 = k.clone()
        k1[:, :, keys] = 0.0
        want, want_l = odf.flash_fwd_window(q0, k1, v, window=window, sinks=sinks, q_offset=off, **mod)
    o, lse = odf.flash_fwd_window(q, k, v, window=window, sinks=sinks, q_offset=off, **mod)
    assert torch.isnan(lse[:, :, sees]).all() and torch.isnan(o[:, :, sees]).all()
    assert torch.isfinite(lse[:, :, ~sees]).all() and torch.isfinite(o[:, :, ~sees]).all()
    blocks = sees.nonzero().flatten() // 256
    apart = ~torch.isin(torch.arange(M, device="cuda") // 256, blocks)
    assert torch.equal(o[:, :, apart], want[:, :, apart]) and torch.equal(lse[:, :, apart], want_l[:, :, apart])
