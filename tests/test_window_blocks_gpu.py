"""Which rows of a sliding-window call a non-finite value can reach: those of 256-row blocks (counted from row 0) with a
row that sees its key, and no others."""
from __future__ import annotations

import pytest
import torch

import odf_b200 as odf
import paged_ref as ref

pytestmark = pytest.mark.gpu


def _reach(M, N, window, sinks, off, keys):
    """(rows that see one of `keys`, rows of the blocks that have such a row)."""
    p = off + torch.arange(M, device="cuda")
    sees = ref.visible(p, torch.arange(N, device="cuda"), N, window, sinks)[:, keys].any(1)
    blocks = torch.zeros(-(-M // 256), dtype=torch.bool, device="cuda")
    blocks[torch.arange(M, device="cuda")[sees] // 256] = True
    return sees, blocks.repeat_interleave(256)[:M]


# M, N, window, sinks, q_offset; heads: few (a query tile per work item, or a split key range) and many
SHAPES = [(2048, 2048, 100, 0, 0), (1000, 1000, 1, 0, 0), (1000, 1000, 128, 3, 0), (1300, 1400, 333, 150, 70),
          (700, 2000, 777, 5, 1300), (600, 500, 50, 0, 0), (515, 515, 10 ** 6, 0, 0), (300, 5000, 4000, 4, 4700)]


@pytest.mark.parametrize("mod", [{}, {"softcap": 20.0}, {"alibi": True}, {"alibi": True, "softcap": 20.0}],
                         ids=["plain", "softcap", "alibi", "alibi_softcap"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "_".join(str(x) for x in s))
def test_blocks_that_do_not_see_a_value_are_untouched(shape, D, mod):
    M, N, window, sinks, off = shape
    for Hq, Hkv in ((2, 1), (160, 2)):
        g = torch.Generator(device="cuda").manual_seed(M + D)
        q, k, v = (torch.randn(s, generator=g, device="cuda").to(torch.bfloat16)
                   for s in ((1, Hq, M, D), (1, Hkv, N, D), (1, Hkv, N, D)))
        want, want_l = odf.flash_fwd_window(q, k, v, window=window, sinks=sinks, q_offset=off, **mod)
        assert torch.isfinite(want).all()
        for block in range(1, -(-M // 256)):  # a block's first key, and the last that a 128-key tile could reach
            for keys in ([off + 256 * block], list(range(off + 256 * block, min(N, off + 256 * block + 128)))):
                keys = [j for j in keys if j < N]
                if not keys:
                    continue
                sees, reach = _reach(M, N, window, sinks, off, keys)
                assert not reach[:256 * block].any()  # the blocks before have no row that sees them
                for bad in (float("nan"), float("inf")):
                    v2 = v.clone()
                    v2[:, :, keys] = bad
                    o, lse = odf.flash_fwd_window(q, k, v2, window=window, sinks=sinks, q_offset=off, **mod)
                    assert torch.equal(lse, want_l)
                    assert torch.equal(o[:, :, ~reach], want[:, :, ~reach]), f"{Hq} heads, keys {keys[0]}..{keys[-1]}"
                    if not mod.get("alibi"):  # with ALiBi, far tiles (weights below 2^-48) are left out
                        assert not torch.isfinite(o[:, :, sees]).any()
                k2 = k.clone()
                k2[:, :, keys] = float("nan")
                o, lse = odf.flash_fwd_window(q, k2, v, window=window, sinks=sinks, q_offset=off, **mod)
                assert torch.equal(o[:, :, ~reach], want[:, :, ~reach])
                assert torch.equal(lse[:, :, ~reach], want_l[:, :, ~reach])
