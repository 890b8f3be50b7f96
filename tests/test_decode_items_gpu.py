"""Decode attention with 112 to 440 work items (sequences x kv-heads), where the kernel chooses between a CTA per item and
items cut into pieces: batches on both sides of that choice, and next to it, against the 64-bit reference."""
from __future__ import annotations

import pytest
import torch

import odf_b200 as odf
import paged_ref as ref

pytestmark = pytest.mark.gpu


def _slices(lens, row_bytes):
    keys = 16 if row_bytes >= 256 else 32
    return [max(1, -(-n // keys)) for n in lens]


def _even(B, n):
    return [n] * B


def _spread(B, n, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(n // 4, 2 * n, (B,), generator=g).tolist()


@pytest.mark.parametrize("kv,D", [("bf16", 128), ("e4m3", 128), ("bf16", 64), ("e4m3", 64)])
@pytest.mark.parametrize("B,Hkv,group", [(14, 8, 2), (37, 4, 8), (100, 4, 1), (112, 1, 12)])
def test_items_whole_and_cut(B, Hkv, group, kv, D):
    row = D * (2 if kv == "bf16" else 1)
    edge = 24 * (16 if row >= 256 else 32)  # an even batch's items stop being whole between this and twice it
    sides = set()
    for lens in (_even(B, edge), _even(B, edge * 3 // 2), _even(B, 2 * edge), _even(B - 1, 40) + [3000], _spread(B, edge, B),
                 _spread(B, 2 * edge, B + 1)):
        slices = _slices(lens, row)
        sides.add(max(slices) <= sum(slices) * Hkv // 280 + 24)
        cache = ref.Cache(lens, Hkv=Hkv, D=D, page=64, kv=kv, seed=B)
        g = torch.Generator(device="cuda").manual_seed(D)
        q = torch.randn((B, Hkv * group, D), generator=g, device="cuda").to(torch.bfloat16)
        args = (q, cache.k, cache.v, cache.table, cache.lens)
        o, lse = odf.paged_decode(*args, k_scale=cache.ks, v_scale=cache.vs, out_dtype=torch.bfloat16)
        ref.check_decode(o, lse, q, cache, what=f"{B} sequences, longest {max(lens)}")
        again, lse2 = odf.paged_decode(*args, k_scale=cache.ks, v_scale=cache.vs, out_dtype=torch.bfloat16)
        assert torch.equal(o, again) and torch.equal(lse, lse2)
    assert sides == {False, True}
    assert odf.device_status() == 0
