"""Appends of many rows on the GPU: from 148 blocks of 64 rows (head_dim 128) or 128 rows (64) on, a thread takes four
rows, and keeps a head's divisors while the head stays.  Every case here is that large, against the definition to the bit.
"""
from __future__ import annotations

import math

import pytest
import torch

import odf_b200 as odf
import paged_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean_status():
    yield
    assert odf.device_status() == 0


def _rows_of_a_block(D):
    return 4 * 256 // (D // 8)


CASES = [
    # B, Hkv, T, D, page: the last block is partly filled in each
    (3, 2, 1603, 128, 16),
    (3, 2, 3205, 64, 64),
    (1, 1, 9500, 128, 7),
    (1400, 7, 1, 128, 16),  # every row another head than the one before
    (1350, 5, 3, 64, 1),
    (4, 3, 811, 128, 1),
]


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("layout", ["HND", "NHD"])
@pytest.mark.parametrize("B,Hkv,T,D,page", CASES)
def test_append_many_rows(kv, layout, B, Hkv, T, D, page):
    assert B * Hkv * T > 147 * _rows_of_a_block(D) and (B * Hkv * T) % _rows_of_a_block(D)
    g = torch.Generator().manual_seed(B + T)
    starts = torch.randint(0, 3 * page, (B,), generator=g)
    counts = torch.randint(0, T + 1, (B,), generator=g)
    for with_counts in (False, True):
        n = counts if with_counts else torch.full((B,), T)
        width = int((starts + T).max() + page - 1) // page
        used = (starts + n + page - 1) // page  # pages of each sequence; entries past them are out of range
        total = int(used.sum()) + 2
        perm = torch.randperm(total, generator=g)
        table = torch.full((B, width), 2 ** 31 - 1, dtype=torch.int64)
        table[torch.arange(width)[None] < used[:, None]] = perm[:total - 2]
        dtype = torch.bfloat16 if kv == "bf16" else torch.float8_e4m3fn
        shape = (total, Hkv, page, D) if layout == "HND" else (total, page, Hkv, D)
        kp, vp = (torch.full(shape, float("nan"), device="cuda").to(dtype) for _ in range(2))
        if layout == "NHD":
            kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
        scales = [torch.rand(Hkv, generator=g).cuda() / 30 + 1e-3 if kv == "e4m3" else None for _ in range(2)]
        k, v = (torch.randn((B, Hkv, T, D), device="cuda").to(torch.bfloat16) for _ in range(2))
        tail = torch.arange(T)[None] >= n[:, None]
        for x in (k, v):
            x.masked_fill_(tail[:, None, :, None].cuda(), float("nan"))
        if kv == "e4m3" and n[0]:
            k[0, 0, 0, :6] = torch.tensor([1e30, -1e30, math.inf, -math.inf, math.nan, 0.0])
        odf.paged_append(k, v, kp, vp, table.to(torch.int32).cuda(), starts.to(torch.int32).cuda(),
                         counts=n.to(torch.int32).cuda() if with_counts else None, k_scale=scales[0], v_scale=scales[1])
        b, t = (~tail).nonzero(as_tuple=True)
        pos = starts[b] + t
        at_page, at_slot = table[b, pos // page].cuda(), (pos % page).cuda()
        for new, pages, scale in ((k, kp, scales[0]), (v, vp, scales[1])):
            rows = new[b.cuda(), :, t.cuda()]  # [written rows, Hkv, D]
            if scale is not None:  # the fp32 quotient, which the kernel rounds
                rows = ref.to_e4m3((rows.float() / scale.view(1, -1, 1)).double())
            want = torch.full((total, Hkv, page, D), float("nan"), device="cuda")
            want[at_page, :, at_slot] = rows.float()
            assert torch.equal(torch.nan_to_num(pages.float(), nan=12345.0), torch.nan_to_num(want, nan=12345.0))


@pytest.mark.parametrize("D", [64, 128])
def test_append_rounds_every_value_as_the_quotient(D):
    """All bf16 values over scales of every kind, at 24576 rows and more."""
    x = torch.arange(65536, device="cuda", dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    scales = [1.0, 1 / 64, 0.015625 * 1.5, 0.1, 1 / 3, 7.123e-3, 0.99999994, 1.0000001, 3e-39, 1e38, 2.0 ** -126, 2.0 ** 127,
              2.0 ** 100, 1.1e-30, 5.0, 1e-45]
    B, Hkv, page = 3, len(scales), 64
    tokens = 65536 // D
    k = x.view(1, 1, tokens, D).expand(B, Hkv, tokens, D).contiguous()
    assert B * Hkv * tokens >= 24576 > 147 * _rows_of_a_block(D)
    s = torch.tensor(scales, device="cuda")
    table = torch.arange(B * tokens // page, device="cuda", dtype=torch.int32).view(B, -1)
    pages = [torch.zeros((B * tokens // page, Hkv, page, D), device="cuda").to(torch.float8_e4m3fn) for _ in range(2)]
    odf.paged_append(k, k.flip(1), pages[0], pages[1], table, torch.zeros(B, device="cuda", dtype=torch.int32),
                     k_scale=s, v_scale=s.flip(0))
    want = torch.nan_to_num(ref.to_e4m3((k[0].float() / s.view(-1, 1, 1)).double()).float(), nan=999.0)
    for held, flipped in ((pages[0], False), (pages[1], True)):
        got = held.float().view(B, tokens // page, Hkv, page, D).transpose(1, 2).reshape(B, Hkv, tokens, D)
        got = got.flip(1) if flipped else got
        for b in range(B):
            assert torch.equal(torch.nan_to_num(got[b], nan=999.0), want)
