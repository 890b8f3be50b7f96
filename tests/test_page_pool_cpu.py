"""The page pool's numbers past 63 bits, and copies that several calls of `extend` ask for, run together."""
from __future__ import annotations

import random

import pytest

import odf_b200 as odf

WRAP = 2 ** 64  # a 64-bit integer of the C side would see 0


@pytest.mark.parametrize("args", [(WRAP + 4, 16), (4, WRAP + 16), (-WRAP + 4, 16), (2 ** 63, 16)])
def test_pool_sizes_do_not_wrap(args):
    with pytest.raises(ValueError):
        odf.PagePool(*args)


def test_pool_calls_do_not_wrap():
    pool = odf.PagePool(8, 16)
    seq = pool.add()
    pool.extend(seq, 40)
    for call in (lambda: pool.extend(seq, WRAP + 1), lambda: pool.extend(seq, -WRAP + 1), lambda: pool.truncate(seq, WRAP + 7),
                 lambda: pool.truncate(seq, -WRAP), lambda: pool.fork(WRAP + seq), lambda: pool.free(WRAP + seq),
                 lambda: pool.extend(WRAP + seq, 1), lambda: pool.truncate(seq - WRAP, 1), lambda: pool.length(WRAP + seq),
                 lambda: pool.pages(WRAP + seq), lambda: pool.table([WRAP + seq])):
        with pytest.raises(ValueError):
            call()
    assert pool.length(seq) == 40 and pool.pages(seq) == [0, 1, 2] and pool.free_pages == 5
