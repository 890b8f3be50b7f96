"""Checks of page copies' pairs: short and long lists refuse the same, and short ones need no memory for the pool."""
from __future__ import annotations

import ctypes as C
import random
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

import odf_b200 as odf
from test_paged_cpu import _copy


def _refusal(pairs, pages):
    """The first thing that is wrong, reading the ids in order; None if nothing is."""
    read, written = set(), set()
    for src, dst in pairs:
        for i, id_ in enumerate((src, dst)):
            if not 0 <= id_ < pages:
                return "outside"
            if i and id_ in written:
                return "twice"
            (written if i else read).add(id_)
            if id_ in read and id_ in written:
                return "read"
    return None


@pytest.mark.parametrize("seed", range(4))
def test_refusals_of_short_and_long_lists(seed):
    rng = random.Random(seed)
    lib = odf.load_library()
    seen = set()
    for _ in range(600):
        n = rng.choice([1, 2, 3, 7, 31, 32, 33, 34, 60])
        pages = rng.choice([2 * n, 3 * n, 5000])
        ids = rng.sample(range(pages), 2 * n)
        pairs = [list(p) for p in zip(ids[:n], ids[n:])]
        for _ in range(rng.randint(1, 2)):  # one or two mistakes
            i, j = rng.randrange(n), rng.randrange(2)
            pairs[i][j] = rng.choice([-1, pages, 2 ** 31 - 1, pairs[rng.randrange(n)][0], pairs[rng.randrange(n)][1]])
        want = _refusal(pairs, pages)
        if want is None:  # it would be launched
            continue
        seen.add((want, n > 32))
        p = _copy(pairs, **{"cache.num_pages": pages})
        assert lib.odf_page_copy_sm100(C.byref(p), None) == odf.ODF_ERR_INVALID_ARG
        assert want in odf.last_error(), (pairs, want, odf.last_error())
    assert len(seen) == 6


SCRIPT = """
import ctypes as C, resource, sys
sys.path[:0] = {paths!r}
import odf_b200 as odf
from test_paged_cpu import _copy
lib = odf.load_library()
p = _copy([(0, 1), (5, 6), (7, 1)], **{{"cache.num_pages": 2 ** 31 - 1}})
size = [int(x.split()[1]) * 1024 for x in open("/proc/self/status") if x.startswith("VmSize")][0]
resource.setrlimit(resource.RLIMIT_AS, (size + (256 << 20),) * 2)
print(lib.odf_page_copy_sm100(C.byref(p), None), odf.last_error())
"""


def test_a_few_pairs_need_no_memory_for_the_pool():
    """A pool of 2^31 - 1 pages, with 256 MB to spare: the pairs are still read (and refused for what they are)."""
    here = Path(__file__).resolve().parent
    paths = [str(here), str(here.parent / "dnn-flash_b200"), str(here.parent / "oracle")]
    out = subprocess.run([sys.executable, "-c", SCRIPT.format(paths=paths)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    assert out.stdout.startswith(f"{odf.ODF_ERR_INVALID_ARG} ") and "twice" in out.stdout, out.stdout
