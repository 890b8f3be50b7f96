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


@pytest.mark.parametrize("seed", range(6))
def test_pairs_of_several_extends_in_one_copy(seed):
    """A step of a serving loop: every live sequence is extended, then the copies run together, then the new tokens are
    written.  Each page that is read by a copy still holds what it held, and no copy reads what another writes."""
    rng = random.Random(seed)
    page, total = rng.choice([1, 4, 7]), 300
    pool = odf.PagePool(total, page)
    memory = [[None] * page for _ in range(total)]
    model = {pool.add(): []}
    fresh = iter(range(10 ** 9))
    gathered = 0
    for _ in range(60):
        for _ in range(rng.randint(0, 3)):  # forks, cuts and ends come between the steps
            seq = rng.choice(list(model))
            what = rng.choice(["fork", "fork", "truncate", "free"])
            if what == "fork" and len(model) < 12:
                model[pool.fork(seq)] = list(model[seq])
            elif what == "truncate":
                n = rng.randint(0, len(model[seq]))
                pool.truncate(seq, n)
                del model[seq][n:]
            elif what == "free" and len(model) > 2:
                pool.free(seq)
                del model[seq]
        before = [list(m) for m in memory]
        live = rng.sample(list(model), rng.randint(1, len(model)))
        grow = {s: rng.randint(0, 2 * page) for s in live}
        pairs = [pair for s in live for pair in pool.extend(s, grow[s])]
        read, written = {s for s, _ in pairs}, [d for _, d in pairs]
        assert len(set(written)) == len(written) and not read & set(written)
        rng.shuffle(pairs)  # one launch: in no order
        for s, d in pairs:
            memory[d] = list(before[s])
        gathered = max(gathered, len(pairs))
        for s in live:
            pages = pool.pages(s)
            for i in range(len(model[s]), len(model[s]) + grow[s]):
                model[s].append(next(fresh))
                memory[pages[i // page]][i % page] = model[s][-1]
        for s, tokens in model.items():
            pages = pool.pages(s)
            assert [memory[pages[i // page]][i % page] for i in range(len(tokens))] == tokens
        if pool.free_pages < 60:
            for s in list(model)[1:]:
                pool.free(s)
                del model[s]
            pool.truncate(list(model)[0], 0)
            model[list(model)[0]].clear()
    assert gathered >= 2 or page == 1
