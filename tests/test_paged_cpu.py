"""Host side of the paged cache: refusals of the entry points (before any CUDA call) and the page pool."""
from __future__ import annotations

import ctypes as C
import random
import subprocess
from pathlib import Path

import numpy as np
import pytest

import odf_b200 as odf

INV, UNS = odf.ODF_ERR_INVALID_ARG, odf.ODF_ERR_UNSUPPORTED
A = 4096  # never dereferenced: validation fails first


def _set(p, over):
    for name, value in over.items():
        at = p
        *path, last = name.split(".")
        for part in path:
            at = getattr(at, part)
        if isinstance(value, (list, tuple)):
            for i, x in enumerate(value):
                getattr(at, last)[i] = x
        else:
            setattr(at, last, value)
    return p


def _cache(c):
    c.k_pages = c.v_pages = c.page_table = A
    c.kv_dtype = odf.ODF_DTYPE_BF16
    c.num_pages, c.heads_kv, c.page_size, c.head_dim, c.max_pages = 8, 2, 16, 64, 4


def _decode(**over):
    p = odf.DecodeParams()
    p.q = p.o = p.lens = p.workspace = A
    p.workspace_bytes = 1 << 30
    p.o_dtype, p.batch, p.heads_q, p.scale = odf.ODF_DTYPE_BF16, 2, 4, 0.125
    _cache(p.cache)
    return _set(p, over)


def _append(**over):
    p = odf.AppendParams()
    p.k = p.v = p.starts = A
    p.batch, p.tokens = 2, 3
    _cache(p.cache)
    return _set(p, over)


CACHE_REFUSALS = [
    ("cache.k_pages", None, INV), ("cache.v_pages", None, INV), ("cache.k_pages", A + 8, INV),
    ("cache.kv_dtype", odf.ODF_DTYPE_F32, UNS), ("cache.num_pages", 0, INV), ("cache.page_size", 0, INV),
    ("cache.page_size", 65537, UNS), ("cache.heads_kv", -1, INV), ("cache.heads_kv", 65536, UNS),
    ("cache.head_dim", 96, UNS), ("cache.k_strides", (2048, 1024, 63), INV), ("cache.v_strides", (2048, -8, 64), INV),
    ("cache.v_strides", (2048, 0, 64), INV), ("cache.page_table", None, INV), ("cache.page_table", A + 2, INV),
    ("cache.max_pages", 0, INV), ("cache.table_stride", 3, INV), ("cache.max_pages", 1 << 28, UNS),
    ("cache.k_scale", A, INV),
]


@pytest.mark.parametrize("field,value,code", CACHE_REFUSALS + [
    ("q", None, INV), ("o", None, INV), ("lens", None, INV), ("batch", 0, INV), ("heads_q", 0, INV), ("heads_q", 3, INV),
    ("o_dtype", 7, UNS), ("scale", float("nan"), INV), ("softcap", -1.0, INV), ("softcap", float("inf"), INV),
    ("window", -1, INV), ("sinks", -1, INV), ("bias_kind", odf.ODF_BIAS_SAME_SHAPE, UNS), ("q", A + 8, INV),
    ("lens", A + 1, INV), ("q_strides", (256, 4), INV), ("o_strides", (256, -64), INV), ("workspace", None, INV),
    ("workspace_bytes", 16, INV), ("workspace", A + 4, INV), ("batch", 1 << 23, UNS),
])
def test_decode_refuses(field, value, code):
    lib = odf.load_library()
    assert lib.odf_paged_decode_sm100(C.byref(_decode(**{field: value})), None) == code
    assert odf.last_error()


@pytest.mark.parametrize("field,value,code", CACHE_REFUSALS + [
    ("k", None, INV), ("v", A + 4, INV), ("starts", None, INV), ("starts", A + 1, INV), ("counts", A + 2, INV),
    ("batch", 0, INV), ("tokens", 0, INV), ("k_strides", (8, 8, 4), INV), ("tokens", 1 << 31, UNS),
])
def test_append_refuses(field, value, code):
    lib = odf.load_library()
    assert lib.odf_paged_append_sm100(C.byref(_append(**{field: value})), None) == code
    assert odf.last_error()


def test_decode_refuses_what_does_not_fit_its_counters():
    """Explicit slopes past 256 heads, a K pool past 64 GB."""
    lib = odf.load_library()
    slopes = (C.c_float * 300)()
    p = _decode(heads_q=300, bias_kind=odf.ODF_BIAS_ALIBI, alibi_slopes=C.cast(slopes, C.c_void_p))
    assert lib.odf_paged_decode_sm100(C.byref(p), None) == UNS and "256" in odf.last_error()
    p = _decode(**{"cache.num_pages": 1 << 24, "cache.k_strides": (4096, 1024, 64)})
    assert lib.odf_paged_decode_sm100(C.byref(p), None) == UNS and "64 GB" in odf.last_error()


def test_headers_compile_as_c(tmp_path):
    src = tmp_path / "use.c"
    src.write_text('#include "odf_paged_sm100.h"\n#include "odf_sm100.h"\n'
                   "int main(void) { odf_decode_params p = {0}; odf_window w = {1, 0, 0};\n"
                   "  return (int)(p.batch + w.sinks) + ODF_ERR_NO_PAGES - 8; }\n")
    include = Path(__file__).resolve().parents[1] / "include"
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Wextra", "-Werror", f"-I{include}", "-c", "-o", str(tmp_path / "use.o"),
                    str(src)], check=True)


def test_null_params():
    lib = odf.load_library()
    for f in (lib.odf_paged_decode_sm100, lib.odf_paged_append_sm100, lib.odf_page_copy_sm100):
        assert f(None, None) == INV
    assert lib.odf_paged_decode_workspace_size(None) == 0


def _copy(ids_, **over):
    p = odf.PageCopyParams()
    _cache(p.cache)
    ids = np.ascontiguousarray(ids_, dtype=np.int32).reshape(-1, 2)
    p.layers, p.k_layer_stride, p.v_layer_stride = 2, 1 << 16, 1 << 16
    p.pairs, p.n_pairs = ids.ctypes.data, len(ids)
    p.keep = ids
    return _set(p, over)


@pytest.mark.parametrize("pairs,over,text", [
    ([(0, 8)], {}, "outside"), ([(-1, 2)], {}, "outside"), ([(0, 2), (1, 2)], {}, "twice"), ([(0, 1), (1, 2)], {}, "read"),
    ([(3, 3)], {}, "read"), ([(1, 2), (0, 1)], {}, "read"), ([(0, 1)], {"layers": 0}, "layers"),
    ([(0, 1)], {"k_layer_stride": 0}, "layer strides"), ([(0, 1)], {"v_layer_stride": 12}, "layer strides"),
    ([(0, 1)], {"pairs": None}, "non-null"), ([(0, 1)], {"n_pairs": -1}, "non-null"), ([(0, 1)], {"n_pairs": 9}, "twice"),
])
def test_copy_refuses(pairs, over, text):
    lib = odf.load_library()
    assert lib.odf_page_copy_sm100(C.byref(_copy(pairs, **over)), None) == INV
    assert text in odf.last_error()


def test_copy_of_nothing_needs_no_device():
    assert odf.load_library().odf_page_copy_sm100(C.byref(_copy([])), None) == odf.ODF_OK


# ------------------------------------------------------------------------------------ page pool
def test_pool_refuses():
    lib = odf.load_library()
    for pages, size in ((0, 16), (-1, 16), (1 << 31, 16), (4, 0), (4, 65537)):
        with pytest.raises(ValueError):
            odf.PagePool(pages, size)
    pool = odf.PagePool(4, 16)
    for call in (lambda: pool.fork(7), lambda: pool.extend(7, 1), lambda: pool.truncate(7, 0), lambda: pool.free(7),
                 lambda: pool.pages(7), lambda: pool.extend(pool.add(), -1), lambda: pool.truncate(pool.add(), 1)):
        with pytest.raises(ValueError):
            call()
    seq = pool.add()
    with pytest.raises(odf.OdfError) as e:
        pool.extend(seq, 65)
    assert e.value.code == odf.ODF_ERR_NO_PAGES and pool.free_pages == 4 and pool.length(seq) == 0
    with pytest.raises(ValueError):
        pool.extend(seq, 1 << 31)
    with pytest.raises(ValueError):
        pool.extend(seq, (1 << 63) - 1)
    pool.extend(seq, 64)
    out = (C.c_int32 * 2)()
    assert lib.odf_page_pool_table(pool._pool, seq, out, 2) == INV
    with pytest.raises(ValueError):
        pool.table([seq], max_pages=3)
    n = C.c_int64()
    assert lib.odf_page_pool_create(4, 16, None) == INV
    assert lib.odf_page_pool_add(None, C.byref(n)) == INV
    assert lib.odf_page_pool_free_pages(None) == 0
    lib.odf_page_pool_destroy(None)


def test_pool_copy_on_write():
    pool = odf.PagePool(6, 4)
    a = pool.add()
    assert pool.extend(a, 6) == [] and pool.pages(a) == [0, 1]
    b = pool.fork(a)
    assert pool.pages(b) == [0, 1] and pool.free_pages == 4
    assert pool.extend(b, 1) == [(1, 2)] and pool.pages(b) == [0, 2]  # the shared half-filled page
    assert pool.extend(a, 1) == []  # now a's alone
    c = pool.fork(a)
    pool.truncate(c, 4)
    assert pool.extend(c, 1) == []  # page 0 is full and stays shared
    assert pool.pages(c) == [0, 3]
    pool.free(a)
    assert pool.free_pages == 6 - 3
    d = pool.fork(c)
    pool.truncate(d, 2)
    assert pool.extend(d, 1) == [(0, 1)]  # cut back into a shared page
    pool.free(b), pool.free(c), pool.free(d)
    assert pool.free_pages == 6


@pytest.mark.parametrize("seed", range(6))
def test_pool_random_against_model(seed):
    """Random calls against a model that keeps every sequence's tokens and carries out the copies."""
    rng = random.Random(seed)
    page, total = rng.choice([1, 3, 8]), rng.choice([5, 40, 200])
    pool = odf.PagePool(total, page)
    memory = [[None] * page for _ in range(total)]
    model = {}
    fresh = iter(range(10 ** 9))

    def run(pairs):
        dst = [d for _, d in pairs]
        assert len(set(dst)) == len(dst) and not set(dst) & {s for s, _ in pairs}
        for s, d in pairs:
            memory[d] = list(memory[s])

    for _ in range(400):
        what = rng.choice(["add", "fork", "extend", "extend", "extend", "truncate", "free", "compact"])
        seq = rng.choice(list(model)) if model else None
        if what == "add" or seq is None:
            model[pool.add()] = []
        elif what == "fork":
            model[pool.fork(seq)] = list(model[seq])
        elif what == "extend":
            n = rng.randint(0, 3 * page)
            before = (pool.free_pages, pool.pages(seq))
            try:
                run(pool.extend(seq, n))
            except odf.OdfError as e:
                assert e.code == odf.ODF_ERR_NO_PAGES and before == (pool.free_pages, pool.pages(seq))
                continue
            pages = pool.pages(seq)
            for i in range(len(model[seq]), len(model[seq]) + n):
                tok = next(fresh)
                model[seq].append(tok)
                memory[pages[i // page]][i % page] = tok
        elif what == "truncate":
            n = rng.randint(0, len(model[seq]))
            pool.truncate(seq, n)
            del model[seq][n:]
        elif what == "free":
            pool.free(seq)
            del model[seq]
        else:
            run(pool.compact())
            used = {p for s in model for p in pool.pages(s)}
            assert used == set(range(len(used)))
        used = {p for s in model for p in pool.pages(s)}
        assert pool.free_pages == total - len(used)
        for s, tokens in model.items():
            pages = pool.pages(s)
            assert pool.length(s) == len(tokens) and len(pages) == -(-len(tokens) // page)
            assert [memory[pages[i // page]][i % page] for i in range(len(tokens))] == tokens
    if model:
        table = pool.table(list(model), max_pages=total)
        for row, s in zip(table.tolist(), model):
            pages = pool.pages(s)
            assert row == pages + [-1] * (total - len(pages))


@pytest.mark.parametrize("pack,cls", [("_PACK_DECODE", odf.DecodeParams), ("_PACK_APPEND", odf.AppendParams),
                                      ("_PACK_COPY", odf.PageCopyParams), ("_PACK_FWD", odf.FwdParams),
                                      ("_PACK_WINDOW", odf.Window)])
def test_packed_structs_are_the_ctypes_ones(pack, cls):
    """Every field of the packed form lands where the ctypes struct (and so the C one) has it."""
    def leaves(c):
        for name, t in c._fields_:
            if issubclass(t, C.Structure):
                yield from leaves(t)
            else:
                n = getattr(t, "_length_", 1)
                yield from [t._type_ if n > 1 else t] * n

    values = [i + 0.5 if t is C.c_float else i + 1 for i, t in enumerate(leaves(cls))]
    raw = getattr(odf, pack)(*values)
    assert len(raw) == C.sizeof(cls)
    at = iter(values)

    def walk(x):
        for name, t in x._fields_:
            v = getattr(x, name)
            if isinstance(v, C.Structure):
                walk(v)
            elif hasattr(t, "_length_"):
                assert list(v) == [next(at) for _ in v], name
            else:
                assert v == next(at), name

    walk(cls.from_buffer_copy(raw))


def test_python_checks_without_a_device():
    import torch

    bf = torch.bfloat16
    cache = torch.zeros((4, 2, 16, 64), dtype=bf)
    table = torch.zeros((2, 2), dtype=torch.int32)
    lens = torch.ones(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        odf.paged_decode(torch.zeros((2, 4, 64), dtype=bf), cache, cache, table, lens)
    with pytest.raises(ValueError, match="rank 3"):
        odf.paged_decode(torch.zeros((2, 4, 1, 64), dtype=bf), cache, cache, table, lens)
    with pytest.raises(ValueError, match="CUDA"):
        odf.paged_append(torch.zeros((2, 2, 1, 64), dtype=bf), torch.zeros((2, 2, 1, 64), dtype=bf), cache, cache, table, lens)
    with pytest.raises(ValueError, match="CUDA"):
        odf.page_copy(cache, cache, [(0, 1)])
