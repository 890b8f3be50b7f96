"""The paged cache on the GPU: decode attention, append and page copies against 64-bit references.

Slots that hold no token are NaN in every cache here, and table entries past a sequence's pages are out
of range, so a kernel that reads either shows it.
"""
from __future__ import annotations

import math

import pytest
import torch

import odf_b200 as odf
import paged_ref as ref

pytestmark = pytest.mark.gpu


def _q(B, Hq, D, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn((B, Hq, D), generator=g, device="cuda").to(torch.bfloat16)


def _decode(cache, q, **kw):
    return odf.paged_decode(q, cache.k, cache.v, cache.table, cache.lens, k_scale=cache.ks, v_scale=cache.vs, **kw)


@pytest.fixture(autouse=True)
def _clean_status():
    yield
    if torch.cuda.is_available():
        assert odf.device_status() == 0


DECODE = [
    # Hq, Hkv, D, page, lens, options
    (4, 4, 64, 16, [1], {}),
    (4, 4, 64, 16, [129], {}),
    (8, 8, 128, 64, [8192], {}),
    (8, 1, 128, 64, [5000, 1], {}),
    (7, 7, 128, 7, [0, 13, 500], {}),
    (6, 2, 64, 1, [1, 2, 3, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 0], {}),
    (64, 8, 128, 16, [1, 4097, 0, 333, 2048, 16, 15, 900], {}),
    (32, 2, 128, 128, [700, 1300], {}),          # 16 query heads to a kv-head
    (48, 2, 64, 32, [700, 41], {}),              # 24
    (80, 1, 128, 32, [515, 64], {}),             # 80
    (16, 8, 128, 256, [1000, 3], {"window": 100}),
    (16, 8, 128, 32, [1000, 50, 4, 0], {"window": 100, "sinks": 4}),
    (8, 8, 64, 16, [1000, 17, 1], {"window": 1}),
    (8, 8, 64, 16, [1000, 17, 1], {"window": 1, "sinks": 1}),
    (8, 4, 128, 48, [777, 95, 96, 97], {"window": 64, "sinks": 33}),
    (8, 4, 128, 48, [777, 95], {"window": 10 ** 10, "sinks": 10 ** 10}),
    (8, 4, 128, 64, [3000, 200], {"sinks": 7}),  # no window: sinks are not read
    (32, 8, 128, 32, [2500, 64], {"softcap": 50.0}),
    (32, 8, 64, 32, [2500, 64], {"softcap": 2.0, "window": 300, "sinks": 2}),
    (16, 4, 128, 16, [1500, 1], {"alibi": True}),
    (12, 4, 64, 16, [900, 77], {"alibi": True, "softcap": 20.0}),
    (4, 2, 128, 16, [400], {"alibi": True, "alibi_slopes": [0.5, 0.0, -0.01, 2.0], "window": 120, "sinks": 5}),
    (8, 2, 128, 16, [300], {"scale": 0.5}),
    (8, 2, 128, 16, [300], {"scale": -0.1}),
    (8, 2, 128, 16, [300], {"scale": 0.0}),
]


def _slopes(options, Hq):
    if not options.get("alibi"):
        return None
    return options.get("alibi_slopes") or odf.alibi_slopes(Hq)


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("case", DECODE, ids=lambda c: f"hq{c[0]}hkv{c[1]}d{c[2]}p{c[3]}n{max(c[4])}" + "".join(c[5]))
def test_decode(case, kv):
    Hq, Hkv, D, page, lens, options = case
    layout = "NHD" if (Hq + page) % 3 == 0 else "HND"
    cache = ref.Cache(lens, Hkv=Hkv, D=D, page=page, kv=kv, layout=layout, seed=Hq + D)
    q = _q(len(lens), Hq, D)
    want = {k: v for k, v in options.items() if k in ("window", "sinks", "softcap", "scale")}
    for out_dtype in (torch.bfloat16, torch.float32):
        o, lse = _decode(cache, q, out_dtype=out_dtype, **options)
        ref.check_decode(o, lse, q, cache, slopes=_slopes(options, Hq), what=f"{kv} {layout} {out_dtype}", **want)


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("D", [64, 128])
def test_decode_random_batches(kv, D):
    """Many sequences of every length: work split over the cache's length and over sequences."""
    g = torch.Generator().manual_seed(D)
    for B, hi, Hkv, group, page in ((1, 30000, 2, 3, 16), (5, 6000, 4, 8, 64), (70, 900, 2, 5, 16), (300, 60, 3, 1, 8),
                                    (200, 20, 4, 2, 16), (90, 5000, 3, 12, 16)):
        lens = torch.randint(0, hi, (B,), generator=g).tolist()
        if hi == 20:
            lens[77], lens[140] = 9000, 1400  # two long ones among many short
        cache = ref.Cache(lens, Hkv=Hkv, D=D, page=page, kv=kv, seed=B)
        q = _q(B, Hkv * group, D, seed=B)
        o, lse = _decode(cache, q, out_dtype=torch.bfloat16)
        ref.check_decode(o, lse, q, cache, what=f"B{B}")
        again, lse2 = _decode(cache, q, out_dtype=torch.bfloat16)
        assert torch.equal(o, again) and torch.equal(lse, lse2)  # the same answer each time


def test_decode_large_scores_and_values():
    """Scores far apart (one key takes all the weight), and a query of the largest bf16 sizes over an 8-bit cache."""
    for kv in ("bf16", "e4m3"):
        cache = ref.Cache([700, 45], Hkv=2, D=128, page=16, kv=kv, seed=3, k_gain=1.0)
        for gain in (1e-30, 30.0, 3e4):
            q = (_q(2, 8, 128).float() * gain).to(torch.bfloat16)
            scale = 0.3 / max(gain, 1.0)
            o, lse = _decode(cache, q, scale=scale, out_dtype=torch.bfloat16)
            ref.check_decode(o, lse, q, cache, scale=scale, what=f"{kv} gain {gain}")


def test_decode_nonfinite_where_visible():
    """NaN in a visible key or value reaches the output, +-inf as the formula has it; other heads are untouched."""
    cache = ref.Cache([100], Hkv=3, D=64, page=16, seed=5)
    page, slot = int(cache.table[0, 2]), 3
    cache.k[page, 0, slot, 5] = float("nan")
    cache.v[page, 1, slot, 7] = float("inf")
    q = _q(1, 3, 64)
    o, lse = _decode(cache, q, out_dtype=torch.float32)
    assert torch.isnan(o[0, 0]).all() and torch.isnan(lse[0, 0])
    assert o[0, 1, 7] == math.inf and torch.isfinite(o[0, 1, :7]).all() and torch.isfinite(o[0, 1, 8:]).all()
    assert torch.isfinite(o[0, 2]).all() and torch.isfinite(lse[0, 1:]).all()
    # out of the window the same keys are not seen
    o, lse = _decode(cache, q, out_dtype=torch.float32, window=100 - 36, sinks=35)
    assert torch.isfinite(o).all() and torch.isfinite(lse).all()


def test_decode_many_heads_with_generated_slopes():
    """More heads than explicit slopes may have: the kernel works them out itself."""
    cache = ref.Cache([300, 20], Hkv=40, D=64, page=16, seed=12)
    q = _q(2, 320, 64)
    o, lse = _decode(cache, q, alibi=True, out_dtype=torch.bfloat16)
    ref.check_decode(o, lse, q, cache, slopes=odf.alibi_slopes(320))


def test_decode_shared_pages_and_repeated_sequences():
    """Tables that name the same pages (a fork before it is written), one of them cut short."""
    cache = ref.Cache([700], Hkv=2, D=128, page=16, seed=13)
    q = _q(3, 8, 128)
    many = ref.Cache.__new__(ref.Cache)
    many.__dict__.update(cache.__dict__)
    many.table = cache.table.expand(3, -1).contiguous()
    many.lens_list = [700, 700, 333]
    many.lens = torch.tensor(many.lens_list, dtype=torch.int32, device="cuda")
    o, lse = _decode(many, q, out_dtype=torch.bfloat16)
    ref.check_decode(o, lse, q, many)


def test_decode_table_wider_than_the_lengths():
    """Room for a million tokens, and one token: what the table could hold is no work."""
    cache = ref.Cache([1, 0, 40], Hkv=2, D=64, page=16, seed=14, max_pages=65536)
    q = _q(3, 4, 64)
    o, lse = _decode(cache, q)
    ref.check_decode(o, lse, q, cache)


def test_decode_strided_and_given_outputs():
    lens = [500, 20]
    cache = ref.Cache(lens, Hkv=2, D=128, page=16, seed=8, max_pages=40)
    wide = torch.full((2, 12, 256), float("nan"), device="cuda", dtype=torch.bfloat16)
    q = wide[:, 1:9, 128:]
    q.copy_(_q(2, 8, 128))
    out = torch.full((2, 16, 128), 7.0, device="cuda", dtype=torch.bfloat16)[:, ::2]
    lse = torch.empty((2, 8), device="cuda")
    table = torch.full((2, 64), -5, dtype=torch.int32, device="cuda")
    table[:, :40] = cache.table
    o, l = odf.paged_decode(q, cache.k, cache.v, table[:, :40], cache.lens, out=out, lse_out=lse)
    assert o is out and l is lse
    ref.check_decode(o, l, q, cache)
    assert (out._base[:, 1::2] == 7).all()
    o, l = odf.paged_decode(q, cache.k, cache.v, table[:, :40], cache.lens, want_lse=False)
    assert l is None
    ref.check_decode(o, None, q, cache)


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
def test_decode_and_append_with_unlike_layouts(kv):
    """K as [page, head, slot], V as [page, slot, head] with a gap between rows; the pages inside a larger pool."""
    cache = ref.Cache([333, 50, 7], Hkv=3, D=64, page=16, kv=kv, seed=21)
    pages = cache.k.shape[0]
    wide = torch.zeros((2 * pages, 16, 3, 64 + 32), device="cuda").to(cache.v.dtype)
    v = wide[::2, :, :, :64].transpose(1, 2)
    v.copy_(cache.v)
    cache.v = v
    q = _q(3, 9, 64)
    o, lse = _decode(cache, q)
    ref.check_decode(o, lse, q, cache)
    k = torch.randn((3, 3, 2, 64), device="cuda").to(torch.bfloat16)
    before = wide.float()
    odf.paged_append(k, k, cache.k, cache.v, cache.table, torch.tensor([3, 0, 5], device="cuda", dtype=torch.int32),
                     k_scale=cache.ks, v_scale=cache.vs)
    got = cache.v[int(cache.table[0, 0]), :, 3:5].float()
    want = k[0].float() if kv == "bf16" else ref.to_e4m3((k[0].float() / cache.vs.view(-1, 1, 1)).double()).float()
    assert torch.equal(got, want)
    assert torch.equal(torch.nan_to_num(wide[1::2].float()), torch.nan_to_num(before[1::2]))
    assert torch.equal(wide[..., 64:].float(), before[..., 64:])


def test_decode_beyond_32_bits():
    """Pages whose byte offsets need more than 32 bits."""
    Hkv, D, page = 8, 128, 64
    row = Hkv * page * D
    pages = (1 << 32) // (row * 2) + 40
    pool = torch.zeros((pages, Hkv, page, D), device="cuda", dtype=torch.bfloat16)
    cache = ref.Cache([1000], Hkv=Hkv, D=D, page=page, seed=9)
    n = 16
    top = torch.arange(pages - n, pages, device="cuda")
    pool[top] = cache.k[cache.table[0, :n].long()]
    vpool = torch.zeros_like(pool)
    vpool[top] = cache.v[cache.table[0, :n].long()]
    table = top.to(torch.int32).view(1, -1)
    q = _q(1, 8, D)
    o, lse = odf.paged_decode(q, pool, vpool, table, cache.lens, out_dtype=torch.bfloat16)
    ref.check_decode(o, lse, q, cache)
    k = torch.randn((1, Hkv, 1, D), device="cuda").to(torch.bfloat16)
    odf.paged_append(k, -k, pool, vpool, table, cache.lens)
    assert torch.equal(pool[pages - 1, :, 1000 % page], k[0, :, 0])
    assert torch.equal(vpool[pages - 1, :, 1000 % page], -k[0, :, 0])
    odf.page_copy(pool, vpool, [(pages - 1, 0), (pages - 2, 5)])
    assert torch.equal(pool[0].view(torch.int16), pool[pages - 1].view(torch.int16))
    assert torch.equal(vpool[5].view(torch.int16), vpool[pages - 2].view(torch.int16))


def test_decode_other_stream_and_two_at_once():
    """Launches on side streams, each with a workspace of its own, give the default stream's results."""
    caches = [ref.Cache([4000 + 100 * i, 37], Hkv=2, D=128, page=16, seed=i) for i in range(2)]
    qs = [_q(2, 8, 128, seed=i) for i in range(2)]
    want = [_decode(c, q) for c, q in zip(caches, qs)]
    spaces = [odf.paged_decode_workspace(2, 8, 2, 128) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for rep in range(5):
        for c, q, w, s in zip(caches, qs, spaces, streams):
            got.append(_decode(c, q, workspace=w, stream=s.cuda_stream))
    got.append(_decode(caches[1], qs[1], stream=streams[0]))  # makes its own workspace there
    torch.cuda.synchronize()
    for i, (o, lse) in enumerate(got[:-1]):
        assert torch.equal(o, want[i % 2][0]) and torch.equal(lse, want[i % 2][1])
    assert torch.equal(got[-1][0], want[1][0])


def test_decode_in_graphs_that_share_a_workspace():
    """Two captured steps (append, then attention) over one workspace, replayed in turn as lengths grow."""
    cache = ref.Cache([100, 0, 515], Hkv=2, D=64, page=16, seed=4, max_pages=40, spare=8)
    spare = [int(x) for x in set(range(cache.k.shape[0])) - set(cache.table[cache.table < 2 ** 30].tolist())]
    cache.table[0, 7], cache.table[1, 0], cache.table[2, 33] = spare[:3]
    ws = odf.paged_decode_workspace(3, 8, 2, 64)
    k, v = (torch.zeros((3, 2, 1, 64), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    q = _q(3, 8, 64)
    outs = [torch.empty((3, 8, 64), device="cuda") for _ in range(2)]
    lses = [torch.empty((3, 8), device="cuda") for _ in range(2)]

    def step(i):
        odf.paged_append(k, v, cache.k, cache.v, cache.table, cache.lens)
        cache.lens.add_(1)
        odf.paged_decode(q, cache.k, cache.v, cache.table, cache.lens, out=outs[i], lse_out=lses[i], workspace=ws,
                         window=300 if i else 0, sinks=3)

    odf.paged_decode(q, cache.k, cache.v, cache.table, cache.lens, workspace=ws)  # sets the device up
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for i, g in enumerate(graphs):
        with torch.cuda.graph(g):
            step(i)
    for n in range(6):
        k.normal_()
        v.normal_()
        q.normal_()
        graphs[n % 2].replay()
        torch.cuda.synchronize()
        cache.lens_list = [x + 1 for x in cache.lens_list]
        assert cache.lens.tolist() == cache.lens_list
        assert torch.equal(cache.rows(1)[0][:, -1].float(), k[1, :, 0].float())
        ref.check_decode(outs[n % 2], lses[n % 2], q, cache, window=300 if n % 2 else 0, sinks=3, what=f"step {n}")
    del graphs


# --------------------------------------------------------------------------------------- append
@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("layout", ["HND", "NHD"])
@pytest.mark.parametrize("B,Hkv,T,D,page", [(1, 1, 1, 64, 16), (3, 2, 1, 128, 1), (4, 3, 37, 64, 7), (2, 8, 300, 128, 64),
                                            (65, 2, 5, 128, 16)])
def test_append(kv, layout, B, Hkv, T, D, page):
    g = torch.Generator().manual_seed(T)
    starts = torch.randint(0, 3 * page, (B,), generator=g).tolist()
    counts = torch.randint(0, T + 1, (B,), generator=g).tolist()
    for with_counts in (False, True):
        n = counts if with_counts else [T] * B
        cache = ref.Cache([a + m for a, m in zip(starts, n)], Hkv=Hkv, D=D, page=page, kv=kv, layout=layout, seed=T)
        k, v = (torch.randn((B, T, Hkv, D), device="cuda").to(torch.bfloat16).transpose(1, 2) for _ in range(2))
        for b in range(B):  # a padded batch: what lies behind a sequence's tokens is not read
            k[b, :, n[b]:] = float("nan")
        if kv == "e4m3" and n[0]:
            k[0, 0, 0, :6] = torch.tensor([1e30, -1e30, math.inf, -math.inf, math.nan, 0.0])
        before = [x.float() for x in (cache.k, cache.v)]
        odf.paged_append(k, v, cache.k, cache.v, cache.table, torch.tensor(starts, dtype=torch.int32, device="cuda"),
                         counts=torch.tensor(n, dtype=torch.int32, device="cuda") if with_counts else None,
                         k_scale=cache.ks, v_scale=cache.vs)
        for new, pages, old, scale in ((k, cache.k, before[0], cache.ks), (v, cache.v, before[1], cache.vs)):
            want = old.double()
            for b in range(B):
                pos = torch.arange(starts[b], starts[b] + n[b], device="cuda")
                x = new[b, :, :n[b]].double()
                if scale is not None:
                    # the quotient in fp32 first: the kernel divides there, and the second rounding is what it stores
                    x = (x.float() / scale.view(-1, 1, 1)).double()
                    x = ref.to_e4m3(x)
                want[cache.table[b][pos // page].long(), :, pos % page] = x.transpose(0, 1)
            assert torch.equal(torch.nan_to_num(pages.float(), nan=12345.0), torch.nan_to_num(want.float(), nan=12345.0))


def test_append_rounds_every_value_as_the_quotient():
    """All bf16 values over scales of every kind: the e4m3 value of the fp32 quotient, ties and subnormals included."""
    x = torch.arange(65536, device="cuda", dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    scales = [1.0, 1 / 64, 0.015625 * 1.5, 0.1, 1 / 3, 7.123e-3, 0.99999994, 1.0000001, 3e-39, 1e38, 2.0 ** -126, 2.0 ** 127,
              2.0 ** 100, 1.1e-30, 5.0, 1e-45]
    Hkv, D, page = len(scales), 128, 64
    tokens = 65536 // D
    k = x.view(1, 1, tokens, D).expand(1, Hkv, tokens, D).contiguous()
    s = torch.tensor(scales, device="cuda")
    table = torch.arange(tokens // page, device="cuda", dtype=torch.int32).view(1, -1)
    pages = [torch.zeros((tokens // page, Hkv, page, D), device="cuda").to(torch.float8_e4m3fn) for _ in range(2)]
    odf.paged_append(k, k.flip(1), pages[0], pages[1], table, torch.zeros(1, device="cuda", dtype=torch.int32),
                     k_scale=s, v_scale=s.flip(0))
    want = ref.to_e4m3((k[0].float() / s.view(-1, 1, 1)).double())
    got = pages[0].transpose(0, 1).reshape(Hkv, tokens, D).float()
    assert torch.equal(torch.nan_to_num(got, nan=999.0), torch.nan_to_num(want.float(), nan=999.0))
    got = pages[1].transpose(0, 1).reshape(Hkv, tokens, D).float().flip(0)
    assert torch.equal(torch.nan_to_num(got, nan=999.0), torch.nan_to_num(want.float(), nan=999.0))


# ----------------------------------------------------------------------------------------- copy
@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("layout", ["HND", "NHD", "padded"])
@pytest.mark.parametrize("layers,P,Hkv,page,D,n", [(0, 9, 3, 7, 64, 3), (1, 4, 1, 1, 128, 2), (3, 40, 2, 16, 64, 17),
                                                   (2, 1100, 1, 2, 64, 500)])
def test_copy(kv, layout, layers, P, Hkv, page, D, n):
    dtype = torch.bfloat16 if kv == "bf16" else torch.float8_e4m3fn
    L = max(layers, 1)

    def make():
        if layout == "HND":
            x = torch.randn((L, P, Hkv, page, D), device="cuda").to(dtype)
        elif layout == "NHD":
            x = torch.randn((L, P, page, Hkv, D), device="cuda").to(dtype).transpose(2, 3)
        else:  # rows with a gap between them
            x = torch.randn((L, P, Hkv, page, D + 32), device="cuda").to(dtype)[..., :D]
        return x if layers else x[0]

    k, v = make(), make()
    g = torch.Generator().manual_seed(n)
    ids = torch.randperm(P, generator=g)
    src, dst = ids[:n], ids[n:2 * n]
    src = src[torch.randint(0, n, (n,), generator=g)]  # a page may be read more than once
    base = [(x._base if x._base is not None else x) for x in (k, v)]
    want = []
    for x in (k, v):
        w = x.float() if layers else x.float()[None]
        w[:, dst] = w[:, src]
        want.append(w if layers else w[0])
    gaps = [b[..., D:].float().clone() for b in base] if layout == "padded" else []
    odf.page_copy(k, v, torch.stack([src, dst], 1))
    assert torch.equal(k.float(), want[0]) and torch.equal(v.float(), want[1])
    for b, g0 in zip(base, gaps):
        assert torch.equal(b[..., D:].float(), g0)
    odf.page_copy(k, v, [])
    assert torch.equal(k.float(), want[0])


def test_copy_captured():
    k, v = (torch.randn((2, 8, 2, 16, 64), device="cuda").to(torch.bfloat16) for _ in range(2))
    odf.page_copy(k, v, [(0, 1)])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        odf.page_copy(k, v, [(2, 7), (3, 6)])
    k.normal_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(k[:, 7], k[:, 2]) and torch.equal(k[:, 6], k[:, 3]) and torch.equal(v[:, 7], v[:, 2])
    del graph


def test_refusals_of_the_binding():
    cache = ref.Cache([20, 30], Hkv=2, D=64, page=16)
    q = _q(2, 4, 64)
    ok = dict(q=q, k_pages=cache.k, v_pages=cache.v, page_table=cache.table, lens=cache.lens)
    for over in (dict(lens=cache.lens.long()), dict(lens=cache.lens[:1]), dict(page_table=cache.table[:1]),
                 dict(page_table=cache.table.long()), dict(q=q.float()), dict(q=q[..., :32]), dict(q=_q(2, 3, 64)),
                 dict(k_pages=cache.k.half()), dict(v_pages=cache.v[:1]), dict(lens=cache.lens.cpu()),
                 dict(k_scale=torch.ones(2, device="cuda")), dict(window=-1), dict(out=torch.empty((2, 4, 63), device="cuda")),
                 dict(alibi=True, alibi_slopes=[1.0]), dict(workspace=torch.zeros(8, dtype=torch.uint8, device="cuda")),
                 dict(lse_out=torch.empty((2, 3), device="cuda"))):
        with pytest.raises(ValueError):
            odf.paged_decode(**{**ok, **over})
    for n in (1, 40):  # few and many pairs take different ways
        for bad in ((0, cache.k.shape[0]), (-1, 0), (0, 2 ** 32 + 1)):
            with pytest.raises(ValueError, match="outside"):
                odf.page_copy(cache.k, cache.v, [bad] * n)
            with pytest.raises(ValueError, match="outside"):
                odf.page_copy(cache.k, cache.v, torch.tensor([bad] * n))
        for bad in ([(0, 1, 2)] * n, [0] * n, torch.rand(n, 2), [(0.5, 1)] * n):
            with pytest.raises(ValueError, match="integers"):
                odf.page_copy(cache.k, cache.v, bad)
        with pytest.raises(ValueError, match="read" if n == 1 else "twice"):
            odf.page_copy(cache.k, cache.v, [(0, 0)] * n)


# ------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
def test_bad_pages_are_reported(kv):
    """A page id out of range, a length beyond the table: no access out of range, a status, other sequences right."""
    cache = ref.Cache([100, 200, 60], Hkv=2, D=64, page=16, kv=kv, seed=6)
    good = cache.table.clone()
    q = _q(3, 4, 64)
    for at, value in (((0, 2), -1), ((0, 6), cache.k.shape[0]), ((0, 0), 2 ** 31 - 1), ((0, 0), -2 ** 31)):
        cache.table = good.clone()
        cache.table[at] = value
        o, lse = _decode(cache, q)
        torch.cuda.synchronize()
        assert odf.device_status() == odf.ODF_ERR_BAD_PAGE
        cache.table = good
        sub = [1, 2]
        part = ref.Cache.__new__(ref.Cache)
        part.__dict__.update(cache.__dict__)
        part.table, part.lens_list = good[sub], [200, 60]
        ref.check_decode(o[sub], lse[sub], q[sub], part)
    lens = cache.lens.clone()
    lens[1] = 10 ** 6
    lens[2] = -5
    o, lse = odf.paged_decode(q, cache.k, cache.v, good, lens, k_scale=cache.ks, v_scale=cache.vs)
    torch.cuda.synchronize()
    assert odf.device_status() == odf.ODF_ERR_BAD_PAGE
    assert (o[2] == 0).all() and (lse[2] == -math.inf).all()
    before = cache.k.float().clone()
    k = torch.randn((3, 2, 4, 64), device="cuda").to(torch.bfloat16)
    for starts, table in (([-3, -2 ** 31, 2 ** 31 - 1], good), ([10 ** 6, 13 * 16, 2 ** 31 - 2], good),
                          ([0, 0, 0], torch.full_like(good, -7))):
        odf.paged_append(k, k, cache.k, cache.v, table, torch.tensor(starts, dtype=torch.int32, device="cuda"),
                         counts=torch.tensor([3, 4, 4], dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        assert odf.device_status() == odf.ODF_ERR_BAD_PAGE
        assert torch.equal(torch.nan_to_num(cache.k.float(), nan=5.0), torch.nan_to_num(before, nan=5.0))
