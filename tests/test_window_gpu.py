"""Sliding-window attention with sinks on the GPU against a 64-bit reference."""
from __future__ import annotations

import json
import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import odf_b200 as odf
import paged_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean_status():
    yield
    assert odf.device_status() == 0


def _qkv(B, Hq, Hkv, M, N, D, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(s, generator=g, device="cuda").to(torch.bfloat16)
            for s in ((B, Hq, M, D), (B, Hkv, N, D), (B, Hkv, N, D))]


def _check(o, lse, q, k, v, *, window, sinks=0, q_offset=0, softcap=0.0, slopes=None, scale=None, rows=None, what=""):
    B, Hq, M, D = q.shape
    G = Hq // k.shape[1]
    rows = torch.arange(M, device="cuda") if rows is None else rows
    sl = None if slopes is None else torch.tensor(slopes, dtype=torch.float64, device="cuda")
    for b in range(B):
        kb, vb = (x[b].double().repeat_interleave(G, 0) for x in (k, v))
        r = ref.attend(q[b][:, rows].double(), kb, vb, q_offset + rows, k.shape[2], window=window, sinks=sinks,
                       scale=1 / math.sqrt(D) if scale is None else scale, slopes=sl, softcap=softcap,
                       out_type=o.dtype)
        ref.check(o[b][:, rows], None if lse is None else lse[b][:, rows], r, f"{what} batch {b}")


CASES = [
    # B, Hq, Hkv, M, N, D, window, sinks, q_offset
    (1, 2, 2, 1, 1, 64, 1, 0, 0),
    (1, 2, 2, 1, 1, 128, 5, 3, 0),
    (1, 4, 4, 512, 512, 64, 100, 4, 0),
    (1, 4, 2, 512, 512, 128, 128, 0, 0),
    (2, 2, 1, 333, 333, 128, 1, 0, 0),
    (2, 2, 1, 333, 333, 128, 1, 1, 0),
    (1, 2, 2, 700, 700, 64, 127, 129, 0),
    (1, 2, 2, 700, 700, 128, 129, 300, 0),
    (1, 2, 2, 257, 257, 128, 10 ** 12, 0, 0),      # plain causal
    (1, 2, 2, 257, 257, 64, 64, 10 ** 12, 0),      # every key a sink
    (1, 3, 1, 130, 1000, 128, 200, 4, 870),        # a chunk
    (1, 3, 1, 1, 1000, 64, 200, 4, 999),           # one token
    (1, 2, 2, 1000, 3000, 128, 777, 16, 2000),
    (1, 2, 2, 300, 2000, 128, 5000, 0, 1700),      # causal chunk
    (1, 2, 2, 300, 2000, 128, 100, 130, 500),      # keys that no row has reached yet
    (1, 2, 2, 600, 400, 128, 100, 0, 0),           # rows past the last key: the last ones see nothing
    (1, 2, 2, 600, 400, 64, 100, 2, 0),            # but the sinks
    (1, 2, 2, 200, 400, 128, 50, 0, 1000),         # no row sees anything
    (1, 2, 2, 200, 400, 64, 50, 7, 1000),          # the sinks only
    (3, 8, 2, 1500, 1500, 128, 384, 128, 0),
    (1, 8, 1, 100, 8192, 128, 4000, 4, 8092),      # few rows, split over the keys
    (1, 4, 1, 40, 9000, 64, 8000, 200, 8960),
    (1, 2, 2, 4096, 4096, 128, 1000, 5, 0),
]
MODS = [{}, {"softcap": 30.0}, {"alibi": True}, {"alibi": True, "softcap": 30.0}]


@pytest.mark.parametrize("mod", range(4), ids=["plain", "softcap", "alibi", "alibi_softcap"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "_".join(str(x) for x in c))
def test_window(case, mod):
    B, Hq, Hkv, M, N, D, window, sinks, off = case
    q, k, v = _qkv(B, Hq, Hkv, M, N, D, seed=M + mod)
    o, lse = odf.flash_fwd_window(q, k, v, window=window, sinks=sinks, q_offset=off,
                                  out_dtype=torch.bfloat16 if mod % 2 else torch.float32, **MODS[mod])
    _check(o, lse, q, k, v, window=window, sinks=sinks, q_offset=off, softcap=MODS[mod].get("softcap", 0.0),
           slopes=odf.alibi_slopes(Hq) if MODS[mod].get("alibi") else None)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("sinks", [0, 4, 200])
def test_keys_that_no_row_sees_may_be_nan(D, sinks):
    """Evicted keys between the sinks and the window, and room for tokens to come."""
    M, N, off, window = 300, 3000, 2000, 500
    q, k, v = _qkv(1, 4, 2, M, N, D, seed=D)
    want, want_l = odf.flash_fwd_window(q, k, v, window=window, sinks=sinks, q_offset=off)
    lo, hi = off - window + 1, off + M
    for bad in (float("nan"), float("inf")):
        for x in (k, v):
            x[:, :, sinks:lo] = bad
            x[:, :, hi:] = bad
        o, lse = odf.flash_fwd_window(q, k, v, window=window, sinks=sinks, q_offset=off)
        assert torch.equal(o, want) and torch.equal(lse, want_l)


def test_window_of_everything_is_the_causal_forward():
    q, k, v = _qkv(2, 4, 2, 700, 700, 128)
    o, lse = odf.flash_fwd_window(q, k, v, window=700)
    o2, lse2 = odf.flash_fwd(q, k, v, causal=True)
    bound = 2.0 ** -7 * v.abs().max()  # two roundings of P to bf16, of values up to the largest
    assert (o - o2).abs().max() <= bound and (lse - lse2).abs().max() <= 1e-4


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("scale", [0.0, -0.1, 0.5, 3.0])
def test_scales_and_far_apart_scores(D, scale):
    """Scores that spread over hundreds (the running max moves late and often), or fall with the scale's sign."""
    q, k, v = _qkv(1, 4, 2, 1200, 1200, D, seed=5)
    k[:, :, 700:720] *= 8.0  # a few keys far above the others, in the middle of the windows
    for sinks in (0, 3):
        o, lse = odf.flash_fwd_window(q, k, v, window=500, sinks=sinks, scale=scale)
        _check(o, lse, q, k, v, window=500, sinks=sinks, scale=scale, what=f"scale {scale} sinks {sinks}")


def test_strides_given_outputs_and_a_side_stream():
    B, H, M, D = 2, 4, 400, 128
    q, k, v = (torch.randn((B, M, H, D), device="cuda").to(torch.bfloat16).transpose(1, 2) for _ in range(3))
    want = odf.flash_fwd_window(q.contiguous(), k.contiguous(), v.contiguous(), window=90, sinks=3, out_dtype=torch.bfloat16)
    out = torch.zeros((B, M, H, D), device="cuda", dtype=torch.bfloat16).transpose(1, 2)
    lse = torch.zeros((B, H, M), device="cuda")
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    odf.flash_fwd_window(q, k, v, window=90, sinks=3, out=out, lse_out=lse, stream=stream)
    got = [odf.flash_fwd_window(q[:, :, -64:], k, v, window=350, sinks=3, q_offset=M - 64, stream=stream.cuda_stream)
           for _ in range(3)]
    torch.cuda.synchronize()
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    for o, l in got:
        _check(o, l, q[:, :, -64:], k, v, window=350, sinks=3, q_offset=M - 64)


def test_captured_and_replayed():
    q, k, v = _qkv(1, 4, 4, 128, 4096, 128)
    out, lse = torch.empty((1, 4, 128, 128), device="cuda"), torch.empty((1, 4, 128), device="cuda")
    kw = dict(window=3000, sinks=4, q_offset=4096 - 128, out=out, lse_out=lse)
    odf.flash_fwd_window(q, k, v, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        odf.flash_fwd_window(q, k, v, **kw)
    for _ in range(2):
        for t in (q, k, v):
            t.normal_()
        graph.replay()
        torch.cuda.synchronize()
        _check(out, lse, q, k, v, window=3000, sinks=4, q_offset=4096 - 128)
    del graph


@pytest.mark.parametrize("D", [64, 128])
def test_random_problems(D):
    g = torch.Generator().manual_seed(D)
    pick = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=g))  # noqa: E731
    for n in range(25):
        M = pick(1, 700)
        off = pick(0, 900) * pick(0, 1)
        N = max(1, off + M + pick(-60, 60))
        Hkv, G = pick(1, 3), pick(1, 4)
        window, sinks, mod = pick(1, 600), pick(0, 1) * pick(0, 300), MODS[pick(0, 3)]
        q, k, v = _qkv(pick(1, 2), Hkv * G, Hkv, M, N, D, seed=n)
        o, lse = odf.flash_fwd_window(q, k, v, window=window, sinks=sinks, q_offset=off, **mod)
        _check(o, lse, q, k, v, window=window, sinks=sinks, q_offset=off, softcap=mod.get("softcap", 0.0),
               slopes=odf.alibi_slopes(Hkv * G) if mod.get("alibi") else None,
               what=f"M{M} N{N} off{off} w{window} s{sinks} {mod}")


def test_long_prompt_sampled_rows():
    q, k, v = _qkv(1, 16, 2, 32768, 32768, 128)
    o, lse = odf.flash_fwd_window(q, k, v, window=4096, sinks=4, out_dtype=torch.bfloat16)
    rows = torch.tensor([0, 1, 4095, 4096, 4099, 4100, 20000, 32767], device="cuda")
    _check(o, lse, q, k, v, window=4096, sinks=4, rows=rows)


def test_checked_build_invariants_hold():
    """Work items, KV entries, ring loads and P.V counts of the window variants, counted in the kernel."""
    root = Path(__file__).resolve().parent.parent
    assert (root / "dnn-flash_b200" / "lib" / "libodf_sm100_checked.so").exists()
    proc = subprocess.run([sys.executable, str(root / "tests" / "checked_window_run.py")], capture_output=True, text=True,
                          timeout=600)
    assert proc.returncode == 0, proc.stderr[-3000:]
    results = [json.loads(line) for line in proc.stdout.splitlines() if line.startswith("{")]
    assert len(results) == 6
    for r in results:
        assert r["rc"] == 0 and r["check_bits"] == 0 and r["status"] == 0, r


# ------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
def test_serving_a_prompt_then_tokens(kv):
    """A prompt in two chunks, its keys appended to the cache, a fork of it, then tokens on both branches:
    every step against attention over all the tokens in 64 bits."""
    Hq, Hkv, D, page, window, sinks = 8, 2, 64, 16, 60, 3
    dtype = torch.bfloat16 if kv == "bf16" else torch.float8_e4m3fn
    pool = odf.PagePool(40, page)
    kp, vp = (torch.full((40, Hkv, page, D), float("nan"), device="cuda").to(dtype) for _ in range(2))
    scale = None if kv == "bf16" else torch.full((Hkv,), 1 / 64.0, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn((1, h, 150, D), generator=g, device="cuda").to(torch.bfloat16) for h in (Hq, Hkv, Hkv))
    a = pool.add()
    for lo, hi in ((0, 90), (90, 150)):
        o, lse = odf.flash_fwd_window(q[:, :, lo:hi], k[:, :, :hi], v[:, :, :hi], window=window, sinks=sinks, q_offset=lo)
        _check(o, lse, q[:, :, lo:hi], k[:, :, :hi], v[:, :, :hi], window=window, sinks=sinks, q_offset=lo)
        odf.page_copy(kp, vp, pool.extend(a, hi - lo))
        start = torch.tensor([lo], dtype=torch.int32, device="cuda")
        odf.paged_append(k[:, :, lo:hi], v[:, :, lo:hi], kp, vp, pool.table([a]).cuda(), start, k_scale=scale, v_scale=scale)
    b = pool.fork(a)
    held = {}
    for s in (a, b):  # what the cache stands for, in 64 bits
        hk, hv = (x[0].double() if kv == "bf16" else ref.to_e4m3(x[0].double() * 64) / 64 for x in (k, v))
        held[s] = [hk, hv]
    ws = odf.paged_decode_workspace(2, Hq, Hkv, D)
    for step in range(20):
        if step == 10:  # another sequence comes and goes, the cache is compacted
            c = pool.add()
            pool.extend(c, 100)
            pool.free(a)
            odf.page_copy(kp, vp, pool.compact())
            pool.free(c)
            odf.page_copy(kp, vp, pool.compact())
        live = [b] if step >= 10 else [a, b]
        n = len(live)
        pairs = [p for s in live for p in pool.extend(s, 1)]
        assert len(pairs) == (1 if step == 0 else 0)  # the fork's half-filled page
        odf.page_copy(kp, vp, pairs)
        nk, nv = (torch.randn((n, Hkv, 1, D), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
        nq = torch.randn((n, Hq, D), generator=g, device="cuda").to(torch.bfloat16)
        table = pool.table(live).cuda()
        lens = torch.tensor([pool.length(s) for s in live], dtype=torch.int32, device="cuda")
        odf.paged_append(nk, nv, kp, vp, table, lens - 1, k_scale=scale, v_scale=scale)
        o, lse = odf.paged_decode(nq, kp, vp, table, lens, window=window, sinks=sinks, k_scale=scale, v_scale=scale,
                                  workspace=ws)
        for i, s in enumerate(live):
            for x, new in zip((0, 1), (nk, nv)):
                row = new[i].double() if kv == "bf16" else ref.to_e4m3(new[i].double() * 64) / 64
                held[s][x] = torch.cat([held[s][x], row], 1)
            hk, hv = (x.repeat_interleave(Hq // Hkv, 0) for x in held[s])
            m = hk.shape[1]
            assert m == pool.length(s)
            r = ref.attend(nq[i].double().unsqueeze(1), hk, hv, torch.tensor([m - 1], device="cuda"), m, window=window,
                           sinks=sinks, scale=1 / math.sqrt(D), p_type=torch.bfloat16, out_type=torch.float32)
            ref.check(o[i].unsqueeze(1), lse[i].unsqueeze(1), r, f"step {step} sequence {i}")
