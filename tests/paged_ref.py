"""64-bit reference of the serving operators, written from their definitions, and the error bounds
that the GPU tests hold the kernels to."""
from __future__ import annotations

import math

import torch

# half a step of each type, relative to the value
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def visible(p, j, n, window, sinks):
    """Truth values [rows, keys]: which of the keys j (of n) the rows at positions p see (window 0: all up to p)."""
    d = p[:, None] - j[None, :]
    seen = (d >= 0) & (j[None, :] < n)
    if window:
        seen &= (d < window) | (j[None, :] < sinks)
    return seen


def attend(q, k, v, p, n, *, window=0, sinks=0, scale, slopes=None, softcap=0.0, p_type=torch.bfloat16,
           out_type=torch.bfloat16):
    """q [H, M, D], k, v [H, N, D] float64; p [M] positions.  Returns (o, lse, o_tol, lse_tol).

    The bounds count what a kernel that is right may lose:
      score    D products summed in fp32 (in any order), the scale, the ALiBi term and the soft-cap:
               ds <= 2^-24 (D + 8) (scale sum|q k| + |bias|) [+ 1e-5 softcap for its tanh]
      LSE      ds, exponentials good to 2^-21, a sum of n terms in fp32 whose longest chain is below n / 16 + 64,
               and the result's own rounding
      O        every weight off by 2 ds + 2^-20 (its own and the sum's) and rounded to p_type, the products
               summed in fp32, the result rounded to out_type
    """
    j = torch.arange(k.shape[1], device=k.device)
    seen = visible(p, j, n, window, sinks)
    k = k.clone()
    v = v.clone()
    hidden = ~seen.any(0)  # keys no row sees may hold anything
    k[:, hidden] = 0
    v[:, hidden] = 0
    s = torch.matmul(q, k.transpose(1, 2)) * scale
    size = torch.matmul(q.abs(), k.abs().transpose(1, 2)) * abs(scale)
    if slopes is not None:
        bias = slopes.view(-1, 1, 1) * (j[None, :] - p[:, None]).double()
        s = s + bias
        size = size + bias.abs()
    ds = 2.0 ** -24 * (k.shape[2] + 8) * size
    if softcap:
        s = softcap * torch.tanh(s / softcap)
        ds = ds + 1e-5 * softcap
    s = s.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1)
    w = torch.exp(s - lse.unsqueeze(-1)).masked_fill(~seen, 0.0)
    o = torch.matmul(w, v)
    mass = torch.matmul(w, v.abs())
    ds = ds.masked_fill(~seen, 0.0).amax(-1) if s.shape[-1] else torch.zeros_like(lse)
    chain = seen.sum(-1).double() / 16 + 64
    lse_tol = ds + 2.0 ** -21 + 2.0 ** -24 * (chain + 4 * torch.where(torch.isinf(lse), 0.0, lse.abs()))
    rel = 2 * ds + 2.0 ** -20 + HALF[p_type] + HALF[out_type] + 2.0 ** -24 * chain
    o_tol = mass * rel.unsqueeze(-1) + 1e-30
    return o, lse, o_tol, lse_tol


def check(o, lse, ref, what=""):
    o_ref, lse_ref, o_tol, lse_tol = ref
    off = (o.double() - o_ref).abs()
    bad = ~(off <= o_tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} outputs off, worst {float((off / o_tol).max()):.2f} of the bound"
    if lse is not None:
        empty = torch.isinf(lse_ref)
        assert torch.equal(torch.isinf(lse) & (lse < 0), empty), f"{what}: empty rows"
        off = (lse.double() - lse_ref).abs()[~empty]
        bad = ~(off <= lse_tol[~empty])
        assert not bad.any(), f"{what}: {int(bad.sum())} LSEs off, worst {float((off / lse_tol[~empty]).max()):.2f}"


def to_e4m3(x):
    """Nearest e4m3 value of float64 x (ties to even), saturated at +-448, as float64; NaN stays."""
    c = x.clamp(-448.0, 448.0)
    e = torch.floor(torch.log2(c.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    return torch.round(c / step) * step


class Cache:
    """A paged cache of sequences with the given lengths, every slot that holds no token filled with NaN."""

    def __init__(self, lens, *, Hkv, D, page, kv="bf16", layout="HND", seed=0, spare=2, max_pages=None, scales=True,
                 device="cuda", k_gain=1.0):
        g = torch.Generator(device=device).manual_seed(seed)
        counts = [-(-n // page) for n in lens]
        total = sum(counts) + spare
        width = max([1] + counts) if max_pages is None else max_pages
        perm = torch.randperm(total, generator=g, device=device).to(torch.int32)
        self.table = torch.full((len(lens), width), 2 ** 31 - 1, dtype=torch.int32, device=device)
        self.lens_list, self.page, self.Hkv, self.D = list(lens), page, Hkv, D
        self.lens = torch.tensor(lens, dtype=torch.int32, device=device)
        shape = (total, Hkv, page, D)
        k, v = (torch.full(shape, float("nan"), device=device, dtype=torch.float32) for _ in range(2))
        at = 0
        for b, (n, c) in enumerate(zip(lens, counts)):
            self.table[b, :c] = perm[at:at + c]
            for i in range(c):
                m = min(page, n - i * page)
                for x, gain in ((k, k_gain), (v, 1.0)):
                    x[int(perm[at + i]), :, :m] = torch.randn((Hkv, m, D), generator=g, device=device) * gain
            at += c
        self.kv = kv
        if kv == "bf16":
            dtype = torch.bfloat16
            self.ks = self.vs = None
        else:
            dtype = torch.float8_e4m3fn
            k, v = k * 60.0, v * 60.0
            self.ks = (torch.rand(Hkv, generator=g, device=device) + 0.5) / 60.0 if scales else None
            self.vs = (torch.rand(Hkv, generator=g, device=device) + 0.5) / 60.0 if scales else None
        if layout == "HND":
            self.k, self.v = k.to(dtype), v.to(dtype)
        else:  # [pages, slots, heads, D] in memory
            self.k, self.v = (x.transpose(1, 2).contiguous().to(dtype).transpose(1, 2) for x in (k, v))

    def rows(self, b):
        """K and V of sequence b as float64 [Hkv, n, D]."""
        n = self.lens_list[b]
        pages = self.table[b, :-(-n // self.page)].long()
        out = []
        for x, s in ((self.k, self.ks), (self.v, self.vs)):
            r = x.float()[pages].double().transpose(0, 1).reshape(self.Hkv, -1, self.D)[:, :n]
            out.append(r if s is None else r * s.double().view(-1, 1, 1))
        return out


def check_decode(o, lse, q, cache, *, window=0, sinks=0, softcap=0.0, slopes=None, scale=None, what=""):
    B, Hq, D = q.shape
    g = Hq // cache.Hkv
    p_type = torch.bfloat16 if cache.kv == "bf16" else torch.float16
    for b, n in enumerate(cache.lens_list):
        if n == 0:
            assert (o[b] == 0).all() and (lse is None or (lse[b] == -math.inf).all()), what
            continue
        k, v = cache.rows(b)
        k, v = (x.repeat_interleave(g, 0) for x in (k, v))
        sl = None if slopes is None else torch.tensor(slopes, dtype=torch.float64, device=q.device)
        ref = attend(q[b].double().unsqueeze(1), k, v, torch.tensor([n - 1], device=q.device), n, window=window, sinks=sinks,
                     scale=scale if scale is not None else 1 / math.sqrt(D), slopes=sl, softcap=softcap, p_type=p_type,
                     out_type=o.dtype)
        check(o[b].unsqueeze(1), None if lse is None else lse[b].unsqueeze(1), ref, f"{what} sequence {b} of {n}")
