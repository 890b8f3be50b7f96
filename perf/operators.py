"""What the serving operators are measured on: windowed prefill attention, attention of one new token
over a paged key-value cache, appending to that cache, and copying its pages.

``run`` computes each operator in plain torch operations in 32 bits, or (``own = True``) through the
framework's Python binding.  Heads, head sizes and lengths are those of the configurations in bench.py
(4 heads x 64 over 512 tokens, 32 heads over 8192 with a soft-cap of 50, 8 heads over 8192 keys, 64 query
and 8 key-value heads over 32768) or generic.
"""
import math
import sys
from pathlib import Path

import torch

own = False

_PACKAGE = Path(__file__).resolve().parents[1] / "dnn-flash_b200"
_E4M3_MAX = 448.0


def _binding():
    if str(_PACKAGE) not in sys.path:
        sys.path.insert(0, str(_PACKAGE))
    import odf_b200

    return odf_b200


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # A short prompt of a small model: latency of one launch.
        {"name": "window_prompt_512", "op": "window", "B": 1, "Hq": 4, "Hkv": 4, "M": 512, "N": 512, "D": 64,
         "window": 100, "sinks": 4, "softcap": 0.0, "alibi": False, "out": "bf16"},
        # The next chunk of two long prompts, odd sizes, against what the cache already holds.
        {"name": "window_chunk_softcap", "op": "window", "B": 2, "Hq": 32, "Hkv": 32, "M": 1000, "N": 8193, "D": 128,
         "window": 2047, "sinks": 16, "softcap": 50.0, "alibi": False, "out": "bf16"},
        # A whole long prompt with grouped heads: the largest prefill.
        {"name": "window_prompt_32k_gqa", "op": "window", "B": 1, "Hq": 64, "Hkv": 8, "M": 32768, "N": 32768, "D": 128,
         "window": 4096, "sinks": 4, "softcap": 0.0, "alibi": False, "out": "bf16"},
        # One user's first tokens: the smallest decode step, all latency.
        {"name": "decode_one_short", "op": "decode", "B": 1, "Hq": 4, "Hkv": 4, "D": 64, "page": 16, "lo": 129,
         "hi": 129, "window": 0, "sinks": 0, "softcap": 0.0, "alibi": False, "kv": "bf16", "out": "bf16"},
        # One user, a long conversation, without grouped heads: split over the cache's length.
        {"name": "decode_one_8k", "op": "decode", "B": 1, "Hq": 8, "Hkv": 8, "D": 128, "page": 64, "lo": 8192,
         "hi": 8192, "window": 0, "sinks": 0, "softcap": 0.0, "alibi": False, "kv": "bf16", "out": "bf16"},
        # A serving batch of users at every point of their conversations: ragged lengths, the largest decode.
        {"name": "decode_batch_ragged", "op": "decode", "B": 64, "Hq": 64, "Hkv": 8, "D": 128, "page": 16, "lo": 1,
         "hi": 8192, "window": 0, "sinks": 0, "softcap": 0.0, "alibi": False, "kv": "bf16", "out": "bf16"},
        # A layer with a sliding window and sinks in such a batch, with a soft-cap.
        {"name": "decode_window_softcap", "op": "decode", "B": 32, "Hq": 32, "Hkv": 8, "D": 128, "page": 32,
         "lo": 700, "hi": 8192, "window": 1024, "sinks": 4, "softcap": 50.0, "alibi": False, "kv": "bf16",
         "out": "bf16"},
        # A few users with very long contexts over a cache held in 8 bits.
        {"name": "decode_32k_e4m3", "op": "decode", "B": 4, "Hq": 64, "Hkv": 8, "D": 128, "page": 64, "lo": 20000,
         "hi": 32768, "window": 0, "sinks": 0, "softcap": 0.0, "alibi": False, "kv": "e4m3", "out": "bf16"},
        # One new token per user of a batch: what every decode step does first, all latency.
        {"name": "append_token", "op": "append", "B": 64, "Hkv": 8, "T": 1, "D": 128, "page": 16, "past": 500,
         "kv": "bf16"},
        # Ragged prompts of a padded batch into an 8-bit cache.
        {"name": "append_prompts_e4m3", "op": "append", "B": 8, "Hkv": 8, "T": 4096, "D": 128, "page": 64, "past": 100,
         "kv": "e4m3"},
        # A fork's partial last page in every layer of a small model: all latency.
        {"name": "copy_fork", "op": "copy", "L": 4, "P": 64, "Hkv": 4, "D": 64, "page": 16, "pairs": 3, "kv": "bf16"},
        # Compaction of a fragmented cache over several layers.
        {"name": "copy_compact", "op": "copy", "L": 4, "P": 384, "Hkv": 8, "D": 128, "page": 64, "pairs": 180,
         "kv": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["window", "decode", "decode", "append", "copy"])
    D = rng.choice([64, 128])
    group = rng.choice([1, 1, 2, 3, 4, 7, 8])
    Hkv = rng.choice([1, 2, 4, 8])
    if op == "window":
        B = rng.choice([1, 1, 2, 3])
        M = _log(rng, 1, 8192)
        N = M if rng.random() < 0.5 else M + _log(rng, 1, 8192)
        return {"op": op, "B": B, "Hq": Hkv * group, "Hkv": Hkv, "M": M, "N": N, "D": D, "window": _log(rng, 1, 4096),
                "sinks": rng.choice([0, 0, 1, 4, 16, _log(rng, 1, 500)]), "softcap": rng.choice([0.0, 0.0, 50.0]),
                "alibi": rng.random() < 0.25, "out": "bf16"}
    page = rng.choice([1, 7, 16, 16, 32, 64, 64, 128, 256])
    kv = rng.choice(["bf16", "bf16", "e4m3"])
    if op == "decode":
        B = _log(rng, 1, 64)
        hi = _log(rng, 1, 32768 if B <= 8 else 8192)
        windowed = rng.random() < 0.4
        return {"op": op, "B": B, "Hq": Hkv * group, "Hkv": Hkv, "D": D, "page": page,
                "lo": rng.choice([0, hi, max(1, hi // 2)]), "hi": hi, "window": _log(rng, 1, 4096) if windowed else 0,
                "sinks": rng.choice([0, 1, 4, 30]) if windowed else 0, "softcap": rng.choice([0.0, 0.0, 50.0]),
                "alibi": rng.random() < 0.25, "kv": kv,
                "out": "bf16"}
    if op == "append":
        B = _log(rng, 1, 64)
        T = rng.choice([1, _log(rng, 1, 32768 // B)])
        return {"op": op, "B": B, "Hkv": Hkv, "T": T, "D": D, "page": page, "past": _log(rng, 1, 1000), "kv": kv}
    P = _log(rng, 8, 384)
    return {"op": op, "L": rng.choice([1, 2, 4]), "P": P, "Hkv": Hkv, "D": D, "page": min(page, 64),
            "pairs": _log(rng, 1, P // 2), "kv": kv}


# ----------------------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)


def _pages(g, shape, kv):
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16)
    if kv == "bf16":
        return x
    # what a cache held in e4m3 stands on: values spread over the type's range (the scale is below)
    return (x.float() * 64.0).clamp(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn)


def _scales(g, heads):
    # per kv-head scales around 1/64, which give the 8-bit values above about unit variance
    return (torch.rand(heads, generator=g, device="cuda") * 0.5 + 0.75) / 64.0


def _tables(g, lens, page, longest):
    """Pages of all sequences in random order: table [B, most pages] (-1 where there is none) and the pages of
    the cache, which has room for every sequence at its longest."""
    counts = [-(-n // page) for n in lens]
    total = len(lens) * -(-longest // page) + 3
    perm = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(1, max(counts))), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = perm[at:at + c]
        at += c
    return table, total


def _lengths(g, B, lo, hi):
    return torch.randint(lo, hi + 1, (B,), generator=g, device="cuda").cpu().tolist()


def prepare(case, seed):
    g = _generator(seed)
    s = {"case": dict(case)}
    bf = torch.bfloat16
    if case["op"] == "window":
        c = case
        s["q"] = torch.randn((c["B"], c["Hq"], c["M"], c["D"]), generator=g, device="cuda", dtype=bf)
        s["k"] = torch.randn((c["B"], c["Hkv"], c["N"], c["D"]), generator=g, device="cuda", dtype=bf)
        s["v"] = torch.randn((c["B"], c["Hkv"], c["N"], c["D"]), generator=g, device="cuda", dtype=bf)
        return s
    if case["op"] == "decode":
        c = case
        lens = _lengths(g, c["B"], c["lo"], c["hi"])
        table, total = _tables(g, lens, c["page"], c["hi"])
        s["lens_list"] = lens
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["table"] = table
        s["q"] = torch.randn((c["B"], c["Hq"], c["D"]), generator=g, device="cuda", dtype=bf)
        s["kp"] = _pages(g, (total, c["Hkv"], c["page"], c["D"]), c["kv"])
        s["vp"] = _pages(g, (total, c["Hkv"], c["page"], c["D"]), c["kv"])
        s["ks"] = _scales(g, c["Hkv"]) if c["kv"] == "e4m3" else None
        s["vs"] = _scales(g, c["Hkv"]) if c["kv"] == "e4m3" else None
        if own:  # a serving loop keeps one workspace for all of its steps
            s["ws"] = _binding().paged_decode_workspace(c["B"], c["Hq"], c["Hkv"], c["D"], device="cuda")
        return s
    if case["op"] == "append":
        c = case
        starts = _lengths(g, c["B"], 0, c["past"])
        counts = _lengths(g, c["B"], (c["T"] + 1) // 2, c["T"]) if c["T"] > 1 else [1] * c["B"]
        table, total = _tables(g, [a + n for a, n in zip(starts, counts)], c["page"],
                               c["past"] + c["T"])
        s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        s["counts"] = torch.tensor(counts, dtype=torch.int32, device="cuda") if c["T"] > 1 else None
        s["starts_list"], s["counts_list"], s["table"] = starts, counts, table
        s["k"] = torch.randn((c["B"], c["Hkv"], c["T"], c["D"]), generator=g, device="cuda", dtype=bf)
        s["v"] = torch.randn((c["B"], c["Hkv"], c["T"], c["D"]), generator=g, device="cuda", dtype=bf)
        s["kp"] = _pages(g, (total, c["Hkv"], c["page"], c["D"]), c["kv"])
        s["vp"] = _pages(g, (total, c["Hkv"], c["page"], c["D"]), c["kv"])
        s["ks"] = _scales(g, c["Hkv"]) if c["kv"] == "e4m3" else None
        s["vs"] = _scales(g, c["Hkv"]) if c["kv"] == "e4m3" else None
        # where each new row goes, which the plain form indexes with: sequence, token, page, slot
        b = torch.cat([torch.full((n,), i) for i, n in enumerate(counts)]).cuda()
        t = torch.cat([torch.arange(n) for n in counts]).cuda()
        pos = s["starts"].long()[b] + t
        s["rows"] = (b, t, table[b, pos // c["page"]].long(), pos % c["page"])
        return s
    c = case
    order = torch.randperm(c["P"], generator=g, device="cuda").cpu()
    s["pairs"] = torch.stack([order[:c["pairs"]], order[c["pairs"]:2 * c["pairs"]]], dim=1).contiguous()
    s["src"], s["dst"] = s["pairs"][:, 0].cuda(), s["pairs"][:, 1].cuda()
    s["kp"] = _pages(g, (c["L"], c["P"], c["Hkv"], c["page"], c["D"]), c["kv"])
    s["vp"] = _pages(g, (c["L"], c["P"], c["Hkv"], c["page"], c["D"]), c["kv"])
    return s


# ------------------------------------------------------------------------------------- plain form
def _dtype(name):
    return torch.bfloat16 if name == "bf16" else torch.float32


def _slopes(heads, dtype):
    h = torch.arange(1, heads + 1, device="cuda", dtype=dtype)
    return torch.exp2(-8.0 * h / heads)


def _attend(q, k, v, p, j, keys, c, scale):
    """q [B, Hkv, G, M, D], k, v [B, Hkv, n, D]; positions p [B or 1, M] of the rows and j [n] of the keys, of which
    `keys` (a number or [B, 1, 1]) exist; fp32."""
    dist = j - p.unsqueeze(-1)  # [B or 1, M, n]
    s = torch.matmul(q, k.transpose(-1, -2).unsqueeze(2)) * scale
    if c["alibi"]:
        slope = _slopes(c["Hq"], torch.float32).view(c["Hkv"], -1, 1, 1)
        s = s + slope * dist[:, None, None].float()
    if c["softcap"]:
        s = c["softcap"] * torch.tanh(s / c["softcap"])
    seen = (dist <= 0) & (j < keys)
    if c["window"]:
        seen = seen & ((dist > -c["window"]) | (j < c["sinks"]))
    s = torch.where(seen[:, None, None], s, float("-inf"))
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == float("-inf"), 0.0, m)
    e = torch.exp(s - m)
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e, v.unsqueeze(2)) / torch.where(total == 0, 1.0, total)
    return o, (m + torch.log(total)).squeeze(-1)


def _plain_window(s):
    c = s["case"]
    B, Hq, M, D = s["q"].shape
    N, Hkv, offset = c["N"], c["Hkv"], c["N"] - c["M"]
    o = torch.empty((B, Hq, M, D), dtype=_dtype(c["out"]), device="cuda")
    lse = torch.empty((B, Hq, M), dtype=torch.float32, device="cuda")
    step = 1024  # rows whose scores are held at once: 64 heads x 1024 x 5120 in fp32 are 1.3 GB
    for i in range(0, M, step):
        n = min(step, M - i)
        lo = max(0, offset + i - c["window"] + 1)
        hi = min(N, offset + i + n)
        first = min(c["sinks"], lo)
        j = torch.cat([torch.arange(first, device="cuda"), torch.arange(lo, hi, device="cuda")])
        k, v = (torch.cat([x[:, :, :first], x[:, :, lo:hi]], dim=2).float() for x in (s["k"], s["v"]))
        q = s["q"][:, :, i:i + n].float().view(B, Hkv, Hq // Hkv, n, D)
        p = torch.arange(offset + i, offset + i + n, device="cuda").view(1, n)
        ob, lb = _attend(q, k, v, p, j, N, c, 1.0 / math.sqrt(D))
        o[:, :, i:i + n] = ob.reshape(B, Hq, n, D).to(o.dtype)
        lse[:, :, i:i + n] = lb.reshape(B, Hq, n)
    return o, lse


def _plain_decode(s):
    c = s["case"]
    B, Hq, D = s["q"].shape
    Hkv = c["Hkv"]
    table = s["table"].long().clamp(min=0)
    n = table.shape[1] * c["page"]
    k, v = (x[table].float().transpose(1, 2).reshape(B, Hkv, n, D) for x in (s["kp"], s["vp"]))
    if s["ks"] is not None:
        k, v = k * s["ks"].view(-1, 1, 1), v * s["vs"].view(-1, 1, 1)
    q = s["q"].float().view(B, Hkv, Hq // Hkv, 1, D)
    lens = s["lens"].long()
    o, lse = _attend(q, k, v, lens.view(B, 1) - 1, torch.arange(n, device="cuda"), lens.view(B, 1, 1), c,
                     1.0 / math.sqrt(D))
    return o.reshape(B, Hq, D).to(_dtype(c["out"])), lse.reshape(B, Hq)


def _values(pages):
    """A cache's contents as values: what is held in e4m3 is exact in bf16."""
    return pages.to(torch.bfloat16) if pages.dtype == torch.float8_e4m3fn else pages


def _plain_append(s):
    b, t, page, slot = s["rows"]
    for new, pages, scale in ((s["k"], s["kp"], s["ks"]), (s["v"], s["vp"], s["vs"])):
        x = new[b, :, t]
        if scale is not None:
            x = (x.float() / scale.view(1, -1, 1)).clamp(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn)
            pages.view(torch.uint8)[page, :, slot] = x.view(torch.uint8)
        else:
            pages[page, :, slot] = x
    return _values(s["kp"]), _values(s["vp"])


def _plain_copy(s):
    for pages in (s["kp"], s["vp"]):
        raw = pages.view(torch.uint8)
        raw[:, s["dst"]] = raw[:, s["src"]]
    return _values(s["kp"]), _values(s["vp"])


# ------------------------------------------------------------------------------------------- run
def run(state):
    c = state["case"]
    if not own:
        return {"window": _plain_window, "decode": _plain_decode, "append": _plain_append,
                "copy": _plain_copy}[c["op"]](state)
    odf = _binding()
    if c["op"] == "window":
        return odf.flash_fwd_window(state["q"], state["k"], state["v"], window=c["window"], sinks=c["sinks"],
                                    q_offset=c["N"] - c["M"], softcap=c["softcap"], alibi=c["alibi"],
                                    out_dtype=_dtype(c["out"]))
    if c["op"] == "decode":
        return odf.paged_decode(state["q"], state["kp"], state["vp"], state["table"], state["lens"],
                                window=c["window"], sinks=c["sinks"], softcap=c["softcap"], alibi=c["alibi"],
                                k_scale=state["ks"], v_scale=state["vs"], out_dtype=_dtype(c["out"]),
                                workspace=state["ws"])
    if c["op"] == "append":
        odf.paged_append(state["k"], state["v"], state["kp"], state["vp"], state["table"], state["starts"],
                         counts=state["counts"], k_scale=state["ks"], v_scale=state["vs"])
    else:
        odf.page_copy(state["kp"], state["vp"], state["pairs"])
    return _values(state["kp"]), _values(state["vp"])


# ------------------------------------------------------------------------------------------ work
def _visible(p, keys, window, sinks):
    """Keys that a row at position p sees."""
    n = min(p + 1, keys)
    if not window:
        return n
    lo = max(0, p - window + 1)
    return max(0, n - lo) + min(sinks, lo, n)


def work(case):
    c = case
    if c["op"] == "window":
        offset = c["N"] - c["M"]
        pairs = sum(_visible(offset + i, c["N"], c["window"], c["sinks"]) for i in range(c["M"]))
        # keys that some row sees: those from the first row's window on, and the sinks before them
        lo = max(0, offset - c["window"] + 1)
        keys = c["N"] - lo + min(c["sinks"], lo)
        es = 2 if c["out"] == "bf16" else 4
        rows = c["B"] * c["Hq"] * c["M"]
        return {"bytes": rows * (c["D"] * (2 + es) + 4) + c["B"] * c["Hkv"] * keys * c["D"] * 4,
                "flops": 4 * c["D"] * c["B"] * c["Hq"] * pairs}
    if c["op"] == "decode":
        # lengths are drawn evenly from lo..hi: the mean number of visible keys
        step = max(1, (c["hi"] - c["lo"]) // 256)
        some = range(c["lo"], c["hi"] + 1, step)
        keys = sum(_visible(n - 1, n, c["window"], c["sinks"]) for n in some) / len(some) * c["B"]
        es = 2 if c["kv"] == "bf16" else 1
        eo = 2 if c["out"] == "bf16" else 4
        return {"bytes": int(keys * c["Hkv"] * c["D"] * 2 * es + c["B"] * c["Hq"] * (c["D"] * (2 + eo) + 4)),
                "flops": int(4 * c["D"] * c["Hq"] * keys)}
    if c["op"] == "append":
        rows = c["B"] * (0.75 * c["T"] if c["T"] > 1 else 1)
        es = 2 if c["kv"] == "bf16" else 1
        return {"bytes": int(rows * c["Hkv"] * c["D"] * 2 * (2 + es)), "flops": 0}
    es = 2 if c["kv"] == "bf16" else 1
    return {"bytes": 2 * 2 * c["pairs"] * c["L"] * c["Hkv"] * c["page"] * c["D"] * es, "flops": 0}


# ----------------------------------------------------------------------------------------- exact
def exact(case, seed):
    """The definitions in 64 bits: softmax through logsumexp, keys picked by the visibility rule."""
    s = prepare(case, seed)
    c = case
    f64 = torch.float64
    if c["op"] in ("append", "copy"):
        outs = []
        for name in ("k", "v"):
            pages = _values(s[name + "p"]).to(f64)
            if c["op"] == "copy":
                for a, b in s["pairs"].tolist():
                    pages[:, b] = pages[:, a]
            else:
                scale = s[name + "s"]
                for b, (start, n) in enumerate(zip(s["starts_list"], s["counts_list"])):
                    for t0 in range(0, n, 1 if n < 64 else n):
                        rows = torch.arange(t0, n if n >= 64 else t0 + 1, device="cuda")
                        x = s[name][b][:, rows].to(f64)  # [Hkv, rows, D]
                        if scale is not None:
                            x = x / scale.to(f64).view(-1, 1, 1)
                            x = _nearest_e4m3(x)
                        at = start + rows
                        pages[s["table"][b][at // c["page"]].long(), :, at % c["page"]] = x.transpose(0, 1)
            outs.append(pages)
        return tuple(outs)
    Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
    G = Hq // Hkv
    slope = torch.tensor([2.0 ** (-8.0 * (h + 1) / Hq) for h in range(Hq)], dtype=f64, device="cuda")

    def rows(qr, kr, vr, dist, seen):
        """qr [Hq, m, D]; kr, vr [Hkv, n, D]; dist = j - p and seen: [m, n]."""
        x = torch.einsum("hgmd,hnd->hgmn", qr.view(Hkv, G, -1, D), kr).reshape(Hq, qr.shape[1], -1) / math.sqrt(D)
        if c["alibi"]:
            x = x + slope.view(-1, 1, 1) * dist
        if c["softcap"]:
            x = torch.tanh(x / c["softcap"]) * c["softcap"]
        x = x.masked_fill(~seen, -math.inf)
        lse = torch.logsumexp(x, -1)
        w = torch.exp(x - lse.unsqueeze(-1)).masked_fill(~seen, 0.0)
        o = torch.einsum("hgmn,hnd->hgmd", w.view(Hkv, G, qr.shape[1], -1), vr).reshape(Hq, -1, D)
        return o, lse

    if c["op"] == "decode":
        o = torch.zeros((c["B"], Hq, D), dtype=f64, device="cuda")
        lse = torch.full((c["B"], Hq), -math.inf, dtype=f64, device="cuda")
        for b, n in enumerate(s["lens_list"]):
            vis = [j for j in range(n) if not c["window"] or n - 1 - j < c["window"] or j < c["sinks"]]
            if not vis:
                continue
            at = torch.tensor(vis, device="cuda")
            page, slot = s["table"][b][at // c["page"]].long(), at % c["page"]
            k, v = (s[x][page, :, slot].to(f64).transpose(0, 1) for x in ("kp", "vp"))
            if s["ks"] is not None:
                k, v = k * s["ks"].to(f64).view(-1, 1, 1), v * s["vs"].to(f64).view(-1, 1, 1)
            dist = (at - (n - 1)).to(f64).view(1, -1)
            ob, lb = rows(s["q"][b].to(f64).unsqueeze(1), k, v, dist, torch.ones_like(dist, dtype=torch.bool))
            o[b], lse[b] = ob[:, 0], lb[:, 0]
        return o, lse
    o = torch.zeros((c["B"], Hq, c["M"], D), dtype=f64, device="cuda")
    lse = torch.empty((c["B"], Hq, c["M"]), dtype=f64, device="cuda")
    offset = c["N"] - c["M"]
    for b in range(c["B"]):
        for i in range(0, c["M"], 512):
            p = torch.arange(offset + i, offset + min(c["M"], i + 512), device="cuda")
            j = torch.arange(c["N"], device="cuda")
            near = ((j > p[0] - c["window"]) | (j < c["sinks"])) & (j <= p[-1])
            j = j[near]
            k, v = (s[x][b][:, near].to(f64) for x in ("k", "v"))
            dist = (j[None, :] - p[:, None])
            seen = (dist <= 0) & ((dist > -c["window"]) | (j[None, :] < c["sinks"]))
            ob, lb = rows(s["q"][b, :, i:i + 512].to(f64), k, v, dist.to(f64), seen)
            o[b, :, i:i + 512], lse[b, :, i:i + 512] = ob, lb
    return o, lse


def _nearest_e4m3(x):
    """x to the nearest value of e4m3 (ties to even), at most 448 in size: steps of 2^(e-3), e >= -6."""
    x = x.clamp(-_E4M3_MAX, _E4M3_MAX)
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step
