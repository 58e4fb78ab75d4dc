"""Performance cases of the quantised key / value cache: writing it, reading it back, attention over its pages (single
tokens, a few tokens, whole chunks) and attention of a batch whose sequences share a prefix.

Head layouts: 56 heads of 128 with as many K/V heads (the wider DiT of this repository's benchmark, whose frames are
written and attended in chunks), and grouped query heads over few K/V heads, as a text encoder in front of it has them.

  listed()             the cases
  draw(rng)            one more case of the same ranges
  prepare(case, seed)  a filled cache, its page table and lengths, and the new rows
  run(state)           one pass: the framework's calls where `own`, else the same by elementary torch in 32 bits
  exact(case, seed)    the result in float64
  work(case)           bytes and operations a pass cannot do without
"""
import math
import os
import random
import sys

import torch

sys.path.insert(0, os.path.abspath("rapid-h3_amd"))   # the package folder of the tree this runs in

own = False

DEV = "cuda"
F32, F64 = torch.float32, torch.float64
FP8 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------- the cases
# batch sequences of `rows` new tokens each; lengths up to `keys` (ragged: spread down to a sixteenth of it)
def listed():
    return [
        # one step of a small batch: every sequence's new token is quantised into its page, then read back
        {"name": "write_step", "kind": "write", "fmt": "int8", "dtype": "bf16", "batch": 16, "rows": 1, "keys": 900, "ragged": True, "hkv": 8, "dim": 128, "page": 64},
        # one draft-size pass of the wider DiT: all its tokens' keys and values kept for the chunks that follow
        {"name": "write_draft", "kind": "write", "fmt": "fp8", "dtype": "bf16", "batch": 1, "rows": 22332, "keys": 22332, "ragged": False, "hkv": 56, "dim": 128, "page": 128},
        # a window of the last tokens handed back to a program that works on values
        {"name": "read_window", "kind": "read", "fmt": "fp8", "dtype": "fp16", "batch": 5, "rows": 333, "keys": 2100, "ragged": True, "hkv": 4, "dim": 64, "page": 16},
        # whole histories of a batch read back
        {"name": "read_all", "kind": "read", "fmt": "int8", "dtype": "bf16", "batch": 8, "rows": 7919, "keys": 7919, "ragged": False, "hkv": 16, "dim": 128, "page": 64},
        # the smallest attention: one sequence, its next token
        {"name": "token_one", "kind": "attend", "fmt": "int8", "dtype": "bf16", "batch": 1, "rows": 1, "keys": 1023, "ragged": False, "causal": True, "lse": False, "hq": 32, "hkv": 8, "dim": 128, "page": 64},
        # a served batch of uneven histories, one token each
        {"name": "token_batch", "kind": "attend", "fmt": "int8", "dtype": "bf16", "batch": 64, "rows": 1, "keys": 8190, "ragged": True, "causal": True, "lse": False, "hq": 32, "hkv": 8, "dim": 128, "page": 64},
        # long histories, a group of 7 query heads to a K/V head
        {"name": "token_long", "kind": "attend", "fmt": "fp8", "dtype": "bf16", "batch": 4, "rows": 1, "keys": 131071, "ragged": False, "causal": True, "lse": False, "hq": 56, "hkv": 8, "dim": 128, "page": 128},
        # a few proposed tokens of each sequence checked at once, log-sum-exp kept for the joining of parts
        {"name": "few_tokens", "kind": "attend", "fmt": "fp8", "dtype": "fp16", "batch": 12, "rows": 5, "keys": 3001, "ragged": True, "causal": True, "lse": True, "hq": 28, "hkv": 4, "dim": 64, "page": 32},
        # a prompt's next chunk against what is cached of it
        {"name": "chunk_causal", "kind": "attend", "fmt": "int8", "dtype": "bf16", "batch": 1, "rows": 2048, "keys": 16384, "ragged": False, "causal": True, "lse": False, "hq": 32, "hkv": 8, "dim": 128, "page": 64},
        # the tokens of a new latent frame of the wider DiT against the draft-size history, itself included
        {"name": "chunk_frame", "kind": "attend", "fmt": "fp8", "dtype": "bf16", "batch": 1, "rows": 1560, "keys": 22332, "ragged": False, "causal": False, "lse": False, "hq": 56, "hkv": 56, "dim": 128, "page": 128},
        # a handful of prompts behind one instruction
        {"name": "shared_small", "kind": "shared", "fmt": "fp8", "dtype": "bf16", "batch": 6, "rows": 1, "keys": 140, "ragged": True, "prefix": 1777, "causal": True, "lse": False, "hq": 32, "hkv": 8, "dim": 128, "page": 64},
        # many continuations of one long context
        {"name": "shared_large", "kind": "shared", "fmt": "int8", "dtype": "bf16", "batch": 64, "rows": 1, "keys": 510, "ragged": True, "prefix": 32768, "causal": True, "lse": False, "hq": 32, "hkv": 8, "dim": 128, "page": 64},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("write", "read", "token", "token", "token", "few", "chunk", "chunk", "shared", "shared"))
    hq, hkv = rng.choice(((56, 56), (32, 8), (56, 8), (28, 4), (16, 16), (8, 1), (12, 4)))
    c = {"kind": "attend", "fmt": rng.choice(("int8", "fp8")), "dtype": rng.choice(("bf16", "bf16", "fp16"))}
    g = {"hq": hq, "hkv": hkv, "dim": rng.choice((128, 128, 64)), "page": rng.choice((16, 32, 64, 128, 256))}
    if kind in ("write", "read"):
        rows = _log(rng, 1, 20000)
        batch = rng.randint(1, max(1, min(64, 20000 // rows)))
        g.pop("hq")
        return {**c, "kind": kind, "batch": batch, "rows": rows, "keys": rows + _log(rng, 1, 2000), "ragged": rng.random() < 0.5, **g}
    tail = {"ragged": rng.random() < 0.6, "causal": rng.random() < 0.7, "lse": rng.random() < 0.4, **g}
    if kind == "chunk":
        rows = _log(rng, 48, 2048)
        keys = rows + _log(rng, 64, 16000)
        batch = rng.randint(1, max(1, min(16, int(6e10 / (rows * keys * hq * g["dim"])))))
        return {**c, "batch": batch, "rows": rows, "keys": keys, **tail}
    rows = 1 if kind == "token" else rng.randint(2, 8) if kind == "few" else rng.choice((1, 1, 3))
    if kind == "shared":
        return {**c, "kind": "shared", "batch": _log(rng, 2, 64), "rows": rows, "prefix": _log(rng, 100, 32768), "keys": rows + _log(rng, 8, 1000), **tail}
    keys = rows + _log(rng, 64, 100000)
    batch = rng.randint(1, max(1, min(64, int(3.5e6 / (keys * hkv)))))
    return {**c, "batch": batch, "rows": rows, "keys": keys, **tail}


def _lengths(case):
    """Cached tokens of each sequence (the new rows included) and its new rows, by the case alone."""
    b, n, rows = case["batch"], case["keys"], case["rows"]
    if not case["ragged"]:
        return [n] * b, [rows] * b
    r = random.Random(b * 1000003 + n)
    lens = [max(1, int(n * 16 ** -r.random())) for _ in range(b)]
    lens[0] = n
    new = [rows if rows < 16 else max(1, int(rows * 4 ** -r.random())) for _ in range(b)]
    return lens, [min(a, c) for a, c in zip(new, lens)]


# ---------------------------------------------------------------- inputs
def _quantise(x, fmt):
    """[..., D] fp32 -> the codes and the fp32 scale of each row."""
    amax = x.abs().amax(-1)
    # the IEEE fp32 quotient: by way of 64 bits, for torch divides a GPU tensor by a number through its reciprocal
    s = (amax.double() / (127.0 if fmt == "int8" else 448.0)).float().clamp_min(1e-12)
    y = x / s[..., None]
    if fmt == "int8":
        return torch.round(y).to(torch.int8), s
    return y.clamp(-448.0, 448.0).to(FP8), s


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 11)
    b, hkv, d, page = case["batch"], case["hkv"], case["dim"], case["page"]
    hq, prefix, dt = case.get("hq", hkv), case.get("prefix", 0), TYPES[case["dtype"]]
    lens, new = _lengths(case)
    width = [-(-n // page) for n in lens]
    pre = -(-prefix // page)
    pages = sum(width) + pre + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    # a row of the table: its pages in any order of the pool, no page (-1) behind them
    table = torch.full((b, max(width)), -1, dtype=torch.int32, device=DEV)
    at = pre
    for i, w in enumerate(width):
        table[i, :w] = order[at:at + w]
        at += w
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    t = cu[-1]
    kc = 2.0 * torch.randn((1, hkv, 1, d), generator=g, device=DEV)   # the offset that keys carry from channel to channel

    def rows(n, h):
        return torch.randn((n, h, d), generator=g, device=DEV)

    s = {"case": dict(case), "table": table, "lens": torch.tensor(lens, dtype=torch.int32, device=DEV),
         "cu": None if len(set(new)) == 1 else torch.tensor(cu, dtype=torch.int32, device=DEV), "rows": t,
         "most": max(new), "prefix": order[:pre].contiguous(), "prefix_len": prefix, "dtype": dt,
         "causal": case.get("causal", False), "lse": case.get("lse", False)}
    if case["kind"] == "write":
        codes = torch.int8 if case["fmt"] == "int8" else FP8
        s["k"], s["v"] = (torch.zeros((pages, hkv, page, d), dtype=torch.int8, device=DEV).view(codes) for _ in range(2))
        s["k_scale"], s["v_scale"] = (torch.zeros((pages, hkv, page), device=DEV) for _ in range(2))
        s["new_k"], s["new_v"] = (rows(t, hkv) + kc[:, :, 0]).to(dt), rows(t, hkv).to(dt)
        return s
    s["k"], s["k_scale"] = _quantise(torch.randn((pages, hkv, page, d), generator=g, device=DEV) + kc, case["fmt"])
    s["v"], s["v_scale"] = _quantise(torch.randn((pages, hkv, page, d), generator=g, device=DEV)
                                     * torch.exp(0.5 * torch.randn((pages, hkv, page, 1), generator=g, device=DEV)), case["fmt"])
    if case["kind"] != "read":
        s["q"] = (rows(t, hq) * 1.5).to(dt)
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    kind = s["case"]["kind"]
    if own:
        return _framework(s, kind)
    if kind == "write":
        _plain_write(s)
    if kind in ("write", "read"):
        return _plain_read(s)
    return _plain_attention(s)


def _framework(s, kind):
    from rapid_h3 import kvcache
    if "cache" not in s:   # made once beside the buffers that it names, as a program keeps it from step to step
        s["cache"] = kvcache.KVCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    cache = s["cache"]
    if kind == "write":
        kvcache.kv_write(cache, s["new_k"], s["new_v"], s["table"], s["lens"], s["cu"])
    if kind in ("write", "read"):
        return kvcache.kv_read(cache, s["table"], s["lens"], s["cu"], rows=s["rows"], dtype=s["dtype"])
    if kind == "shared":
        return kvcache.kv_attention_shared(s["q"], cache, s["prefix"], s["prefix_len"], s["table"], s["lens"], s["cu"],
                                           causal=s["causal"], lse=s["lse"])
    return kvcache.kv_attention(s["q"], cache, s["table"], s["lens"], s["cu"], causal=s["causal"], lse=s["lse"])


def _places(s):
    """Of each new row: its sequence, its number in it, the sequence's new rows."""
    b, t = s["table"].shape[0], s["rows"]
    at = torch.arange(t, device=DEV)
    if s["cu"] is None:
        n = t // b
        return at // n, at % n, torch.full((b,), n, device=DEV), torch.arange(b, device=DEV) * n
    cu = s["cu"].long()
    seq = torch.searchsorted(cu[1:].contiguous(), at, right=True)
    return seq, at - cu[seq], cu[1:] - cu[:-1], cu[:-1]


def _slots(s):
    seq, i, n, _ = _places(s)
    pos = s["lens"].long()[seq] - n[seq] + i
    page = s["k"].shape[2]
    return s["table"].long()[seq, pos // page], pos % page


def _plain_write(s):
    p, o = _slots(s)
    for x, codes, scale in ((s["new_k"], s["k"], s["k_scale"]), (s["new_v"], s["v"], s["v_scale"])):
        c, f = _quantise(x.float(), s["case"]["fmt"])
        codes.view(torch.int8).transpose(1, 2)[p, o] = c.view(torch.int8)
        scale.transpose(1, 2)[p, o] = f


def _plain_read(s):
    p, o = _slots(s)
    return [(codes.view(torch.uint8).transpose(1, 2)[p, o].view(codes.dtype).float() * scale.transpose(1, 2)[p, o][..., None]).to(s["dtype"])
            for codes, scale in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"]))]


def _gather(codes, scale, table):
    """The pages of a table [B, W] as fp32 values [B, H, W * page, D]."""
    t = table.long().clamp_min(0)
    x = codes.view(torch.uint8)[t].view(codes.dtype).float() * scale[t][..., None]
    b, w, h, page, d = x.shape
    return x.transpose(1, 2).reshape(b, h, w * page, d)


def _plain_attention(s):
    c = s["case"]
    b, hkv, d, g = c["batch"], c["hkv"], c["dim"], c["hq"] // c["hkv"]
    seq, i, n, first = _places(s)
    most = s["most"]
    step = torch.arange(most, device=DEV)
    rows = (first[:, None] + step).clamp_max(s["rows"] - 1)
    q = s["q"].float()[rows].reshape(b, most, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, g * most, d) * d ** -0.5
    k, v = _gather(s["k"], s["k_scale"], s["table"]), _gather(s["v"], s["v_scale"], s["table"])
    at = torch.arange(k.shape[2], device=DEV)
    lens = s["lens"].long()
    v = torch.where((at < lens[:, None])[:, None, :, None], v, 0.0)
    last = lens[:, None] - n[:, None] + step + 1 if s["causal"] else lens[:, None].expand(b, most)
    hidden = at >= torch.minimum(last, lens[:, None])[:, :, None]
    x = torch.matmul(q, k.transpose(2, 3)).reshape(b, hkv, g, most, -1)
    x = x.masked_fill(hidden[:, None, None], -math.inf).reshape(b, hkv, g * most, -1)
    if c["kind"] == "shared":
        # the common keys, against all rows of a K/V head at once
        pk, pv = (_gather(a, f, s["prefix"][None])[0, :, :s["prefix_len"]] for a, f in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])))
        qa = q.transpose(0, 1).reshape(hkv, b * g * most, d)
        y = torch.matmul(qa, pk.transpose(1, 2))
        y = y.reshape(hkv, b, g * most, -1).transpose(0, 1)
        x = torch.cat([y, x], 3)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    if c["kind"] == "shared":
        pa = p[..., :s["prefix_len"]].transpose(0, 1).reshape(hkv, b * g * most, -1)
        o = torch.matmul(pa, pv).reshape(hkv, b, g * most, d).transpose(0, 1) + torch.matmul(p[..., s["prefix_len"]:], v)
    else:
        o = torch.matmul(p, v)
    o = torch.where(total > 0, o / total, 0.0)
    o = o.reshape(b, hkv * g, most, d)[seq, :, i].to(s["dtype"])
    if not s["lse"]:
        return o
    e = (torch.log(total) + m).reshape(b, hkv * g, most)[seq, :, i]
    return o, e


# ---------------------------------------------------------------- the result in 64 bits
def _e4m3(y):
    """Float64 values to the nearest e4m3 value, halves to even."""
    y = y.clamp(-448.0, 448.0)
    _, e = torch.frexp(y)
    grid = torch.ldexp(torch.ones_like(y), (e - 1).clamp_min(-6) - 3)
    return torch.round(y / grid) * grid


def exact(case, seed):
    s = prepare(case, seed)
    lens, new = _lengths(case)
    page, hkv, d = case["page"], case["hkv"], case["dim"]
    table = s["table"].tolist()
    if case["kind"] == "write":
        out = []
        for x in (s["new_k"], s["new_v"]):
            x = x.to(F64)
            f = (x.abs().amax(-1, keepdim=True) / (127 if case["fmt"] == "int8" else 448)).clamp_min(1e-12).to(F32).to(F64)
            y = (x / f).to(F32).to(F64)   # the quotient that is rounded to a code is the fp32 one, by definition
            out.append((torch.round(y) if case["fmt"] == "int8" else _e4m3(y)) * f)
        return out

    def values(pages, n):
        """The first n positions of a list of pages, as [H, n, D] float64."""
        got = []
        for codes, scale in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])):
            at = torch.tensor(pages, dtype=torch.int64, device=DEV)
            x = codes.view(torch.uint8).index_select(0, at).view(codes.dtype).to(F64) * scale.index_select(0, at).to(F64)[..., None]
            got.append(x.permute(1, 0, 2, 3).reshape(hkv, len(pages) * page, d)[:, :n])
        return got

    if case["kind"] == "read":
        parts = [[x[:, n - r:].transpose(0, 1) for x in values(row[:-(-n // page)], n)] for row, n, r in zip(table, lens, new)]
        return [torch.cat([p[j] for p in parts]) for j in range(2)]

    hq = case["hq"]
    group = hq // hkv
    common = values(s["prefix"].tolist(), s["prefix_len"]) if case["kind"] == "shared" else None
    outs, sums, at = [], [], 0
    for row, n, r in zip(table, lens, new):
        k, v = values(row[:-(-n // page)], n)
        if common:
            k, v = torch.cat([common[0], k], 1), torch.cat([common[1], v], 1)
        q = s["q"][at:at + r].to(F64)
        at += r
        o, e = torch.empty((r, hq, d), dtype=F64, device=DEV), torch.empty((r, hq), dtype=F64, device=DEV)
        place = torch.arange(k.shape[1], device=DEV)[None]
        own_row = k.shape[1] - r + torch.arange(r, device=DEV)[:, None]
        for h in range(hq):
            x = torch.mm(q[:, h], k[h // group].t().contiguous()) / math.sqrt(d)
            if case["causal"]:
                x = x.masked_fill(place > own_row, -math.inf)
            e[:, h] = torch.logsumexp(x, 1)
            o[:, h] = torch.mm(torch.exp(x - e[:, h:h + 1]), v[h // group])
        outs.append(o)
        sums.append(e)
    o = torch.cat(outs)
    return (o, torch.cat(sums)) if case["lse"] else o


# ---------------------------------------------------------------- what a pass has to move and compute
def work(case):
    lens, new = _lengths(case)
    hkv, d, t = case["hkv"], case["dim"], sum(new)
    cached = 2 * hkv * (d + 4)           # bytes of one token in the cache: codes and scales of key and value
    if case["kind"] == "write":
        return {"bytes": t * (2 * hkv * d * 2 + cached + 2 * hkv * d * 2), "flops": 0}
    if case["kind"] == "read":
        return {"bytes": t * (cached + 2 * hkv * d * 2), "flops": 0}
    hq, prefix = case["hq"], case.get("prefix", 0)
    pairs = sum(r * (n + prefix) - (r * (r - 1) // 2 if case["causal"] else 0) for n, r in zip(lens, new))
    return {"bytes": (sum(lens) + prefix) * cached + t * hq * (2 * d * 2 + (4 if case["lse"] else 0)), "flops": 4 * d * hq * pairs}
