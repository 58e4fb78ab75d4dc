"""Performance cases of a serving step around the key / value cache: page tables and slot maps from request lengths, the norm
and rotation of queries and keys, the same with the rows written into the cache in one pass, a cache in 4 bits (written, read
back), and attention over it.

Head layouts: 56 heads of 128 with as many K/V heads (the wider DiT of this repository's benchmark, whose frames are written and
attended in chunks), and grouped query heads over few K/V heads, as a text encoder in front of it has them.

The 4-bit format: groups of 32 channels of a row share a power of two 2^e, the least with amax <= 7 * 2^e (e within +-125), kept
as the byte e + 127; a value is an e2m1 code (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign bit) nearest to x / 2^e, ties to the even code,
magnitudes past 6 to 6; two codes to a byte, the lower channel in the low half.

  listed()             the cases
  draw(rng)            one more case of the same ranges
  prepare(case, seed)  a pool of pages with its table and lengths, a filled cache, the new rows
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
EPS = 1e-6
GROUP = 32                                            # channels that share a scale
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ---------------------------------------------------------------- the cases
# pages: `batch` sequences of up to `keys` cached positions; a share `done` of them ends, of the others a share `prompts` brings up
#   to `rows` positions, the rest one
# rope: `rows` rows at positions up to `far`; rot: rotated channels; scaling: how the frequencies are stretched for long contexts
# the others: `rows` new rows to each of `batch` sequences, whose lengths reach up to `keys` (ragged: spread down to a sixteenth of it)
def listed():
    return [
        # one step of a small served batch: a token each, one request has ended
        {"name": "pages_step", "kind": "pages", "batch": 16, "keys": 900, "rows": 1, "prompts": 0.0, "done": 0.07, "page": 64},
        # many requests at once, some bring whole prompts and some have ended
        {"name": "pages_prompts", "kind": "pages", "batch": 700, "keys": 6000, "rows": 3001, "prompts": 0.15, "done": 0.1, "page": 16},
        # a few tokens deep in a long context whose frequencies are stretched by parts
        {"name": "rope_tokens", "kind": "rope", "dtype": "bf16", "rows": 8, "far": 131071, "hq": 32, "hkv": 8, "dim": 128, "rot": 128,
         "layout": "half", "norm": True, "scaling": "parts"},
        # the draft pass of the wider DiT: every token's queries and keys, 96 of 128 channels rotated
        {"name": "rope_draft", "kind": "rope", "dtype": "bf16", "rows": 22332, "far": 22332, "hq": 56, "hkv": 56, "dim": 128, "rot": 96,
         "layout": "half", "norm": True, "scaling": None},
        # a batch's next tokens go from the projection into a 4-bit cache
        {"name": "step_tokens", "kind": "step", "fmt": "fp4", "dtype": "bf16", "batch": 24, "rows": 1, "keys": 5001, "ragged": True, "hq": 32,
         "hkv": 8, "dim": 128, "page": 64, "rot": 128, "layout": "half", "norm": True, "scaling": None},
        # prompts on their way into an int8 cache, pairs of neighbouring channels rotated in half of each head
        {"name": "step_prompts", "kind": "step", "fmt": "int8", "dtype": "fp16", "batch": 3, "rows": 8003, "keys": 9001, "ragged": False, "hq": 56,
         "hkv": 8, "dim": 128, "page": 32, "rot": 64, "layout": "interleaved", "norm": False, "scaling": "linear"},
        # a few tokens' keys and values quantised into their pages, then read back
        {"name": "write4_few", "kind": "write", "fmt": "fp4", "dtype": "fp16", "batch": 5, "rows": 7, "keys": 700, "ragged": True, "hkv": 4, "dim": 64,
         "page": 16},
        # one draft-size pass of the wider DiT: all its tokens' keys and values kept for the chunks that follow
        {"name": "write4_draft", "kind": "write", "fmt": "fp4", "dtype": "bf16", "batch": 1, "rows": 22332, "keys": 22332, "ragged": False, "hkv": 56,
         "dim": 128, "page": 128},
        # one sequence, its next token, log-sum-exp kept for the joining of parts
        {"name": "attend4_one", "kind": "attend", "fmt": "fp4", "dtype": "fp16", "batch": 1, "rows": 1, "keys": 2047, "ragged": False, "causal": True,
         "lse": True, "hq": 28, "hkv": 4, "dim": 64, "page": 32},
        # a served batch of uneven histories, one token each
        {"name": "attend4_batch", "kind": "attend", "fmt": "fp4", "dtype": "bf16", "batch": 64, "rows": 1, "keys": 16381, "ragged": True, "causal": True,
         "lse": False, "hq": 32, "hkv": 8, "dim": 128, "page": 64},
        # a prompt's next chunk against what is cached of it
        {"name": "attend4_chunk", "kind": "attend", "fmt": "fp4", "dtype": "bf16", "batch": 1, "rows": 2048, "keys": 16384, "ragged": False,
         "causal": True, "lse": False, "hq": 32, "hkv": 8, "dim": 128, "page": 64},
        # a few proposed tokens of each of many continuations of one long context
        {"name": "attend4_shared", "kind": "shared", "fmt": "fp4", "dtype": "bf16", "batch": 40, "rows": 3, "keys": 601, "ragged": True,
         "prefix": 24001, "causal": True, "lse": False, "hq": 56, "hkv": 8, "dim": 128, "page": 64},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("pages", "rope", "step", "step", "write", "token", "token", "chunk", "chunk", "shared"))
    page = rng.choice((16, 32, 64, 128, 256))
    if kind == "pages":
        return {"kind": "pages", "batch": _log(rng, 1, 700), "keys": _log(rng, 10, 6000), "rows": _log(rng, 1, 3001),
                "prompts": rng.choice((0.0, 0.15)), "done": rng.choice((0.0, 0.1)), "page": page}
    hq, hkv = rng.choice(((56, 56), (32, 8), (56, 8), (28, 4), (16, 16), (8, 1), (12, 4)))
    dim = rng.choice((128, 128, 64))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    turn = {"rot": rng.choice((dim, dim, dim // 2, dim // 4 * 3)), "layout": rng.choice(("half", "interleaved")), "norm": rng.random() < 0.7,
            "scaling": rng.choice((None, "linear", "base", "parts"))}
    if kind == "rope":
        return {"kind": "rope", "dtype": dtype, "rows": _log(rng, 1, 20000), "far": _log(rng, 30000, 1000000), "hq": hq, "hkv": hkv, "dim": dim, **turn}
    c = {"kind": "attend", "fmt": "fp4", "dtype": dtype}
    g = {"hq": hq, "hkv": hkv, "dim": dim, "page": page}
    if kind in ("write", "step"):
        rows = _log(rng, 1, 15000)
        batch = rng.randint(1, max(1, min(64, 15000 // rows)))
        c = {**c, "kind": kind, "batch": batch, "rows": rows, "keys": rows + _log(rng, 1, 2000), "ragged": rng.random() < 0.5, **g}
        if kind == "write":
            c.pop("hq")
            return c
        return {**c, "fmt": rng.choice(("fp4", "fp4", "int8", "fp8")), **turn}
    tail = {"ragged": rng.random() < 0.6, "causal": rng.random() < 0.7, "lse": rng.random() < 0.4, **g}
    if kind == "chunk":
        rows = _log(rng, 48, 2048)
        keys = min(rows + _log(rng, 64, 14000), int(1.28e11 / (rows * hq * dim)))
        batch = rng.randint(1, max(1, min(16, int(6e10 / (rows * keys * hq * dim)))))
        return {**c, "batch": batch, "rows": rows, "keys": keys, **tail}
    rows = rng.choice((1, 1, 1, 2, 5))
    if kind == "shared":
        return {**c, "kind": "shared", "batch": _log(rng, 2, 40), "rows": rows, "prefix": _log(rng, 100, 24000), "keys": rows + _log(rng, 8, 600), **tail}
    keys = rows + _log(rng, 64, 100000)
    batch = rng.randint(1, max(1, min(64, int(3.5e6 / (keys * hkv)))))
    return {**c, "batch": batch, "rows": rows, "keys": keys, **tail}


def _lengths(case):
    """Cached positions of each sequence (the new rows included) and its new rows, by the case alone."""
    b, n, rows = case["batch"], case["keys"], case["rows"]
    if not case["ragged"]:
        return [n] * b, [rows] * b
    r = random.Random(b * 1000003 + n)
    lens = [max(1, int(n * 16 ** -r.random())) for _ in range(b)]
    lens[0] = n
    new = [rows if rows < 16 else max(1, int(rows * 4 ** -r.random())) for _ in range(b)]
    return lens, [min(a, c) for a, c in zip(new, lens)]


def _requests(case):
    """Of each sequence of a pages case: positions cached before the step, new ones, whether it has ended before it."""
    b, n = case["batch"], case["keys"]
    r = random.Random(b * 1000003 + n * 17 + case["rows"])
    lens = [max(1, int(n * 16 ** -r.random())) for _ in range(b)]
    done = [r.random() < case["done"] for _ in range(b)]
    new = [max(1, int(case["rows"] * 4 ** -r.random())) if r.random() < case["prompts"] else 1 for _ in range(b)]
    new = [0 if d and r.random() < 0.5 else c for c, d in zip(new, done)]   # the other half of the ended ones' places is taken at once
    lens[0], new[0], done[0] = n, max(case["rows"], new[0]), False
    return lens, new, done


def _frequencies(case):
    """[rot / 2] fp64 radians to a position, and the factor of the rotated values."""
    rot, kind = case["rot"], case["scaling"]
    base, factor, original = 10000.0, 4.0, 8192
    if kind == "base":
        base *= factor ** (rot / (rot - 2))
    inv = base ** (-torch.arange(0, rot, 2, dtype=F64) / rot)
    if kind == "linear":
        inv = inv / factor
    if kind != "parts":
        return inv, 1.0
    # what turns often within the original length keeps its frequency, what turns less than once is stretched
    turns = original * inv / (2 * math.pi)
    keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
    return inv * keep + inv / factor * (1.0 - keep), 0.1 * math.log(factor) + 1.0


# ---------------------------------------------------------------- inputs
def _pow2(e):
    """2^e as fp32, by its bits (e within +-126)."""
    return ((e.int() + 127) << 23).view(F32)


def _quantise4(x):
    """[..., D] fp32 -> the codes [..., D / 2] and the scale bytes [..., D / 32]."""
    y = x.unflatten(-1, (-1, GROUP))
    m, e = torch.frexp(y.abs().amax(-1))
    e = (e - 3 + (m > 0.875).int()).clamp(-125, 125)
    y = (y * _pow2(-e)[..., None]).flatten(-2)
    a = y.abs()
    c = ((a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte() + (a > 2.5).byte() + (a >= 3.5).byte() + (a > 5.0).byte()
         + 8 * (y < 0).byte())
    c = c.unflatten(-1, (-1, 2))
    return c[..., 0] | (c[..., 1] << 4), (e + 127).byte()


def _quantise(x, fmt):
    """[..., D] fp32 -> the codes and the scales."""
    if fmt == "fp4":
        return _quantise4(x)
    amax = x.abs().amax(-1)
    # the IEEE fp32 quotient: by way of 64 bits, for torch divides a GPU tensor by a number through its reciprocal
    s = (amax.double() / (127.0 if fmt == "int8" else 448.0)).float().clamp_min(1e-12)
    y = x / s[..., None]
    return (torch.round(y).to(torch.int8) if fmt == "int8" else y.clamp(-448.0, 448.0).to(FP8)), s


def _pairs():
    """[256, 2]: the values of a byte's two codes."""
    v = torch.tensor(E2M1 + tuple(-x for x in E2M1), device=DEV)
    at = torch.arange(256, device=DEV)
    return torch.stack([v[at & 15], v[at >> 4]], 1)


def _values(codes, scale):
    """Codes with their scales -> fp32 values [..., D]."""
    if codes.dtype == torch.uint8:
        v = _pairs().index_select(0, codes.reshape(-1).int()).view(*codes.shape[:-1], -1, GROUP)
        return (v * _pow2(scale.int() - 127)[..., None]).flatten(-2)
    return codes.float() * scale[..., None]


def _new_cache(case, pages):
    hkv, page, d = case["hkv"], case["page"], case["dim"]
    if case["fmt"] == "fp4":
        return [torch.zeros((pages, hkv, page, d // n), dtype=torch.uint8, device=DEV) for n in (2, 2, GROUP, GROUP)]
    codes = torch.int8 if case["fmt"] == "int8" else FP8
    return ([torch.zeros((pages, hkv, page, d), dtype=torch.int8, device=DEV).view(codes) for _ in range(2)]
            + [torch.zeros((pages, hkv, page), device=DEV) for _ in range(2)])


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 11)
    kind = case["kind"]
    if kind == "pages":
        return _prepare_pages(case, g)
    d, dt = case["dim"], TYPES[case["dtype"]]
    hkv = case["hkv"]
    hq = case.get("hq", hkv)
    kc = 2.0 * torch.randn((1, hkv, 1, d), generator=g, device=DEV)   # the offset that keys carry from channel to channel

    def rows(n, h):
        return torch.randn((n, h, d), generator=g, device=DEV)

    s = {"case": dict(case), "dtype": dt}
    if kind in ("rope", "step"):
        inv, factor = _frequencies(case)
        s["inv"], s["factor"], s["norm"], s["layout"] = inv.to(DEV), factor, case["norm"], case["layout"]
        s["qw"], s["kw"] = ((1.0 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(dt) if case["norm"] else None for _ in range(2))
    if kind == "rope":
        t = case["rows"]
        s["positions"] = torch.randint(0, case["far"] + 1, (t,), generator=g, device=DEV).to(torch.int32)
        s["positions"][0] = case["far"]
        # views of one projection's rows
        qkv = torch.cat([rows(t, hq) * 1.5, rows(t, hkv) + kc[:, :, 0], rows(t, hkv)], 1).to(dt)
        s["q"], s["new_k"], _ = qkv.split([hq, hkv, hkv], 1)
        return s

    b, page, prefix = case["batch"], case["page"], case.get("prefix", 0)
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
    s.update({"table": table, "lens": torch.tensor(lens, dtype=torch.int32, device=DEV),
              "cu": None if len(set(new)) == 1 else torch.tensor(cu, dtype=torch.int32, device=DEV), "rows": t,
              "most": max(new), "prefix": order[:pre].contiguous(), "prefix_len": prefix,
              "causal": case.get("causal", False), "lse": case.get("lse", False)})
    if kind in ("write", "step"):
        s["k"], s["v"], s["k_scale"], s["v_scale"] = _new_cache(case, pages)
        if kind == "step":   # views of one projection's rows
            qkv = torch.cat([rows(t, hq) * 1.5, rows(t, hkv) + kc[:, :, 0], rows(t, hkv)], 1).to(dt)
            s["q"], s["new_k"], s["new_v"] = qkv.split([hq, hkv, hkv], 1)
        else:
            s["new_k"], s["new_v"] = (rows(t, hkv) + kc[:, :, 0]).to(dt), rows(t, hkv).to(dt)
        return s
    s["k"], s["k_scale"] = _quantise(torch.randn((pages, hkv, page, d), generator=g, device=DEV) + kc, case["fmt"])
    s["v"], s["v_scale"] = _quantise(torch.randn((pages, hkv, page, d), generator=g, device=DEV)
                                     * torch.exp(0.5 * torch.randn((pages, hkv, page, 1), generator=g, device=DEV)), case["fmt"])
    s["q"] = (rows(t, hq) * 1.5).to(dt)
    return s


def _prepare_pages(case, g):
    """The pool and table as the step finds them, in one block of memory, and a copy that each pass begins with."""
    b, page = case["batch"], case["page"]
    lens, new, done = _requests(case)
    have = [-(-n // page) for n in lens]
    width = max(max(have), max(-(-(n + m) // page) for n, m in zip(lens, new))) + 1
    pages = sum(have) + sum(-(-m // page) + 1 for m in new) + 5
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    whole = torch.empty(b * width + b + pages + 2, dtype=torch.int32, device=DEV)
    table, n, free, state = whole.split([b * width, b, pages, 2])
    table = table.view(b, width)
    table.fill_(-1)
    at = 0
    for i, w in enumerate(have):
        table[i, :w] = order[at:at + w]
        at += w
    free.fill_(-1)
    free[:pages - at] = order[at:]
    n.copy_(torch.tensor(lens, dtype=torch.int32))
    state.copy_(torch.tensor([pages - at, 0], dtype=torch.int32))
    return {"case": dict(case), "whole": whole, "before": whole.clone(), "table": table, "lens": n, "free": free, "state": state,
            "new": torch.tensor(new, dtype=torch.int32, device=DEV), "done": torch.tensor(done, dtype=torch.bool, device=DEV),
            "rows": sum(new), "page": page}


# ---------------------------------------------------------------- one pass
def run(s):
    kind = s["case"]["kind"]
    if own:
        return _framework(s, kind)
    if kind == "pages":
        return _plain_pages(s)
    if kind == "rope":
        cos, sin = _angles(s, s["positions"])
        return [_plain_turn(s, x, w, cos, sin) for x, w in ((s["q"], s["qw"]), (s["new_k"], s["kw"]))]
    if kind == "step":
        seq, i, n, _ = _places(s)
        cos, sin = _angles(s, s["lens"].long()[seq] - n[seq] + i)
        q, k = (_plain_turn(s, x, w, cos, sin) for x, w in ((s["q"], s["qw"]), (s["new_k"], s["kw"])))
        _plain_write(s, k, s["new_v"])
        return [q] + _plain_read(s)
    if kind == "write":
        _plain_write(s, s["new_k"], s["new_v"])
        return _plain_read(s)
    return _plain_attention(s)


def _framework(s, kind):
    from rapid_h3 import kvcache, rope
    if kind == "pages":
        if "pool" not in s:   # made once beside the buffers that it names, as a program keeps it from step to step
            s["pool"] = kvcache.KVPages(s["free"], s["state"], s["page"])
        s["whole"].copy_(s["before"])
        cu, positions, slots = kvcache.kv_extend(s["pool"], s["table"], s["lens"], s["new"], s["rows"], s["done"])
        return [s["table"], s["lens"], s["free"], s["state"], cu, positions, slots]
    if kind in ("rope", "step") and "rotary" not in s:
        s["rotary"] = rope.Rotary(s["inv"], s["case"]["layout"], s["factor"])
    eps = EPS if s.get("norm") else None
    if kind == "rope":
        return list(rope.qk_norm_rope(s["q"], s["new_k"], s["positions"], s["rotary"], s["qw"], s["kw"], eps))
    if "cache" not in s:
        s["cache"] = kvcache.KVCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    cache = s["cache"]
    if kind == "step":
        q = kvcache.kv_write_rope(cache, s["q"], s["new_k"], s["new_v"], s["table"], s["lens"], s["cu"], s["rotary"], s["qw"], s["kw"], eps)
        return [q, *kvcache.kv_read(cache, s["table"], s["lens"], s["cu"], rows=s["rows"], dtype=s["dtype"])]
    if kind == "write":
        kvcache.kv_write(cache, s["new_k"], s["new_v"], s["table"], s["lens"], s["cu"])
        return kvcache.kv_read(cache, s["table"], s["lens"], s["cu"], rows=s["rows"], dtype=s["dtype"])
    if kind == "shared":
        return kvcache.kv_attention_shared(s["q"], cache, s["prefix"], s["prefix_len"], s["table"], s["lens"], s["cu"],
                                           causal=s["causal"], lse=s["lse"])
    return kvcache.kv_attention(s["q"], cache, s["table"], s["lens"], s["cu"], causal=s["causal"], lse=s["lse"])


def _plain_pages(s):
    """Ended sequences give their pages back, in the order of the table; then every sequence takes what its new positions need off
    the end of the free list, in order."""
    s["whole"].copy_(s["before"])
    table, lens, free, state, page = s["table"], s["lens"], s["free"], s["state"], s["page"]
    b, width = table.shape
    at = torch.arange(width, device=DEV)
    have = (lens + page - 1) // page
    back = (s["done"][:, None] & (at < have[:, None]) & (table >= 0)).reshape(-1)
    held = state[0].long()
    spare = torch.cat([free, free.new_zeros(1)])
    spare[torch.where(back, held + torch.cumsum(back, 0) - 1, free.numel())] = table.reshape(-1)
    free.copy_(spare[:-1])
    held = held + back.sum()
    table.masked_fill_(back.view(b, width), -1)
    start = torch.where(s["done"], 0, lens)
    end = start + s["new"]
    p0, p1 = ((start + page - 1) // page).clamp_max(width), ((end + page - 1) // page).clamp_max(width)
    need = p1 - p0
    first = torch.cumsum(need, 0) - need
    take = (at >= p0[:, None]) & (at < p1[:, None])
    place = held - 1 - (first[:, None] + at - p0[:, None])
    table.copy_(torch.where(take, torch.where(place >= 0, free[place.clamp(0, free.numel() - 1)], -1), table))
    lens.copy_(end)
    total = need.sum()
    state.copy_(torch.stack([(held - total).clamp_min(0), (total - held).clamp_min(0)]))
    cu = torch.cat([end.new_zeros(1), torch.cumsum(s["new"], 0).int()])
    row = torch.arange(s["rows"], device=DEV)
    seq = torch.searchsorted(cu[1:].contiguous(), row.int(), right=True)
    inside = seq < b
    seq = seq.clamp_max(b - 1)
    pos = torch.where(inside, start[seq] + row - cu[seq], -1)
    entry = torch.where(inside & (pos < width * page), table[seq, (pos // page).clamp(0, width - 1)], -1)
    slots = torch.where(entry >= 0, entry.long() * page + pos % page, -1)
    return [table, lens, free, state, cu, pos.int(), slots]


def _angles(s, positions):
    """Cosines and sines [rows, rot / 2] in 32 bits, of angles in 64."""
    a = positions.double()[:, None] * s["inv"]
    return (torch.cos(a) * s["factor"]).float(), (torch.sin(a) * s["factor"]).float()


def _plain_turn(s, x, w, cos, sin):
    """The RMS norm of each head's row and its rotation, rounded once."""
    x = x.float()
    if s["norm"]:
        # the squares are summed in 64 bits: what is quantised afterwards lies next to the codes' borders
        r = (x.double().square().mean(-1, keepdim=True) + EPS).rsqrt().float()
        x = x * r * w.float()
    half = cos.shape[1]
    cos, sin = cos[:, None], sin[:, None]
    if s["layout"] == "half":
        a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
    else:
        a, b, rest = x[..., 0:2 * half:2], x[..., 1:2 * half:2], x[..., 2 * half:]
        y = torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)
    return y.to(s["dtype"])


def _places(s):
    """Of each new row: its sequence, its number in it; the sequences' new rows and first ones."""
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


def _bytes(codes):
    return codes if codes.dtype == torch.float32 else codes.view(torch.uint8)


def _plain_write(s, k, v):
    p, o = _slots(s)
    for x, codes, scale in ((k, s["k"], s["k_scale"]), (v, s["v"], s["v_scale"])):
        c, f = _quantise(x.float(), s["case"]["fmt"])
        _bytes(codes).transpose(1, 2)[p, o] = _bytes(c)
        scale.transpose(1, 2)[p, o] = f


def _plain_read(s):
    p, o = _slots(s)
    return [_values(_bytes(codes).transpose(1, 2)[p, o].view(codes.dtype), scale.transpose(1, 2)[p, o]).to(s["dtype"])
            for codes, scale in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"]))]


def _gather(codes, scale, table):
    """The pages of a table [B, W] as fp32 values [B, H, W * page, D]."""
    t = table.long().clamp_min(0)
    x = _values(codes[t], scale[t])
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
def _pow2_64(e):
    """2^e in float64, by its bits."""
    return ((e.long() + 1023) << 52).view(F64)


def _decoded(codes, scale):
    """Float64 values of codes with their scales, without a table: sign, exponent and mantissa of each code."""
    if codes.dtype != torch.uint8:
        return codes.to(F64) * scale.to(F64)[..., None]
    c = torch.stack([codes.int() & 15, codes.int() >> 4], -1).flatten(-2)
    e, m = (c >> 1) & 3, (c & 1).to(F64)
    mag = torch.where(e == 0, 0.5 * m, (1.0 + 0.5 * m) * _pow2_64(e - 1))
    x = torch.where(c >= 8, -mag, mag).unflatten(-1, (-1, GROUP))
    return (x * _pow2_64(scale.int() - 127)[..., None]).flatten(-2)


def _nearest(y, bits, least, most):
    """Float64 values to the nearest with `bits` bits behind the leading one, from the exponent `least` on, halves to even."""
    y = y.clamp(-most, most)
    _, e = torch.frexp(y)
    grid = _pow2_64((e - 1).clamp_min(least) - bits)
    return torch.round(y / grid) * grid


def _stored(x, fmt):
    """What a row of values reads back as."""
    x = x.to(F64)
    if fmt == "fp4":
        y = x.unflatten(-1, (-1, GROUP))
        e = torch.ceil(torch.log2(y.abs().amax(-1, keepdim=True) / 7.0)).clamp(-125, 125)
        f = _pow2_64(e)
        return (_nearest(y / f, 1, 0, 6.0) * f).flatten(-2)
    f = (x.abs().amax(-1, keepdim=True) / (127 if fmt == "int8" else 448)).clamp_min(1e-12).to(F32).to(F64)
    y = (x / f).to(F32).to(F64)   # the quotient that is rounded to a code is the fp32 one, by definition
    return (torch.round(y) if fmt == "int8" else _nearest(y, 3, -6, 448.0)) * f


def _turned(case, x, w, positions, inv, factor):
    x = x.to(F64)
    if case["norm"]:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.to(F64)
    at = positions.to(F64)[:, None, None] * inv
    z = torch.polar(torch.full_like(at, factor), at)
    rot = case["rot"]
    body, rest = x[..., :rot], x[..., rot:]
    if case["layout"] == "half":
        c = torch.complex(body[..., :rot // 2].contiguous(), body[..., rot // 2:].contiguous()) * z
        return torch.cat([c.real, c.imag, rest], -1)
    c = torch.view_as_complex(body.unflatten(-1, (-1, 2)).contiguous()) * z
    return torch.cat([torch.view_as_real(c).flatten(-2), rest], -1)


def _exact_pages(s):
    """The same step on Python's lists."""
    table, free, page = s["table"].tolist(), s["free"].tolist(), s["page"]
    lens, new, done = s["lens"].tolist(), s["new"].tolist(), s["done"].tolist()
    held, lacking = s["state"].tolist()[0], 0
    for row, n, d in zip(table, lens, done):
        for i in range(-(-n // page) if d else 0):
            if row[i] >= 0:
                free[held] = row[i]
                held += 1
                row[i] = -1
    cu, positions, slots, ends = [0], [], [], []
    for row, n, m, d in zip(table, lens, new, done):
        n = 0 if d else n
        for i in range(-(-n // page), min(-(-(n + m) // page), len(row))):
            if held:
                held -= 1
                row[i] = free[held]
            else:
                row[i] = -1
                lacking += 1
        for p in range(n, n + m):
            entry = row[p // page] if p // page < len(row) else -1
            positions.append(p)
            slots.append(entry * page + p % page if entry >= 0 else -1)
        cu.append(cu[-1] + m)
        ends.append(n + m)
    return [torch.tensor(x, dtype=t, device=DEV) for x, t in ((table, torch.int32), (ends, torch.int32), (free, torch.int32),
                                                              ([held, lacking], torch.int32), (cu, torch.int32), (positions, torch.int32),
                                                              (slots, torch.int64))]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "pages":
        return _exact_pages(s)
    if case["kind"] == "rope":
        return [_turned(case, x, w, s["positions"], s["inv"], s["factor"]) for x, w in ((s["q"], s["qw"]), (s["new_k"], s["kw"]))]
    lens, new = _lengths(case)
    if case["kind"] == "write":
        return [_stored(x, case["fmt"]) for x in (s["new_k"], s["new_v"])]
    if case["kind"] == "step":
        at = torch.cat([torch.arange(n - r, n, device=DEV) for n, r in zip(lens, new)])
        # keys are rounded to the rows' type in between, and a code next to a border goes by that
        return [_turned(case, s["q"], s["qw"], at, s["inv"], s["factor"]), None, _stored(s["new_v"], case["fmt"])]
    page, hkv, d = case["page"], case["hkv"], case["dim"]
    table = s["table"].tolist()

    def values(pages, n):
        """The first n positions of a list of pages, as [H, n, D] float64."""
        at = torch.tensor(pages, dtype=torch.int64, device=DEV)
        return [_decoded(codes.index_select(0, at), scale.index_select(0, at)).permute(1, 0, 2, 3).reshape(hkv, len(pages) * page, d)[:, :n]
                for codes, scale in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"]))]

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
    if case["kind"] == "pages":
        lens, new, done = _requests(case)
        page = case["page"]
        back = sum(-(-n // page) for n, d in zip(lens, done) if d)
        taken = sum(-(-((0 if d else n) + m) // page) - -(-(0 if d else n) // page) for n, m, d in zip(lens, new, done))
        # a page given back: its entry read and cleared, a place of the list written; one taken: read there, an entry written
        return {"bytes": len(lens) * (4 + 4 + 1 + 4 + 4) + back * 12 + taken * 8 + sum(new) * (4 + 8), "flops": 0}
    hkv, d = case["hkv"], case["dim"]
    if case["kind"] == "rope":
        n = case["rows"] * (case["hq"] + hkv) * d
        return {"bytes": 2 * n * 2 + 4 * case["rows"], "flops": 3 * n + (4 * n if case["norm"] else 0)}
    lens, new = _lengths(case)
    t = sum(new)
    # bytes of one position in the cache: codes and scales of key and value
    cached = 2 * hkv * (d // 2 + d // GROUP if case["fmt"] == "fp4" else d + 4)
    if case["kind"] in ("write", "step"):
        hq = case.get("hq", 0)
        return {"bytes": t * (2 * hkv * d * 2 + 2 * hq * d * 2 + 2 * cached + 2 * hkv * d * 2), "flops": 0}
    hq, prefix = case["hq"], case.get("prefix", 0)
    pairs = sum(r * (n + prefix) - (r * (r - 1) // 2 if case["causal"] else 0) for n, r in zip(lens, new))
    return {"bytes": (sum(lens) + prefix) * cached + t * hq * (2 * d * 2 + (4 if case["lse"] else 0)), "flops": 4 * d * hq * pairs}
