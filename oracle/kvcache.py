"""The paged key / value cache restated plainly: quantising rows into pages, reading them back, attention over the values in
64 bits (torch, any device), with the bounds that the arithmetic of a 16-bit kernel gives."""
import math

import torch

FP8 = torch.float8_e4m3fn
QMAX = {torch.int8: 127.0, FP8: 448.0}


def quantise(x, code):
    """[..., D] -> codes and fp32 scales [...]: s = max(amax / QMAX, 1e-12), round half even of the fp32 quotient; a row
    with an infinity or a NaN: s = NaN, codes 0."""
    x = x.float()
    amax = x.abs().amax(-1)
    bad = ~torch.isfinite(x).all(-1)
    # the IEEE fp32 quotient (torch divides a GPU tensor by a number through its reciprocal; 64 bits rounded once are exact)
    s = (amax.double() / QMAX[code]).float().clamp_min(1e-12)
    s = torch.where(bad, torch.nan, s)
    y = torch.where(bad[..., None], 0.0, x / s[..., None])
    q = torch.round(y).to(torch.int8) if code == torch.int8 else y.clamp(-448.0, 448.0).to(FP8)
    return q, s


def rows_of(lens, cu, rows, batch):
    """(sequence, position) of each row, None where no sequence has it; position may be negative."""
    if cu is None:
        n = rows // batch
        return [(r // n, lens[r // n] - n + r % n) for r in range(rows)]
    got = [None] * rows
    for b in range(batch):
        for r in range(cu[b], cu[b + 1]):
            got[r] = (b, lens[b] - (cu[b + 1] - cu[b]) + r - cu[b])
    return got


def slot(table, pages, page, b, pos):
    """(page, offset) of a position, None where nothing is."""
    if pos < 0 or pos >= len(table[b]) * page:
        return None
    p = table[b][pos // page]
    return (p, pos % page) if 0 <= p < pages else None


def gather(cache, table, n):
    """The first n positions of a list of pages as float64 keys, values [H, n, D] and a mask of those that are there."""
    page = cache.k.shape[2]
    at = torch.tensor([table[i // page] for i in range(n)], dtype=torch.int64, device=cache.k.device)
    off = torch.arange(n, device=at.device) % page
    here = (at >= 0) & (at < cache.k.shape[0])
    at = torch.where(here, at, 0)
    out = []
    for codes, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        x = codes.view(torch.uint8)[at, :, off].view(codes.dtype).double() * scale[at, :, off].double()[..., None]
        out.append(x.transpose(0, 1))
    return out[0], out[1], here


def attention(q, cache, table, lens, cu=None, causal=True, scale=None, prefix=None, prefix_len=0):
    """float64 out [T, Hq, D] and log-sum-exp [T, Hq] of kv_attention / kv_attention_shared (lists for table, lens, cu,
    prefix), the weighted magnitudes sum_j p_j |v_j| [T, Hq, D] and the error bound of a row's scores [T, Hq] (fp32 sums of
    exact products). Rows that no sequence has are NaN."""
    t, hq, d = q.shape
    b = len(lens)
    hkv = cache.k.shape[1]
    g = hq // hkv
    dev = q.device
    scale = d ** -0.5 if scale is None else scale
    o = torch.full((t, hq, d), math.nan, dtype=torch.float64, device=dev)
    mag = o.clone()
    lse = torch.full((t, hq), math.nan, dtype=torch.float64, device=dev)
    err = lse.clone()
    for i in range(b):
        r0, r1 = (i * (t // b), (i + 1) * (t // b)) if cu is None else (cu[i], cu[i + 1])
        n = r1 - r0
        if n == 0:
            continue
        parts = [gather(cache, table[i], lens[i])]
        if prefix_len:
            parts.insert(0, gather(cache, prefix, prefix_len))
        k, v = (torch.cat([p[j] for p in parts], 1) for j in range(2))
        here = torch.cat([p[2] for p in parts])
        place = torch.cat([torch.full((prefix_len,), -1 << 40, device=dev), torch.arange(lens[i], device=dev)])
        last = lens[i] - n + torch.arange(n, device=dev) if causal else torch.full((n,), lens[i], device=dev)
        see = (place[None] <= last[:, None]) & here[None]                          # [n, keys]
        for h in range(hq):
            kh, vh = k[h // g], v[h // g]
            x = (q[r0:r1, h].double() @ kh.t()) * scale
            x = torch.where(see, x, -math.inf)
            m = x.amax(1, keepdim=True) if x.shape[1] else torch.full((n, 1), -math.inf, dtype=torch.float64, device=dev)
            p = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
            # a NaN that a row does not see stays out of its sums
            w = p.sum(1, keepdim=True)
            p = torch.where(w > 0, p / w, p)
            for dst, val in ((o, vh), (mag, vh.abs())):
                clean = torch.nan_to_num(val, nan=0.0)
                r = p @ clean
                nan_seen = (see & torch.isnan(val).any(1)[None]).any(1)
                r[nan_seen] = math.nan
                dst[r0:r1, h] = r
            both = (see & (torch.isnan(kh).any(1) | torch.isnan(vh).any(1))[None]).any(1)
            e = (torch.log(w) + m)[:, 0]
            e[both] = math.nan
            lse[r0:r1, h] = e
            a = (q[r0:r1, h].double().abs() @ torch.nan_to_num(kh, nan=0.0).abs().t()) * abs(scale)
            a = torch.where(see, a, 0.0)
            # D + 8 roundings of fp32 sums and products, and of the score and reference in base 2 (twice the magnitude)
            err[r0:r1, h] = (d + 16) * 2.0 ** -24 * (a.amax(1) if a.shape[1] else 0.0) + 2.0 ** -20
    return o, lse, mag, err
