"""The 4-bit form of the paged key / value cache (rapid_h3.kvcache) on the GPU: codes and scale bytes bit for bit against the plain
restatement, values read back, attention (both kernels, whole and in parts, with and without a shared prefix) against float64 over
the stored values."""
import math

import pytest
import torch

from oracle import kvcache as ok
from rapid_h3 import kvcache as kv

pytestmark = pytest.mark.gpu

FP4 = torch.float4_e2m1fn_x2
FORMS = ["token", "chunk"]          # both kernels, whichever the sizes would choose
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _pool(dev, pages, heads, page, dim, seed, garbage=False):
    """A cache full of quantised random values; garbage: every byte 255 (the codes -6, the scales NaN)."""
    if garbage:
        k, v = (torch.full((pages, heads, page, dim // 2), 255, dtype=torch.uint8, device=dev) for _ in range(2))
        return kv.KVCache(k, v, *(torch.full((pages, heads, page, dim // 32), 255, dtype=torch.uint8, device=dev) for _ in range(2)))
    g = _gen(seed)
    kc = 2.0 * torch.randn(1, heads, 1, dim, generator=g)
    k, ks = ok.quantise4(torch.randn(pages, heads, page, dim, generator=g) + kc)
    v, vs = ok.quantise4(torch.randn(pages, heads, page, dim, generator=g) * torch.exp(torch.randn(pages, heads, page, 1, generator=g)))
    return kv.KVCache(*(t.to(dev) for t in (k, v, ks, vs)))


def _bytes(c):
    return [t.view(torch.uint8) for t in (c.k, c.v, c.k_scale, c.v_scale)]


def _tables(pages, width, batch, seed):
    """Disjoint pages in any order, one list per sequence."""
    p = torch.randperm(pages, generator=_gen(seed + 99)).tolist()
    return [p[b * width:(b + 1) * width] for b in range(batch)]


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _cu(new):
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return cu


def _check(out, ref, mag, err, form, keys):
    """|out - ref| within the output's rounding (half a step of its type), the weights' (to bf16 in the chunk kernel for bf16 results,
    else to two bf16 terms) and the fp32 sums' (2^-24 to a key) of sum p |v|, and the scores' error e (at most (exp(2 e) - 1) of the
    same sum). bf16 has 8 significant bits: a value in [1, 2) lies within 2^-8 of one, a rounding is off by 2^-8 of the value at most
    (torch.finfo(bf16).eps / 2), a second term's of what the first left by 2^-8 of that. Below its smallest normal number a type's steps
    stay as they are there: half of one is tiny * eps / 2 (fp16 2^-25)."""
    eps = torch.finfo(out.dtype).eps / 2
    weight = 2.0 ** -8 if form != "token" and out.dtype == BF else 2.0 ** -16
    o = out.double()
    known = ~torch.isnan(ref)
    assert torch.equal(torch.isnan(o), ~known)
    tol = eps * ref.abs() * 1.01 + (weight + (keys + 64) * 2.0 ** -24 + torch.expm1(2 * err)[..., None]) * mag * 1.05 + torch.finfo(out.dtype).tiny * eps
    bad = known & ((o - ref).abs() > tol)
    assert not bad.any(), (int(bad.sum()), float(((o - ref).abs() / tol)[known].max()))


def _check_lse(lse, ref, err):
    known = ~torch.isnan(ref)
    assert torch.equal(torch.isnan(lse), ~known)
    e = lse.double()
    inf = known & torch.isinf(ref)
    assert torch.equal(e[inf], ref[inf])
    fin = known & ~inf
    tol = err + 2.0 ** -22 * ref.abs() + 2.0 ** -20
    assert ((e - ref).abs() <= tol)[fin].all(), float(((e - ref).abs() / tol)[fin].max())


# ---------------------------------------------------------------- writing and reading
def _rows(n, heads, dim, dtype, seed, strided, dev):
    g = _gen(seed)
    x = torch.randn(n, heads, dim, generator=g) * torch.exp(2 * torch.randn(n, heads, 1, generator=g))
    x = x.to(dtype).to(dev)
    if strided:   # a view of a wider buffer: heads and rows apart
        w = torch.zeros(n, heads, dim + 8, dtype=dtype, device=dev)
        w[..., :dim] = x
        x = w[..., :dim]
    return x


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("heads,dim,page,lens,new,strided", [
    (3, 128, 64, [1], [1], False),
    (1, 64, 16, [17, 5, 33], [17, 3, 16], True),
    (2, 128, 32, [0, 40, 7, 64], [0, 33, 9, 1], False),        # a sequence without rows, one with more rows than positions
    (5, 64, 256, [300], [300], True),
    (8, 128, 128, [130, 1, 77], [2, 1, 0], False),
])
def test_write_and_read(dev, dtype, heads, dim, page, lens, new, strided):
    b = len(lens)
    width = max(-(-max(lens) // page), 1) + 1
    pages = b * width + 2
    table = _tables(pages, width, b, 5)
    if b > 1:
        table[1][0] = -1                                       # an absent page
    cu = _cu(new)
    even = len(set(new)) == 1
    rows = cu[-1] + (0 if even else 3)                         # three rows that no sequence has
    k, v = _rows(rows, heads, dim, dtype, 1, strided, dev), _rows(rows, heads, dim, dtype, 2, strided, dev)
    c = _pool(dev, pages, heads, page, dim, 3)
    want = [t.clone() for t in _bytes(c)]
    args = (_i32(table, dev), _i32(lens, dev), None if even else _i32(cu, dev))
    kv.kv_write(c, k, v, *args)
    got_k, got_v = kv.kv_read(c, *args, rows=rows, dtype=dtype)
    keep = torch.full((rows, heads, dim), 7.0, dtype=dtype, device=dev)
    kept = (keep, keep.clone())
    kv.kv_read(c, *args, out=kept)
    for x, codes, scales, got, left in ((k, want[0], want[2], got_k, kept[0]), (v, want[1], want[3], got_v, kept[1])):
        q, s = ok.quantise4(x)
        for r, where in enumerate(ok.rows_of(lens, None if even else cu, rows, b)):
            at = where and ok.slot(table, pages, page, *where)
            if at:
                codes[at[0], :, at[1]] = q[r]
                scales[at[0], :, at[1]] = s[r]
                value = ok.values4(q[r], s[r]).to(dtype)
                assert torch.equal(got[r], value) and torch.equal(left[r], value), r
            else:
                assert (got[r] == 0).all(), r
                assert (left[r] == (7.0 if where is None else 0.0)).all(), r
    for x, y in zip(want, _bytes(c)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_write_special_rows(dev, dim, dtype):
    """Every code, the halfway points between codes, zeros of both signs, group maxima on both sides of 7 * 2^e, the smallest and
    largest magnitudes, groups that are far apart."""
    fin = torch.finfo(dtype)
    at = torch.arange(dim)
    g = _gen(0)
    ladder = torch.tensor([0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7])
    rows = [torch.zeros(dim), -torch.zeros(dim), torch.full((dim,), fin.tiny), torch.full((dim,), fin.max), torch.full((dim,), -fin.max),
            ladder[at % 16], -ladder[at % 16] * 2.0 ** 5, ladder[at % 16] * 2.0 ** -10,
            ladder[at % 16] * (1 + fin.eps), ladder[at % 16] * (1 - fin.eps / 2), torch.where(at % 32 == 0, 7.0, 0.25),
            torch.where(at % 32 == 0, 7.0 * (1 + fin.eps), 0.25), torch.where(at < 32, 2.0 ** -14, 2.0 ** 12) * ladder[at % 16],
            torch.randn(dim, generator=g) * 1e-4, torch.randn(dim, generator=g), torch.randn(dim, generator=g) * 1e3]
    if dtype != HF:
        rows += [torch.randn(dim, generator=g) * f for f in (1e-37, 1e-30, 1e30, 1e37)]
    x = torch.stack(rows)[:, None].to(dtype).to(dev)
    n = x.shape[0]
    c = kv.kv_cache(4, 1, 16, dim, FP4, dev)
    args = (_i32([[2, 0]], dev), _i32([n], dev))
    kv.kv_write(c, x, x.flip(0), *args)
    for codes, scale, y in ((_bytes(c)[0], _bytes(c)[2], x), (_bytes(c)[1], _bytes(c)[3], x.flip(0))):
        q, s = ok.quantise4(y)
        got = torch.cat([codes[2, 0], codes[0, 0]])[:n], torch.cat([scale[2, 0], scale[0, 0]])[:n]
        assert torch.equal(got[0], q[:, 0]) and torch.equal(got[1], s[:, 0])
    k, _ = kv.kv_read(c, *args, rows=n, dtype=F32)
    assert torch.equal(k.double(), ok.values4(*ok.quantise4(x)))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_positions_that_are_not_finite(dev, dim, dtype, bad):
    """An infinity or a NaN in a head's key or value marks the position for that head: NaN in both, the others as ever."""
    x, y = (torch.randn(5, 3, dim, generator=_gen(i)).to(dtype) for i in range(2))
    x[1, 0, dim - 1] = bad
    y[3, 2, 0] = bad
    c = _pool(dev, 3, 3, 16, dim, 0, garbage=True)
    args = (_i32([[1]], dev), _i32([5], dev))
    kv.kv_write(c, x.to(dev), y.to(dev), *args)
    codes = [t[1, :, :5].transpose(0, 1).cpu() for t in _bytes(c)]
    marked = torch.zeros(5, 3, dtype=torch.bool)
    marked[1, 0] = marked[3, 2] = True
    for z, q, s, mark in ((x, codes[0], codes[2], 255), (y, codes[1], codes[3], 0)):
        want_q, want_s = ok.quantise4(torch.where(marked[..., None], 0.0, z.float()))
        assert torch.equal(q, torch.where(marked[..., None], 0, want_q)) and torch.equal(s, torch.where(marked[..., None], mark, want_s))
    for got in kv.kv_read(c, *args, rows=5, dtype=dtype):
        assert torch.equal(torch.isnan(got).all(-1).cpu(), marked) and torch.equal(torch.isnan(got).any(-1).cpu(), marked)


# ---------------------------------------------------------------- attention
CASES = [
    # hq, hkv, dim, page, lens, new, causal: single tokens
    (4, 1, 128, 16, [1], [1], True),
    (8, 8, 128, 64, [15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129], [1] * 11, True),
    (7, 1, 64, 32, [100, 0, 1, 257], [1] * 4, True),                     # a sequence with no key
    (16, 2, 128, 256, [1000, 3, 700], [1] * 3, False),
    # a few tokens: ragged, more rows than positions (rows that see nothing), sequences without rows
    (8, 2, 128, 64, [40, 2, 129, 5], [3, 4, 0, 5], True),
    (6, 2, 64, 16, [200, 33], [5, 5], True),
    (32, 1, 128, 128, [300, 20], [1, 1], True),                          # 32 rows to a K/V head
    # many rows
    (4, 4, 128, 64, [200], [200], True),
    (6, 2, 128, 32, [300, 70, 1], [130, 70, 1], True),
    (5, 1, 64, 64, [500, 77], [50, 77], False),
    (3, 1, 64, 16, [130, 64], [129, 64], True),
    (8, 1, 128, 128, [40, 400], [60, 17], True),                         # more rows than positions
    (2, 2, 128, 256, [64, 1024, 0], [64, 65, 40], True),
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention(dev, dtype, form, case):
    hq, hkv, dim, page, lens, new, causal = CASES[case]
    b = len(lens)
    width = max(-(-max(lens) // page), 1)
    pages = b * width + 3
    table = _tables(pages, width, b, case)
    cu = None if len(set(new)) == 1 else _cu(new)
    c = _pool(dev, pages, hkv, page, dim, case)
    q = (2.0 * torch.randn(sum(new), hq, dim, generator=_gen(case + 50))).to(dtype).to(dev)
    out, lse = kv.kv_attention(q, c, _i32(table, dev), _i32(lens, dev), None if cu is None else _i32(cu, dev), causal=causal, lse=True,
                               form=form)
    ref, rl, mag, err = ok.attention(q, c, table, lens, cu, causal)
    _check(out, ref, mag, err, form, max(lens))
    _check_lse(lse, rl, err)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows,hq,hkv,lens,page", [
    (1, 8, 2, [20011], 64),              # one sequence on many workgroups
    (1, 8, 8, [9000, 31, 4001, 1, 0, 2500], 16),   # uneven histories: items begin and end inside a workgroup's share
    (2, 14, 2, [5000, 5001, 200], 128),
    (40, 4, 1, [9001], 64),              # key ranges of the chunk kernel
    (100, 2, 2, [3000, 20], 32),
])
@pytest.mark.parametrize("form", FORMS)
def test_attention_in_parts(dev, dim, form, rows, hq, hkv, lens, page):
    b = len(lens)
    width = -(-max(lens) // page)
    table = _tables(b * width, width, b, 1)
    c = _pool(dev, b * width, hkv, page, dim, 8)
    q = (2.0 * torch.randn(b * rows, hq, dim, generator=_gen(9))).to(BF).to(dev)
    args = (_i32(table, dev), _i32(lens, dev))
    out, lse = kv.kv_attention(q, c, *args, lse=True, form=form)
    ref, rl, mag, err = ok.attention(q, c, table, lens)
    _check(out, ref, mag, err, form, max(lens))
    _check_lse(lse, rl, err)
    again = kv.kv_attention(q, c, *args, form=form)
    assert torch.equal(out.view(torch.int16), again.view(torch.int16))          # the same bits every time


@pytest.mark.parametrize("dtype,dim", [(BF, 128), (HF, 64)])
@pytest.mark.parametrize("rows,lens,page", [(1, [33, 5, 0], 16), (3, [70, 9], 64), (1, [1000], 32), (70, [90, 71], 16), (80, [40], 32)])
@pytest.mark.parametrize("form", FORMS)
def test_unwritten_pool_stays_out(dev, dtype, dim, form, rows, lens, page):
    """What lies behind the sequences, in absent pages and in rows that a causal limit hides (codes and scale bytes 255) reaches no
    row that does not see it; a marked position makes those NaN that do."""
    b, hq, hkv = len(lens), 4, 2
    width = max(-(-max(lens) // page), 1) + 1
    table = _tables(b * width, width, b, 2)
    c = _pool(dev, b * width, hkv, page, dim, 0, garbage=True)
    g = _gen(11)
    total = sum(lens)
    x = torch.randn(total, hkv, dim, generator=g).to(dtype)
    y = torch.randn(total, hkv, dim, generator=g).to(dtype)
    cu = _cu(lens)
    if lens[0] > 3:        # the last position of the first sequence holds a NaN key, the one before it an infinite value
        x[cu[1] - 1, 0, 3] = math.nan
        y[cu[1] - 2, 1, 7] = math.inf
    args = (_i32(table, dev), _i32(lens, dev))
    if total:
        kv.kv_write(c, x.to(dev), y.to(dev), *args, _i32(cu, dev))
    if lens[0] > page:     # a page in the middle of what is visible goes away
        table[0][0] = b * width
    q = torch.randn(b * rows, hq, dim, generator=g).to(dtype).to(dev)
    out, lse = kv.kv_attention(q, c, _i32(table, dev), _i32(lens, dev), lse=True, form=form)
    ref, rl, mag, err = ok.attention(q, c, table, lens)
    _check(out, ref, mag, err, form, max(lens))
    _check_lse(lse, rl, err)


@pytest.mark.parametrize("b,rows,hq,hkv,prefix,lens,dim,page", [
    (2, 1, 8, 2, 100, [5, 40], 128, 64),            # few rows on both sides
    (3, 2, 4, 1, 1777, [0, 3, 200], 64, 16),        # a sequence with nothing of its own
    (24, 1, 16, 2, 3001, None, 128, 64),            # many rows on the prefix, few on each sequence
    (2, 70, 4, 2, 333, [90, 75], 128, 32),          # many on both
    (5, 1, 4, 4, 1, [1, 2, 3, 4, 5], 64, 256),
    (3, 1, 4, 4, 0, [7, 2, 3], 128, 64),            # no prefix after all
])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("form", [None] + FORMS)
def test_shared_prefix(dev, dtype, form, b, rows, hq, hkv, prefix, lens, dim, page):
    lens = lens or [1 + 17 * i for i in range(b)]
    width = max(-(-max(lens) // page), 1)
    pre = -(-prefix // page)
    pages = b * width + pre + 1
    table = _tables(pages, width, b, 3)
    used = {p for t in table for p in t}
    common = [p for p in range(pages) if p not in used][:pre]
    c = _pool(dev, pages, hkv, page, dim, 12)
    q = (2.0 * torch.randn(b * rows, hq, dim, generator=_gen(13))).to(dtype).to(dev)
    for causal in (True, False):
        out, lse = kv.kv_attention_shared(q, c, _i32(common, dev), prefix, _i32(table, dev), _i32(lens, dev), causal=causal, lse=True,
                                         form=form)
        ref, rl, mag, err = ok.attention(q, c, table, lens, None, causal, prefix=common, prefix_len=prefix)
        _check(out, ref, mag, err, form, prefix + max(lens))
        _check_lse(lse, rl, err)


@pytest.mark.parametrize("form", FORMS)
def test_many_sequences(dev, form):
    """More sequences than a wavefront has lanes, uneven, some without rows or without keys, alone and behind a prefix."""
    b, hq, hkv, dim, page = 200, 4, 2, 64, 16
    new = [(i * 7) % 4 for i in range(b)]
    lens = [(i * i) % 97 for i in range(b)]
    cu = _cu(new)
    width = 7
    table = _tables(b * width + 10, width, b, 21)
    used = {p for t in table for p in t}
    common = [p for p in range(b * width + 10) if p not in used]
    c = _pool(dev, b * width + 10, hkv, page, dim, 22)
    q = torch.randn(cu[-1], hq, dim, generator=_gen(23)).to(BF).to(dev)
    args = (_i32(table, dev), _i32(lens, dev), _i32(cu, dev))
    out, lse = kv.kv_attention(q, c, *args, lse=True, form=form)
    ref, rl, mag, err = ok.attention(q, c, table, lens, cu)
    _check(out, ref, mag, err, form, 97)
    _check_lse(lse, rl, err)
    out, lse = kv.kv_attention_shared(q, c, _i32(common, dev), 155, *args, lse=True, form=form)
    ref, rl, mag, err = ok.attention(q, c, table, lens, cu, prefix=common, prefix_len=155)
    _check(out, ref, mag, err, form, 252)
    _check_lse(lse, rl, err)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rows,gap", [(600, 40), (600, 13), (100, 25), (2, 30)])
def test_rising_scores(dev, dim, form, rows, gap):
    """Scores that rise by `gap` (base 2) from one stretch of keys to the next, and such that begin far below: references move, in
    whole and divided items."""
    hkv, page, n = 2, 64, 1500
    keys = torch.zeros(n, hkv, dim)
    keys[:, :, 0] = (torch.arange(n) // 100)[:, None] * 1.0
    keys[:, 1] *= -1.0
    c = kv.kv_cache(30, hkv, page, dim, FP4, dev)
    table = _tables(30, 24, 1, 4)
    args = (_i32(table, dev), _i32([n], dev))
    kv.kv_write(c, keys.to(BF).to(dev), torch.randn(n, hkv, dim, generator=_gen(5)).to(BF).to(dev), *args)
    q = torch.zeros(rows, 4, dim)
    q[..., 0] = gap * math.log(2) * dim ** 0.5
    q = q.to(BF).to(dev)
    out, lse = kv.kv_attention(q, c, *args, lse=True, form=form)
    ref, rl, mag, err = ok.attention(q, c, table, [n])
    _check(out, ref, mag, err, form, n)
    _check_lse(lse, rl, err)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rows", [2, 100, 600])
@pytest.mark.parametrize("gap", [5, 7, 8, 9, 11, 12])
def test_scores_that_rise_a_little(dev, dim, form, rows, gap):
    """Rises about as far as a reference stays where it is."""
    test_rising_scores(dev, dim, form, rows, gap)


@pytest.mark.parametrize("dim", [64, 128])
def test_time_of_scores_that_rise_a_little(dev, dim):
    """Keys that score 10 (base 2) over a share's first ones move the reference once, as such do that score 20 over: the same time, where
    doing every half's softmax again took 1.8 to 1.9 times as long. So many sequences that a workgroup has all keys of one."""
    b, rows, heads, page, n = 256, 128, 2, 64, 8192
    c = _pool(dev, n // page, heads, page, dim, 3)
    for t in (c.k, c.k_scale):
        t.view(torch.uint8).zero_()
    key = torch.zeros(dim)
    key[0] = 6.0
    codes, scales = ok.quantise4(key)
    c.k.view(torch.uint8)[1:], c.k_scale.view(torch.uint8)[1:] = codes.to(dev), scales.to(dev)
    q = torch.zeros(b * rows, heads, dim, dtype=BF, device=dev)
    q[..., 0] = 1.0
    args = (torch.arange(n // page, dtype=torch.int32, device=dev).expand(b, -1).contiguous(), _i32([n] * b, dev))
    best = {10: math.inf, 20: math.inf}
    for _ in range(8):
        for gap in best:
            a, z = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(4):
                kv.kv_attention(q, c, *args, causal=False, scale=gap * math.log(2) / 6, form="chunk")
            z.record()
            z.synchronize()
            best[gap] = min(best[gap], a.elapsed_time(z))
    assert best[10] < 1.4 * best[20], best


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rows", [1, 90])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_query_magnitudes(dev, form, rows, dtype):
    """Query rows of every size beside each other, zeros and infinities among them: each has its own result."""
    n, dim, page = 300, 128, 32
    sizes = [0.0, 1e-7, 1e-3, 1.0, 30.0, 3e3] if dtype == HF else [0.0, 1e-30, 1e-10, 1.0, 1e3, 1e8, 1e30]
    g = _gen(40)
    q = torch.randn(rows, 8, dim, generator=g) * torch.tensor([sizes[i % len(sizes)] for i in range(rows * 8)]).view(rows, 8, 1)
    q = q.to(dtype)
    q[0, 3, 5] = math.nan
    c = _pool(dev, 10, 2, page, dim, 41)
    table = _tables(10, 10, 1, 42)
    out, lse = kv.kv_attention(q.to(dev), c, _i32(table, dev), _i32([n], dev), lse=True, form=form)
    ref, rl, mag, err = ok.attention(torch.nan_to_num(q, nan=0.0).to(dev), c, table, [n])
    assert torch.isnan(out[0, 3]).all() and torch.isnan(lse[0, 3])
    keep = torch.ones(rows, 8, dtype=torch.bool, device=dev)
    keep[0, 3] = False
    # rows whose scores' error is past what the bound is for (a key's share is then any) only have to be finite
    sure = keep & (err < 0.1)
    for a in (ref, mag):
        a[~sure] = 0.0
    assert torch.isfinite(out[keep]).all()
    _check(torch.where(sure[..., None], out, 0.0), ref, mag, torch.where(sure, err, 0.0), form, n)
    assert ((lse.double() - rl).abs() <= err + 2.0 ** -22 * rl.abs() + 2.0 ** -20)[sure].all()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rows,n,prefix_len", [(1, 200, 0), (1, 20011, 0), (100, 3001, 0), (3, 100, 9000), (200, 90, 700)])
@pytest.mark.parametrize("size", [2.0 ** 120, 2.0 ** 60, 2.0 ** -60, 2.0 ** -80])
def test_value_magnitudes(dev, form, rows, n, prefix_len, size):
    """Values of very large and very small size: bf16 results keep their precision."""
    hkv, dim, page = 2, 64, 32
    width, pre = -(-n // page), -(-prefix_len // page)
    c = _pool(dev, width + pre, hkv, page, dim, 50)
    v = torch.randn(width + pre, hkv, page, dim, generator=_gen(51)) * size
    codes, scale = ok.quantise4(v.to(BF))
    c.v.copy_(codes.to(dev))
    c.v_scale.copy_(scale.to(dev))
    table = [list(range(pre, pre + width))]
    q = torch.randn(rows, 4, dim, generator=_gen(52)).to(BF).to(dev)
    args = (_i32(table, dev), _i32([n], dev))
    if prefix_len:
        out = kv.kv_attention_shared(q, c, _i32(list(range(pre)), dev), prefix_len, *args, form=form)
    else:
        out = kv.kv_attention(q, c, *args, form=form)
    ref, _, mag, err = ok.attention(q, c, table, [n], prefix=list(range(pre)), prefix_len=prefix_len)
    _check(out, ref, mag, err, form, n + prefix_len)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rise,low", [(11, 128), (0, 0)])
def test_sums_of_the_largest_values(dev, dim, form, rise, low):
    """Very many keys on one wave, all of the same weight but a first stretch `rise` (base 2) below, with the largest values that the
    format holds: their sums, not yet divided, stay finite. So many sequences that a workgroup has all keys of one; they share pages."""
    b, heads, page, n = 96, 8, 64, (1 << 15) + 128
    pages = -(-n // page)
    c = kv.kv_cache(pages, heads, page, dim, FP4, dev)
    codes, scales = ok.quantise4(torch.full((dim,), 6 * 2.0 ** 125))
    c.v.view(torch.uint8)[:] = codes.to(dev)
    c.v_scale.view(torch.uint8)[:] = scales.to(dev)
    key = torch.zeros(dim)
    key[0] = 6.0
    codes, scales = ok.quantise4(key)
    c.k.view(torch.uint8)[low // page:] = codes.to(dev)
    c.k_scale.view(torch.uint8)[:] = scales.to(dev)
    q = torch.zeros(b, heads, dim, dtype=BF, device=dev)
    q[..., 0] = 1.0
    table = torch.arange(pages, dtype=torch.int32, device=dev).expand(b, pages).contiguous()
    scale = rise * math.log(2) / 6.0
    out, lse = kv.kv_attention(q, c, table, _i32([n] * b, dev), scale=scale, lse=True, form=form)
    ref = torch.full((b, heads, dim), 6 * 2.0 ** 125, dtype=torch.float64, device=dev)
    err = torch.full((b, heads), 2.0 ** -20, dtype=torch.float64, device=dev)   # a score is one product, scaled and less a reference: 3 roundings
    _check(out, ref, ref, err, form, n)
    _check_lse(lse, torch.full_like(err, math.log(low + (n - low) * 2.0 ** rise)), err)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rows,prefix_len", [(3, 0), (90, 0), (90, 300)])
def test_fp16_results_are_rounded_once(dev, dim, form, rows, prefix_len):
    """fp16 results differ from float64 by little more than their own rounding."""
    n, page, hkv = 700, 64, 2
    width, pre = -(-n // page), -(-prefix_len // page)
    c = _pool(dev, width + pre, hkv, page, dim, 30)
    table = [list(range(pre, pre + width))]
    q = torch.randn(rows, 8, dim, generator=_gen(31)).to(HF).to(dev)
    args = (_i32(table, dev), _i32([n], dev))
    if prefix_len:
        out = kv.kv_attention_shared(q, c, _i32(list(range(pre)), dev), prefix_len, *args, form=form)
    else:
        out = kv.kv_attention(q, c, *args, form=form)
    ref, _, mag, err = ok.attention(q, c, table, [n], prefix=list(range(pre)), prefix_len=prefix_len)
    _check(out, ref, mag, err, form, n + prefix_len)


# ---------------------------------------------------------------- layouts, contents, sizes
def test_layouts(dev):
    """Pages and heads of a cache apart, query rows and results strided, a wider table, out over q."""
    pages, heads, page, dim, n = 9, 2, 32, 128, 130
    whole = torch.zeros(pages, 3, heads + 1, page, dim // 2 + dim // 32 + 12, dtype=torch.uint8, device=dev)
    flat = whole.view(pages, 3, heads + 1, -1)
    span, scales = page * dim // 2, page * dim // 32

    def codes(i):
        return flat[:, i, :heads, :span].view(pages, heads, page, dim // 2)

    def scale(i):
        return flat[:, i, :heads, span:span + scales].view(pages, heads, page, dim // 32)
    far = kv.KVCache(codes(0), codes(1), scale(0), scale(1))
    near = kv.kv_cache(pages, heads, page, dim, FP4, dev)
    x, y = (torch.randn(n, heads, dim, generator=_gen(i)).to(BF).to(dev) for i in range(2))
    table = _i32([[4, 8, 1, 0, 7, 3, 2]], dev)[:, :5]
    lens = _i32([n], dev)
    for c in (far, near):
        kv.kv_write(c, x, y, table, lens)
    for a, b in zip(kv.kv_read(far, table, lens, rows=n), kv.kv_read(near, table, lens, rows=n)):
        assert torch.equal(a, b)
    assert (whole[:, 2] == 0).all() and (whole[:, :, heads] == 0).all()
    for rows in (1, 100):
        q = torch.randn(rows, 6, 3, dim, generator=_gen(9)).to(BF).to(dev)[:, :, 1]
        want = kv.kv_attention(q, near, table, lens)
        out = torch.zeros(rows, 7, dim, dtype=BF, device=dev)[:, :6]
        assert kv.kv_attention(q, far, table, lens, out=out) is out and torch.equal(out, want)
        kv.kv_attention(q, far, table, lens, out=q)
        assert torch.equal(q, want)


def test_rows_that_no_sequence_has_stay(dev):
    c = _pool(dev, 4, 2, 16, 64, 1)
    table, lens, cu = _i32([[0, 1], [2, 3]], dev), _i32([20, 30], dev), _i32([2, 3, 5], dev)
    q = torch.randn(9, 4, 64, generator=_gen(2)).to(BF).to(dev)
    for form in FORMS:
        out = torch.full_like(q, 5.0)
        kv.kv_attention(q, c, table, lens, cu, out=out, form=form)
        assert (out[:2] == 5).all() and (out[5:] == 5).all()
        assert torch.equal(out[2:5], kv.kv_attention(q[2:5], c, table, lens, cu - 2, form=form))


def test_bad_contents_stay_inside(dev):
    """Lengths beyond the table, negative ones, page numbers that are none, row offsets that fall or pass the end: clamped or
    absent, and the sequences beside them keep their results."""
    pages, page, dim = 6, 16, 64
    c = _pool(dev, pages, 2, page, dim, 43)
    before = [t.clone() for t in _bytes(c)]
    table = [[0, 1], [-7, 2 ** 31 - 1], [2, pages], [3, 4]]
    lens = [10 ** 9, 20, 32, -5]
    for rows, form in ((1, "token"), (30, "token"), (1, "chunk"), (30, "chunk")):
        q = torch.randn(4 * rows, 4, dim, generator=_gen(44)).to(BF).to(dev)
        out = kv.kv_attention(q, c, _i32(table, dev), _i32(lens, dev), causal=False, form=form)
        ref, _, mag, err = ok.attention(q, c, table, [32, 20, 32, 0], None, False)
        _check(out, ref, mag, err, form, 32)
        assert (out[rows:2 * rows] == 0).all() and (out[3 * rows:] == 0).all()
    q = torch.randn(6, 4, dim, generator=_gen(45)).to(BF).to(dev)
    x = torch.randn(6, 2, dim, generator=_gen(46)).to(BF).to(dev)
    bad = _i32([2, -3, 5, 1, 99], dev)
    dead = _i32([[-1, pages]] * 4, dev)
    kv.kv_write(c, x, x, dead, _i32([20] * 4, dev), bad)
    assert all(torch.equal(a, b) for a, b in zip(before, _bytes(c)))
    kv.kv_read(c, dead, _i32([20] * 4, dev), bad, rows=6)
    for form in FORMS:
        kv.kv_attention(q, c, dead, _i32([20] * 4, dev), bad, form=form)
        kv.kv_attention_shared(q, c, _i32([9, -1, 2], dev), 40, dead, _i32([20] * 4, dev), bad, form=form)
    torch.cuda.synchronize()


def test_offsets_past_32_bits(dev):
    """Pages beyond 4 GiB of codes."""
    heads, page, dim = 8, 256, 128
    pages = (5 << 30) // (heads * page * dim // 2)
    k, v = (torch.empty((pages, heads, page, dim // 2), dtype=torch.uint8, device=dev) for _ in range(2))
    c = kv.KVCache(k, v, *(torch.empty((pages, heads, page, dim // 32), dtype=torch.uint8, device=dev) for _ in range(2)))
    table, lens = [[pages - 1, 0, pages - 2], [1, pages - 3, 2]], [600, 700]
    g = _gen(60)
    x, y = (torch.randn(1300, heads, dim, generator=g).to(BF).to(dev) for _ in range(2))
    args = (_i32(table, dev), _i32(lens, dev), _i32([0, 600, 1300], dev))
    kv.kv_write(c, x, y, *args)
    for a, b in zip((x, y), kv.kv_read(c, *args, rows=1300)):
        assert torch.equal(b, ok.values4(*ok.quantise4(a)).to(BF))
    for rows, form in ((1, None), (50, "chunk")):
        q = torch.randn(2 * rows, 8, dim, generator=g).to(BF).to(dev)
        out = kv.kv_attention(q, c, *args[:2], form=form)
        ref, _, mag, err = ok.attention(q, c, table, lens)
        _check(out, ref, mag, err, form, 700)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rows,prefix_len", [(1, 0), (1, 500), (60, 0)])
def test_captured_steps(dev, form, rows, prefix_len):
    """A step captured once follows new inputs, lengths and page tables on every replay; two captured steps run at once on two
    streams."""
    b, hq, hkv, dim, page = 2, 4, 2, 128, 32

    def step(c, q, k, v, tab, lens, ptab):
        kv.kv_write(c, k, v, tab, lens)
        if prefix_len:
            return kv.kv_attention_shared(q, c, ptab, prefix_len, tab, lens, form=form)
        return kv.kv_attention(q, c, tab, lens, form=form)
    steps = []
    for which in range(2):
        c = _pool(dev, 80, hkv, page, dim, 80 + which)
        g = _gen(81 + which)
        q, k, v = (torch.randn(b * rows, h, dim, generator=g).to(BF).to(dev) for h in (hq, hkv, hkv))
        tab, ptab = _i32(_tables(60, 30, b, which), dev), _i32(list(range(60, 76)), dev)
        args = (c, q, k, v, tab, _i32([700, 130], dev), ptab)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step(*args)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*args)
        steps.append((graph, out, args, torch.cuda.Stream()))
    for replay in range(3):
        want = []
        for graph, out, args, _ in steps:
            c, q, k, v, tab, lens, ptab = args
            for t in (q, k, v):
                t.copy_(torch.randn(t.shape, generator=_gen(replay + 7)).to(BF))
            lens.copy_(torch.tensor([60 + 300 * replay, 959 - replay], dtype=torch.int32))
            tab.copy_(tab.flip(1))
            want.append(step(*args).clone())
            out.zero_()
        torch.cuda.synchronize()
        for graph, _, _, stream in steps:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (_, out, _, _), w in zip(steps, want):
            assert torch.equal(out.view(torch.int16), w.view(torch.int16)), replay


def test_bytes_and_named_types(dev):
    """Tensors of torch's 4-bit and exponent types and plain bytes are the same to a cache."""
    c = kv.kv_cache(3, 2, 16, 64, FP4, dev)
    assert c.k.dtype == FP4 and c.k_scale.dtype == torch.float8_e8m0fnu and c.dim == 64 and c.k.shape == (3, 2, 16, 32)
    d = kv.KVCache(*_bytes(c))
    x = torch.randn(4, 2, 64, generator=_gen(1)).to(BF).to(dev)
    args = (_i32([[1]], dev), _i32([4], dev))
    kv.kv_write(d, x, x, *args)
    assert torch.equal(kv.kv_read(c, *args, rows=4)[0], ok.values4(*ok.quantise4(x)).to(BF))


@pytest.mark.parametrize("fmt", [torch.int8, torch.float8_e4m3fn, torch.float4_e2m1fn_x2])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_beyond_the_last_cache(dev, fmt, dtype):
    """Calls of so many rows that they are streamed leave what calls of parts of them leave, bit for bit."""
    n, heads, dim, page = 9001, 64, 128, 64
    pages = -(-n // page)
    g = torch.Generator(device=dev).manual_seed(5)
    k, v = (torch.randn(n, heads, dim, generator=g, device=dev).to(dtype) for _ in range(2))
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(6)).to(torch.int32).to(dev)[None]
    one, parts = (kv.kv_cache(pages, heads, page, dim, fmt, dev) for _ in range(2))
    kv.kv_write(one, k, v, table, _i32([n], dev))
    step = 1000                          # 65 MB of 32-bit K and V
    for at in range(0, n, step):
        end = min(at + step, n)
        kv.kv_write(parts, k[at:end], v[at:end], table, _i32([end], dev))
    for x, y in zip((one.k, one.v, one.k_scale, one.v_scale), (parts.k, parts.v, parts.k_scale, parts.v_scale)):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    rk, rv = kv.kv_read(one, table, _i32([n], dev), rows=n, dtype=dtype)
    for at in range(0, n, step):
        end = min(at + step, n)
        pk, pv = kv.kv_read(parts, table, _i32([end], dev), rows=end - at, dtype=dtype)
        assert torch.equal(rk[at:end], pk) and torch.equal(rv[at:end], pv)


@pytest.mark.parametrize("fmt", [torch.int8, torch.float8_e4m3fn, torch.float4_e2m1fn_x2])
def test_time_of_fp32_rows_beyond_the_last_cache(dev, fmt):
    """A call of many fp32 rows takes no longer than calls of parts of them that the last cache holds (streamed past it such rows took 1.17
    times as long to write and 1.3 to read)."""
    n, heads, dim, page, step = 12288, 56, 128, 64, 4096
    c = kv.kv_cache(n // page, heads, page, dim, fmt, dev)
    k, v = (torch.randn(n, heads, dim, device=dev) for _ in range(2))
    table = torch.arange(n // page, dtype=torch.int32, device=dev)[None]
    ends = [_i32([at + step], dev) for at in range(0, n, step)]
    calls = {("write", 1): lambda: kv.kv_write(c, k, v, table, ends[-1]),
             ("write", 3): lambda: [kv.kv_write(c, k[i * step:(i + 1) * step], v[i * step:(i + 1) * step], table, e) for i, e in enumerate(ends)],
             ("read", 1): lambda: kv.kv_read(c, table, ends[-1], out=(k, v)),
             ("read", 3): lambda: [kv.kv_read(c, table, e, out=(k[i * step:(i + 1) * step], v[i * step:(i + 1) * step])) for i, e in enumerate(ends)]}
    best = dict.fromkeys(calls, math.inf)
    for _ in range(8):
        for what, call in calls.items():
            a, z = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            call()
            a.record()
            for _ in range(4):
                call()
            z.record()
            z.synchronize()
            best[what] = min(best[what], a.elapsed_time(z))
    assert best["read", 1] < 1.12 * best["read", 3] and best["write", 1] < 1.12 * best["write", 3], best
