"""The paged, quantised key / value cache (rapid_h3.kvcache) on the GPU: codes and scales bit for bit against the plain
restatement, values read back, attention (both kernels, whole and in parts, with and without a shared prefix) against float64
over the stored values."""
import math

import pytest
import torch

from oracle import kvcache as ok
from rapid_h3 import kvcache as kv

pytestmark = pytest.mark.gpu

I8, F8 = torch.int8, torch.float8_e4m3fn
FORMS = ["token", "chunk"]          # both kernels, whichever the sizes would choose
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _pool(dev, fmt, pages, heads, page, dim, seed, garbage=False):
    """A cache full of quantised random values; garbage: full of what an unwritten pool may hold instead (NaN codes, NaN and
    infinite scales)."""
    if garbage:
        k, v = (torch.full((pages, heads, page, dim), 0x7f, dtype=torch.uint8, device=dev).view(fmt) for _ in range(2))
        ks = torch.full((pages, heads, page), math.nan, device=dev)
        ks[:, :, ::3] = math.inf
        return kv.KVCache(k, v, ks, ks.clone())
    g = _gen(seed)
    kc = 2.0 * torch.randn(1, heads, 1, dim, generator=g)
    k, ks = ok.quantise(torch.randn(pages, heads, page, dim, generator=g) + kc, fmt)
    v, vs = ok.quantise(torch.randn(pages, heads, page, dim, generator=g) * torch.exp(torch.randn(pages, heads, page, 1, generator=g)), fmt)
    return kv.KVCache(*(t.to(dev) for t in (k, v, ks, vs)))


def _tables(pages, width, batch, seed):
    """Disjoint pages in any order, one list per sequence."""
    p = torch.randperm(pages, generator=_gen(seed + 99)).tolist()
    return [p[b * width:(b + 1) * width] for b in range(batch)]


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _check(out, ref, mag, err, terms):
    """|out - ref| within the output's rounding (half a step of its type), `terms` f16 roundings of the weights and values
    (2^-11 each of sum p |v|), and the scores' error e (at most (exp(2 e) - 1) of the same sum)."""
    eps = torch.finfo(out.dtype).eps / 2
    o = out.double()
    known = ~torch.isnan(ref)
    assert torch.equal(torch.isnan(o), ~known)
    tol = eps * ref.abs() * 1.01 + (terms * 2.0 ** -11 + torch.expm1(2 * err)[..., None]) * mag * 1.05 + 1e-30
    bad = known & ((o - ref).abs() > tol)
    assert not bad.any(), (int(bad.sum()), float(((o - ref).abs() / tol)[known].max()))


def _check_lse(lse, ref, err):
    known = ~torch.isnan(ref)
    assert torch.equal(torch.isnan(lse), ~known)
    e = lse.double()
    inf = known & torch.isinf(ref)
    assert torch.equal(e[inf], ref[inf])
    fin = known & ~inf
    tol = err + 2.0 ** -22 * ref.abs() + 2.0 ** -21
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


@pytest.mark.parametrize("fmt", [I8, F8])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("heads,dim,page,lens,new,strided", [
    (3, 128, 64, [1], [1], False),
    (1, 64, 16, [17, 5, 33], [17, 3, 16], True),
    (2, 128, 32, [0, 40, 7, 64], [0, 33, 9, 1], False),        # a sequence without rows, one with more rows than positions
    (5, 64, 256, [300], [300], True),
    (8, 128, 128, [130, 1, 77], [2, 1, 0], False),
])
def test_write_and_read(dev, fmt, dtype, heads, dim, page, lens, new, strided):
    b = len(lens)
    width = max(-(-max(lens) // page), 1) + 1
    pages = b * width + 2
    table = _tables(pages, width, b, 5)
    if b > 1:
        table[1][0] = -1                                       # an absent page
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    rows = cu[-1] + 3                                          # three rows that no sequence has
    even = len(set(new)) == 1
    if even:
        rows = cu[-1]
    k, v = _rows(rows, heads, dim, dtype, 1, strided, dev), _rows(rows, heads, dim, dtype, 2, strided, dev)
    c = _pool(dev, fmt, pages, heads, page, dim, 3)
    want = [t.clone() for t in (c.k.view(torch.uint8), c.v.view(torch.uint8), c.k_scale, c.v_scale)]
    args = (_i32(table, dev), _i32(lens, dev), None if even else _i32(cu, dev))
    kv.kv_write(c, k, v, *args)
    got_k, got_v = kv.kv_read(c, *args, rows=rows, dtype=dtype)
    keep = torch.full((rows, heads, dim), 7.0, dtype=dtype, device=dev)
    kept = (keep, keep.clone())
    kv.kv_read(c, *args, out=kept)
    for x, codes, scales, got, left in ((k, want[0], want[2], got_k, kept[0]), (v, want[1], want[3], got_v, kept[1])):
        q, s = ok.quantise(x, fmt)
        for r, where in enumerate(ok.rows_of(lens, None if even else cu, rows, b)):
            at = where and ok.slot(table, pages, page, *where)
            if at:
                codes[at[0], :, at[1]] = q[r].view(torch.uint8)
                scales[at[0], :, at[1]] = s[r]
                value = (q[r].float() * s[r][:, None]).to(dtype)
                assert torch.equal(got[r], value) and torch.equal(left[r], value), r
            else:
                assert (got[r] == 0).all(), r
                assert (left[r] == (7.0 if where is None else 0.0)).all(), r
    for x, y in zip(want, (c.k.view(torch.uint8), c.v.view(torch.uint8), c.k_scale, c.v_scale)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("fmt", [I8, F8])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_write_special_rows(dev, fmt, dtype):
    """Zeros of both signs, the smallest and largest magnitudes, halfway quotients, infinities and NaN."""
    d, page = 128, 16
    big = torch.finfo(dtype).max
    rows = [torch.zeros(d), -torch.zeros(d), torch.full((d,), torch.finfo(dtype).tiny), torch.full((d,), big),
            torch.arange(d) - 63.5, (torch.arange(d) - 64.0) * 2.0, torch.randn(d, generator=_gen(0)) * 1e-6,
            torch.linspace(-448, 448, d), torch.randn(d, generator=_gen(1)), torch.randn(d, generator=_gen(2)),
            torch.randn(d, generator=_gen(3))]
    rows[8][5] = math.inf
    rows[9][127] = math.nan
    rows[10][0], rows[10][1] = -math.inf, math.nan
    x = torch.stack(rows)[:, None].to(dtype).to(dev)
    n = x.shape[0]
    c = kv.kv_cache(1, 1, page, d, fmt, dev)
    args = (_i32([[0]], dev), _i32([n], dev))
    kv.kv_write(c, x, x.flip(0).contiguous(), *args)
    for y, codes, scales in ((x, c.k, c.k_scale), (x.flip(0), c.v, c.v_scale)):
        q, s = ok.quantise(y, fmt)
        assert torch.equal(codes[0, 0, :n].view(torch.uint8), q[:, 0].view(torch.uint8))
        assert torch.equal(torch.nan_to_num(scales[0, 0, :n], nan=-1.0), torch.nan_to_num(s[:, 0], nan=-1.0))
    got, _ = kv.kv_read(c, *args, rows=n, dtype=F32)
    # 127 * fl(max / 127) lies above the largest fp32 value: that row, and only that, may read back as infinite
    assert torch.isnan(got[8:]).all() and torch.isfinite(got[:3]).all() and torch.isfinite(got[4:8]).all()
    assert torch.equal(got[3], ok.quantise(x, fmt)[0][3].float() * ok.quantise(x, fmt)[1][3][:, None])


def test_write_many_sequences(dev):
    """More sequences than a wavefront has lanes, some of them without rows: every row finds its own."""
    b, page, heads, dim = 1500, 16, 2, 64
    new = [(i * 7) % 4 for i in range(b)]
    lens = [n + i % 13 for i, n in enumerate(new)]
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    pages = b
    table = [[i] for i in range(b)]
    x = torch.randn(cu[-1], heads, dim, generator=_gen(4)).to(BF).to(dev)
    c = kv.kv_cache(pages, heads, page, dim, I8, dev)
    args = (_i32(table, dev), _i32(lens, dev), _i32(cu, dev))
    kv.kv_write(c, x, -x, *args)
    q, s = ok.quantise(x, I8)
    where = ok.rows_of(lens, cu, cu[-1], b)
    p = torch.tensor([w[0] for w in where], device=dev)
    o = torch.tensor([w[1] for w in where], device=dev)
    assert torch.equal(c.k[p, :, o], q) and torch.equal(c.v[p, :, o], -q) and torch.equal(c.k_scale[p, :, o], s)
    assert int((c.k_scale != 0).sum()) == cu[-1] * heads
    k, v = kv.kv_read(c, *args, rows=cu[-1])
    assert torch.equal(k, (q.float() * s[..., None]).to(BF)) and torch.equal(v, -k)


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


@pytest.mark.parametrize("fmt", [I8, F8])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention(dev, fmt, dtype, form, case):
    hq, hkv, dim, page, lens, new, causal = CASES[case]
    b = len(lens)
    width = max(-(-max(lens) // page), 1)
    pages = b * width + 3
    table = _tables(pages, width, b, case)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    even = len(set(new)) == 1
    t = cu[-1]
    c = _pool(dev, fmt, pages, hkv, page, dim, case)
    q = (2.0 * torch.randn(t, hq, dim, generator=_gen(case + 50))).to(dtype).to(dev)
    out, lse = kv.kv_attention(q, c, _i32(table, dev), _i32(lens, dev), None if even else _i32(cu, dev), causal=causal, lse=True,
                               form=form)
    ref, rl, mag, err = ok.attention(q, c, table, lens, None if even else cu, causal)
    _check(out, ref, mag, err, 3.1)
    _check_lse(lse, rl, err)


@pytest.mark.parametrize("fmt", [I8, F8])
@pytest.mark.parametrize("rows,hq,hkv,lens,page", [
    (1, 8, 2, [20011], 64),              # one sequence on many workgroups
    (1, 8, 8, [9000, 31, 4001, 1, 0, 2500], 16),   # uneven histories: items begin and end inside a workgroup's share
    (2, 14, 2, [5000, 5001, 200], 128),
    (40, 4, 1, [9001], 64),              # key ranges of the chunk kernel
    (100, 2, 2, [3000, 20], 32),
])
@pytest.mark.parametrize("form", FORMS)
def test_attention_in_parts(dev, fmt, form, rows, hq, hkv, lens, page):
    b, dim = len(lens), 128
    width = -(-max(lens) // page)
    table = _tables(b * width, width, b, 1)
    c = _pool(dev, fmt, b * width, hkv, page, dim, 8)
    q = (2.0 * torch.randn(b * rows, hq, dim, generator=_gen(9))).to(BF).to(dev)
    args = (_i32(table, dev), _i32(lens, dev))
    out, lse = kv.kv_attention(q, c, *args, lse=True, form=form)
    ref, rl, mag, err = ok.attention(q, c, table, lens)
    _check(out, ref, mag, err, 3.1)
    _check_lse(lse, rl, err)
    again = kv.kv_attention(q, c, *args, form=form)
    assert torch.equal(out.view(torch.int16), again.view(torch.int16))          # the same bits every time


@pytest.mark.parametrize("fmt", [I8, F8])
@pytest.mark.parametrize("rows,lens,page", [(1, [33, 5, 0], 16), (3, [70, 9], 64), (1, [1000], 32), (70, [90, 71], 16), (80, [40], 32)])
@pytest.mark.parametrize("form", FORMS)
def test_unwritten_pool_stays_out(dev, fmt, form, rows, lens, page):
    """What lies behind the sequences, in absent pages and in rows that a causal limit hides (NaN codes, NaN and infinite
    scales) reaches no row that does not see it."""
    b, hq, hkv, dim = len(lens), 4, 2, 128
    width = max(-(-max(lens) // page), 1) + 1
    table = _tables(b * width, width, b, 2)
    c = _pool(dev, fmt, b * width, hkv, page, dim, 0, garbage=True)
    g = _gen(11)
    total = sum(lens)
    x = torch.randn(total, hkv, dim, generator=g).to(BF)
    y = torch.randn(total, hkv, dim, generator=g).to(BF)
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    if lens[0] > 3:        # the last position of the first sequence holds a NaN key, the one before it a NaN value
        x[cu[1] - 1, 0, 3] = math.nan
        y[cu[1] - 2, 1, 7] = math.inf
    args = (_i32(table, dev), _i32(lens, dev))
    if total:
        kv.kv_write(c, x.to(dev), y.to(dev), *args, _i32(cu, dev))
    if lens[0] > page:     # a page in the middle of what is visible goes away
        table[0][0] = b * width
    q = torch.randn(b * rows, hq, dim, generator=g).to(BF).to(dev)
    out, lse = kv.kv_attention(q, c, _i32(table, dev), _i32(lens, dev), lse=True, form=form)
    ref, rl, mag, err = ok.attention(q, c, table, lens)
    _check(out, ref, mag, err, 3.1)
    _check_lse(lse, rl, err)


@pytest.mark.parametrize("fmt", [I8, F8])
@pytest.mark.parametrize("b,rows,hq,hkv,prefix,lens,dim,page", [
    (2, 1, 8, 2, 100, [5, 40], 128, 64),            # few rows on both sides
    (3, 2, 4, 1, 1777, [0, 3, 200], 64, 16),        # a sequence with nothing of its own
    (24, 1, 16, 2, 3000, None, 128, 64),            # many rows on the prefix, few on each sequence
    (2, 70, 4, 2, 333, [90, 75], 128, 32),          # many on both
    (5, 1, 4, 4, 1, [1, 2, 3, 4, 5], 64, 256),
    (3, 1, 4, 4, 0, [7, 2, 3], 128, 64),            # no prefix after all
])
@pytest.mark.parametrize("form", [None] + FORMS)
def test_shared_prefix(dev, fmt, form, b, rows, hq, hkv, prefix, lens, dim, page):
    lens = lens or [1 + 17 * i for i in range(b)]
    width = max(-(-max(lens) // page), 1)
    pre = -(-prefix // page)
    pages = b * width + pre + 1
    table = _tables(pages, width, b, 3)
    used = {p for t in table for p in t}
    common = [p for p in range(pages) if p not in used][:pre]
    c = _pool(dev, fmt, pages, hkv, page, dim, 12)
    q = (2.0 * torch.randn(b * rows, hq, dim, generator=_gen(13))).to(HF).to(dev)
    for causal in (True, False):
        out, lse = kv.kv_attention_shared(q, c, _i32(common, dev), prefix, _i32(table, dev), _i32(lens, dev), causal=causal, lse=True,
                                         form=form)
        ref, rl, mag, err = ok.attention(q, c, table, lens, None, causal, prefix=common, prefix_len=prefix)
        _check(out, ref, mag, err, 3.1)
        _check_lse(lse, rl, err)


@pytest.mark.parametrize("form", FORMS)
def test_many_sequences(dev, form):
    """More sequences than a wavefront has lanes, uneven, some without rows or without keys, alone and behind a prefix."""
    b, hq, hkv, dim, page = 200, 4, 2, 64, 16
    new = [(i * 7) % 4 for i in range(b)]
    lens = [(i * i) % 97 for i in range(b)]
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    width = 7
    table = _tables(b * width + 10, width, b, 21)
    used = {p for t in table for p in t}
    common = [p for p in range(b * width + 10) if p not in used]
    c = _pool(dev, F8, b * width + 10, hkv, page, dim, 22)
    q = torch.randn(cu[-1], hq, dim, generator=_gen(23)).to(BF).to(dev)
    args = (_i32(table, dev), _i32(lens, dev), _i32(cu, dev))
    out, lse = kv.kv_attention(q, c, *args, lse=True, form=form)
    ref, rl, mag, err = ok.attention(q, c, table, lens, cu)
    _check(out, ref, mag, err, 3.1)
    _check_lse(lse, rl, err)
    out, lse = kv.kv_attention_shared(q, c, _i32(common, dev), 155, *args, lse=True, form=form)
    ref, rl, mag, err = ok.attention(q, c, table, lens, cu, prefix=common, prefix_len=155)
    _check(out, ref, mag, err, 3.1)
    _check_lse(lse, rl, err)


def test_prefix_and_sequences_on_their_own_kernels(dev):
    """A prefix long enough for the chunk kernel before sequences that take the token kernel."""
    b, hq, hkv, dim, page, prefix = 64, 8, 2, 128, 256, 60001
    lens = [1 + 5 * i for i in range(b)]
    pre = -(-prefix // page)
    table = _tables(2 * b + pre, 2, b, 24)
    used = {p for t in table for p in t}
    common = [p for p in range(2 * b + pre) if p not in used]
    c = _pool(dev, I8, 2 * b + pre, hkv, page, dim, 25)
    q = torch.randn(b, hq, dim, generator=_gen(26)).to(BF).to(dev)
    out, lse = kv.kv_attention_shared(q, c, _i32(common, dev), prefix, _i32(table, dev), _i32(lens, dev), lse=True)
    ref, rl, mag, err = ok.attention(q, c, table, lens, prefix=common, prefix_len=prefix)
    _check(out, ref, mag, err, 3.1)
    _check_lse(lse, rl, err)


@pytest.mark.parametrize("fmt", [I8, F8])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rows,hkv", [(1, 1), (9, 2), (70, 2), (400, 1)])
def test_fp16_results_are_rounded_once(dev, fmt, dim, form, rows, hkv):
    """fp16 results: the weights in two f16 terms (2^-22 of each, and sums in fp32: with 2^-20 of sum p |v| for both) leave little
    beside the rounding of the result."""
    n, page = 777, 32
    width = -(-n // page)
    table = _tables(2 * width, width, 2, 3)
    c = _pool(dev, fmt, 2 * width, hkv, page, dim, 6)
    q = torch.randn(2 * rows, 2 * hkv, dim, generator=_gen(7)).to(HF).to(dev)
    out = kv.kv_attention(q, c, _i32(table, dev), _i32([n, n - 300], dev), form=form)
    ref, _, mag, err = ok.attention(q, c, table, [n, n - 300])
    _check(out, ref, mag, err, 2.0 ** -9)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rows", [1, 50])
def test_query_magnitudes(dev, dtype, form, rows):
    """Query rows of every magnitude their type has, zero rows, and infinite or NaN ones, which change no other row."""
    c = _pool(dev, I8, 4, 1, 64, 128, 20)
    top = 100 if dtype == BF else 14
    q = torch.randn(6 * rows, 1, 128, generator=_gen(21))
    q *= torch.logspace(-top, 2, 6 * rows, base=2.0)[:, None, None]
    q[1], q[2, 0, 5], q[3, 0, 0] = 0.0, math.nan, math.inf
    q = q.to(dtype).to(dev)
    table, lens = [[0, 2]] * 6, [100] * 6
    out, lse = kv.kv_attention(q, c, _i32(table, dev), _i32(lens, dev), causal=False, lse=True, form=form)
    ref, rl, mag, err = ok.attention(q, c, table, lens, None, False)
    assert torch.isnan(out[2]).all() and torch.isnan(lse[2]).all()
    keep = [i for i in range(6 * rows) if i not in (2, 3)]
    _check(out[keep], ref[keep], mag[keep], err[keep], 3.1)
    _check_lse(lse[keep], rl[keep], err[keep])


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rows", [1, 60])
def test_extreme_scores_and_scales(dev, form, rows):
    """One key far above the others (their probabilities vanish), whose values are far smaller than theirs: value scales within
    2^24 of each other keep the weights' full precision."""
    dim, page, n = 128, 32, 200
    g = _gen(30)
    x, y = torch.randn(n, 1, dim, generator=g), torch.randn(n, 1, dim, generator=g)
    x[77] *= 40.0
    y *= torch.logspace(-6, 6, n, base=2.0)[torch.randperm(n, generator=g)][:, None, None]
    y[77] *= 1e-3
    c = kv.kv_cache(7, 1, page, dim, I8, dev)
    args = (_i32([[6, 0, 3, 2, 5, 4, 1]], dev), _i32([n], dev))
    kv.kv_write(c, x.to(dev), y.to(dev), *args)
    q = torch.cat([3.0 * torch.randn(rows, 2, dim, generator=g) + x[77] / 8]).to(BF).to(dev)
    out, lse = kv.kv_attention(q, c, *args, lse=True, causal=False, form=form)
    ref, rl, mag, err = ok.attention(q, c, [[6, 0, 3, 2, 5, 4, 1]], [n], None, False)
    _check(out, ref, mag, err, 3.1)
    _check_lse(lse, rl, err)


@pytest.mark.parametrize("fmt", [I8, F8])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rows,hkv,gap", [(600, 4, 70), (600, 4, 23), (100, 2, 45), (2, 2, 40)])
def test_rising_scores(dev, fmt, dim, form, rows, hkv, gap):
    """Scores that rise again and again along the keys, for some rows by far more than the weights' range, for others downwards or
    not at all, and a page that is not there."""
    page, n = 64, 1500
    g = _gen(41)
    u = torch.randn(dim, generator=g)
    u = u / u.norm() * 8.0
    rise = torch.cumsum((torch.rand(n, generator=g) < 1.0 / gap).float(), 0)
    k = rise[:, None, None] * u + 0.3 * torch.randn(n, hkv, dim, generator=g)
    v = torch.randn(n, hkv, dim, generator=g)
    width = -(-n // page)
    table = _tables(width, width, 1, 5)
    c = kv.kv_cache(width, hkv, page, dim, fmt, dev)
    kv.kv_write(c, k.to(dev), v.to(dev), _i32(table, dev), _i32([n], dev))
    table[0][9] = -1
    share = torch.tensor([0.3, 2.0, -1.0, 0.0])[torch.randint(0, 4, (rows, hkv), generator=g)]
    q = (share[..., None] * u + 0.3 * torch.randn(rows, hkv, dim, generator=g)).to(BF).to(dev)
    out, lse = kv.kv_attention(q, c, _i32(table, dev), _i32([n], dev), lse=True, causal=False, form=form)
    ref, rl, mag, err = ok.attention(q, c, table, [n], None, False)
    _check(out, ref, mag, err, 3.1)
    _check_lse(lse, rl, err)


# ---------------------------------------------------------------- neighbours of another magnitude
def _call(q, c, table, lens, cu, prefix, prefix_len, dev, **kw):
    """kv_attention or, with a prefix, kv_attention_shared, by lists."""
    args = (_i32(table, dev), _i32(lens, dev), None if cu is None else _i32(cu, dev))
    if prefix_len:
        return kv.kv_attention_shared(q, c, _i32(prefix, dev), prefix_len, *args, **kw)
    return kv.kv_attention(q, c, *args, **kw)


@pytest.mark.parametrize("fmt", [I8, F8])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("big", [2.0 ** 13, 2.0 ** 17, 2.0 ** 30, 1e12, 1e30])
@pytest.mark.parametrize("b,rows,prefix_len", [(1, 60, 0), (2, 300, 0), (6, 1, 333), (5, 40, 700)])
def test_rows_beside_far_larger_ones(dev, fmt, dim, form, big, b, rows, prefix_len):
    """A query row's result is its own, however large a finite row beside it is: of its sequence, or of another that shares the
    prefix."""
    hq, hkv, page = 4, 2, 32
    lens = [350 - 7 * i for i in range(b)]
    width, pre = 11, -(-prefix_len // page)
    table = _tables(b * width, width, b, 31)
    common = list(range(b * width, b * width + pre))
    c = _pool(dev, fmt, b * width + pre, hkv, page, dim, 32)
    q = 2.0 * torch.randn(b * rows, hq, dim, generator=_gen(33))
    at = [0, 3 * (b * rows) // 4]
    q[at] *= big
    q = q.to(BF).to(dev)
    out, lse = _call(q, c, table, lens, None, common, prefix_len, dev, lse=True, form=form)
    ref, rl, mag, err = ok.attention(q, c, table, lens, prefix=common, prefix_len=prefix_len)
    rest = [i for i in range(b * rows) if i not in at]
    _check(out[rest], ref[rest], mag[rest], err[rest], 3.1)
    _check_lse(lse[rest], rl[rest], err[rest])
    assert bool(torch.isfinite(out[at]).all()) and bool(torch.isfinite(lse[at]).all())


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rows", [1, 90])
def test_small_rows_beside_a_large_one_fp16(dev, form, rows):
    """The same for fp16 rows over the whole of that type's range, with scores that matter from large keys."""
    c = kv.kv_cache(5, 1, 64, 128, I8, dev)
    g = _gen(34)
    x, y = 2000.0 * torch.randn(300, 1, 128, generator=g), torch.randn(300, 1, 128, generator=g)
    args = (_i32([[0, 1, 2, 3, 4]], dev), _i32([300], dev))
    kv.kv_write(c, x.to(dev), y.to(dev), *args)
    q = 1e-3 * torch.randn(rows, 3, 128, generator=g)
    q[:, 0] *= 2.0 ** -8
    q[rows // 2, 1] = 30000.0 * torch.sign(q[rows // 2, 1])
    q = q.to(HF).to(dev)
    out = kv.kv_attention(q, c, *args, causal=False, form=form)
    ref, _, mag, err = ok.attention(q, c, [[0, 1, 2, 3, 4]], [300], None, False)
    keep = torch.ones(rows, 3, dtype=torch.bool, device=dev)
    keep[rows // 2, 1] = False
    _check(out[keep], ref[keep], mag[keep], err[keep], 2.0 ** -9)


@pytest.mark.parametrize("fmt", [I8, F8])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("rows", [1, 90])
def test_scores_of_every_size(dev, fmt, dtype, form, sign, rows):
    """Scores c 2^e (base 2, c of 1 to 16, or all negative) up to the largest of fp32: the row is the mean of its largest keys'
    values, also where a score's last place is more than the distance between a maximum and its reference."""
    n, dim, page = 200, 64, 32
    g = _gen(35)
    code = sign * torch.randint(1, 17, (n,), generator=g)
    k = torch.zeros(n, dim)
    k[:, 0] = code
    k = torch.cat([k, torch.zeros(24, dim)]).reshape(7, 1, page, dim).to(fmt)
    v, vs = ok.quantise(torch.randn(7, 1, page, dim, generator=g), fmt)
    c = kv.KVCache(k.to(dev), v.to(dev), torch.ones(7, 1, page, device=dev), vs.to(dev))
    values = (v.double() * vs.double()[..., None]).reshape(224, dim)[:n]
    see = torch.arange(n) <= n - rows + torch.arange(rows)[:, None]
    top = torch.where(see, code, -99).amax(1, keepdim=True)
    w = (see & (code == top)).double()
    ref = ((w @ values) / w.sum(1, keepdim=True)).to(dev)[:, None]
    mag = ((w @ values.abs()) / w.sum(1, keepdim=True)).to(dev)[:, None]
    for e in [*range(6, 15)] + ([*range(15, 48), 60, 90, 99, 101, 110, 120, 123] if dtype == BF else []):
        q = torch.zeros(rows, 1, dim)
        q[:, :, 0] = 2.0 ** e
        out, lse = kv.kv_attention(q.to(dtype).to(dev), c, _i32([list(range(7))], dev), _i32([n], dev), scale=math.log(2.0), lse=True,
                                   form=form)
        _check(out, ref, mag, torch.zeros(rows, 1, dtype=torch.float64, device=dev), 3.1)
        rl = (math.log(2.0) * top.double() * 2.0 ** e + torch.log(w.sum(1, keepdim=True))).to(dev)
        assert ((lse.double() - rl).abs() <= 2.0 ** -21 * rl.abs() + 2.0 ** -20).all(), e


def _outlier_values(dev, fmt, dim, n, rows, factor, at, hidden, seed, slack=0.0):
    """A cache of one sequence whose value at position `at` is `factor` times the others, with queries that either may not see it
    (hidden) or see it with about 1 / factor of the other keys' probability (or 2^-slack of that)."""
    page, hkv = 32, 2
    g = _gen(seed)
    width = -(-n // page)
    u = torch.randn(dim, generator=g)
    u = u / u.norm()
    x = torch.randn(n, hkv, dim, generator=g)
    y = torch.randn(n, hkv, dim, generator=g) * torch.exp(0.5 * torch.randn(n, hkv, 1, generator=g))
    y[at] *= factor
    if not hidden:
        x[at] = -u * (math.log(factor) + slack * math.log(2.0)) / 8.0 * dim ** 0.5
    q = 0.5 * torch.randn(rows, 2 * hkv, dim, generator=g)
    q = q - (q @ u)[..., None] * u + 8.0 * u
    if not hidden:
        others = torch.arange(n) != at
        x[others] -= (x[others] @ u)[..., None] * u
    table = _tables(width, width, 1, seed)
    c = kv.kv_cache(width, hkv, page, dim, fmt, dev)
    kv.kv_write(c, x.to(dev), y.to(dev), _i32(table, dev), _i32([n], dev))
    return c, table, q


@pytest.mark.parametrize("fmt", [I8, F8])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("factor", [2.0 ** 18, 2.0 ** 24, 2.0 ** 60, 1e30])
@pytest.mark.parametrize("rows,dim,dtype", [(4, 128, BF), (4, 64, HF), (90, 64, BF), (90, 128, HF)])
def test_values_beside_far_larger_hidden_ones(dev, fmt, form, factor, rows, dim, dtype):
    """What a causal row may not see does not touch its result: the last position's value is larger by any factor."""
    n = 300
    c, table, q = _outlier_values(dev, fmt, dim, n, rows, factor, n - 1, True, 36)
    q = q.to(dtype).to(dev)
    out, lse = kv.kv_attention(q, c, _i32(table, dev), _i32([n], dev), lse=True, form=form)
    ref, rl, mag, err = ok.attention(q, c, table, [n])
    _check(out[:-1], ref[:-1], mag[:-1], err[:-1], 3.1)
    _check_lse(lse, rl, err)


@pytest.mark.parametrize("fmt", [I8, F8])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("factor", [2.0 ** 24, 2.0 ** 60])
@pytest.mark.parametrize("at", [0, 150, 299])
@pytest.mark.parametrize("slack", [0.0, -6.0])
@pytest.mark.parametrize("rows,dim,dtype", [(4, 128, BF), (90, 64, BF), (90, 128, HF)])
def test_values_beside_far_larger_unlikely_ones(dev, fmt, form, factor, at, slack, rows, dim, dtype):
    """A value larger by a factor that its probability is smaller by: it and the others count as much as they do."""
    n = 300
    c, table, q = _outlier_values(dev, fmt, dim, n, rows, factor, at, False, 37, slack)
    q = q.to(dtype).to(dev)
    out, lse = kv.kv_attention(q, c, _i32(table, dev), _i32([n], dev), causal=False, lse=True, form=form)
    ref, rl, mag, err = ok.attention(q, c, table, [n], None, False)
    _check(out, ref, mag, err, 3.1)
    _check_lse(lse, rl, err)


@pytest.mark.parametrize("fmt", [I8, F8])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rows", [2, 70])
def test_values_of_every_size_and_zero_ones(dev, fmt, form, rows):
    """Values that grow from key to key through all of their type's range, and rows of zeros between them, whose scale is the
    quantiser's least: each causal row has its own largest."""
    n, dim, page = 90, 128, 16
    g = _gen(38)
    x = 0.3 * torch.randn(n, 1, dim, generator=g)
    y = torch.randn(n, 1, dim, generator=g) * torch.logspace(-30, 60, n, base=2.0)[:, None, None]
    y[::7] = 0.0
    c = kv.kv_cache(6, 1, page, dim, fmt, dev)
    args = (_i32([[5, 3, 0, 1, 2, 4]], dev), _i32([n], dev))
    kv.kv_write(c, x.to(dev), y.to(dev), *args)
    q = torch.randn(rows, 3, dim, generator=g).to(BF).to(dev)
    out, lse = kv.kv_attention(q, c, *args, lse=True, form=form)
    ref, rl, mag, err = ok.attention(q, c, [[5, 3, 0, 1, 2, 4]], [n])
    _check(out, ref, mag, err, 3.1)
    _check_lse(lse, rl, err)


@pytest.mark.parametrize("b,first", [(1, 1), (5, 2), (70, 3), (300, 40)])
def test_rows_in_front_of_the_first_sequence(dev, b, first):
    """cu[0] > 0: the rows in front of it are no sequence's; nor is any row where all offsets lie behind the rows."""
    hq, hkv, dim, page = 4, 2, 64, 16
    new = [1 + i % 3 for i in range(b)]
    lens = [n + i % 11 for i, n in enumerate(new)]
    cu = [first]
    for n in new:
        cu.append(cu[-1] + n)
    rows = cu[-1] + 2
    table = [[i] for i in range(b)]
    x = torch.randn(rows, hkv, dim, generator=_gen(50)).to(BF).to(dev)
    c = kv.kv_cache(b, hkv, page, dim, I8, dev)
    args = (_i32(table, dev), _i32(lens, dev), _i32(cu, dev))
    kv.kv_write(c, x, -x, *args)
    assert int((c.k_scale != 0).sum()) == (cu[-1] - first) * hkv
    k, v = kv.kv_read(c, *args, rows=rows)
    q, s = ok.quantise(x, I8)
    want = (q.float() * s[..., None]).to(BF)
    mine = slice(first, cu[-1])
    assert torch.equal(k[mine], want[mine]) and torch.equal(v[mine], -want[mine])
    assert not k[:first].any() and not k[cu[-1]:].any()
    q = torch.randn(rows, hq, dim, generator=_gen(51)).to(BF).to(dev)
    for form in FORMS:
        out = torch.full_like(q, 5.0)
        kv.kv_attention(q, c, *args, out=out, form=form)
        assert bool((out[:first] == 5.0).all()) and bool((out[cu[-1]:] == 5.0).all())
        ref, _, mag, err = ok.attention(q[mine], c, table, lens, [i - first for i in cu])
        _check(out[mine], ref, mag, err, 3.1)
        out.fill_(5.0)
        kv.kv_attention(q, c, args[0], args[1], args[2] + rows, out=out, form=form)
        assert bool((out == 5.0).all())


@pytest.mark.parametrize("form,b,new,prefix_len", [("token", 5, 3, 333), ("chunk", 5, 3, 333), ("chunk", 3, 50, 90), (None, 5, 3, 333),
                                                   (None, 64, 1, 60001)])
@pytest.mark.parametrize("first", [0, 2])
def test_shared_rows_that_no_sequence_has(dev, form, b, new, prefix_len, first):
    """Rows in front of cu[0] and behind cu[B] of a call with a prefix: neither their results nor, whatever they hold, those of the
    other rows are touched."""
    hq, hkv, dim, page = 8, 2, 128, 256
    lens = [1 + 5 * i for i in range(b)]
    pre = -(-prefix_len // page)
    table = _tables(2 * b + pre, 2, b, 24)
    used = {p for t in table for p in t}
    common = [p for p in range(2 * b + pre) if p not in used]
    c = _pool(dev, I8, 2 * b + pre, hkv, page, dim, 25)
    cu = [first + new * i for i in range(b + 1)]
    mine = slice(cu[0], cu[-1])
    q = torch.randn(cu[-1] + 9, hq, dim, generator=_gen(26)).to(BF).to(dev)
    got = []
    for other in (1.0, 1e30, math.nan, math.inf):
        q[:cu[0]], q[cu[-1]:] = other, other
        out = torch.full_like(q, 5.0)
        _call(q, c, table, lens, cu, common, prefix_len, dev, out=out, form=form)
        assert bool((out[:cu[0]] == 5.0).all()) and bool((out[cu[-1]:] == 5.0).all())
        got.append(out[mine].clone())
    assert all(torch.equal(got[0].view(torch.int16), x.view(torch.int16)) for x in got[1:])
    cu0 = [x - first for x in cu]
    ref, _, mag, err = ok.attention(q[mine], c, table, lens, cu0, prefix=common, prefix_len=prefix_len)
    _check(got[0], ref, mag, err, 3.1)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("fmt,dim", [(I8, 64), (F8, 128)])
@pytest.mark.parametrize("lens,cu,rows", [
    ([40, 25, 33], [0, 5, 12, 30], 20),           # the last sequence's rows end behind the call's
    ([40, 25, 33], [-7, 5, 12, 20], 20),          # the first one's begin in front of them
    ([40, 25, 33], [-300, -4, 2, 400], 20),
    ([60, 48, 33], [0, 12, 24, 30], 30),          # sequences that have outgrown their tables
    ([90, 47, 33], [0, 12, 24, 30], 30),
    ([60, 100, 90], None, 30),
])
def test_rows_outside_the_call_or_the_table(dev, fmt, dim, form, lens, cu, rows):
    """A row's position is lens[b] - (cu[b + 1] - cu[b]) + i also where the call has only some of the sequence's rows, or the table
    not all of its positions: what it does not have is skipped, read as 0 and not seen, and nothing else is written or read in its
    place."""
    b, hq, hkv, page = 3, 4, 2, 16
    table = [[4, 7, 1], [0, 3, 8], [2, 6, 5]]                    # 48 positions
    longer = [t + [-1] * 4 for t in table]                       # the oracle's: absent pages behind them
    whole = [rows // b * i for i in range(b + 1)] if cu is None else cu
    c = _pool(dev, fmt, 9, hkv, page, dim, 52)
    before = [t.clone() for t in (c.k.view(torch.uint8), c.v.view(torch.uint8), c.k_scale, c.v_scale)]
    args = (_i32(table, dev), _i32(lens, dev), None if cu is None else _i32(cu, dev))
    x, y = _rows(rows, hkv, dim, BF, 53, False, dev), _rows(rows, hkv, dim, BF, 54, False, dev)
    place = {}                                                   # row -> (page, offset) or None, of rows that a sequence has
    for i in range(b):
        for r in range(max(whole[i], 0), min(whole[i + 1], rows)):
            place[r] = ok.slot(longer, 9, page, i, lens[i] - whole[i + 1] + r)
    got = kv.kv_read(c, *args, rows=rows, dtype=F32)
    for t, codes, scales in ((got[0], before[0], before[2]), (got[1], before[1], before[3])):
        for r in range(rows):
            at = place.get(r)
            want = codes[at[0], :, at[1]].view(fmt).float() * scales[at[0], :, at[1]][:, None] if at else torch.zeros_like(t[r])
            assert torch.equal(t[r], want), r
    kv.kv_write(c, x, y, *args)
    for t, codes, scales in ((x, before[0], before[2]), (y, before[1], before[3])):
        q, s = ok.quantise(t, fmt)
        for r, at in place.items():
            if at:
                codes[at[0], :, at[1]], scales[at[0], :, at[1]] = q[r].view(torch.uint8), s[r]
    for t, u in zip(before, (c.k.view(torch.uint8), c.v.view(torch.uint8), c.k_scale, c.v_scale)):
        assert torch.equal(t, u)
    # attention: the oracle over all rows that the offsets name, of which the call has some
    q = torch.randn(max(whole[-1], rows) - whole[0], hq, dim, generator=_gen(55)).to(BF).to(dev)
    mine = slice(-whole[0], -whole[0] + rows)
    for causal in (True, False):
        out, lse = kv.kv_attention(q[mine], c, *args, causal=causal, lse=True, form=form)
        ref, rl, mag, err = (t[mine] for t in ok.attention(q, c, longer, [min(n, 48) if not causal else n for n in lens],
                                                           [i - whole[0] for i in whole], causal))
        # Value rows here differ by up to e^+-6 and some weights vanish beside others. A weight is at least 2^10 for the row's largest
        # (in the units that f16 has it in), and off by half of f16's last place, 2^-25, where it is small: 2^-35 of the largest
        # value for each of a row's up to 48 keys, also in a channel where the large ones hold 0.
        most = max(float(t.max()) for t in ok.gather(c, sum(table, []), 144)[1].abs())
        far = (out.double() - ref).abs() <= 48 * 2.0 ** -35 * most
        _check(torch.where(far, ref.to(BF), out), ref, mag, err, 3.1)
        _check_lse(lse, rl, err)


@pytest.mark.parametrize("form", FORMS)
def test_axes_of_length_one(dev, form):
    """One head, one row, one page and one table entry: the stride of such an axis is no one's, whatever number it is."""
    def odd(t):   # the same tensor with other strides at its axes of length 1
        return t.as_strided(t.shape, [s if n > 1 else 12345 + 7 * i for i, (n, s) in enumerate(zip(t.shape, t.stride()))])
    c = _pool(dev, I8, 1, 1, 64, 128, 56)
    d = kv.KVCache(odd(c.k), c.v, odd(c.k_scale), c.v_scale)
    x, y = (torch.randn(1, 1, 128, generator=_gen(57 + i)).to(BF).to(dev) for i in range(2))
    table, lens = _i32([[0]], dev), _i32([50], dev)
    kv.kv_write(c, x, y, table, lens)
    want = [t.clone() for t in (c.k, c.v, c.k_scale, c.v_scale)]
    kv.kv_write(d, odd(x), y, odd(table), lens)
    assert all(torch.equal(t, u) for t, u in zip(want, (d.k, d.v, d.k_scale, d.v_scale)))
    got = (odd(torch.zeros_like(x)), odd(torch.zeros_like(y)))
    kv.kv_read(d, odd(table), lens, out=got)
    assert all(torch.equal(t, u) for t, u in zip(got, kv.kv_read(c, table, lens)))
    q = torch.randn(1, 1, 128, generator=_gen(59)).to(BF).to(dev)
    out = odd(torch.zeros_like(q))
    kv.kv_attention(odd(q), d, odd(table), lens, out=out, form=form)
    assert torch.equal(out, kv.kv_attention(q, c, table, lens, form=form))


@pytest.mark.parametrize("fmt", [I8, F8])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rows,n,prefix_len", [(1, 200, 0), (1, 20011, 0), (100, 3000, 0), (3, 100, 9000), (200, 90, 700)])
def test_values_near_the_largest(dev, fmt, form, rows, n, prefix_len):
    """Values of 2^126 at most, which many keys' weights times them, before the division by the weights' sum, are far past fp32."""
    hq, hkv, dim, page = 4, 2, 128, 64
    width, pre = -(-n // page), -(-prefix_len // page)
    g = _gen(43)
    k, ks = ok.quantise(0.2 * torch.randn(width + pre, hkv, page, dim, generator=g), fmt)
    v, vs = ok.quantise((torch.rand(width + pre, hkv, page, dim, generator=g) - 0.3) * 2.0 ** 126, fmt)
    c = kv.KVCache(*(t.to(dev) for t in (k, v, ks, vs)))
    table, common = [list(range(pre, pre + width))], list(range(pre))
    q = torch.randn(rows, hq, dim, generator=g).to(BF).to(dev)
    out, lse = _call(q, c, table, [n], None, common, prefix_len, dev, lse=True, form=form)
    ref, rl, mag, err = ok.attention(q, c, table, [n], prefix=common, prefix_len=prefix_len)
    _check(out, ref, mag, err, 3.1)
    _check_lse(lse, rl, err)


@pytest.mark.parametrize("fmt", [I8, F8])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("form,dtype,terms", [("token", BF, 1), ("chunk", BF, 3), ("token", HF, 2.0 ** -10), ("chunk", HF, 2.0 ** -10)])
@pytest.mark.parametrize("rows,prefix_len", [(3, 0), (90, 0), (90, 300)])
def test_roundings_of_each_kernel(dev, fmt, dim, form, dtype, terms, rows, prefix_len):
    """No more than each kernel's own f16 roundings, 2^-11 of a product each, before that of the result: one of the weight in the
    token kernel, three (weight, value scale, scaled value) in the chunk kernel, for fp16 results two terms of the weight (2^-22,
    and 2^-22 for fp32 sums)."""
    n, page = 777, 32
    width, pre = -(-n // page), -(-prefix_len // page)
    c = _pool(dev, fmt, 2 * width + pre, 2, page, dim, 62)
    table, common = _tables(2 * width, width, 2, 63), list(range(2 * width, 2 * width + pre))
    lens = [n, n - 300]
    q = torch.randn(2 * rows, 4, dim, generator=_gen(64)).to(dtype).to(dev)
    out = _call(q, c, table, lens, None, common, prefix_len, dev, form=form)
    ref, _, mag, err = ok.attention(q, c, table, lens, prefix=common, prefix_len=prefix_len)
    _check(out, ref, mag, err, terms)


def test_layouts(dev):
    """A cache that is a view of a buffer of several layers, strided queries and output, a wider table, out over q."""
    pages, heads, page, dim, hq = 9, 2, 32, 128, 6
    whole = [torch.zeros((pages, 3, heads, page, dim), dtype=torch.int8, device=dev) for _ in range(2)]
    scale = [torch.zeros((pages, 3, heads, page), device=dev) for _ in range(2)]
    c = kv.KVCache(whole[0][:, 1], whole[1][:, 1], scale[0][:, 1], scale[1][:, 1])
    lens, table = [70, 33], [[8, 1, 4, 2], [0, 6, 3, 7]]
    tab = torch.full((2, 11), -1, dtype=torch.int32, device=dev)
    tab[:, :4] = _i32(table, dev)
    ln = _i32(lens, dev)
    qkv = torch.randn(103, hq + 2 * heads, dim, generator=_gen(40)).to(BF).to(dev)
    cu = _i32([0, 70, 103], dev)
    kv.kv_write(c, qkv[:, hq:hq + heads], qkv[:, hq + heads:], tab[:, :4], ln, cu)
    assert not any(t[:, i].any() for t in whole + scale for i in (0, 2))
    q = qkv[:, :hq]
    ref, rl, mag, err = ok.attention(q, c, table, lens, [0, 70, 103])
    wide = torch.full((103, hq, dim + 64), 5.0, dtype=BF, device=dev)
    kv.kv_attention(q, c, tab[:, :4], ln, cu, out=wide[..., 64:])
    _check(wide[..., 64:], ref, mag, err, 3.1)
    assert (wide[..., :64] == 5.0).all()
    want = wide[..., 64:].clone()
    kv.kv_attention(q, c, tab, ln, cu, out=q)                  # the same positions by a longer table; out over q
    _check(q, ref, mag, err, 3.1)
    assert torch.equal(q, want)


@pytest.mark.parametrize("form", [None] + FORMS)
@pytest.mark.parametrize("rows", [1, 21, 300])
@pytest.mark.parametrize("prefix_len", [0, 333])
def test_out_over_q_and_repeated_rows(dev, form, rows, prefix_len):
    """The result written over q, and q given as one row repeated without memory of its own (stride 0): the same bits as apart."""
    b, hq, hkv, dim, page = 3, 6, 2, 128, 64
    c = _pool(dev, I8, 40, hkv, page, dim, 60)
    table, lens, prefix = _i32([[1, 2, 3], [30, 5, 6], [7, 8, 39]], dev), _i32([190, 64, 5], dev), _i32([9, 20, 11, 12, 13, 14], dev)

    def call(q, out=None):
        if prefix_len:
            return kv.kv_attention_shared(q, c, prefix, prefix_len, table, lens, out=out, form=form)
        return kv.kv_attention(q, c, table, lens, out=out, form=form)
    q = torch.randn(b * rows, hq, dim, generator=_gen(61)).to(BF).to(dev)
    want = call(q)
    same = q.clone()
    assert call(same, out=same) is same and torch.equal(same.view(torch.int16), want.view(torch.int16))
    one = q[:1].expand(b * rows, hq, dim)
    assert torch.equal(call(one).view(torch.int16), call(one.contiguous()).view(torch.int16))


def test_rows_that_no_sequence_has_stay(dev):
    c = _pool(dev, I8, 4, 1, 16, 64, 41)
    for rows, cu, form in ((5, [0, 1, 3], "token"), (90, [0, 40, 83], "chunk"), (90, [0, 40, 83], "token")):
        q = torch.randn(rows, 2, 64, generator=_gen(42)).to(BF).to(dev)
        out = torch.full_like(q, 9.0)
        kv.kv_attention(q, c, _i32([[0, 1], [2, 3]], dev), _i32([20, 30], dev), _i32(cu, dev), out=out, form=form)
        assert (out[cu[-1]:] == 9.0).all() and not (out[:cu[-1]] == 9.0).all(-1).any()
        ref, _, mag, err = ok.attention(q[:cu[-1]], c, [[0, 1], [2, 3]], [20, 30], cu)
        _check(out[:cu[-1]], ref, mag, err, 3.1)


def test_bad_contents_stay_inside(dev):
    """Lengths beyond the table, negative ones, page numbers that are none, row offsets that fall or pass the end: clamped or
    absent, and the sequences beside them keep their results."""
    pages, page, dim = 6, 16, 64
    c = _pool(dev, I8, pages, 2, page, dim, 43)
    before = [t.clone() for t in (c.k, c.v, c.k_scale, c.v_scale)]
    table = [[0, 1], [-7, 2 ** 31 - 1], [2, pages], [3, 4]]
    lens = [10 ** 9, 20, 32, -5]
    for rows, form in ((1, "token"), (30, "token"), (1, "chunk"), (30, "chunk")):
        q = torch.randn(4 * rows, 4, dim, generator=_gen(44)).to(BF).to(dev)
        out = kv.kv_attention(q, c, _i32(table, dev), _i32(lens, dev), causal=False, form=form)
        ref, _, mag, err = ok.attention(q, c, table, [32, 20, 32, 0], None, False)
        _check(out, ref, mag, err, 3.1)
        assert (out[rows:2 * rows] == 0).all() and (out[3 * rows:] == 0).all()
    q = torch.randn(6, 4, dim, generator=_gen(45)).to(BF).to(dev)
    x = torch.randn(6, 2, dim, generator=_gen(46)).to(BF).to(dev)
    bad = _i32([2, -3, 5, 1, 99], dev)                         # rows 0 .. 5 of sequence 1 by clamping, 1 .. 5 of sequence 3 again
    dead = _i32([[-1, pages]] * 4, dev)
    kv.kv_write(c, x, x, dead, _i32([20] * 4, dev), bad)
    assert all(torch.equal(a, b) for a, b in zip(before, (c.k, c.v, c.k_scale, c.v_scale)))
    kv.kv_read(c, dead, _i32([20] * 4, dev), bad, rows=6)
    for form in FORMS:
        kv.kv_attention(q, c, dead, _i32([20] * 4, dev), bad, form=form)
        kv.kv_attention_shared(q, c, _i32([9, -1, 2], dev), 40, dead, _i32([20] * 4, dev), bad, form=form)
    torch.cuda.synchronize()


@pytest.mark.parametrize("fmt", [I8, F8])
def test_offsets_past_32_bits(dev, fmt):
    """Pages beyond 4 GiB of codes."""
    heads, page, dim = 8, 256, 128
    pages = (5 << 30) // (heads * page * dim)
    k, v = (torch.empty((pages, heads, page, dim), dtype=torch.int8, device=dev).view(fmt) for _ in range(2))
    c = kv.KVCache(k, v, *(torch.empty((pages, heads, page), device=dev) for _ in range(2)))
    table, lens = [[pages - 1, 0, pages - 2], [1, pages - 3, 2]], [600, 700]
    cu = [0, 600, 1300]
    g = _gen(60)
    x, y = (torch.randn(1300, heads, dim, generator=g).to(BF).to(dev) for _ in range(2))
    args = (_i32(table, dev), _i32(lens, dev), _i32(cu, dev))
    kv.kv_write(c, x, y, *args)
    gk, gv = kv.kv_read(c, *args, rows=1300)
    for a, b in ((x, gk), (y, gv)):
        q, s = ok.quantise(a, fmt)
        assert torch.equal(b, (q.float() * s[..., None]).to(BF))
    q = torch.randn(2, 8, dim, generator=g).to(BF).to(dev)
    out = kv.kv_attention(q, c, *args[:2])
    ref, _, mag, err = ok.attention(q, c, table, lens)
    _check(out, ref, mag, err, 3.1)
    q = torch.randn(100, 8, dim, generator=g).to(BF).to(dev)
    out = kv.kv_attention(q, c, *args[:2], form="chunk")
    ref, _, mag, err = ok.attention(q, c, table, lens)
    _check(out, ref, mag, err, 3.1)


# ---------------------------------------------------------------- together, streams, graphs
def test_generation(dev):
    """A prompt is written and attended in two chunks, then tokens one by one, in a batch of uneven prompts behind a common
    instruction: every step equals float64 attention over the stored values, and the values are the inputs' to half a step."""
    b, hq, hkv, dim, page = 3, 8, 2, 128, 16
    c = kv.kv_cache(40, hkv, page, dim, I8, dev)
    prefix_len, pre = 50, [39, 38, 37, 36]
    table = _tables(36, 9, b, 70)
    tab, ptab = _i32(table, dev), _i32(pre, dev)
    lens = torch.zeros(b, dtype=torch.int32, device=dev)
    g = _gen(71)
    kept = [torch.zeros(0, hkv, dim) for _ in range(b)]

    def rows(n):
        return (torch.randn(n, h, dim, generator=g).to(BF).to(dev) for h in (hq, hkv, hkv))
    _, k, v = rows(prefix_len)
    kv.kv_write(c, k, v, ptab[None], _i32([prefix_len], dev))
    for new in ([70, 33, 1], [40, 2, 7], [1, 1, 1], [1, 1, 1], [1, 1, 1]):
        n = _i32(new, dev)
        cu = torch.cat([torch.zeros(1, dtype=torch.int32, device=dev), n.cumsum(0).int()])
        lens += n
        q, k, v = rows(sum(new))
        kv.kv_write(c, k, v, tab, lens, cu)
        out, lse = kv.kv_attention_shared(q, c, ptab, prefix_len, tab, lens, cu, lse=True)
        at = lens.tolist()
        ref, rl, mag, err = ok.attention(q, c, table, at, cu.tolist(), prefix=pre, prefix_len=prefix_len)
        _check(out, ref, mag, err, 3.1)
        _check_lse(lse, rl, err)
        for i, part in enumerate(k.cpu().split(new)):
            kept[i] = torch.cat([kept[i], part.float()])
    whole = torch.cat([torch.zeros(1, dtype=torch.int32, device=dev), lens.cumsum(0).int()])
    got, _ = kv.kv_read(c, tab, lens, whole, rows=int(whole[-1]), dtype=F32)
    want = torch.cat(kept)
    step = want.abs().amax(-1, keepdim=True) / 127
    assert ((got.cpu() - want).abs() <= step * (0.5 + 2.0 ** -15)).all()


def _step(c, q, k, v, tab, lens, ptab=None, prefix_len=0, form=None):
    kv.kv_write(c, k, v, tab, lens)
    if prefix_len:
        return kv.kv_attention_shared(q, c, ptab, prefix_len, tab, lens, form=form)
    return kv.kv_attention(q, c, tab, lens, form=form)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rows,prefix_len", [(1, 0), (1, 500), (60, 0)])
def test_captured_steps(dev, form, rows, prefix_len):
    """A step captured once follows new inputs, lengths and page tables on every replay; two captured steps run at once on two
    streams."""
    b, hq, hkv, dim, page = 2, 4, 2, 128, 32
    steps = []
    for which in range(2):
        c = _pool(dev, I8, 80, hkv, page, dim, 80 + which)
        g = _gen(81 + which)
        q, k, v = (torch.randn(b * rows, h, dim, generator=g).to(BF).to(dev) for h in (hq, hkv, hkv))
        tab, ptab = _i32(_tables(60, 30, b, which), dev), _i32(list(range(60, 76)), dev)
        lens = _i32([700, 130], dev)
        args = (c, q, k, v, tab, lens, ptab, prefix_len, form)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            _step(*args)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _step(*args)
        steps.append((graph, out, args, torch.cuda.Stream()))
    for replay in range(3):
        want = []
        for graph, out, (c, q, k, v, tab, lens, ptab, n, _), _ in steps:
            for t in (q, k, v):
                t.copy_(torch.randn(t.shape, generator=_gen(replay + 7)).to(BF))
            lens.copy_(torch.tensor([60 + 300 * replay, 959 - replay], dtype=torch.int32))
            tab.copy_(tab.flip(1))
            want.append(_step(c, q, k, v, tab, lens, ptab, n, form).clone())
            out.zero_()
        torch.cuda.synchronize()
        for graph, _, _, stream in steps:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (_, out, _, _), w in zip(steps, want):
            assert torch.equal(out.view(torch.int16), w.view(torch.int16)), replay


def test_two_streams(dev):
    """Two calls at once on streams of their own."""
    c = _pool(dev, F8, 200, 2, 64, 128, 90)
    tab, lens = _i32(_tables(200, 100, 2, 9), dev), _i32([6400, 3001], dev)
    qs = [torch.randn(2, 8, 128, generator=_gen(91 + i)).to(BF).to(dev) for i in range(2)]
    want = [kv.kv_attention(q, c, tab, lens) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(kv.kv_attention(qs[i], c, tab, lens))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, x) for x in g)
