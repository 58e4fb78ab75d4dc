"""The norm and rotation of query and key heads (rapid_h3.rope), alone and on their way into a key / value cache
(kvcache.kv_write_rope), on the GPU against the plain restatement and float64."""
import math

import numpy as np
import pytest
import torch

from oracle import kvcache as ok
from oracle import rope as orope
from rapid_h3 import kvcache as kv
from rapid_h3 import rope

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
FMT = [torch.int8, torch.float8_e4m3fn, torch.float4_e2m1fn_x2]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _rows(t, heads, dim, dtype, seed, dev):
    """Views of one projection's rows, one for each entry of heads."""
    g = _gen(seed)
    x = torch.randn(t, sum(heads), dim, generator=g) * torch.exp(torch.randn(t, sum(heads), 1, generator=g))
    return x.to(dtype).to(dev).split(heads, 1)


def _check(got, x, args):
    """Within the result's rounding of the float64 one (half a step of its type; fp32 rows: see below) and the fp32 steps before it:
    the norm's factor, its product, the weight's, cosine and sine, their products and the sum, 2^-24 each of the pair's magnitude."""
    positions, freq, layout, factor, weight, eps = args
    ref = orope.turned64(x, *args)
    y = orope.turned64(x, positions, None, layout, factor, weight, eps) if eps is not None else x.double()
    mag = y.abs()
    if freq is not None:   # of a pair, what both members bring
        u, w, rest = orope._pairs(mag, freq.shape[0], layout)
        mag = orope._back((u + w) * factor, (u + w) * factor, rest, layout)
    f = torch.finfo(x.dtype)
    tol = f.eps / 2 * ref.abs() * 1.01 + 8 * 2.0 ** -24 * mag + f.tiny * f.eps
    assert ((got.double() - ref).abs() <= tol).all(), float(((got.double() - ref).abs() / tol).max())


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("t,hq,hk,dim,rot,eps,how", [
    (1, 1, 1, 128, 128, 1e-6, {}),
    (1, 32, 8, 128, 128, None, {}),
    (3, 28, 4, 64, 64, 1e-5, dict(scaling="linear", stretch=4.0)),
    (67, 5, 3, 128, 96, 1e-6, dict(scaling="base", stretch=8.0)),
    (130, 12, 4, 64, 16, 1e-6, dict(base=500000.0)),
    (1100, 7, 7, 64, 48, None, dict(scaling="parts", stretch=4.0, original=8192)),
    (1027, 9, 1, 128, 64, 1e-6, dict(scaling="parts", stretch=16.0, original=4096)),
    (5, 3, 2, 128, 0, 1e-6, None),                              # the norm alone
])
def test_norm_rope(dev, dtype, layout, t, hq, hk, dim, rot, eps, how):
    q, k, _ = _rows(t, [hq, hk, hk], dim, dtype, 1, dev)
    pos = torch.randint(0, 200000, (t,), generator=_gen(2)).to(torch.int32)
    pos[0], pos[-1] = 0, 1 << 30
    pos = pos.to(dev)
    turn = rope.rotary(rot, layout, dev, **how) if how is not None else None
    qw, kw = ((1 + 0.3 * torch.randn(dim, generator=_gen(3 + i))).to(dtype).to(dev) if eps else None for i in range(2))
    got = rope.qk_norm_rope(q, k, pos, turn, qw, kw, eps)
    freq, factor = (turn.freq, turn.factor) if turn else (None, 1.0)
    for x, y, w in ((q, got[0], qw), (k, got[1], kw)):
        args = (pos, freq, layout, factor, w, eps)
        _check(y, x, args)
        want = orope.turned(x, *args)
        # the steps are defined to the bit but for the last one of 64-bit results that are rounded to fp32, whose neighbours then
        # differ by 2^-23 of them: no more than one value in a thousand of a 16-bit result, or of fp32 ones one row or angle in 2^20
        off = (y != want).double().mean().item()
        assert off <= 1e-3, off
    a, b = q.clone(), k.clone()
    back = rope.qk_norm_rope(a, b, pos, turn, qw, kw, eps, out=(a, b))
    assert back[0] is a and back[1] is b
    assert torch.equal(a, got[0]) and torch.equal(b, got[1])
    alone, none = rope.qk_norm_rope(q, None, pos, turn, qw, None, eps)
    assert none is None and torch.equal(alone, got[0])


def test_weights_in_fp32_and_none(dev):
    q, k = _rows(9, [4, 2], 128, BF, 5, dev)
    pos = torch.arange(9, dtype=torch.int32, device=dev)
    turn = rope.rotary(128, "half", dev)
    w = (1 + 0.3 * torch.randn(128, generator=_gen(6))).to(BF).to(dev)
    wide = rope.qk_norm_rope(q, k, pos, turn, w.float(), w.float(), 1e-6)
    near = rope.qk_norm_rope(q, k, pos, turn, w, w, 1e-6)
    assert all(torch.equal(a, b) for a, b in zip(wide, near))
    plain = rope.qk_norm_rope(q, k, pos, turn, None, None, 1e-6)
    ones = rope.qk_norm_rope(q, k, pos, turn, torch.ones_like(w), torch.ones_like(w), 1e-6)
    assert all(torch.equal(a, b) for a, b in zip(plain, ones))


def test_rows_that_are_not_finite_stay_alone(dev):
    """Zeros, infinities and NaN in one head's row change no other; without a norm they change no other channel pair."""
    x, = _rows(6, [4], 64, BF, 7, dev)
    x = x.contiguous()
    turn = rope.rotary(32, "half", dev)
    pos = torch.arange(6, dtype=torch.int32, device=dev) * 1000
    want = {eps: rope.qk_norm_rope(x, None, pos, turn, None, None, eps)[0] for eps in (None, 1e-6)}
    y = x.clone()
    y[1, 2, 40], y[3, 0, 5], y[4, 1] = math.inf, math.nan, 0.0
    for eps, w in want.items():
        got = rope.qk_norm_rope(y, None, pos, turn, None, None, eps)[0]
        same = torch.ones(6, 4, 64, dtype=torch.bool, device=dev)
        for r, h in ((1, 2), (3, 0), (4, 1)):
            same[r, h] = False
        assert torch.equal(got[same], w[same]) and (got[4, 1] == 0).all()
        if eps is None:
            assert torch.isinf(got[1, 2, 40]) and torch.isfinite(got[1, 2]).sum() == 63
            assert torch.isnan(got[3, 0, [5, 21]]).all() and torch.isfinite(got[3, 0]).sum() == 62


def test_inverse_rotation(dev):
    """Frequencies of the other sign turn back."""
    q, = _rows(40, [6], 128, F32, 8, dev)
    pos = torch.randint(0, 100000, (40,), generator=_gen(9)).to(torch.int32).to(dev)
    for layout in rope.LAYOUTS:
        freq, _ = rope.frequencies(128)
        there, back = (rope.Rotary((s * freq).to(dev), layout) for s in (1, -1))
        y = rope.qk_norm_rope(rope.qk_norm_rope(q, None, pos, there)[0], None, pos, back)[0]
        # two rotations of fp32 steps: 2 * 4 roundings of the pair's magnitude
        u, w, _ = orope._pairs(q.double().abs(), 64, layout)
        assert ((y.double() - q.double()).abs() <= 10 * 2.0 ** -24 * orope._back(2 * (u + w), 2 * (u + w), u[..., :0], layout)).all()


# ---------------------------------------------------------------- into the cache
@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("hq,hkv,dim,page,lens,new,rot,layout,eps,first", [
    (32, 8, 128, 64, [1, 77, 64], [1, 1, 1], 128, "half", 1e-6, 0),
    (7, 1, 64, 16, [40, 5, 33], [17, 9, 16], 32, "interleaved", None, 777),   # a sequence with more rows than positions
    (4, 4, 128, 32, [0, 300, 7], [0, 290, 7], 96, "half", 1e-5, 0),
    (2, 2, 64, 256, [1500], [1400], 0, "half", 1e-6, 5),                       # the norm alone
    (3, 1, 128, 128, [1500, 2], [1200, 1], 64, "interleaved", 1e-6, -3),
])
def test_write_rope_is_both(dev, fmt, dtype, hq, hkv, dim, page, lens, new, rot, layout, eps, first):
    """The same bits as the rotation, then the write: queries, codes and scales."""
    b = len(lens)
    width = max(-(-max(lens) // page), 1) + 1
    pages = b * width + 1
    perm = torch.randperm(pages, generator=_gen(4)).tolist()
    table = [perm[i * width:(i + 1) * width] for i in range(b)]
    if b > 1:
        table[1][0] = -1
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    even = len(set(new)) == 1
    t = cu[-1] + (0 if even else 3)
    q, k, v = _rows(t, [hq, hkv, hkv], dim, dtype, 5, dev)
    args = (_i32(table, dev), _i32(lens, dev), None if even else _i32(cu, dev))
    turn = rope.rotary(rot, layout, dev) if rot else None
    qw, kw = ((1 + 0.3 * torch.randn(dim, generator=_gen(3 + i))).to(dtype).to(dev) if eps else None for i in range(2))
    one, two = (kv.kv_cache(pages, hkv, page, dim, fmt, dev) for _ in range(2))
    got = kv.kv_write_rope(one, q, k, v, *args, turn, qw, kw, eps, first=first)
    where = ok.rows_of(lens, None if even else cu, t, b)
    pos = _i32([w[1] + first if w else 0 for w in where], dev)
    wq, wk = rope.qk_norm_rope(q, k, pos, turn, qw, kw, eps)
    kv.kv_write(two, wk, v, *args)
    for x, y in zip((one.k, one.v, one.k_scale, one.v_scale), (two.k, two.v, two.k_scale, two.v_scale)):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    mine = torch.tensor([w is not None for w in where], device=dev)
    assert torch.equal(got[mine], wq[mine]) and (got[~mine] == 0).all()
    keep = torch.full_like(q, 3.0)
    assert kv.kv_write_rope(one, q, k, v, *args, turn, qw, kw, eps, first=first, out=keep) is keep
    assert torch.equal(keep[mine], wq[mine]) and (keep[~mine] == 3).all()
    x = q.clone()
    kv.kv_write_rope(one, x, k, v, *args, turn, qw, kw, eps, first=first, out=x)
    assert torch.equal(x[mine], wq[mine]) and torch.equal(x[~mine], q[~mine])


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("first", [0, 777])
def test_rows_past_the_table_turn_by_their_positions(dev, fmt, ragged, first):
    """Sequences that have outgrown their tables: rows that begin behind the last page, or in it and go on behind it, are written
    nowhere, and their queries turn by the positions that kv_extend gives them, however the rows are split over calls."""
    hq, hkv, dim, page = 4, 2, 64, 16
    had, new = ([95, 10, 3, 1 << 29], [5, 10, 4, 3]) if ragged else ([95, 10, 3, 1 << 29], [4] * 4)
    b, t = len(new), sum(new)
    pool = kv.kv_pages(8, page, dev)
    table, lens = _i32([[p] for p in range(b)], dev), _i32(had, dev)
    cu, positions, slots = kv.kv_extend(pool, table, lens, _i32(new, dev), t)
    assert positions.tolist() == [p for n, m in zip(had, new) for p in range(n, n + m)]
    q, k, v = _rows(t, [hq, hkv, hkv], dim, BF, 5, dev)
    turn = rope.rotary(dim, "half", dev)
    one, two, parts = (kv.kv_cache(8, hkv, page, dim, fmt, dev) for _ in range(3))
    got = kv.kv_write_rope(one, q, k, v, table, lens, cu if ragged else None, turn, eps=1e-6, first=first)
    wq, wk = rope.qk_norm_rope(q, k, positions + first, turn, eps=1e-6)
    assert torch.equal(got, wq)
    kv.kv_write(two, wk, v, table, lens, cu if ragged else None)
    bounds = cu.tolist()
    for i, n in enumerate(had):                  # one row to a call
        for j in range(new[i]):
            r = bounds[i] + j
            x = kv.kv_write_rope(parts, q[r:r + 1], k[r:r + 1], v[r:r + 1], table[i:i + 1], _i32([n + j + 1], dev), None, turn, eps=1e-6, first=first)
            assert torch.equal(x, wq[r:r + 1]), (i, j)
    for x, y, z in zip(*((c.k, c.v, c.k_scale, c.v_scale) for c in (one, two, parts))):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)) and torch.equal(x.view(torch.uint8), z.view(torch.uint8))


def _rows_at_a_border(n, dim, eps, seed):
    """fp32 rows whose inverse root mean square lies at the middle of two fp32 numbers, as near as their squares' sum in 64 bits can tell:
    three channels are chosen for it, each taking what the one before it left."""
    r = np.random.default_rng(seed)
    x = r.standard_normal((n, dim)).astype(np.float32)
    for row in x:
        last = r.choice(dim, 3, replace=False)
        row[last] = 0.0
        rest = (row.astype(np.longdouble) ** 2).sum()
        near = np.float32(1 / np.sqrt((rest + 1 + r.random()) / dim + eps))
        middle = np.longdouble(near) + np.longdouble(np.spacing(near)) / 2
        left = dim * (1 / middle ** 2 - np.longdouble(eps)) - rest
        for i in last:
            y = np.float32(np.sqrt(left))
            row[i] = y if np.longdouble(y) ** 2 <= left else np.nextafter(y, np.float32(0))
            left -= np.longdouble(row[i]) ** 2
    return torch.from_numpy(x)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rot", [(128, 128), (128, 96), (64, 64), (64, 16), (128, 0)])
def test_write_rope_is_both_where_the_norm_is_at_a_border(dev, dim, rot, layout):
    """The same bits also of fp32 rows whose norm would be rounded to another number if its squares were summed in another order."""
    n, heads, page = 300, 3, 64
    k = _rows_at_a_border(n * heads, dim, 1e-6, 1).view(n, heads, dim).to(dev)
    turn = rope.rotary(rot, layout, dev) if rot else None
    table, lens = _i32([range(5)], dev), _i32([n], dev)
    one, two = (kv.kv_cache(5, heads, page, dim, FMT[0], dev) for _ in range(2))
    pos = torch.arange(n, dtype=torch.int32, device=dev)
    kv.kv_write_rope(one, k, k, k, table, lens, None, turn, eps=1e-6)
    kv.kv_write(two, rope.qk_norm_rope(k, None, pos, turn, eps=1e-6)[0], k, table, lens)
    for x, y in zip((one.k, one.v, one.k_scale, one.v_scale), (two.k, two.v, two.k_scale, two.v_scale)):
        assert torch.equal(x, y)


def test_captured(dev):
    """A captured call follows new rows, positions, lengths and tables on every replay, beside another on its own stream."""
    steps = []
    for which in range(2):
        q, k, v = (x.contiguous() for x in _rows(6, [4, 2, 2], 128, BF, which, dev))
        c = kv.kv_cache(12, 2, 16, 128, FMT[2], dev)
        args = (_i32([[0, 1, 2], [3, 4, 5]], dev), _i32([20, 40], dev))
        turn = rope.rotary(128, "half", dev)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            kv.kv_write_rope(c, q, k, v, *args, rotary=turn, eps=1e-6)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = kv.kv_write_rope(c, q, k, v, *args, rotary=turn, eps=1e-6)
        steps.append((graph, out, c, q, k, v, args, turn, torch.cuda.Stream()))
    for replay in range(3):
        want = []
        for i, (graph, out, c, q, k, v, args, turn, _) in enumerate(steps):
            for j, x in enumerate((q, k, v)):
                x.copy_(torch.randn(x.shape, generator=_gen(10 * replay + 3 * i + j)).to(BF))
            args[0].copy_(torch.randperm(12, generator=_gen(replay))[:6].view(2, 3).int())
            args[1].copy_(torch.tensor([7 + 13 * replay, 48 - replay], dtype=torch.int32))
            d = kv.kv_cache(12, 2, 16, 128, FMT[2], dev)
            want.append((kv.kv_write_rope(d, q, k, v, *args, rotary=turn, eps=1e-6), d))
            out.zero_()
            c.k.view(torch.uint8).zero_()
            c.v.view(torch.uint8).zero_()
            c.k_scale.view(torch.uint8).zero_()
            c.v_scale.view(torch.uint8).zero_()
        torch.cuda.synchronize()
        for graph, *_, s in steps:
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for (_, out, c, *_), (w, d) in zip(steps, want):
            assert torch.equal(out, w)
            for x, y in ((c.k, d.k), (c.v, d.v), (c.k_scale, d.k_scale), (c.v_scale, d.v_scale)):
                assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), replay


def test_bad_contents_stay_inside(dev):
    """Lengths, tables and offsets that are none write nothing outside."""
    c = kv.kv_cache(4, 2, 16, 64, FMT[0], dev)
    q, k, v = _rows(6, [4, 2, 2], 64, BF, 1, dev)
    turn = rope.rotary(64, "half", dev)
    for table, lens, cu in (([[-1, 9]] * 2, [20, -4], None), ([[4, 2 ** 31 - 1]] * 2, [10 ** 9, 32], [0, 99, 3]), ([[-5, -1]] * 2, [-10 ** 9, 2], [5, -3, 2])):
        kv.kv_write_rope(c, q, k, v, _i32(table, dev), _i32(lens, dev), None if cu is None else _i32(cu, dev), rotary=turn)
    torch.cuda.synchronize()
    assert not c.k.any() and not c.k_scale.any()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_beyond_the_last_cache(dev, dtype, layout):
    """Calls of so many rows that they are streamed leave what calls of parts of them leave, bit for bit."""
    n, hq, hkv, dim, page = 9001, 96, 32, 128, 64
    g = torch.Generator(device=dev).manual_seed(5)
    q, k, v = (torch.randn(n, h, dim, generator=g, device=dev).to(dtype) for h in (hq, hkv, hkv))
    turn = rope.rotary(96, layout, dev)
    weight = (1 + 0.1 * torch.randn(dim, generator=g, device=dev)).to(dtype)
    positions = torch.arange(n, dtype=torch.int32, device=dev)
    gq, gk = rope.qk_norm_rope(q, k, positions, turn, weight, weight, 1e-6)
    pages = -(-n // page)
    table = torch.arange(pages, dtype=torch.int32, device=dev)[None]
    cache, parts = (kv.kv_cache(pages, hkv, page, dim, FMT[2], dev) for _ in range(2))
    wq = kv.kv_write_rope(cache, q, k, v, table, _i32([n], dev), None, turn, weight, weight, 1e-6)
    assert torch.equal(wq, gq)
    for at in range(0, n, 500):
        end = min(at + 500, n)
        pq, pk = rope.qk_norm_rope(q[at:end], k[at:end], positions[at:end].clone(), turn, weight, weight, 1e-6)
        assert torch.equal(gq[at:end], pq) and torch.equal(gk[at:end], pk)
        kv.kv_write(parts, pk, v[at:end], table, _i32([end], dev))
    for x, y in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), (parts.k, parts.v, parts.k_scale, parts.v_scale)):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
