"""Page tables and slot maps made on the GPU (kvcache.kv_extend) against the same steps on lists, alone and with the calls that use
them: a served batch from its prompts over its tokens to new requests in the places of ended ones."""
import random

import pytest
import torch

from oracle import kvcache as ok
from oracle import rope as orope
from rapid_h3 import kvcache as kv
from rapid_h3 import rope

pytestmark = pytest.mark.gpu


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


class Lists:
    """A pool, a table and lengths as lists."""

    def __init__(self, pages, page, b, w):
        self.free, self.held, self.lacking, self.page = list(range(pages - 1, -1, -1)), pages, 0, page
        self.table, self.lens = [[-1] * w for _ in range(b)], [0] * b

    def extend(self, new, rows, done):
        page = self.page
        for row, n, d in zip(self.table, self.lens, done):
            if d:
                for i in range(min(-(-n // page), len(row))):
                    if 0 <= row[i] < len(self.free) and self.held < len(self.free):
                        self.free[self.held] = row[i]
                        self.held += 1
                    row[i] = -1
        cu, positions, slots, self.lacking = [0], [], [], 0
        for b, (row, m, d) in enumerate(zip(self.table, new, done)):
            n = 0 if d else self.lens[b]
            for i in range(-(-n // page), min(-(-(n + m) // page), len(row))):
                if self.held:
                    self.held -= 1
                    row[i] = self.free[self.held]
                else:
                    row[i] = -1
                    self.lacking += 1
            for p in range(n, n + m):
                at = row[p // page] if p // page < len(row) else -1
                positions.append(p)
                slots.append(at * page + p % page if at >= 0 else -1)
            cu.append(cu[-1] + m)
            self.lens[b] = n + m
        tail = [-1] * (rows - len(slots))
        return cu, (positions + tail)[:rows], (slots + tail)[:rows]


def _same(pool, table, lens, lists):
    assert table.tolist() == lists.table and lens.tolist() == lists.lens
    assert pool.state.tolist() == [lists.held, lists.lacking] and pool.free.tolist() == lists.free


@pytest.mark.parametrize("pages,page,b,w,most,seed", [
    (5, 16, 1, 3, 20, 0),                # one sequence, past its table and the pool's end
    (40, 64, 7, 9, 130, 1),
    (300, 16, 64, 12, 60, 2),            # the pool runs out now and then
    (4000, 32, 1500, 40, 300, 3),        # sequences in more than one turn of the sums, rows in a second launch
    (9000, 16, 3000, 9, 40, 4),          # more than are kept near
    (2000, 256, 30, 80, 9000, 5),        # many pages come back at once
])
def test_steps(dev, pages, page, b, w, most, seed):
    r = random.Random(seed)
    pool, lists = kv.kv_pages(pages, page, dev), Lists(pages, page, b, w)
    wide = torch.full((b, w + 3), -7, dtype=torch.int32, device=dev)
    table = wide[:, :w]                  # a row of the table has a neighbour
    table.fill_(-1)
    lens = torch.zeros(b, dtype=torch.int32, device=dev)
    for step in range(6):
        new = [r.choice((0, 1, 1, r.randint(0, most))) if step else r.randint(0, most) for _ in range(b)]
        done = [r.random() < 0.2 for _ in range(b)] if step else [False] * b
        rows = max(0, sum(new) + r.choice((0, 0, 5, -3)))
        got = kv.kv_extend(pool, table, lens, _i32(new, dev), rows, torch.tensor(done, device=dev) if step else None)
        want = lists.extend(new, rows, done)
        for x, y in zip(got, want):
            assert x.tolist() == y, step
        _same(pool, table, lens, lists)
        assert (wide[:, w:] == -7).all()


class Cut(Lists):
    """Lists whose sequences also take rows back (a negative number of new ones)."""

    def extend(self, new, rows, done):
        page, cut = self.page, [not d and m < 0 for m, d in zip(new, done)]
        for b, row in enumerate(self.table):     # what comes back of all sequences, in their order, before anything is taken
            n = self.lens[b]
            keep = 0 if done[b] else max(n + new[b], 0) if cut[b] else n
            for i in range(-(-keep // page), min(-(-n // page), len(row))):
                if 0 <= row[i] < len(self.free) and self.held < len(self.free):
                    self.free[self.held] = row[i]
                    self.held += 1
                row[i] = -1
            self.lens[b] = keep
        return super().extend([max(m, 0) for m in new], rows, [False] * len(new))


@pytest.mark.parametrize("pages,page,b,w,most,seed", [
    (5, 16, 1, 3, 20, 0),
    (40, 64, 7, 9, 130, 1),
    (300, 16, 64, 12, 60, 2),
    (4000, 32, 1500, 40, 300, 3),
    (9000, 16, 3000, 9, 40, 4),
    (2000, 256, 30, 80, 9000, 5),
])
def test_rows_taken_back(dev, pages, page, b, w, most, seed):
    """Steps in which some sequences grow, others lose their last rows, some more than they have, some end: no page is lost."""
    r = random.Random(seed)
    pool, lists = kv.kv_pages(pages, page, dev), Cut(pages, page, b, w)
    table, lens = torch.full((b, w), -1, dtype=torch.int32, device=dev), torch.zeros(b, dtype=torch.int32, device=dev)
    for step in range(6):
        new = [r.choice((0, 1, r.randint(0, most), -1, -r.randint(0, most), -r.randint(0, 3 * most))) if step else r.randint(0, most) for _ in range(b)]
        done = [r.random() < 0.1 for _ in range(b)] if step else [False] * b
        rows = sum(max(m, 0) for m in new) + 2
        got = kv.kv_extend(pool, table, lens, _i32(new, dev), rows, torch.tensor(done, device=dev) if step else None)
        for x, y in zip(got, lists.extend(new, rows, done)):
            assert x.tolist() == y, step
        _same(pool, table, lens, lists)
        owned = table[table >= 0].tolist()
        assert sorted(owned + pool.free[:int(pool.state[0])].tolist()) == list(range(pages)), step


def test_drafts_and_a_pool_that_runs_out(dev):
    """Drafts that are not accepted go back with their pages, step after step; a step that lacked pages is undone and made again when
    another sequence has ended; the smallest number takes back everything."""
    page, pages = 16, 6
    pool = kv.kv_pages(pages, page, dev)
    table, lens = torch.full((2, 5), -1, dtype=torch.int32, device=dev), torch.zeros(2, dtype=torch.int32, device=dev)
    kv.kv_extend(pool, table, lens, _i32([15, 10], dev), 25)
    for _ in range(20):                          # four drafts each, of which one or none is kept
        kv.kv_extend(pool, table, lens, _i32([20, 4], dev), 24)
        kv.kv_extend(pool, table, lens, _i32([-20, -4], dev), 0)
    assert pool.state.tolist() == [4, 0] and lens.tolist() == [15, 10] and (table[:, 1:] == -1).all()
    before = table.tolist()
    kv.kv_extend(pool, table, lens, _i32([50, 40], dev), 90)
    assert pool.state.tolist() == [0, 3]
    kv.kv_extend(pool, table, lens, _i32([-50, -40], dev), 0)
    assert pool.state.tolist() == [4, 0] and lens.tolist() == [15, 10] and table.tolist() == before
    _, positions, slots = kv.kv_extend(pool, table, lens, _i32([50, 0], dev), 50, torch.tensor([False, True], device=dev))
    assert pool.state.tolist() == [1, 0] and positions.tolist() == list(range(15, 65)) and (slots >= 0).all()
    cu, _, _ = kv.kv_extend(pool, table, lens, _i32([-2 ** 31, 3], dev), 3)
    assert cu.tolist() == [0, 0, 3] and lens.tolist() == [0, 3] and pool.state.tolist() == [5, 0] and (table[0] == -1).all()


def test_captured_steps_that_take_rows_back(dev):
    """A captured step takes rows back on the replays whose numbers say so."""
    pages, page, b, w, rows = 60, 16, 6, 8, 250
    pool, lists = kv.kv_pages(pages, page, dev), Cut(pages, page, b, w)
    table, lens = torch.full((b, w), -1, dtype=torch.int32, device=dev), torch.zeros(b, dtype=torch.int32, device=dev)
    new, done = torch.zeros(b, dtype=torch.int32, device=dev), torch.zeros(b, dtype=torch.bool, device=dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = kv.kv_extend(pool, table, lens, new, rows, done)
    r = random.Random(8)
    for replay in range(8):
        n, d = [r.randint(-20 if replay else 0, 40) for _ in range(b)], [replay > 2 and r.random() < 0.2 for _ in range(b)]
        new.copy_(_i32(n, dev))
        done.copy_(torch.tensor(d, device=dev))
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(got, lists.extend(n, rows, d)):
            assert x.tolist() == y, replay
        _same(pool, table, lens, lists)


@pytest.mark.parametrize("fmt", [torch.int8, torch.float4_e2m1fn_x2])
def test_drafts_that_are_not_accepted_leave_nothing(dev, fmt):
    """A batch whose every step writes and attends three drafted rows to each sequence, of which one to three are kept: what the kept rows gave,
    and what a step over the whole history then gives, are the bits of a batch that never drafted."""
    b, hq, hkv, dim, page, pages, w, steps = 3, 4, 2, 64, 16, 24, 6, 12
    turn = rope.rotary(dim, "half", dev)
    r = random.Random(5)
    kept = [[r.randint(1, 3) for _ in range(b)] for _ in range(steps)]
    kept[0] = [3, 3, 3]
    g = torch.Generator().manual_seed(6)
    most = 3 * steps
    whole = [torch.randn(b, most, h, dim, generator=g).to(torch.bfloat16).to(dev) for h in (hq, hkv, hkv)]
    other = [torch.randn(b, 3, h, dim, generator=g).to(torch.bfloat16).to(dev) for h in (hq, hkv, hkv)]    # of drafts that are wrong

    def run(drafts):
        cache, pool = kv.kv_cache(pages, hkv, page, dim, fmt, dev), kv.kv_pages(pages, page, dev)
        table, lens = torch.full((b, w), -1, dtype=torch.int32, device=dev), torch.zeros(b, dtype=torch.int32, device=dev)
        at, outs = [0] * b, []
        for keep in kept:
            n = [3] * b if drafts else keep
            q, k, v = (torch.cat([torch.cat([x[i, at[i]:at[i] + keep[i]], y[i, keep[i]:n[i]]]) for i in range(b)]) for x, y in zip(whole, other))
            cu, _, slots = kv.kv_extend(pool, table, lens, _i32(n, dev), sum(n))
            assert (slots >= 0).all()
            out = kv.kv_attention(kv.kv_write_rope(cache, q, k, v, table, lens, cu, turn), cache, table, lens, cu, form="token")
            first = cu.tolist()
            outs += [out[first[i]:first[i] + keep[i]] for i in range(b)]
            if drafts:
                kv.kv_extend(pool, table, lens, _i32([a - c for a, c in zip(keep, n)], dev), 0)
            at = [a + c for a, c in zip(at, keep)]
            assert lens.tolist() == at and int(pool.state[0]) == pages - sum(-(-a // page) for a in at)
        q = torch.cat([whole[0][i, :1] for i in range(b)])
        return outs, kv.kv_attention(q, cache, table, lens, form="token")
    (a, last_a), (c, last_c) = run(True), run(False)
    assert torch.equal(last_a, last_c)
    for x, y in zip(a, c):
        # other rows beside a row may change its last bits: on either side the result's rounding, 2^-8 of it, and one of each weight to f16
        # or finer, 2^-11 of the largest value
        assert ((x.double() - y.double()).abs() <= 2.0 ** -7 * y.double().abs() + 2.0 ** -10 * float(whole[2].abs().max())).all()


def test_bad_contents_stay_inside(dev):
    """Counts beyond the list, negative lengths and rows, entries that are no pages, pages given back twice."""
    b, w, pages, page = 4, 3, 6, 16
    whole = torch.full((64,), 99, dtype=torch.int32, device=dev)
    free, state, table, lens = whole[4:4 + pages], whole[12:14], whole[20:32].view(b, w), whole[40:44]
    free.copy_(_i32([3, 2 ** 31 - 1, -4, 5, 1, 0], dev))
    for held in (10 ** 9, -5, 3):
        state.copy_(_i32([held, 0], dev))
        table.copy_(_i32([[2 ** 31 - 1, -1, 4], [-9, 7, 1], [2, 2, 2], [1, 1, 1]], dev))
        lens.copy_(_i32([-3, 10 ** 9, 2 ** 31 - 1, 33], dev))
        pool = kv.KVPages(free, state, page)
        cu, positions, slots = kv.kv_extend(pool, table, lens, _i32([5, -7, 2 ** 31 - 1, 20], dev), 40,
                                            torch.tensor([True, True, False, True], device=dev))
        assert cu.tolist()[:3] == [0, 5, 5] and 0 <= pool.state[0] <= pages
        assert ((positions >= -1) & (positions <= 1 << 30)).all()
    assert all((whole[a:z] == 99).all() for a, z in ((0, 4), (10, 12), (14, 20), (32, 40), (44, 64)))


def test_slots_of_no_page(dev):
    """Entries of the table and of the pool that are no pages are places to none: slots stay inside the cache."""
    page = 16
    pool = kv.KVPages(_i32([9, 8, 4, 2], dev), _i32([3, 0], dev), page)      # taken: 4, 8, 9
    table, lens = _i32([[3, 4, -1, -1], [1, -1, -1, -1], [7, -1, -1, -1]], dev), _i32([20, 16, 2], dev)
    cu, positions, slots = kv.kv_extend(pool, table, lens, _i32([20, 20, 2], dev), 43)
    # sequence 0: positions 20 to 31 in page 4, which is none, 32 to 39 in the pool's 4, none; 1: in 8 and 9, none; 2: in 7, none
    assert positions.tolist() == [*range(20, 40), *range(16, 36), 2, 3, -1] and slots.tolist() == [-1] * 43
    lens.copy_(_i32([3, 16, 2], dev))
    _, _, slots = kv.kv_extend(pool, table, lens, _i32([2, 0, 0], dev), 2)
    assert slots.tolist() == [3 * page + 3, 3 * page + 4]


def test_no_rows(dev):
    pool = kv.kv_pages(4, 16, dev)
    table, lens = torch.full((2, 2), -1, dtype=torch.int32, device=dev), torch.zeros(2, dtype=torch.int32, device=dev)
    cu, positions, slots = kv.kv_extend(pool, table, lens, _i32([0, 0], dev), 0)
    assert cu.tolist() == [0, 0, 0] and positions.numel() == slots.numel() == 0 and pool.state.tolist() == [4, 0]


def test_empty_batch(dev):
    pool = kv.kv_pages(4, 16, dev)
    none = torch.empty(0, dtype=torch.int32, device=dev)
    cu, positions, slots = kv.kv_extend(pool, none.view(0, 3), none, none, 5)
    assert cu.tolist() == [0] and positions.tolist() == slots.tolist() == [-1] * 5 and slots.dtype == torch.int64
    assert pool.state.tolist() == [4, 0]


def test_captured(dev):
    """A captured step goes on from what it finds on every replay."""
    pages, page, b, w = 60, 16, 6, 8
    pool, lists = kv.kv_pages(pages, page, dev), Lists(pages, page, b, w)
    table, lens = torch.full((b, w), -1, dtype=torch.int32, device=dev), torch.zeros(b, dtype=torch.int32, device=dev)
    new, done = torch.zeros(b, dtype=torch.int32, device=dev), torch.zeros(b, dtype=torch.bool, device=dev)
    rows = 50
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = kv.kv_extend(pool, table, lens, new, rows, done)
    r = random.Random(7)
    for replay in range(5):
        n, d = [r.randint(0, 9) for _ in range(b)], [replay > 1 and r.random() < 0.4 for _ in range(b)]
        new.copy_(_i32(n, dev))
        done.copy_(torch.tensor(d, device=dev))
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(got, lists.extend(n, rows, d)):
            assert x.tolist() == y, replay
        _same(pool, table, lens, lists)


@pytest.mark.parametrize("fmt", [torch.int8, torch.float8_e4m3fn, torch.float4_e2m1fn_x2])
@pytest.mark.parametrize("graphs", [False, True])
def test_a_served_batch(dev, fmt, graphs):
    """Prompts behind a common instruction, tokens one by one, requests that end and others in their places: tables from lengths, the
    rotated queries and written keys of each step, attention over the cache, all against float64 over what the cache then holds."""
    b, hq, hkv, dim, page, prefix_len = 4, 8, 2, 128, 16, 37
    pages, w, room = 70, 14, 200
    g = torch.Generator().manual_seed(11)
    cache, pool = kv.kv_cache(pages, hkv, page, dim, fmt, dev), kv.kv_pages(pages, page, dev)
    turn = rope.rotary(dim, "half", dev, scaling="parts", stretch=4.0, original=4096)
    qw, kw = ((1 + 0.2 * torch.randn(dim, generator=g)).to(torch.bfloat16).to(dev) for _ in range(2))

    def rows(n):
        return (torch.randn(n, h, dim, generator=g).to(torch.bfloat16).to(dev) for h in (hq, hkv, hkv))
    # the instruction: a sequence of its own table
    ptab, plen = torch.full((1, 3), -1, dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    kv.kv_extend(pool, ptab, plen, _i32([prefix_len], dev), prefix_len)
    _, k, v = rows(prefix_len)
    q = torch.zeros(prefix_len, hq, dim, dtype=torch.bfloat16, device=dev)
    kv.kv_write_rope(cache, q, k, v, ptab, plen, None, turn, qw, kw, 1e-6)

    table, lens = torch.full((b, w), -1, dtype=torch.int32, device=dev), torch.zeros(b, dtype=torch.int32, device=dev)
    new, done = torch.zeros(b, dtype=torch.int32, device=dev), torch.zeros(b, dtype=torch.bool, device=dev)
    q, k, v = rows(room)

    def step():
        cu, positions, slots = kv.kv_extend(pool, table, lens, new, room, done)
        turned = kv.kv_write_rope(cache, q, k, v, table, lens, cu, turn, qw, kw, 1e-6, first=prefix_len)
        out, lse = kv.kv_attention_shared(turned, cache, ptab[0], prefix_len, table, lens, cu, lse=True)
        return cu, positions, slots, turned, out, lse
    if graphs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
    for n, d in (([60, 17, 0, 90], [0] * 4), ([1, 1, 50, 1], [0] * 4), ([1] * 4, [0] * 4), ([33, 1, 0, 1], [1, 0, 1, 0]), ([1, 1, 20, 1], [0] * 4)):
        new.copy_(_i32(n, dev))
        done.copy_(torch.tensor(d, dtype=torch.bool))
        for x, y in zip((q, k, v), rows(room)):
            x.copy_(y)
        if graphs:
            graph.replay()
        else:
            got = step()
        torch.cuda.synchronize()
        cu, positions, slots, turned, out, lse = got
        t, at, tab = sum(n), lens.tolist(), table.tolist()
        assert cu.tolist()[-1] == t and (turned[t:] == 0).all() and (out[t:] == 0).all()
        args = (positions[:t] + prefix_len, turn.freq, "half", turn.factor)
        want = orope.turned64(q[:t], *args, qw, 1e-6)
        assert ((turned[:t].double() - want).abs() <= 2.0 ** -8 * 1.01 * want.abs() + 2.0 ** -20).all()
        # where the slots say, the cache holds the step's keys and values
        where = slots[:t].tolist()
        assert [(tab[i][p // page] * page + p % page) for i in range(b) for p in range(at[i] - n[i], at[i])] == where
        codes = cache.v.view(torch.uint8).transpose(1, 2).flatten(0, 1)[slots[:t]]
        want_codes = ok.quantise4(v[:t])[0] if fmt == torch.float4_e2m1fn_x2 else ok.quantise(v[:t], fmt)[0].view(torch.uint8)
        assert torch.equal(codes, want_codes)
        ref, rl, mag, err = ok.attention(turned[:t], cache, tab, at, cu.tolist(), prefix=ptab[0].tolist(), prefix_len=prefix_len)
        # a bf16 result's half step, and the weights' roundings: to f16 three times at most, or to bf16 once
        weight = 2.0 ** -8 if fmt == torch.float4_e2m1fn_x2 else 3.1 * 2.0 ** -11
        tol = 2.0 ** -8 * 1.01 * ref.abs() + (weight + torch.expm1(2 * err)[..., None]) * mag * 1.05 + 1e-30
        assert ((out[:t].double() - ref).abs() <= tol).all()
        assert ((lse[:t].double() - rl).abs() <= err + 2.0 ** -22 * rl.abs() + 2.0 ** -20).all()


def test_two_graphs_and_a_stream_of_its_own(dev):
    """Steps of two batches, captured each in a graph of one memory pool, replayed in turn on a stream that is not theirs, with eager
    steps of a third between: every one as if it were alone."""
    hq, hkv, dim, page, room, b = 8, 2, 64, 16, 40, 3
    turn = rope.rotary(dim, "interleaved", dev)

    class Batch:
        def __init__(self, seed):
            g = torch.Generator().manual_seed(seed)
            self.cache, self.pool = kv.kv_cache(40, hkv, page, dim, torch.float4_e2m1fn_x2, dev), kv.kv_pages(40, page, dev)
            self.table, self.lens = torch.full((b, 8), -1, dtype=torch.int32, device=dev), torch.zeros(b, dtype=torch.int32, device=dev)
            self.new = torch.zeros(b, dtype=torch.int32, device=dev)
            self.rows = [torch.randn(room, h, dim, generator=g).to(torch.bfloat16).to(dev) for h in (hq, hkv, hkv)]

        def step(self):
            cu, positions, slots = kv.kv_extend(self.pool, self.table, self.lens, self.new, room)
            q = kv.kv_write_rope(self.cache, *self.rows, self.table, self.lens, cu, turn)
            return positions, slots, q, kv.kv_attention(q, self.cache, self.table, self.lens, cu)
    counts = [[9, 30, 1], [1, 1, 1], [0, 17, 2], [1, 1, 1]]
    want = {}
    for seed in range(3):
        x = Batch(seed)
        for i, n in enumerate(counts):
            x.new.copy_(_i32(n, dev))
            want[seed, i] = [t.clone() for t in x.step()]
    torch.cuda.synchronize()

    batches, graphs, outs = [Batch(seed) for seed in range(3)], [], []
    for x in batches[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            outs.append(x.step())
        graphs.append(graph)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i, n in enumerate(counts):
            for seed, x in enumerate(batches):
                x.new.copy_(_i32(n, dev))
                if seed < 2:
                    graphs[seed].replay()
                    got = outs[seed]
                else:
                    got = x.step()
                side.synchronize()
                for t, w in zip(got, want[seed, i]):
                    assert torch.equal(t, w), (seed, i)
