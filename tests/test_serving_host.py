"""CPU tests of the serving step's entry points (rh3_kv_extend, rh3_qk_norm_rope, rh3_kv_write_rope, the 4-bit cache): what they
refuse, with which message, before touching the device; the frequencies; the oracles' own properties."""
import contextlib
import ctypes
import math
import os
import subprocess
import sys

import pytest
import torch

from oracle import kvcache as ok
from oracle import rope as orope
from rapid_h3 import _native as nat
from rapid_h3 import kvcache as kv
from rapid_h3 import rope

FAKE = 0x1000          # never dereferenced: validation fails first


def _desc(**kw):
    d = dict(k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE, page_stride=4 * 64 * 64, head_stride=64 * 64, scale_page_stride=4 * 64 * 4,
             scale_head_stride=64 * 4, pages=10, heads=4, page=64, dim=128, format=nat.RH3_KV_FP4)
    d.update(kw)
    return nat.KvCacheDesc(**d)


ROPE = ("q q_st q_sh qo qo_st qo_sh k k_st k_sh ko ko_st ko_sh q_heads k_heads rows dim dtype positions "
        "freq rot interleaved factor norm eps qw kw wide").split()


def _rope(**kw):
    d = dict(zip(ROPE, (FAKE, 1024, 128, FAKE, 1024, 128, FAKE, 256, 128, FAKE, 256, 128, 8, 2, 3, 128, 1, FAKE, FAKE, 128, 0, 1.0, 1, 1e-6, FAKE,
                        FAKE, 0)))
    d.update(kw)
    return nat.lib().rh3_qk_norm_rope(rope._ARGS.pack(*d.values()), None)


WRITE = ("q q_st q_sh qo qo_st qo_sh k k_st k_sh v v_st v_sh q_heads dtype rows table table_stride width lens cu batch first "
         "freq rot interleaved factor norm eps qw kw wide").split()


def _write_rope(desc=None, **kw):
    d = dict(zip(WRITE, (FAKE, 1024, 128, FAKE, 1024, 128, FAKE, 512, 128, FAKE, 512, 128, 8, 1, 6, FAKE, 8, 8, FAKE, 0, 2, 0, FAKE, 128, 0, 1.0, 1,
                         1e-6, FAKE, FAKE, 0)))
    d.update(kw)
    desc = desc or _desc()                      # held until the call returns
    return nat.lib().rh3_kv_write_rope(ctypes.addressof(desc), kv._WRITE_ROPE.pack(*d.values()), None)


EXTEND = "free pages state page table table_stride width lens more done batch cu positions slots rows ws n".split()


def _extend(**kw):
    d = dict(zip(EXTEND, (FAKE, 10, FAKE, 64, FAKE, 8, 8, FAKE, FAKE, 0, 3, FAKE, FAKE, FAKE, 5, FAKE, 1 << 20)))
    d.update(kw)
    return nat.lib().rh3_kv_extend(kv._EXTEND.pack(*d.values()), None)


@pytest.mark.parametrize("change,message", [
    (dict(rows=-1), "-1 rows"), (dict(dim=96), "head dim 96"), (dict(rot=24), "24 rotated"), (dict(rot=144), "144 rotated"),
    (dict(rot=-16), "-16 rotated"), (dict(freq=0), "no frequencies"), (dict(rot=0, norm=0), "neither a norm"), (dict(freq=FAKE + 4), "8-byte"),
    (dict(qw=FAKE + 8), "16-byte"), (dict(dtype=4), "row type 4"), (dict(positions=0), "no positions"), (dict(q=0), "null q"),
    (dict(ko=0), "null k's result"), (dict(k_st=100), "k must be 16-byte"), (dict(q=FAKE + 8), "q must be 16-byte"),
    (dict(qo_st=0), "q's result share memory"), (dict(ko_sh=0), "k's result share memory"), (dict(q_heads=70000), "70000 and 2 heads"),
    (dict(k_heads=-1), "8 and -1 heads"), (dict(rows=1 << 31), "rows"),
])
def test_rope_refusals(change, message):
    assert _rope(**change) == 1 and message in nat.last_error(), nat.last_error()


@pytest.mark.parametrize("change,message", [
    (dict(rows=7), "do not divide"), (dict(table=0), "null page table"), (dict(rot=24), "24 rotated"), (dict(q_heads=0), "0 query heads"),
    (dict(first=1 << 40), "first position"), (dict(dtype=0), "row type 0"), (dict(v=0), "null v"), (dict(v_sh=4), "v must be"),
    (dict(qo_st=0), "q's result share memory"), (dict(rot=0, norm=0), "neither a norm"), (dict(batch=0), "0 sequences"),
])
def test_write_rope_refusals(change, message):
    assert _write_rope(**change) == 1 and message in nat.last_error(), nat.last_error()


@pytest.mark.parametrize("change,message", [
    (dict(format=3), "format 3"), (dict(dim=96), "head dim 96"), (dict(k=None), "null cache array"), (dict(head_stride=64 * 64 + 8), "16-byte"),
    (dict(scale_head_stride=64 * 4 + 4), "16-byte"), (dict(scale_page_stride=1028), "16-byte"), (dict(k_scale=FAKE + 4), "16-byte"), (dict(page=24), "page of 24"),
])
def test_four_bit_cache_refusals(change, message):
    assert _write_rope(_desc(**change)) == 1 and message in nat.last_error(), nat.last_error()
    lib, d = nat.lib(), _desc(**change)
    assert lib.rh3_kv_write(ctypes.addressof(d), FAKE, 512, 128, FAKE, 512, 128, 1, 6, FAKE, 8, 8, FAKE, None, 2, None) == 1
    assert message in nat.last_error()


@pytest.mark.parametrize("change,message", [
    (dict(pages=0), "0 pages"), (dict(page=48), "page of 48"), (dict(rows=-1), "-1 rows"), (dict(batch=0), "0 sequences"),
    (dict(batch=65537), "65537 sequences"), (dict(width=0), "table of 0"), (dict(table_stride=7), "stride 7"),
    (dict(batch=65536, width=1 << 15, table_stride=1 << 15), "page table of 32768"), (dict(free=0), "null pool"), (dict(cu=0), "null pool"), (dict(lens=0), "null pool"),
    (dict(positions=0), "null positions"), (dict(ws=0), "workspace"), (dict(n=8), "workspace"), (dict(ws=FAKE + 4), "workspace"),
])
def test_extend_refusals(change, message):
    assert _extend(**change) == 1 and message in nat.last_error(), nat.last_error()


def test_nothing_to_do_is_no_call():
    assert _rope(rows=0, q=0, k=0) == 0 and _rope(q_heads=0, k_heads=0, q=0, k=0) == 0
    assert _write_rope(rows=0, q=0) == 0 and _write_rope(rows=0, batch=0, q=0, table=0, lens=0) == 0
    assert _extend(rows=0, batch=0, table=0) == 0
    size = nat.lib().rh3_kv_extend_workspace_bytes
    assert size(0) == size(65537) == size(-1) == 0 and size(1) == 24 and size(65536) == 12 * 65537


def test_null_arguments():
    lib = nat.lib()
    for call in (lambda: lib.rh3_qk_norm_rope(None, None), lambda: lib.rh3_kv_extend(None, None),
                 lambda: lib.rh3_kv_write_rope(ctypes.addressof(_desc()), None, None)):
        assert call() == 1 and "null arguments" in nat.last_error()


def test_wrappers_refuse(monkeypatch):
    codes, scales = torch.zeros((4, 2, 64, 64), dtype=torch.uint8), torch.zeros((4, 2, 64, 4), dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="no CPU path"):
        kv.KVCache(codes, codes, scales, scales)
    for bad, message in (((codes, codes, scales[..., :2], scales), "scales of 4-bit"), ((codes, codes, scales.float(), scales), "scales of 4-bit"),
                         ((codes[..., :48], codes[..., :48], scales, scales), "head dim"), ((codes, codes, scales[:, :, :, ::2], scales), "scales of 4-bit")):
        with pytest.raises(RuntimeError, match=message):
            kv.KVCache(*bad)
    with pytest.raises(TypeError, match="codes"):
        kv.KVCache(codes, codes.view(torch.int8), scales, scales)
    free, state = torch.zeros(4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for bad, message in (((free.long(), state, 64), "free must be"), ((free, state[:1], 64), "state must be"), ((free, state, 48), "pages of"),
                         ((free, state, 64), "no CPU path"), ((free[:0], state, 64), "free must be")):
        with pytest.raises(RuntimeError, match=message):
            kv.KVPages(*bad)
    freq, _ = rope.frequencies(64)
    for bad, message in (((freq.float(),), "fp64"), ((freq[:12],), "multiple of 8"), ((freq[None],), "fp64"), ((freq,), "no CPU path"),
                         ((torch.cat([freq, freq, freq]),), "8 to 64")):
        with pytest.raises(RuntimeError, match=message):
            rope.Rotary(*bad)
    with pytest.raises(ValueError, match="layout"):
        rope.Rotary(freq, "both")
    x = torch.zeros((3, 2, 128), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        rope.qk_norm_rope(x, None, None, None, eps=1e-6)
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    turn = rope.Rotary(freq)
    for name in ("freq", "rot", "factor"):
        with pytest.raises(AttributeError, match="cannot be changed"):
            setattr(turn, name, 1)
    pool = kv.KVPages(free, state, 64)
    with pytest.raises(AttributeError, match="cannot be changed"):
        pool.free = free
    pos = torch.zeros(3, dtype=torch.int32)
    for call, error, message in (
            (lambda: rope.qk_norm_rope(x, None, pos, None), ValueError, "nothing to do"),
            (lambda: rope.qk_norm_rope(x, None, pos, turn, x[0, 0]), ValueError, "without eps"),
            (lambda: rope.qk_norm_rope(x, None, pos, turn, x[0, 0, :64], None, 1e-6), RuntimeError, "norm weights"),
            (lambda: rope.qk_norm_rope(x, None, pos, turn, x[0, 0], x[0, 0].float(), 1e-6), RuntimeError, "of one type"),
            (lambda: rope.qk_norm_rope(x, None, pos.long(), turn), RuntimeError, "positions"),
            (lambda: rope.qk_norm_rope(x, None, pos[:2], turn), RuntimeError, "positions"),
            (lambda: rope.qk_norm_rope(x, x[:2], pos, turn), RuntimeError, "k must be"),
            (lambda: rope.qk_norm_rope(x, x.half(), pos, turn), RuntimeError, "k must be"),
            (lambda: rope.qk_norm_rope(x, None, pos, turn, out=(x[:2], None)), RuntimeError, "out for q"),
            (lambda: rope.qk_norm_rope(x[..., ::2], None, pos, turn), RuntimeError, "contiguous last dim"),
            (lambda: rope.qk_norm_rope(x[..., :96], None, pos, turn), RuntimeError, "64 or 128"),
            (lambda: rope.qk_norm_rope(x[..., :32], None, pos, turn), RuntimeError, "64 or 128"),
            (lambda: rope.qk_norm_rope(x.double(), None, pos, turn), RuntimeError, "bf16, fp16 or fp32")):
        with pytest.raises(error, match=message):
            call()
    table, n = torch.zeros((3, 2), dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    for call, error, message in (
            (lambda: kv.kv_extend(pool, table.long(), n, n, 3), RuntimeError, "table must be"),
            (lambda: kv.kv_extend(pool, table, n[:2], n, 3), RuntimeError, "lens must be"),
            (lambda: kv.kv_extend(pool, table, n, n.long(), 3), RuntimeError, "new must be"),
            (lambda: kv.kv_extend(pool, table, n, n, 3, n), RuntimeError, "done must be"),
            (lambda: kv.kv_extend(pool, table, n, n, -1), ValueError, "-1 rows")):
        with pytest.raises(error, match=message):
            call()
    cache = kv.KVCache(codes, codes.clone(), scales, scales.clone())
    assert cache.dim == 128 and cache.page == 64
    with pytest.raises(TypeError, match="of one number of rows"):
        kv.kv_write_rope(cache, x[:2], x, x, table, n, rotary=turn)
    with pytest.raises(TypeError, match="of one number of rows"):
        kv.kv_write_rope(cache, x.half(), x, x, table, n, rotary=turn)
    with pytest.raises(RuntimeError, match="at most 64 channels"):
        kv.kv_write_rope(kv.KVCache(codes[..., :32].contiguous(), codes[..., 32:].contiguous(), scales[..., :2].contiguous(), scales[..., 2:].contiguous()),
                         x[..., :64], x[..., :64], x[..., :64], table, n, rotary=rope.Rotary(rope.frequencies(128)[0]))


def test_extend_of_an_empty_batch_lacks_no_pages(monkeypatch):
    """pool.state[1] is of the last call, also where that had no sequences."""
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    pool = kv.KVPages(torch.arange(4, dtype=torch.int32), torch.tensor([3, 7], dtype=torch.int32), 16)
    none = torch.empty(0, dtype=torch.int32)
    kv.kv_extend(pool, none.view(0, 3), none, none, 2)
    assert pool.state.tolist() == [3, 0]


def test_workspace_is_of_the_caches_format(monkeypatch):
    """A call allocates what its own format and query type need: caches of 8-bit codes nothing for the 4-bit kernels' plans. Without them the
    size is enough for all."""
    size, of = nat.lib().rh3_kv_attention_workspace_bytes, nat.RH3_KV_SIZE_OF
    formats, types = (nat.RH3_KV_INT8, nat.RH3_KV_E4M3, nat.RH3_KV_FP4), (nat.RH3_DTYPE_BF16, nat.RH3_DTYPE_F16)
    for hq, heads, dim, rows, cap, batch, prefix in ((32, 8, 128, 1, 16384, 1, 0), (32, 8, 128, 128, 4096, 16, 0), (28, 4, 64, 512, 65536, 4, 0),
                                                     (32, 8, 128, 384, 65536, 4, 0), (56, 8, 128, 120, 640, 40, 24001)):
        for form in (nat.RH3_KV_BY_SIZE, nat.RH3_KV_TOKEN, nat.RH3_KV_CHUNK):
            n = {(f, t): size(hq, heads, dim, rows, cap, batch, 1, prefix, form + of(f, t)) for f in formats for t in types}
            assert max(n.values()) == size(hq, heads, dim, rows, cap, batch, 1, prefix, form) > 0
            assert len({n[f, t] for f in formats[:2] for t in types}) == 1
    # one token: slots for the parts of two workgroups to a CU, or three
    a, b = (size(32, 8, 128, 1, 16384, 1, 1, 0, of(f, types[0])) for f in (nat.RH3_KV_INT8, nat.RH3_KV_FP4))
    assert 3 * a == 2 * b and a % (2 * 2 * 16 * (128 + 2) * 4) == 0
    assert size(32, 8, 128, 1, 16384, 1, 1, 0, of(3, types[0])) == 0

    given = []
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    monkeypatch.setattr(kv, "_on", lambda gpu: contextlib.nullcontext())
    monkeypatch.setattr(kv, "_stream", lambda gpu: None)
    monkeypatch.setattr(nat, "call", lambda name, *args: given.append(args[-2]))
    codes, scales = torch.zeros((4, 2, 64, 128), dtype=torch.int8), torch.zeros((4, 2, 64))
    byte, four = torch.zeros((4, 2, 64, 64), dtype=torch.uint8), torch.zeros((4, 2, 64, 4), dtype=torch.uint8)
    table, lens = torch.zeros((3, 2), dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    kv._workspace_bytes.cache_clear()
    for dtype, t in ((torch.bfloat16, types[0]), (torch.float16, types[1])):
        q = torch.zeros((3, 8, 128), dtype=dtype)
        for args, f in (((codes, codes, scales, scales), formats[0]), ((codes.view(kv.FP8),) * 2 + (scales, scales), formats[1]), ((byte, byte, four, four), formats[2])):
            kv.kv_attention(q, kv.KVCache(*args), table, lens)
            assert given[-1] == size(8, 2, 128, 3, 128, 3, 1, 0, of(f, t))
    kv._workspace_bytes.cache_clear()


def test_a_torch_without_the_four_bit_types():
    """8-bit caches, and 4-bit ones of bytes, need no torch that names the 4-bit and exponent types."""
    code = ("import torch; del torch.float4_e2m1fn_x2, torch.float8_e8m0fnu; from rapid_h3 import kvcache as kv; torch.Tensor.is_cuda = True; "
            "assert kv.kv_cache(2, 1, device='cpu').dim == 128 and kv.kv_cache(2, 1, dtype=kv.FP8, device='cpu').dim == 128; "
            "x, s = torch.zeros((2, 1, 16, 32), dtype=torch.uint8), torch.zeros((2, 1, 16, 2), dtype=torch.uint8); assert kv.KVCache(x, x, s, s).dim == 64")
    path = os.pathsep.join([os.path.dirname(os.path.dirname(kv.__file__)), os.environ.get("PYTHONPATH", "")])
    r = subprocess.run([sys.executable, "-c", code], env={**os.environ, "PYTHONPATH": path}, capture_output=True, text=True, timeout=110)
    assert r.returncode == 0, r.stderr


def test_frequencies():
    f, one = rope.frequencies(128)
    assert one == 1.0 and f.dtype == torch.float64 and torch.equal(f, 10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64))
    g, _ = rope.frequencies(128, scaling="linear", stretch=4.0)
    assert torch.equal(g, f / 4)
    g, _ = rope.frequencies(128, scaling="base", stretch=8.0)
    assert g[0] == 1.0 and abs(g[-1] * 8 / f[-1] - 1) < 1e-12
    g, factor = rope.frequencies(128, scaling="parts", stretch=4.0, original=8192)
    turns = 8192 * f / (2 * math.pi)
    assert torch.equal(g[turns >= 32], f[turns >= 32]) and torch.allclose(g[turns <= 1], f[turns <= 1] / 4, rtol=1e-14, atol=0)
    assert (g <= f).all() and (g >= f / 4 * (1 - 1e-14)).all() and abs(factor - (0.1 * math.log(4) + 1)) < 1e-15
    for bad in (dict(rot=3), dict(rot=2), dict(rot=128, scaling="other"), dict(rot=128, scaling="parts"), dict(rot=128, stretch=0.5),
                dict(rot=128, scaling="parts", original=100, low=4, high=4)):
        with pytest.raises(ValueError):
            rope.frequencies(**bad)


def test_four_bit_oracle():
    """Every code comes back from its own value, whatever the power of two; an error is half a step at most."""
    grid = torch.tensor(ok.E2M1, dtype=torch.float64)
    x = torch.cat([grid, -grid, grid, -grid])
    for e in (-120, -5, 0, 7, 120):
        c, s = ok.quantise4((x * 2.0 ** e)[None])
        assert int(s) == e + 127 and torch.equal(ok.values4(c, s)[0], x * 2.0 ** e)
    x = torch.randn(50, 128, dtype=torch.float64, generator=torch.Generator().manual_seed(0))
    c, s = ok.quantise4(x)
    y = x.unflatten(-1, (-1, 32)) / ok._pow2(s.int() - 127)[..., None]
    amax = y.abs().amax(-1)
    assert (amax <= 7).all() and (amax > 3.5).all()
    step = torch.where(y.abs() < 2, 0.25, torch.where(y.abs() < 4, 0.5, 1.0))
    back = ok.values4(c, s).unflatten(-1, (-1, 32)) / ok._pow2(s.int() - 127)[..., None]
    assert ((back - y).abs() <= step).all()


def test_rope_oracles_agree():
    """The restatement step by step is float64's within its roundings; a rotation keeps a pair's length; position 0 changes nothing."""
    x = torch.randn(20, 3, 64, generator=torch.Generator().manual_seed(1))
    freq, _ = rope.frequencies(48)
    pos = torch.arange(20) * 7001
    for layout in rope.LAYOUTS:
        for eps in (None, 1e-6):
            a, b = (f(x, pos, freq, layout, 1.25, None, eps) for f in (orope.turned, orope.turned64))
            assert ((a.double() - b).abs() <= 1e-6 * (1 + b.abs())).all()
        y = orope.turned64(x, pos, freq, layout, 1.0, None, None)
        before, after = (torch.hypot(*orope._pairs(z.double(), 24, layout)[:2]) for z in (x, y))
        assert (before - after).abs().max() < 1e-12
        assert torch.equal(orope.turned(x, pos * 0, freq, layout, 1.0, None, None), x)
