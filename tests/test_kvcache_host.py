"""CPU tests of the key / value cache's entry points: what they refuse, with which message, before touching the device."""
import ctypes

import pytest
import torch

from rapid_h3 import _native as nat
from rapid_h3 import kvcache as kv

FAKE = 0x1000          # never dereferenced: validation fails first


def _desc(**kw):
    d = dict(k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE, page_stride=4 * 64 * 128, head_stride=64 * 128,
             scale_page_stride=4 * 64, scale_head_stride=64, pages=10, heads=4, page=64, dim=128, format=0)
    d.update(kw)
    return nat.KvCacheDesc(**d)


def _write(desc, name="rh3_kv_write", rows=6, k=FAKE, v=FAKE, k_st=512, k_sh=128, dtype=1, table=FAKE, stride=8, width=8, lens=FAKE,
           cu=None, batch=2):
    return getattr(nat.lib(), name)(ctypes.addressof(desc), k, k_st, k_sh, v, 512, 128, dtype, rows, table, stride, width, lens, cu,
                                    batch, None)


def _attend(desc, rows=2, q=FAKE, q_st=1024, hq=8, dtype=1, table=FAKE, stride=8, width=8, lens=FAKE, cu=None, batch=2, out=FAKE,
            prefix=None, prefix_len=0, form=0, ws=FAKE, n=1 << 40):
    return nat.lib().rh3_kv_attention(ctypes.addressof(desc), q, q_st, 128, hq, dtype, rows, table, stride, width, lens, cu, batch, 1,
                                      0.1, out, 1024, 128, None, prefix, prefix_len, form, ws, n, None)


@pytest.mark.parametrize("change,message", [
    (dict(k=None), "null cache array"), (dict(v_scale=None), "null cache array"), (dict(format=2), "format"),
    (dict(dim=96), "head dim 96"), (dict(page=48), "page of 48"), (dict(page=512), "page of 512"), (dict(page=8), "page of 8"),
    (dict(pages=0), "0 pages"), (dict(heads=0), "0 heads"), (dict(k=FAKE + 8), "16-byte aligned"),
    (dict(head_stride=100), "16-byte aligned"), (dict(scale_page_stride=6), "16-byte aligned"),
    (dict(page_stride=-8192), "negative stride"),
])
def test_cache_refusals(change, message):
    for call in (_write, lambda d: _write(d, "rh3_kv_read"), _attend):
        assert call(_desc(**change)) == 1 and message in nat.last_error(), nat.last_error()


@pytest.mark.parametrize("change,message", [
    (dict(rows=-1), "-1 rows"), (dict(table=None), "null page table"), (dict(lens=None), "null page table"),
    (dict(batch=0), "0 sequences"), (dict(batch=70000, rows=70000), "70000 sequences"), (dict(rows=7), "do not divide"),
    (dict(width=0), "page table of 0"), (dict(stride=7), "stride 7"), (dict(width=1 << 25, stride=1 << 25), "page table of"),
])
def test_sequence_refusals(change, message):
    for call in (_write, lambda d, **kw: _write(d, "rh3_kv_read", **kw), _attend):
        assert call(_desc(), **change) == 1 and message in nat.last_error(), nat.last_error()


def test_row_refusals():
    for name in ("rh3_kv_write", "rh3_kv_read"):
        for change, message in ((dict(k=None), "null rows"), (dict(v=FAKE + 2), "16-byte aligned"), (dict(k_st=500), "multiples of 8"),
                                (dict(k_sh=129), "multiples of 8"), (dict(dtype=4), "row type 4")):
            assert _write(_desc(), name, **change) == 1 and message in nat.last_error(), nat.last_error()
    for change, message in ((dict(q=None), "null q"), (dict(out=None), "null q or out"), (dict(q=FAKE + 8), "16-byte"),
                            (dict(q_st=1028), "multiples of 8"), (dict(dtype=2), "query type 2"), (dict(hq=6), "do not divide over"),
                            (dict(hq=0), "do not divide over"), (dict(prefix_len=5), "without pages"),
                            (dict(prefix=FAKE, prefix_len=-1), "prefix of -1"), (dict(ws=None), "workspace"), (dict(n=64), "workspace"),
                            (dict(ws=FAKE + 4), "workspace"), (dict(form=3), "form 3"), (dict(form=-1), "form -1")):
        assert _attend(_desc(), **change) == 1 and message in nat.last_error(), nat.last_error()


def test_no_rows_is_no_call():
    assert _write(_desc(), rows=0, k=None, v=None) == 0
    assert _write(_desc(), "rh3_kv_read", rows=0, k=None, v=None) == 0
    assert _attend(_desc(), rows=0, q=None, out=None, ws=None, n=0) == 0


def test_workspace_holds_every_part():
    """More rows, positions or a prefix never need less; nothing to compute needs nothing."""
    size = nat.lib().rh3_kv_attention_workspace_bytes
    assert size(8, 4, 128, 0, 512, 2, 1, 0, 0) == 0 and size(6, 4, 128, 2, 512, 2, 1, 0, 0) == 0 and size(8, 0, 128, 2, 512, 2, 1, 0, 0) == 0
    for rows, batch, form in ((1, 1, 0), (64, 64, 0), (64, 2, 1), (64, 2, 2), (5000, 1, 0)):
        n = size(8, 4, 128, rows, 128000, batch, 1, 0, form)
        assert size(8, 4, 128, rows, 128000, batch, 1, 3000, form) > n
        assert size(8, 4, 128, rows, 128000, batch, 0, 0, form) >= n


def test_wrappers_refuse():
    k = torch.zeros((4, 2, 64, 128), dtype=torch.int8)
    s = torch.zeros((4, 2, 64))
    with pytest.raises(RuntimeError, match="no CPU path"):
        kv.KVCache(k, k, s, s)
    for bad, message in (((k, k[:, :1], s, s), "one layout"), ((k[..., :96], k[..., :96], s, s), "head dim"),
                         ((k[:, :, :48], k[:, :, :48], s, s), "pages of"), ((k, k, s[:, :, :32], s), "scales must be"),
                         ((k, k, s, s.double()), "scales must be"), ((k.transpose(1, 2), k.transpose(1, 2), s, s), "pages of"),
                         ((k[..., ::2], k[..., ::2], s, s), "contiguous")):
        with pytest.raises(RuntimeError, match=message):
            kv.KVCache(*bad)
    with pytest.raises(TypeError, match="codes"):
        kv.KVCache(k.float(), k.float(), s, s)
    with pytest.raises(TypeError, match="codes"):
        kv.KVCache(k, k.view(torch.float8_e4m3fn), s, s)

    class Cache:
        heads, dim, page, device, gpu = 2, 128, 64, torch.device("cpu"), -1
    x = torch.zeros((3, 2, 128), dtype=torch.bfloat16)
    t, n = torch.zeros((3, 1), dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        kv.kv_write(Cache, x, x, t, n)
    with pytest.raises(RuntimeError, match="no CPU path"):
        kv.kv_attention(x, Cache, t, n)
    with pytest.raises(RuntimeError, match="kv_write: k must be"):
        kv.kv_write(Cache, x[..., :64], x, t, n)
    with pytest.raises(RuntimeError, match="multiple of 2 heads"):
        kv.kv_attention(x[:, :1], Cache, t, n)
    with pytest.raises(TypeError, match="bf16 or fp16"):
        kv.kv_attention(x.float(), Cache, t, n)
    with pytest.raises(ValueError, match="form 'both'"):
        kv.kv_attention(x, Cache, t, n, form="both")
    with pytest.raises(RuntimeError, match="does not fit"):
        kv.kv_attention_shared(x, Cache, torch.zeros(2, dtype=torch.int32), 129, t, n)
    with pytest.raises(RuntimeError, match="prefix must be"):
        kv.kv_attention_shared(x, Cache, torch.zeros(2), 1, t, n)
    with pytest.raises(RuntimeError, match="table must be"):
        kv._seqs("f", Cache, t.long(), n, None, -1)
    with pytest.raises(RuntimeError, match="lens must be"):
        kv._seqs("f", Cache, t, n[:2], None, -1)
    with pytest.raises(RuntimeError, match="cu must be"):
        kv._seqs("f", Cache, t, n, n, -1)


def test_read_needs_its_number_of_rows():
    """With offsets, whose last only the GPU knows, kv_read takes no number of its own choice."""
    class Cache:
        heads, dim, page, device, gpu = 2, 128, 64, torch.device("cpu"), -1
    t, n = torch.zeros((3, 1), dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="rows .* must be given"):
        kv.kv_read(Cache, t, n, torch.tensor([0, 2, 3, 9], dtype=torch.int32))


def test_join_refusal_comes_before_any_launch():
    """More (row, head) pairs behind a prefix than the join's grid holds: refused as an argument, with nothing launched (on a machine
    without a GPU a launch would be another error)."""
    rows = 1 << 21
    assert _attend(_desc(), rows=rows, hq=64, prefix=FAKE, prefix_len=100, n=1 << 62) == 1
    assert f"{rows} rows of 64 heads" in nat.last_error()


def test_sizes_past_64_bits_are_refused():
    """Widths and head counts whose products with the page or the rows would not fit 64 bits; the workspace has no size for them."""
    for call in (_write, lambda d, **kw: _write(d, "rh3_kv_read", **kw), _attend):
        for width in (1 << 58, 1 << 60, (1 << 62) + 8):
            assert call(_desc(), width=width, stride=width) == 1 and "page table of" in nat.last_error()
    for rows, hq in ((8, 1 << 62), (1 << 20, 1 << 46), (1 << 30, 8)):
        assert _attend(_desc(), rows=rows, hq=hq, n=(1 << 63) - 1) == 1 and f"{rows} rows of {hq} heads" in nat.last_error()
    size = nat.lib().rh3_kv_attention_workspace_bytes
    good = dict(hq=8, heads=4, dim=128, rows=2, cap=512, batch=2, even=1, prefix=0, form=0)
    assert size(*good.values()) > 0
    for bad in (dict(hq=1 << 62), dict(dim=96), dict(rows=1 << 40), dict(cap=1 << 40), dict(batch=1 << 20), dict(prefix=-1), dict(prefix=1 << 40)):
        assert size(*{**good, **bad}.values()) == 0, bad


def test_workspace_size_is_of_the_calls_gpu(monkeypatch):
    """The size depends on the GPU's number of CUs: kept per GPU, and asked for with the call's GPU as the current one."""
    now = [0]

    class On:
        def __init__(self, gpu):
            self.gpu = gpu

        def __enter__(self):
            self.before, now[0] = now[0], self.gpu

        def __exit__(self, *_):
            now[0] = self.before

    class Lib:
        @staticmethod
        def rh3_kv_attention_workspace_bytes(*sizes):
            return 1000 * (1 + now[0])

    class Row:          # a tensor of a GPU, as far as the wrapper looks
        ndim, shape, dtype, is_cuda = 3, (2, 4, 128), torch.bfloat16, True

        def __init__(self, gpu):
            self.gpu = gpu

        def stride(self, i=None):
            return (512, 128, 1) if i is None else (512, 128, 1)[i]

        def get_device(self):
            return self.gpu

        def data_ptr(self):
            return FAKE
    sizes = []
    monkeypatch.setattr(kv, "_on", On)
    monkeypatch.setattr(kv, "_stream", lambda gpu: None)
    monkeypatch.setattr(kv, "_seqs", lambda *a: (FAKE, 1, 1, FAKE, None, 2))
    monkeypatch.setattr(nat, "lib", lambda: Lib)
    monkeypatch.setattr(nat, "call", lambda name, *args: sizes.append(args[-2]))

    class Cache:
        heads, dim, page, device, _ref = 2, 128, 64, torch.device("cpu"), None
    kv._workspace_bytes.cache_clear()
    for gpu in (0, 1, 0):
        kv.kv_attention(Row(gpu), Cache, None, None, out=Row(gpu))
    kv._workspace_bytes.cache_clear()
    assert sizes == [1000, 2000, 1000]


def test_cache_attributes_stay(monkeypatch):
    """The kernels read the addresses that a KVCache was made with, so its tensors cannot be exchanged."""
    k, s = torch.zeros((4, 2, 64, 128), dtype=torch.int8), torch.zeros((4, 2, 64))
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    c = kv.KVCache(k, k.clone(), s, s.clone())
    monkeypatch.undo()
    for name in ("k", "v", "k_scale", "v_scale", "page", "heads"):
        with pytest.raises(AttributeError, match="cannot be changed"):
            setattr(c, name, getattr(c, name))
    assert c.k is k and c.k_scale is s


def test_results_do_not_share_memory():
    """Rows repeated without memory of their own (stride 0) may be read, not written."""
    for change in (dict(k_st=0), dict(k_sh=0)):
        assert _write(_desc(), "rh3_kv_read", **change) == 1 and "share memory" in nat.last_error()
    for change in (dict(o_st=0), dict(o_sh=0)):
        assert _attend_out(_desc(), **change) == 1 and "out share memory" in nat.last_error()


def _attend_out(desc, o_st=1024, o_sh=128):
    return nat.lib().rh3_kv_attention(ctypes.addressof(desc), FAKE, 1024, 128, 8, 1, 2, FAKE, 8, 8, FAKE, None, 2, 1, 0.1, FAKE, o_st,
                                      o_sh, None, None, 0, 0, FAKE, 1 << 40, None)


def test_no_sequences_is_no_call():
    """An empty batch: no rows of no sequences."""
    for name in ("rh3_kv_write", "rh3_kv_read"):
        assert _write(_desc(), name, rows=0, batch=0, k=None, v=None, table=None, lens=None) == 0
        assert _write(_desc(), name, rows=3, batch=0) == 1 and "0 sequences" in nat.last_error()
    assert _attend(_desc(), rows=0, batch=0, q=None, out=None, ws=None, n=0, table=None, lens=None) == 0
