"""A paged, quantised key / value cache and the attention over it, on the HIP kernels (librh3: rh3_kv_*).

For programs that keep keys and values from call to call: the past frames of a video generated in chunks, a prompt's tokens
in a text encoder in front of the DiT, a long context that many continuations share. Keys and values are quantised once, as
they are written, by the row quantizers' rule over one head (s = max(amax / QMAX, 1e-12), round half even of x / s, QMAX 127
or 448), and attention reads the codes where they lie. The reference has no counterpart.

Every call names its sequences alike:
  table [B, W] int32   the pages of each sequence in order; an entry outside [0, pages) is an absent page, and so is what lies
                       past the table
  lens [B] int32       cached positions of each sequence, the rows of this call included
  cu [B + 1] int32     where each sequence's rows begin and end among the call's rows; None: the same number each
The rows of a sequence are its last positions: row i of n is position lens[b] - n + i. The three live on the GPU and are read
by the kernels, so a captured call follows what is written into them between replays. Rows in front of cu[0] and behind cu[B]
are not read and stay as they are; of rows that cu names but the call does not have, it takes none.
"""
import contextlib
import ctypes
import functools

import torch

from . import _native as nat

FP8 = torch.float8_e4m3fn
_ROW = {torch.bfloat16: nat.RH3_DTYPE_BF16, torch.float16: nat.RH3_DTYPE_F16, torch.float32: nat.RH3_DTYPE_F32}
_FORM = {None: nat.RH3_KV_BY_SIZE, "token": nat.RH3_KV_TOKEN, "chunk": nat.RH3_KV_CHUNK}
_HERE = contextlib.nullcontext()


def _st(t, axis):
    """The stride of an axis; 0 for one of length 1, whose stride may be any number and is not used."""
    return t.stride(axis) if t.shape[axis] > 1 else 0


class KVCache:
    """The pages of one layer: k, v [P, heads, page, dim] int8 or float8_e4m3fn codes, k_scale, v_scale [P, heads, page]
    fp32 (page 16 to 256, a power of two; dim 64 or 128; views of larger buffers whose pages and heads lie apart are fine,
    k like v and k_scale like v_scale). Where a position holds something, no code is NaN and a scale is finite and not
    negative, or NaN for a row that is (as kv_write leaves them). The tensors are kept and used as they are; the attributes
    cannot be changed."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "pages", "heads", "page", "dim", "device", "gpu", "_desc", "_ref")

    def __init__(self, k, v, k_scale, v_scale):
        if k.ndim != 4 or v.shape != k.shape or any(_st(v, i) != _st(k, i) for i in range(4)):
            raise RuntimeError(f"KVCache: k and v must be [pages, heads, page, dim] of one layout, got {tuple(k.shape)} and {tuple(v.shape)}")
        p, h, n, d = k.shape
        if k.dtype not in (torch.int8, FP8) or v.dtype != k.dtype:
            raise TypeError(f"KVCache: codes must be int8 or float8_e4m3fn, got {k.dtype} and {v.dtype}")
        if d not in (64, 128) or n not in (16, 32, 64, 128, 256):
            raise RuntimeError(f"KVCache: head dim 64 or 128 and pages of 16, 32, 64, 128 or 256 positions, got {d} and {n}")
        if k.stride(3) != 1 or k.stride(2) != d:
            raise RuntimeError("KVCache: a head's positions in a page must be contiguous")
        for s in (k_scale, v_scale):
            if s.shape != (p, h, n) or s.dtype != torch.float32 or s.stride(2) != 1:
                raise RuntimeError("KVCache: scales must be fp32 [pages, heads, page] with a contiguous last dim")
        if any(_st(v_scale, i) != _st(k_scale, i) for i in range(2)):
            raise RuntimeError("KVCache: k_scale and v_scale must have one layout")
        if not k.is_cuda or any(t.device != k.device for t in (v, k_scale, v_scale)):
            raise RuntimeError("KVCache: the four tensors must be on one GPU (no CPU path)")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.pages, self.heads, self.page, self.dim, self.device = p, h, n, d, k.device
        self.gpu = k.get_device()
        self._desc = nat.KvCacheDesc(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), _st(k, 0), _st(k, 1),
                                     _st(k_scale, 0), _st(k_scale, 1), p, h, n, d,
                                     nat.RH3_KV_INT8 if k.dtype == torch.int8 else nat.RH3_KV_E4M3)
        self._ref = ctypes.addressof(self._desc)

    def __setattr__(self, name, value):
        if hasattr(self, "_ref"):   # the kernels would go on with the addresses taken at first
            raise AttributeError(f"KVCache: {name} cannot be changed; make a new KVCache")
        object.__setattr__(self, name, value)


def kv_cache(pages, heads, page=64, dim=128, dtype=torch.int8, device="cuda"):
    """A new cache of zeros."""
    def codes():
        return torch.zeros((pages, heads, page, dim), dtype=torch.int8, device=device).view(dtype)

    def scales():
        return torch.zeros((pages, heads, page), dtype=torch.float32, device=device)
    return KVCache(codes(), codes(), scales(), scales())


# The small calls (a token of one sequence is 12 us of GPU work in two launches) are bound by what the host does: shapes, strides
# and devices are asked for once a call, devices as numbers, and the workspace's size once for each set of sizes.
def _on(index):
    """The tensors' GPU as the current one for a launch, where it is another."""
    return _HERE if index == torch._C._cuda_getDevice() else torch.cuda.device(index)


_stream = torch._C._cuda_getCurrentRawStream


def _seqs(name, cache, table, lens, cu, gpu):
    """The sequences' arguments of a call after its rows: table, its stride and width, lens, cu, batch."""
    if table.ndim != 2 or table.dtype != torch.int32 or (table.stride(1) != 1 and table.shape[1] > 1):
        raise RuntimeError(f"{name}: table must be int32 [batch, pages of a sequence] with a contiguous last dim")
    b, w = table.shape
    if lens.dtype != torch.int32 or lens.ndim != 1 or lens.numel() != b or not lens.is_contiguous():
        raise RuntimeError(f"{name}: lens must be contiguous int32 [{b}]")
    if table.get_device() != gpu or lens.get_device() != gpu or cache.gpu != gpu:
        raise RuntimeError(f"{name}: the cache, the rows, table and lens must be on one GPU")
    if cu is None:
        return table.data_ptr(), table.stride(0), w, lens.data_ptr(), None, b
    if cu.dtype != torch.int32 or cu.ndim != 1 or cu.numel() != b + 1 or not cu.is_contiguous() or cu.get_device() != gpu:
        raise RuntimeError(f"{name}: cu must be contiguous int32 [{b + 1}] on the rows' GPU")
    return table.data_ptr(), table.stride(0), w, lens.data_ptr(), cu.data_ptr(), b


def _rows(name, what, x, cache):
    """Rows of keys or values: their number and strides."""
    if x.ndim == 3:
        t, h, d = x.shape
        st, sh, sd = x.stride()
        if h == cache.heads and d == cache.dim and sd == 1:
            if not x.is_cuda:
                raise RuntimeError(f"{name}: {what} must be on a GPU (no CPU path)")
            return t, st if t > 1 else 0, sh if h > 1 else 0
    raise RuntimeError(f"{name}: {what} must be [rows, {cache.heads}, {cache.dim}] with a contiguous last dim, got {tuple(x.shape)}")


def _rows_call(name, entry, what, cache, k, v, table, lens, cu):
    t, k_st, k_sh = _rows(name, what[0], k, cache)
    tv, v_st, v_sh = _rows(name, what[1], v, cache)
    dt, gpu = _ROW.get(k.dtype), k.get_device()
    if tv != t or v.dtype != k.dtype or dt is None or v.get_device() != gpu:
        raise TypeError(f"{name}: {what[0]} and {what[1]} must be of one shape, device and type (bf16, fp16 or fp32)")
    seqs = _seqs(name, cache, table, lens, cu, gpu)
    with _on(gpu):
        nat.call(entry, cache._ref, k.data_ptr(), k_st, k_sh, v.data_ptr(), v_st, v_sh, dt, t, *seqs, _stream(gpu))


def kv_write(cache, k, v, table, lens, cu=None):
    """Quantise rows k, v [rows, heads, dim] (bf16, fp16 or fp32, strided ok) into their positions. Rows at a negative
    position, past the table or in an absent page are skipped; a row that holds an infinity or a NaN is kept as NaN (its scale).
    A position that two rows of a call name (a page that sequences share, or that a table names twice) ends with a mixture of
    them."""
    _rows_call("kv_write", "rh3_kv_write", ("k", "v"), cache, k, v, table, lens, cu)


def kv_read(cache, table, lens, cu=None, rows=None, dtype=torch.bfloat16, out=None):
    """The values (code * scale, rounded once to dtype) of the last cu[b + 1] - cu[b] positions of each sequence, packed as
    kv_write takes them: k, v [rows, heads, dim]. rows: how many in all (cu[B], which only the GPU knows and has to be given
    with cu; without cu by default one of each sequence). Positions that hold nothing read as 0. out: a pair of tensors to write into."""
    if out is None:
        if rows is None and cu is not None:
            raise ValueError("kv_read: with cu, rows (cu[B], how many in all) or out must be given")
        n = table.shape[0] if rows is None else int(rows)
        if dtype not in _ROW:
            raise TypeError(f"kv_read: bf16, fp16 or fp32 values, got {dtype}")
        alloc = torch.empty if cu is None else torch.zeros      # rows that no sequence has are not written
        out = alloc((2, n, cache.heads, cache.dim), dtype=dtype, device=cache.device).unbind(0)
    k, v = out
    _rows_call("kv_read", "rh3_kv_read", ("out[0]", "out[1]"), cache, k, v, table, lens, cu)
    return k, v


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(gpu, *sizes):
    """Of a call on this GPU, which is the current one: the number of its CUs counts."""
    return nat.lib().rh3_kv_attention_workspace_bytes(*sizes)


def _attention(name, q, cache, prefix, prefix_len, table, lens, cu, causal, scale, out, lse, form):
    f = _FORM.get(form)
    if f is None:
        raise ValueError(f"{name}: form {form!r} (None, 'token' or 'chunk')")
    if q.ndim != 3 or q.shape[2] != cache.dim or q.stride(2) != 1 or q.shape[1] % cache.heads or not q.shape[1]:
        raise RuntimeError(f"{name}: q must be [rows, a multiple of {cache.heads} heads, {cache.dim}] with a contiguous last dim, got "
                           f"{tuple(q.shape)}")
    dt = _ROW.get(q.dtype)
    if dt is None or dt == nat.RH3_DTYPE_F32:
        raise TypeError(f"{name}: q must be bf16 or fp16, got {q.dtype}")
    if not q.is_cuda:
        raise RuntimeError(f"{name}: q must be on a GPU (no CPU path)")
    gpu, dev = q.get_device(), cache.device
    t, hq, d = q.shape
    q_st, q_sh, _ = q.stride()
    seqs = _seqs(name, cache, table, lens, cu, gpu)
    alloc = torch.empty if cu is None else torch.zeros          # rows that no sequence has are not written
    if out is None:
        out = alloc((t, hq, d), dtype=q.dtype, device=dev)
        o_st, o_sh = hq * d, d
    else:
        if out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1 or out.get_device() != gpu:
            raise RuntimeError(f"{name}: out must be like q, with a contiguous last dim")
        o_st, o_sh, _ = out.stride()
    if t == 1:
        q_st = o_st = 0
    if hq == 1:
        q_sh = o_sh = 0
    sums = alloc((t, hq), dtype=torch.float32, device=dev) if lse else None
    with _on(gpu):
        n = _workspace_bytes(gpu, hq, cache.heads, d, t, seqs[2] * cache.page, seqs[5], cu is None, prefix_len, f)
        ws = torch.empty(n, dtype=torch.uint8, device=dev)
        nat.call("rh3_kv_attention", cache._ref, q.data_ptr(), q_st, q_sh, hq, dt, t, *seqs, causal, d ** -0.5 if scale is None else scale,
                 out.data_ptr(), o_st, o_sh, None if sums is None else sums.data_ptr(), None if prefix is None else prefix.data_ptr(),
                 prefix_len, f, ws.data_ptr(), n, _stream(gpu))
    return (out, sums) if lse else out


def kv_attention(q, cache, table, lens, cu=None, causal=True, scale=None, out=None, lse=False, form=None):
    """Attention of q [rows, q heads, dim] (bf16 or fp16, strided ok) over the cached positions of each row's sequence ->
    out like q; query head h reads K/V head h // (q heads // heads). causal: row i of n sees positions up to
    lens[b] - n + i. scale: dim ** -0.5 by default. lse=True: also the log-sum-exp [rows, q heads] fp32 of the scaled scores.
    A row that sees no key gives 0 and -inf. form: "token" or "chunk", the kernel for few or for many query rows to a K/V head;
    by default the sizes decide, with the table's width in the place of the lengths, which only the GPU knows."""
    return _attention("kv_attention", q, cache, None, 0, table, lens, cu, causal, scale, out, lse, form)


def kv_attention_shared(q, cache, prefix, prefix_len, table, lens, cu=None, causal=True, scale=None, out=None, lse=False,
                        form=None):
    """kv_attention of a batch whose sequences all begin with the first prefix_len (an int) positions of the pages `prefix`
    (int32 [pages]): every row sees them, then its sequence's own positions (table, lens: without the prefix). The prefix is
    read once for the whole batch."""
    prefix_len = int(prefix_len)
    if prefix.ndim != 1 or prefix.dtype != torch.int32 or not prefix.is_contiguous() or prefix.get_device() != q.get_device():
        raise RuntimeError("kv_attention_shared: prefix must be contiguous int32 [pages] on q's GPU")
    if not 0 <= prefix_len <= prefix.numel() * cache.page:
        raise RuntimeError(f"kv_attention_shared: prefix_len {prefix_len} does not fit {prefix.numel()} pages of {cache.page}")
    return _attention("kv_attention_shared", q, cache, prefix, prefix_len, table, lens, cu, causal, scale, out, lse, form)
