"""Position rotations of queries and keys, and their RMS norm for each head in the same pass (librh3: rh3_qk_norm_rope), for rows at
any positions: heads of 64 or 128 channels, as many query heads as there are, rotated whole or in part. With the write into a
key / value cache in the same pass: kvcache.kv_write_rope. A row has one position. (attention.rms_rope_ is the DiT block's form: a table
of bf16 coefficients for tokens 0 .. S, which may turn by positions on several axes, the norm's result rounded in between.)

Of a row x of a head: y = (x * r) * w with r = 1 / sqrt(mean x^2 + eps), made in 64 bits and rounded to fp32 once; then pairs (a, b) of
the first rot channels become (a cos - b sin, b cos + a sin) in fp32, with the cosine and sine of position * freq[i] (a product in
64 bits, so far positions keep their angle) times `factor`, each rounded to fp32 once; one rounding to the rows' type at the end.
"""
import math
import struct

import torch

from . import _native as nat
from ._rows import _ROW, _on, _stream

LAYOUTS = ("half", "interleaved")
_TURN = "3qdqd3q"                                # rh3_turn
_ARGS = struct.Struct("=18q" + _TURN)            # rh3_rope_args


class Rotary:
    """What turns a head: freq [rot / 2] fp64 on the rows' GPU, radians to a position; layout "half" pairs channels i and i + rot / 2,
    "interleaved" 2 i and 2 i + 1; factor multiplies the cosines and sines. rot, twice freq's length, is a multiple of 16 and at most
    the head's dim; channels from rot on keep their place. The tensor is kept and used as it is; the attributes cannot be changed."""

    __slots__ = ("freq", "layout", "factor", "rot", "gpu", "_args")

    def __init__(self, freq, layout="half", factor=1.0):
        if freq.ndim != 1 or freq.dtype != torch.float64 or (freq.shape[0] > 1 and freq.stride(0) != 1):
            raise RuntimeError(f"Rotary: freq must be contiguous fp64 [rot / 2], got {freq.dtype} {tuple(freq.shape)}")
        if freq.shape[0] % 8 or not 8 <= freq.shape[0] <= 64:
            raise RuntimeError(f"Rotary: 8 to 64 frequencies, a multiple of 8, got {freq.shape[0]}")
        if layout not in LAYOUTS:
            raise ValueError(f"Rotary: layout {layout!r} ('half' or 'interleaved')")
        if not freq.is_cuda:
            raise RuntimeError("Rotary: freq must be on a GPU (no CPU path)")
        self.freq, self.layout, self.factor, self.rot, self.gpu = freq, layout, float(factor), 2 * freq.shape[0], freq.get_device()
        self._args = (freq.data_ptr(), self.rot, layout == "interleaved", self.factor)

    def __setattr__(self, name, value):
        if hasattr(self, "_args"):
            raise AttributeError(f"Rotary: {name} cannot be changed; make a new Rotary")
        object.__setattr__(self, name, value)


def frequencies(rot, base=10000.0, scaling=None, stretch=1.0, original=None, low=1.0, high=32.0):
    """freq [rot / 2] fp64 (on the CPU) and factor for Rotary: base ** (-2 i / rot), stretched for contexts `stretch` times as long as
    trained:
      None      as they are
      "linear"  all divided by stretch (positions squeezed together)
      "base"    base * stretch ** (rot / (rot - 2)): the lowest frequency is divided by stretch, the highest stays
      "parts"   by how often a frequency turns within the original length: over `high` times it stays, under `low` it is divided by
                stretch, a straight line in between; factor 0.1 ln(stretch) + 1. (The line is over the number of turns. Models that draw
                it over the channel's number, or have another factor or none, give Rotary their own frequencies and factor.)"""
    if rot < 4 or rot % 2:
        raise ValueError(f"frequencies: rot {rot} (an even number from 4 on)")
    if scaling not in (None, "linear", "base", "parts"):
        raise ValueError(f"frequencies: scaling {scaling!r} (None, 'linear', 'base' or 'parts')")
    if scaling == "parts" and (original is None or not low < high):
        raise ValueError("frequencies: 'parts' needs the original length, and low < high")
    if not stretch >= 1.0:
        raise ValueError(f"frequencies: stretch {stretch} (1 or more)")
    if scaling == "base":
        base = base * stretch ** (rot / (rot - 2))
    freq = float(base) ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if scaling == "linear":
        freq = freq / stretch
    if scaling != "parts":
        return freq, 1.0
    keep = ((original * freq / (2.0 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
    return freq * keep + freq / stretch * (1.0 - keep), 0.1 * math.log(stretch) + 1.0


def rotary(rot, layout="half", device="cuda", **how):
    """A Rotary of frequencies(rot, **how)."""
    freq, factor = frequencies(rot, **how)
    return Rotary(freq.to(device), layout, factor)


def _turn(name, rotary, q_weight, k_weight, eps, dim, dtype, gpu):
    """rh3_turn of a Rotary and a norm: freq, rot, interleaved, factor, norm, eps, the weights, their width."""
    if eps is None:
        if rotary is None:
            raise ValueError(f"{name}: neither a rotary nor eps: nothing to do")
        if q_weight is not None or k_weight is not None:
            raise ValueError(f"{name}: weights without eps (eps=None is no norm)")
    if rotary is not None and (rotary.gpu != gpu or rotary.rot > dim):
        raise RuntimeError(f"{name}: rotary must be on the rows' GPU and turn at most {dim} channels, got {rotary.rot}")
    wide, at = None, [0, 0]
    for i, w in enumerate((q_weight, k_weight)):
        if w is not None:
            t = w.dtype
            if w.shape != (dim,) or (t != dtype and t != torch.float32) or not w.is_contiguous() or w.get_device() != gpu:
                raise RuntimeError(f"{name}: norm weights must be contiguous [{dim}] of the rows' type or fp32, on their GPU")
            if wide is not None and wide != (t == torch.float32):
                raise RuntimeError(f"{name}: the norm weights must be of one type")
            wide, at[i] = t == torch.float32, w.data_ptr()
    freq, rot, interleaved, factor = (0, 0, False, 1.0) if rotary is None else rotary._args
    return freq, rot, interleaved, factor, eps is not None, 0.0 if eps is None else eps, at[0], at[1], bool(wide)


def _rows_of(name, what, x):
    """rh3_head_rows of rows [rows, heads, dim] (strides 0 for axes of length 1), and their sizes."""
    if x.ndim != 3 or x.dtype not in _ROW or not x.is_cuda:
        raise RuntimeError(f"{name}: {what} must be [rows, heads, 64 or 128] bf16, fp16 or fp32 on a GPU (no CPU path), got {x.dtype} "
                           f"{tuple(x.shape)}")
    t, h, d = x.shape
    st, sh, sd = x.stride()
    if sd != 1 or (d != 128 and d != 64):
        raise RuntimeError(f"{name}: {what} must be [rows, heads, 64 or 128] with a contiguous last dim, got {(t, h, d)}")
    return (x.data_ptr(), st if t > 1 else 0, sh if h > 1 else 0), t, h, d


def _result(name, what, x, t, h, d, out):
    """A new result like rows x, or `out`, checked; and its rh3_head_rows."""
    if out is None:
        out = torch.empty_strided((t, h, d), (h * d, d, 1), dtype=x.dtype, device=x.device)
        return out, (out.data_ptr(), h * d, d)
    rows, to, ho, do = _rows_of(name, f"out for {what}", out)
    if (to, ho, do) != (t, h, d) or out.dtype != x.dtype or out.get_device() != x.get_device():
        raise RuntimeError(f"{name}: out for {what} must be like it")
    return out, rows


def qk_norm_rope(q, k, positions, rotary, q_weight=None, k_weight=None, eps=None, out=None):
    """The norm (eps: a number; None: no norm) and rotation (None: no rotation) of q [rows, q heads, dim] and k [rows, k heads, dim]
    (bf16, fp16 or fp32, strided ok; k may be None) at positions [rows] int32 -> new tensors like them, or `out`, a pair. out may lie
    exactly over q and k."""
    name = "qk_norm_rope"
    qr, t, hq, dim = _rows_of(name, "q", q)
    dtype, gpu = q.dtype, q.get_device()
    at = 0
    if rotary is not None:
        if positions.dtype != torch.int32 or positions.shape != (t,) or not positions.is_contiguous() or positions.get_device() != gpu:
            raise RuntimeError(f"{name}: positions must be contiguous int32 [{t}] on the rows' GPU")
        at = positions.data_ptr()
    turn = _turn(name, rotary, q_weight, k_weight, eps, dim, dtype, gpu)
    qo, ko = (None, None) if out is None else out
    qo, qor = _result(name, "q", q, t, hq, dim, qo)
    kr = kor = (0, 0, 0)
    hk = 0
    if k is not None:
        kr, tk, hk, dk = _rows_of(name, "k", k)
        if tk != t or dk != dim or k.dtype != dtype or k.get_device() != gpu:
            raise RuntimeError(f"{name}: k must be of q's rows, dim, type and GPU")
        ko, kor = _result(name, "k", k, t, hk, dim, ko)
    args = _ARGS.pack(*qr, *qor, *kr, *kor, hq, hk, t, dim, _ROW[dtype], at, *turn)
    with _on(gpu):
        nat.call("rh3_qk_norm_rope", args, _stream(gpu))
    return qo, ko if k is not None else None
