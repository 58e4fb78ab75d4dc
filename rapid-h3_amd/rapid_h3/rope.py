"""Position rotations of queries and keys, and their RMS norm for each head in the same pass (librh3: rh3_qk_norm_rope), for rows at
any positions: heads of 64 or 128 channels, as many query heads as there are, rotated whole or in part. With the write into a
key / value cache in the same pass: kvcache.kv_write_rope. (attention.rms_rope_ is the DiT block's form: a table of bf16 coefficients
for tokens 0 .. S, the norm's result rounded in between.)

Of a row x of a head: y = (x * r) * w with r = 1 / sqrt(mean x^2 + eps), made in 64 bits and rounded to fp32 once; then pairs (a, b) of
the first rot channels become (a cos - b sin, b cos + a sin) in fp32, with the cosine and sine of position * freq[i] (a product in
64 bits, so far positions keep their angle) times `factor`, each rounded to fp32 once; one rounding to the rows' type at the end.
"""
import math

import torch

from . import _native as nat
from ._rows import _ROW, _on, _stream

LAYOUTS = ("half", "interleaved")


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
                stretch, a straight line in between; factor 0.1 ln(stretch) + 1"""
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
    """The entry points' arguments for a Rotary and a norm: freq, rot, interleaved, factor, norm, eps, the weights, their width."""
    if rotary is not None and (rotary.gpu != gpu or rotary.rot > dim):
        raise RuntimeError(f"{name}: rotary must be on the rows' GPU and turn at most {dim} channels, got {rotary.rot}")
    wide = None
    for w in (q_weight, k_weight):
        if w is None:
            continue
        if eps is None:
            raise ValueError(f"{name}: weights without eps (eps=None is no norm)")
        if w.shape != (dim,) or w.dtype not in (dtype, torch.float32) or w.stride(0) != 1 or w.get_device() != gpu:
            raise RuntimeError(f"{name}: norm weights must be contiguous [{dim}] of the rows' type or fp32, on their GPU")
        if wide is not None and wide != (w.dtype == torch.float32):
            raise RuntimeError(f"{name}: the norm weights must be of one type")
        wide = w.dtype == torch.float32
    if rotary is None and eps is None:
        raise ValueError(f"{name}: neither a rotary nor eps: nothing to do")
    return (*(rotary._args if rotary is not None else (None, 0, False, 1.0)), eps is not None, 0.0 if eps is None else float(eps),
            nat.ptr(q_weight), nat.ptr(k_weight), bool(wide))


def _heads(name, what, x, like=None):
    """Strides of rows [rows, heads, dim]; 0 for an axis of length 1."""
    if x.ndim != 3 or x.shape[2] not in (64, 128) or x.stride(2) != 1 or x.dtype not in _ROW:
        raise RuntimeError(f"{name}: {what} must be [rows, heads, 64 or 128] bf16, fp16 or fp32 with a contiguous last dim, got {x.dtype} "
                           f"{tuple(x.shape)}")
    if like is not None and (x.shape[0] != like.shape[0] or x.shape[2] != like.shape[2] or x.dtype != like.dtype or x.get_device() != like.get_device()):
        raise RuntimeError(f"{name}: {what} must be of q's rows, dim, type and GPU")
    if not x.is_cuda:
        raise RuntimeError(f"{name}: {what} must be on a GPU (no CPU path)")
    st, sh, _ = x.stride()
    return st if x.shape[0] > 1 else 0, sh if x.shape[1] > 1 else 0


def _result(name, what, x, out):
    if out is None:
        return torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if out.shape != x.shape or out.dtype != x.dtype or out.stride(2) != 1 or out.get_device() != x.get_device():
        raise RuntimeError(f"{name}: out for {what} must be like it, with a contiguous last dim")
    return out


def qk_norm_rope(q, k, positions, rotary, q_weight=None, k_weight=None, eps=None, out=None):
    """The norm (eps: a number; None: no norm) and rotation (None: no rotation) of q [rows, q heads, dim] and k [rows, k heads, dim]
    (bf16, fp16 or fp32, strided ok; k may be None) at positions [rows] int32 -> new tensors like them, or `out`, a pair. out may lie
    exactly over q and k."""
    name = "qk_norm_rope"
    q_st, q_sh = _heads(name, "q", q)
    gpu = q.get_device()
    t, hq, dim = q.shape
    turn = _turn(name, rotary, q_weight, k_weight, eps, dim, q.dtype, gpu)
    if rotary is not None and (positions.dtype != torch.int32 or positions.shape != (t,) or not positions.is_contiguous() or positions.get_device() != gpu):
        raise RuntimeError(f"{name}: positions must be contiguous int32 [{t}] on the rows' GPU")
    qo, ko = (None, None) if out is None else out
    qo = _result(name, "q", q, qo)
    keys = (None, 0, 0, None, 0, 0, 0)
    if k is not None:
        k_st, k_sh = _heads(name, "k", k, q)
        ko = _result(name, "k", k, ko)
        keys = (k.data_ptr(), k_st, k_sh, ko.data_ptr(), *_heads(name, "out for k", ko), k.shape[1])
    with _on(gpu):
        nat.call("rh3_qk_norm_rope", q.data_ptr(), q_st, q_sh, qo.data_ptr(), *_heads(name, "out for q", qo), hq, *keys, t, dim, _ROW[q.dtype],
                 None if rotary is None else positions.data_ptr(), *turn, _stream(gpu))
    return qo, ko if k is not None else None
