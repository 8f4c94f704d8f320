"""Rotary position embedding: half and interleaved layouts, part of the head, scalings for long contexts.

The reference rotates whole heads in the half layout from cosine and sine rows that the caller gathers
(``rotary_emb_fwd``, ``slora/models/llama/triton_kernel/rotary_emb.py:8-71``); ``LoraBatchOps.lora_get_qkv(rope=(cos,
sin))`` does the same in the expand's epilogue.  Here a :class:`RotaryTable` holds the frequencies, the kernel takes
positions, and angles are reduced in 64 bits, so positions far out keep their angle.
"""
from __future__ import annotations

import math

import torch

from . import _lib

LAYOUTS = {"half": 0, "interleaved": 1}


def _frequencies(dim, base, scaling):
    """Radians per position of each of the ``dim / 2`` pairs, and the factor on cosines and sines."""
    freq = [base ** (-2.0 * i / dim) for i in range(dim // 2)]
    if scaling is None:
        return freq, 1.0
    kind = scaling.get("type", scaling.get("rope_type"))
    known = {"linear": {"factor"}, "ntk": {"factor"},
             "yarn": {"factor", "original_max_position", "beta_fast", "beta_slow", "attention_factor"},
             "llama3": {"factor", "low_freq_factor", "high_freq_factor", "original_max_position"}}
    if kind not in known:
        raise RuntimeError(f"rotary scaling {kind!r} is none of {sorted(known)}")
    extra = set(scaling) - known[kind] - {"type", "rope_type"}
    if extra:
        raise RuntimeError(f"rotary scaling {kind!r} does not take {sorted(extra)}")
    try:
        factor = float(scaling["factor"])
        if not factor >= 1.0 or math.isinf(factor):
            raise RuntimeError(f"rotary scaling factor {factor} must be at least 1")
        if kind == "linear":                     # positions shrunk
            return [f / factor for f in freq], 1.0
        if kind == "ntk":                        # the base grown so that the slowest pair is shrunk by the factor
            if dim <= 2:
                raise RuntimeError("ntk scaling needs more than one pair")
            wide = base * factor ** (dim / (dim - 2.0))
            return [wide ** (-2.0 * i / dim) for i in range(dim // 2)], 1.0
        span = float(scaling["original_max_position"])
        if not span >= 1.0:
            raise RuntimeError(f"original_max_position {span} must be at least 1")
        if kind == "yarn":
            # pairs that turn more than beta_fast times within the original span stay, those below beta_slow shrink, a ramp
            # over the pair's index between; the factor makes up for the flatter softmax of longer contexts
            fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))

            def pair(turns):
                return dim * math.log(span / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

            low, high = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), dim - 1)
            out = []
            for i, f in enumerate(freq):
                ramp = min(1.0, max(0.0, (i - low) / max(high - low, 0.001)))
                out.append(f / factor * ramp + f * (1.0 - ramp))
            return out, float(scaling.get("attention_factor", 0.1 * math.log(factor) + 1.0))
        # llama3: by wavelength: long ones shrink, short ones stay, smoothly between
        low, high = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        if not 0.0 < low < high:
            raise RuntimeError("llama3 scaling needs 0 < low_freq_factor < high_freq_factor")
        out = []
        for f in freq:
            wave = 2.0 * math.pi / f
            if wave > span / low:
                out.append(f / factor)
            elif wave < span / high:
                out.append(f)
            else:
                smooth = (span / wave - low) / (high - low)
                out.append((1.0 - smooth) * f / factor + smooth * f)
        return out, 1.0
    except KeyError as e:
        raise RuntimeError(f"rotary scaling {kind!r} needs {e.args[0]!r}") from None


class RotaryTable:
    """Frequencies of a model's rotary embedding, made once per model.

    ``rotary_dim`` (default: the whole head; a multiple of 16) is the part of each head that turns, its first elements;
    ``layout`` pairs element ``i`` with ``i + rotary_dim / 2`` (``"half"``) or ``2i`` with ``2i + 1`` (``"interleaved"``).
    ``scaling``: ``None`` or a dict with a ``"type"``:

    * ``{"type": "linear", "factor"}``
    * ``{"type": "ntk", "factor"}``
    * ``{"type": "yarn", "factor", "original_max_position"[, "beta_fast", "beta_slow", "attention_factor"]}``
    * ``{"type": "llama3", "factor", "low_freq_factor", "high_freq_factor", "original_max_position"}``
    """

    def __init__(self, head_dim, rotary_dim=None, base=10000.0, layout="half", scaling=None, device="cuda"):
        rotary_dim = head_dim if rotary_dim is None else int(rotary_dim)
        if head_dim not in (64, 128, 256):
            raise RuntimeError(f"No suitable kernel. head_dim={head_dim} (64, 128 or 256)")
        if rotary_dim % 16 or not 16 <= rotary_dim <= head_dim:
            raise RuntimeError(f"No suitable kernel. rotary_dim={rotary_dim} (a multiple of 16 up to head_dim={head_dim})")
        if layout not in LAYOUTS:
            raise RuntimeError(f"rotary layout {layout!r} is none of {sorted(LAYOUTS)}")
        if not base > 1.0:
            raise RuntimeError(f"rotary base {base} must be above 1")
        self.head_dim, self.rotary_dim, self.layout = int(head_dim), rotary_dim, layout
        self.inv_freq, self.factor = _frequencies(rotary_dim, float(base), scaling)
        # turns per position: the kernel reduces whole turns away before it goes to 32 bits
        self.turns = torch.tensor([f / (2.0 * math.pi) for f in self.inv_freq], dtype=torch.float64, device=device)
        self.turns_ptr, self.layout_code = self.turns.data_ptr(), LAYOUTS[layout]


def _rows(t, name, head_dim):
    """Shape of ``t`` ``[tokens, heads, head_dim]``, its heads contiguous, and the stride of its tokens."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 3 or shape[2] != head_dim or stride[2] != 1 or (shape[1] > 1 and stride[1] != head_dim):
        raise RuntimeError(f"{name} must be [tokens, heads, {head_dim}] with contiguous heads")
    return shape, stride[0]


def _positions(positions, tokens):
    if positions.dtype != torch.int64 or positions.shape != (tokens,) or not positions.is_contiguous():
        raise RuntimeError("positions must be a contiguous int64 tensor with one entry per token")
    return positions


def rotary(table, positions, q, k=None, q_out=None, k_out=None, inverse=False):
    """Turn ``q`` ``[T, heads, head_dim]`` (and ``k``) by their tokens' positions (int64 ``[T]``).

    In place unless ``q_out`` / ``k_out`` are given; returns ``(q_out, k_out)``.  ``inverse=True`` turns back (the
    gradient's direction).  C entry ``slora_rotary``.
    """
    out, call = _rotary_call(table, positions, q, k, q_out, k_out, inverse)
    _lib.call(*call)
    return out


def _rotary_call(table, positions, q, k=None, q_out=None, k_out=None, inverse=False):
    """The checks of :func:`rotary`, and what is left to do as the arguments of ``_lib.call``."""
    ctx = _lib.device_of(q, positions, table.turns, k, q_out, k_out)
    d, dtype = table.head_dim, q.dtype
    shape, q_stride = _rows(q, "q", d)
    if q_out is None:
        q_out, qo_stride = q, q_stride
    else:
        out_shape, qo_stride = _rows(q_out, "q_out", d)
        if out_shape != shape or q_out.dtype != dtype:
            raise RuntimeError("q_out must have q's shape and dtype")
    _positions(positions, shape[0])
    k_heads = k_stride = ko_stride = kp = kop = 0
    if k is not None:
        k_shape, k_stride = _rows(k, "k", d)
        if k_out is None:
            k_out, ko_stride = k, k_stride
        else:
            out_shape, ko_stride = _rows(k_out, "k_out", d)
            if out_shape != k_shape or k_out.dtype != dtype:
                raise RuntimeError("k_out must have k's shape and dtype")
        if k_shape[0] != shape[0] or k.dtype != dtype:
            raise RuntimeError("k must have q's tokens and dtype")
        k_heads, kp, kop = k_shape[1], k.data_ptr(), k_out.data_ptr()
    elif k_out is not None:
        raise RuntimeError("k_out without k")
    return (q_out, k_out), (ctx, _lib.lib.slora_rotary, q_out.data_ptr(), kop, q.data_ptr(), kp, shape[0], shape[1], k_heads, d,
                            table.rotary_dim, qo_stride, ko_stride, q_stride, k_stride, positions.data_ptr(), table.turns_ptr,
                            table.factor, table.layout_code, int(inverse), _lib.dtype_code(dtype))
