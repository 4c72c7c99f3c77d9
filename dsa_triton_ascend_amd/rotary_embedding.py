"""Rotary positions on MI355X: what produces ``query_rope`` / ``key_rope`` of
the attention operators and rotates the indexer's queries and keys.

``rotary_embedding`` turns a slice of every head of a query and, in the same
launch, of a key; ``rotary_frequencies`` gives its frequencies, plain or
scaled for contexts longer than the trained one.  The reference has no such
operator: it takes rotated inputs.

Angles ``position * inv_freq`` are formed in 64 bits inside the kernel, so
positions up to 2^31 are exact to fp32 and no table is kept.
"""
import math

import torch
from torch.autograd.forward_ad import unpack_dual

from . import _lib

SCALINGS = ("none", "linear", "ntk", "yarn")


def rotary_frequencies(dim, base=10000.0, scaling="none", factor=1.0, original_max_position=4096, beta_fast=32.0,
                       beta_slow=1.0, mscale=1.0, mscale_all_dim=0.0, device=None):
    """Inverse frequencies of ``dim`` rotary columns and the scale of their
    outputs: ``(inv_freq, attention_scale)``, a float64 tensor of ``dim / 2``
    values on ``device`` (default: the current GPU) and a float.

    scaling ``"none"``: ``base ** (-2i / dim)``.  ``"linear"``: those divided
    by ``factor`` (positions interpolated).  ``"ntk"``: the base multiplied by
    ``factor ** (dim / (dim - 2))``, which divides the lowest frequency by
    ``factor`` and keeps the highest.  ``"yarn"``: columns that turn more than
    ``beta_fast`` times within ``original_max_position`` keep their frequency,
    those that turn less than ``beta_slow`` times get the interpolated one, a
    linear ramp over the columns between; attention_scale is
    ``m(mscale) / m(mscale_all_dim)`` with ``m(x) = 0.1 x ln(factor) + 1``
    (1 for a factor up to 1).  It is 1.0 for every other scaling.
    """
    if int(dim) != dim or dim < 2 or dim % 2:
        raise ValueError(f"dim must be even and at least 2, got {dim}")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}, got {scaling}")
    if not (base > 0 and factor > 0 and original_max_position > 0):
        raise ValueError("base, factor and original_max_position must be positive")
    dim, base, factor = int(dim), float(base), float(factor)
    half = dim // 2
    scale = 1.0
    if scaling == "ntk" and factor != 1.0:
        if dim == 2:
            raise ValueError("ntk scaling needs at least 4 columns")
        base *= factor ** (dim / (dim - 2))
    freq = [base ** (-2.0 * i / dim) for i in range(half)]
    if scaling == "linear":
        freq = [f / factor for f in freq]
    elif scaling == "yarn":
        if not (beta_fast > beta_slow > 0):
            raise ValueError("yarn scaling needs beta_fast > beta_slow > 0")
        if base == 1.0:
            raise ValueError("yarn scaling needs a base other than 1")

        def column(turns):  # column pair that makes this many turns within the original context
            return dim * math.log(original_max_position / (turns * 2 * math.pi)) / (2 * math.log(base))

        low = max(math.floor(column(beta_fast)), 0)
        high = min(math.ceil(column(beta_slow)), dim - 1)
        for i in range(half):
            ramp = min(1.0, max(0.0, (i - low) / max(high - low, 0.001)))
            freq[i] = freq[i] / factor * ramp + freq[i] * (1.0 - ramp)

        def m(x):
            return 0.1 * x * math.log(factor) + 1.0 if factor > 1.0 else 1.0

        scale = m(mscale) / m(mscale_all_dim)
    if device is None:
        device = torch.device("cuda", torch.cuda.current_device())
    return torch.tensor(freq, dtype=torch.float64, device=device), scale


_RANK = {"BSND": 4, "TND": 3}
_DTYPE = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16, torch.float32: _lib.DTYPE_FP32}


def _overlaps_itself(t):
    """Whether two elements of a strided tensor may share an address."""
    reach = 0
    for n, s in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n > 1), key=lambda x: x[1]):
        if s <= reach:
            return True
        reach += (n - 1) * s
    return False


def _share_memory(a, a_start, b, b_start, cols):
    """Whether the columns a_start .. a_start + cols of a's heads and b_start ..
    of b's share memory (both checked by ``_overlaps_itself``)."""
    size = a.element_size()
    counts = {}  # how often each stride may be taken
    for n, s in zip(a.shape[:-1], a.stride()):
        lo, hi = counts.get(s * size, (0, 0))
        counts[s * size] = lo - (n - 1), hi
    for n, s in zip(b.shape[:-1], b.stride()):
        lo, hi = counts.get(s * size, (0, 0))
        counts[s * size] = lo, hi + (n - 1)
    steps = sorted(((s, lo, hi) for s, (lo, hi) in counts.items() if lo != hi), reverse=True)
    budget = 1000  # descending strides leave each a few counts; if not, the answer is yes

    def reaches(k, first, last):
        nonlocal budget
        if k == len(steps):
            return first <= 0 <= last
        s, lo, hi = steps[k]
        least, most = (sum(x[0] * x[i] for x in steps[k + 1:]) for i in (1, 2))
        for x in range(max(lo, -((most - first) // s)), min(hi, (last - least) // s) + 1):
            budget -= 1
            if budget < 0 or reaches(k + 1, first - x * s, last - x * s):
                return True
        return False

    apart = b.data_ptr() + b_start * size - a.data_ptr() - a_start * size
    return reaches(0, -apart - cols * size + 1, -apart + cols * size - 1)


def _side(t, start, inplace):
    """Output and C arguments of one rotated tensor [(B,) S, N, D]."""
    if t._is_zerotensor():  # (a gradient without memory)
        t = torch.zeros(t.shape, dtype=t.dtype, device=t.device)
    st = t.stride()
    if st[-1] != 1 and t.shape[-1] != 1:  # columns apart
        t = t.contiguous()
        st = t.stride()
    shape = t.shape
    out = t if inplace else torch.empty(shape, dtype=t.dtype, device=t.device)
    so = out.stride()
    if len(shape) == 4:
        return t, out, (t.data_ptr(), out.data_ptr(), st[0], st[1], st[2], so[0], so[1], so[2], shape[2], shape[3], start)
    return t, out, (t.data_ptr(), out.data_ptr(), 0, st[0], st[1], 0, so[0], so[1], shape[1], shape[2], start)


_NO_KEY = (None, None) + (0,) * 9


def _rotate(query, key, positions, inv_freq, interleaved, q_start, k_start, scale, inverse, inplace):
    """Launch on checked arguments; returns the rotated query and key."""
    result = _lib.calls().rotate(query, key, positions, inv_freq, interleaved, q_start, k_start, scale,
                                 "BSND" if query.dim() == 4 else "TND", inverse, inplace)
    if result is not None:
        return result
    query, q_out, q_args = _side(query, q_start, inplace)
    k_out, k_args = None, _NO_KEY
    if key is not None:
        key, k_out, k_args = _side(key, k_start, inplace)
    shape = query.shape
    b, s = (shape[0], shape[1]) if len(shape) == 4 else (1, shape[0])
    if b == 0 or s == 0:
        return q_out, k_out
    index = query.get_device()
    status = _lib.call_on(
        index, _lib.load().dsa_rope, *q_args, *k_args, positions.data_ptr(), positions.dtype == torch.int64,
        len(shape) == 3 or positions.dim() == 2, inv_freq.data_ptr(), b, s, 2 * inv_freq.shape[0], interleaved, inverse,
        _DTYPE[query.dtype], scale, _lib.raw_stream(index))
    if status:
        _lib.check(status, "dsa_rope")
    if inplace:
        _lib.changed(*(t for t in (q_out, k_out) if t is not None))
    return q_out, k_out


def rotary_embedding(query, key=None, positions=None, inv_freq=None, interleaved=False, rotary_offset=0,
                     key_rotary_offset=None, attention_scale=1.0, layout="BSND", inverse=False, inplace=False):
    """Rotary positions of ``query`` and, if given, ``key``.

    query [B, S, N, D] (layout "BSND") or [T, N, D] ("TND"), bfloat16, float16
    or float32; key of the same batch and tokens with its own heads and
    columns.  ``positions``: int32 or int64, [B, S], [S] (the same for every
    sequence) or [T].  ``inv_freq`` (``rotary_frequencies``): R / 2 values;
    the R columns from ``rotary_offset`` (for the key ``key_rotary_offset``,
    by default the same) are rotated, the others come through unchanged.
    Pairs are columns (2i, 2i + 1) if ``interleaved``, else (i, i + R / 2).
    Rotated columns are multiplied by ``attention_scale``.  ``inverse`` rotates
    by the opposite angles.

    Returns ``(query_out, key_out)`` (key_out is None without a key), new
    contiguous tensors, or with ``inplace`` the inputs themselves (views of one
    projection too, if their rotated columns share no memory).  Strided
    views are read as they are if a head's columns are next to each other.
    Differentiable in query and key, any number of times, in both modes (not
    in place; ``inv_freq`` gets no gradient).
    """
    result = _lib.calls().rotate(query, key, positions, inv_freq, interleaved, rotary_offset, key_rotary_offset,
                                 attention_scale, layout, inverse, inplace)
    if result is not None:
        return result
    rank = _RANK.get(layout)
    if rank is None:
        raise ValueError(f"layout must be BSND or TND, got {layout}")
    if positions is None or inv_freq is None:
        raise ValueError("positions and inv_freq are required")
    shape = query.shape
    if len(shape) != rank:
        raise ValueError(f"query must be {'[T, N, D]' if rank == 3 else '[B, S, N, D]'}, got {tuple(shape)}")
    lead = shape[:rank - 2]
    if query.dtype not in _DTYPE:
        raise ValueError(f"query dtype must be bfloat16, float16 or float32, got {query.dtype}")
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"positions must be int32 or int64, got {positions.dtype}")
    if inv_freq.dim() != 1 or inv_freq.shape[0] < 1:
        raise ValueError(f"inv_freq must be a vector, got {tuple(inv_freq.shape)}")
    rot = 2 * inv_freq.shape[0]
    if positions.shape != lead and positions.shape != lead[-1:]:
        raise ValueError(f"positions must have shape {tuple(lead)}, or {tuple(lead[-1:])} for all sequences, "
                         f"got {tuple(positions.shape)}")
    if key_rotary_offset is None:
        key_rotary_offset = rotary_offset
    if key is not None:
        if key.dim() != rank or key.shape[:rank - 2] != lead:
            raise ValueError(f"key must have the query's batch and tokens, got {tuple(key.shape)}")
        if key.dtype != query.dtype:
            raise ValueError(f"key dtype {key.dtype} differs from query dtype {query.dtype}")
    for name, t, start in (("query", query, rotary_offset), ("key", key, key_rotary_offset)):
        if t is not None and (int(start) != start or not 0 <= start <= t.shape[-1] - rot):
            raise ValueError(f"the {rot} rotary columns from {start} do not lie inside the {t.shape[-1]} of {name}")
    grad = (torch.is_grad_enabled() and (query.requires_grad or (key is not None and key.requires_grad))
            or any(t is not None and unpack_dual(t).tangent is not None for t in (query, key)))
    if inplace:
        if grad:
            raise ValueError("inplace is for inference: the inputs require grad or carry tangents")
        for name, t in (("query", query), ("key", key)):
            if t is not None and ((t.stride(-1) != 1 and t.shape[-1] != 1) or _overlaps_itself(t)):
                raise ValueError(f"inplace needs a {name} whose head columns are next to each other and whose "
                                 "elements do not share memory")
        if key is not None and key.numel() and query.numel() and (
                key.data_ptr() == query.data_ptr()
                or _share_memory(query, rotary_offset, key, key_rotary_offset, rot)):
            raise ValueError("inplace needs a key and a query of their own: they share memory")
    _lib.same_device(query, key, positions, inv_freq)
    if not positions.is_contiguous():
        positions = positions.contiguous()
    if inv_freq.dtype != torch.float64 or not inv_freq.is_contiguous():
        inv_freq = inv_freq.to(torch.float64).contiguous()
    args = (positions, inv_freq, bool(interleaved), int(rotary_offset), int(key_rotary_offset),
            float(attention_scale), bool(inverse))
    if grad:
        from .autograd import RotaryEmbeddingFunction
        return RotaryEmbeddingFunction.apply(query, key, *args)
    return _rotate(query, key, *args, inplace)


class RotaryEmbedding(torch.nn.Module):
    """``rotary_embedding`` with frequencies of its own (a buffer made once by
    ``rotary_frequencies`` on ``device``, moved with the module)."""

    def __init__(self, dim, base=10000.0, scaling="none", factor=1.0, original_max_position=4096, beta_fast=32.0,
                 beta_slow=1.0, mscale=1.0, mscale_all_dim=0.0, interleaved=False, rotary_offset=0,
                 key_rotary_offset=None, layout="BSND", device=None):
        super().__init__()
        inv_freq, self.attention_scale = rotary_frequencies(
            dim, base, scaling, factor, original_max_position, beta_fast, beta_slow, mscale, mscale_all_dim, device)
        self.register_buffer("inv_freq", inv_freq, persistent=False)
        self.interleaved = interleaved
        self.rotary_offset = rotary_offset
        self.key_rotary_offset = key_rotary_offset
        self.layout = layout

    def _apply(self, fn, recurse=True):
        # a cast of the module (half(), bfloat16()) leaves the frequencies in 64 bits
        freq = self.inv_freq
        super()._apply(fn, recurse)
        if self.inv_freq.dtype != torch.float64:
            self.inv_freq = freq.to(self.inv_freq.device)
        return self

    def forward(self, query, key=None, positions=None):
        return rotary_embedding(query, key, positions, self.inv_freq, interleaved=self.interleaved,
                                rotary_offset=self.rotary_offset, key_rotary_offset=self.key_rotary_offset,
                                attention_scale=self.attention_scale, layout=self.layout)

    construct = forward
