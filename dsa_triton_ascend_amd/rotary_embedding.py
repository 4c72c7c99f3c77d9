"""Rotary positions on MI355X: what produces ``query_rope`` / ``key_rope`` of
the attention operators and rotates the indexer's queries and keys.

``rotary_embedding`` turns a slice of every head of a query and, in the same
launch, of a key; ``rotary_frequencies`` gives its frequencies, plain or
scaled for contexts longer than the trained one.  The reference has no such
operator: it takes rotated inputs.

Angles ``position * inv_freq`` are formed in 64 bits inside the kernel, so any
position of an int32 or int64 tensor is exact to fp32 and no table is kept.
"""
import math

import torch

from . import _lib
from .sparse_flash_attention import _check_device, _expect_shape

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


def _heads(t, layout, name):
    """(batch, tokens, heads, columns) of a BSND or TND tensor."""
    if t.dim() != (3 if layout == "TND" else 4):
        raise ValueError(f"{name} must be {'[T, N, D]' if layout == 'TND' else '[B, S, N, D]'}, got {tuple(t.shape)}")
    return (1,) + tuple(t.shape) if layout == "TND" else tuple(t.shape)


def _strides(t):
    """Batch, token and head strides in elements; None if the columns of a
    head are not next to each other."""
    s = t.stride()
    if s[-1] != 1 and t.shape[-1] != 1:
        return None
    return (0,) + s[:2] if t.dim() == 3 else s[:3]


def _overlaps_itself(t):
    """Whether two elements of a strided tensor may share an address."""
    reach = 0
    for n, s in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n > 1), key=lambda x: x[1]):
        if s <= reach:
            return True
        reach += (n - 1) * s
    return False


def _rotate(query, key, positions, inv_freq, interleaved, q_start, k_start, scale, layout, inverse, inplace):
    """Launch on checked arguments; returns the rotated query and key."""
    outs, args = [], []
    for t, start in ((query, q_start), (key, k_start)):
        if t is None:
            outs.append(None)
            args += [None, None] + [0] * 9
            continue
        b, s, n, d = _heads(t, layout, "tensor")
        st = _strides(t)
        if st is None:
            t = t.contiguous()
            st = _strides(t)
        out = t if inplace else torch.empty(t.shape, dtype=t.dtype, device=t.device)
        outs.append(out)
        args += [t.data_ptr(), out.data_ptr(), *st, *_strides(out), n, d, start]
    b, s = _heads(query, layout, "query")[:2]
    if query.numel() == 0:
        return outs
    per_seq = layout == "TND" or positions.dim() == 2
    with _lib.on_device(query.device):
        status = _lib.load().dsa_rope(
            *args, positions.data_ptr(), 1 if positions.dtype == torch.int64 else 0, 1 if per_seq else 0,
            inv_freq.data_ptr(), b, s, 2 * inv_freq.numel(), 1 if interleaved else 0, 1 if inverse else 0,
            _lib.dtype_code(query.dtype), scale, _lib.stream_handle(query.device))
    _lib.check(status, "dsa_rope")
    return outs


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
    contiguous tensors, or with ``inplace`` the inputs themselves.  Strided
    views are read as they are if a head's columns are next to each other.
    Differentiable in query and key (not in place).
    """
    if layout not in ("BSND", "TND"):
        raise ValueError(f"layout must be BSND or TND, got {layout}")
    if positions is None or inv_freq is None:
        raise ValueError("positions and inv_freq are required")
    b, s, n, d = _heads(query, layout, "query")
    if query.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError(f"query dtype must be bfloat16, float16 or float32, got {query.dtype}")
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"positions must be int32 or int64, got {positions.dtype}")
    if inv_freq.dim() != 1 or inv_freq.numel() < 1:
        raise ValueError(f"inv_freq must be a vector, got {tuple(inv_freq.shape)}")
    rot = 2 * inv_freq.numel()
    if positions.dim() != 1 or positions.shape[0] != s:
        _expect_shape(positions, (s,) if layout == "TND" else (b, s), "positions")
    if key_rotary_offset is None:
        key_rotary_offset = rotary_offset
    checks = [("query", query, d, rotary_offset)]
    if key is not None:
        kb, ks, _, kd = _heads(key, layout, "key")
        if (kb, ks) != (b, s):
            raise ValueError(f"key must have the query's batch and tokens, got {tuple(key.shape)}")
        if key.dtype != query.dtype:
            raise ValueError(f"key dtype {key.dtype} differs from query dtype {query.dtype}")
        checks.append(("key", key, kd, key_rotary_offset))
    for name, t, cols, start in checks:
        if int(start) != start or not 0 <= start <= cols - rot:
            raise ValueError(f"the {rot} rotary columns from {start} do not lie inside the {cols} of {name}")
    grad = torch.is_grad_enabled() and (query.requires_grad or (key is not None and key.requires_grad))
    if inplace:
        if grad:
            raise ValueError("inplace is for inference: the inputs require grad")
        for name, t, _, _ in checks:
            if _strides(t) is None or _overlaps_itself(t):
                raise ValueError(f"inplace needs a {name} whose head columns are next to each other and whose "
                                 "elements do not share memory")
        if key is not None and key.numel() and query.numel() and key.data_ptr() == query.data_ptr():
            raise ValueError("inplace needs a key and a query of their own")
    _check_device(query, key, positions, inv_freq)
    positions = positions.contiguous()
    inv_freq = inv_freq.to(torch.float64).contiguous()
    args = (positions, inv_freq, bool(interleaved), int(rotary_offset), int(key_rotary_offset),
            float(attention_scale), layout)
    if grad:
        from .autograd import RotaryEmbeddingFunction
        return RotaryEmbeddingFunction.apply(query, key, *args, bool(inverse))
    out = tuple(_rotate(query, key, *args, bool(inverse), inplace))
    if inplace:
        torch.autograd.graph.increment_version([t for _, t, _, _ in checks])
    return out


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
