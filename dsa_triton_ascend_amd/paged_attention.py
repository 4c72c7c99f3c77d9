"""Attention of each sequence's newest tokens over a paged cache on MI355X:
the dense counterpart of ``sparse_flash_attention``'s paged decode, for layers
and contexts where every cached token is attended.

Two forms: grouped heads over key and value caches, and the MLA-absorb form
over the latent cache of the sparse operators (value = key[..., :D], one key
head, rope parts of 64 columns).  The reference has no such operator; argument
names, masks, zero rows and the return triple are those of
``sparse_flash_attention``.
"""
import torch

from . import _lib
from .sparse_flash_attention import INT64_MAX, _band_args, _expect_shape, _seq_tensor

_GROUPED_D = (64, 128, 256)
_LATENT_D = (128, 256, 512)
_D_ROPE = 64


def paged_attention(query, key, value, block_table, actual_seq_lengths_kv, scale_value=1.0, query_rope=None,
                    key_rope=None, actual_seq_lengths_query=None, sparse_mode=3, pre_tokens=INT64_MAX,
                    next_tokens=INT64_MAX, return_softmax_lse=False):
    """Attention of the newest S1 tokens of B sequences over their pages.

    query [B, S1, N1, D], bfloat16 or float16.  Grouped form: key and value
    [pages, page_size, N2, D], D in (64, 128, 256), N1 a multiple of N2, no
    rope parts.  Latent form: ``value`` None, key [pages, page_size, 1, D], D
    in (128, 256, 512), query_rope [B, S1, N1, 64] and key_rope [pages,
    page_size, 1, 64].  Caches are contiguous and start at a multiple of 16
    bytes; a query that does not is copied.  ``block_table`` [B, max_blocks]; entries outside the
    cache read as zero rows; all of it may name up to 2^35 tokens.  ``actual_seq_lengths_kv`` [B]: cached tokens, the
    new ones included.  ``actual_seq_lengths_query`` [B]: new tokens (S1 by
    default); later rows give zeros.

    sparse_mode 3: new token s1 sees the first act_kv - act_q + s1 + 1 tokens;
    0: all act_kv.  ``pre_tokens`` / ``next_tokens`` select a band around the
    diagonal, as in ``sparse_flash_attention`` (a sliding window of w tokens:
    pre_tokens = w - 1); tokens outside every row's band are not read.  A value
    that one new token of a sequence sees and another does not has weight zero
    for the latter, so it must be finite there; rows that see no token are zero
    whatever the values.

    Returns ``(attention_out, softmax_max, softmax_sum)``: the output in the
    query's shape and dtype, the statistics [B, N2, S1, N1 / N2] in float32,
    zeros unless ``return_softmax_lse``.  Inference only.
    """
    result = _lib.calls().attention(query, key, value, block_table, actual_seq_lengths_kv, scale_value, query_rope,
                                    key_rope, actual_seq_lengths_query, sparse_mode, pre_tokens, next_tokens,
                                    return_softmax_lse)
    if result is not None:
        return result
    pre_tokens, next_tokens = _band_args(pre_tokens, next_tokens)
    if sparse_mode not in (0, 3):
        raise ValueError("Only sparse_mode 0 (full) / 3 (rightDownCausal) supported")
    latent = value is None
    if latent and (query_rope is None or key_rope is None):
        raise ValueError("the latent form (value=None) needs query_rope and key_rope")
    if not latent and (query_rope is not None or key_rope is not None):
        raise ValueError("the grouped form takes no rope parts: rotate query and key instead")
    q_shape, k_shape = query.shape, key.shape
    if len(q_shape) != 4 or len(k_shape) != 4:
        raise ValueError(f"query must be [B, S1, N1, D] and key [pages, page_size, N2, D], got {tuple(q_shape)} "
                         f"and {tuple(k_shape)}")
    B, S1, N1, D = q_shape
    pages, page, N2, kd = k_shape
    if kd != D:
        raise ValueError(f"key must have the query's {D} columns, got {kd}")
    if D not in (_LATENT_D if latent else _GROUPED_D):
        raise ValueError(f"D must be one of {_LATENT_D if latent else _GROUPED_D}, got {D}")
    if latent and N2 != 1:
        raise ValueError(f"the latent form has one key head, got {N2}")
    if N1 < 1 or N2 < 1 or N1 % N2:
        raise ValueError(f"query heads ({N1}) must be a multiple of key heads ({N2})")
    dtype = query.dtype
    if dtype is torch.bfloat16:
        code = _lib.DTYPE_BF16
    elif dtype is torch.float16:
        code = _lib.DTYPE_FP16
    else:
        raise ValueError(f"query dtype must be bfloat16 or float16, got {dtype}")
    if latent:
        if query_rope.shape[:-1] != q_shape[:-1] or query_rope.shape[-1] != _D_ROPE:
            _expect_shape(query_rope, (B, S1, N1, _D_ROPE), "query_rope")
        if key_rope.shape[:-1] != k_shape[:-1] or key_rope.shape[-1] != _D_ROPE:
            _expect_shape(key_rope, (pages, page, 1, _D_ROPE), "key_rope")
        others = (("key", key), ("query_rope", query_rope), ("key_rope", key_rope))
    else:
        if value.shape != k_shape:
            _expect_shape(value, k_shape, "value")
        others = (("key", key), ("value", value))
    for name, t in others:
        if t.dtype != dtype:
            raise ValueError(f"{name} dtype {t.dtype} differs from query dtype {dtype}")
    if block_table is None or actual_seq_lengths_kv is None:
        raise ValueError("block_table and actual_seq_lengths_kv are required")
    if block_table.dim() != 2 or block_table.shape[0] < B:
        raise ValueError(f"block_table must be [B, max_blocks] with B={B} rows, got {tuple(block_table.shape)}")
    _lib.no_derivatives("paged_attention", query, *(t for _, t in others))
    index = _lib.same_device(query, key, value, query_rope, key_rope, block_table)
    dev = query.device
    act_k = _lengths(actual_seq_lengths_kv, dev)
    act_q = None if actual_seq_lengths_query is None else _lengths(actual_seq_lengths_query, dev)
    if act_k.numel() != B or (act_q is not None and act_q.numel() != B):
        raise ValueError("actual sequence length arrays must have one entry per batch")
    for name, t in others:
        if name != "query_rope" and not t.is_contiguous():
            raise ValueError(f"the {name} cache must be contiguous (a copy of it would be made at every call)")
    table = _int32(block_table)
    if not table.is_contiguous():
        table = table.contiguous()
    q = _rows(query)
    qr = _rows(query_rope) if latent else None
    out = q.new_empty(q_shape)
    smax = torch.empty((B, N2, S1, N1 // N2), dtype=torch.float32, device=dev)
    ssum = torch.empty_like(smax)
    if q.numel() == 0:
        return out, smax, ssum
    wide = table.shape[1]
    if key.numel() == 0 or wide == 0:  # no page at all: no row sees a token
        return out.zero_(), smax.zero_(), ssum.zero_()
    lib = _lib.load()
    nbytes = _lib.call_on(index, lib.dsa_paged_attn_workspace_size, B, S1, N1, N2, D, latent, wide, page)
    ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=dev)
    status = _lib.call_on(
        index, lib.dsa_paged_attn, q.data_ptr(), qr.data_ptr() if latent else None, key.data_ptr(),
        key_rope.data_ptr() if latent else None, None if latent else value.data_ptr(), out.data_ptr(),
        smax.data_ptr(), ssum.data_ptr(), None if act_q is None else act_q.data_ptr(), act_k.data_ptr(),
        table.data_ptr(), B, S1, N1, N2, D, _D_ROPE if latent else 0, pages, page, wide, sparse_mode, pre_tokens,
        next_tokens, code, float(scale_value), bool(return_softmax_lse), ws.data_ptr(), nbytes, _lib.raw_stream(index))
    if status:
        _lib.check(status, "dsa_paged_attn")
    return out, smax, ssum


def _rows(t):
    """The tensor as the kernels read it: contiguous, 16 bytes at a time."""
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _int32(t):
    if t.dtype is torch.int64:  # what 32 bits do not hold is as far outside as they go, not another value inside
        t = t.clamp(-2 ** 31, 2 ** 31 - 1)
    return t if t.dtype is torch.int32 else t.to(dtype=torch.int32)


def _lengths(x, device):
    if isinstance(x, torch.Tensor):
        x = _int32(x)
        if x.device == device and x.is_contiguous():
            return x
    return _seq_tensor(x, device)


class PagedAttention(torch.nn.Module):
    """Module wrapper of ``paged_attention`` (the options at construction, the
    tensors at the call)."""

    def __init__(self, scale_value=1.0, sparse_mode=3, return_softmax_lse=False, pre_tokens=INT64_MAX,
                 next_tokens=INT64_MAX):
        super().__init__()
        self.scale_value = scale_value
        self.sparse_mode = sparse_mode
        self.return_softmax_lse = return_softmax_lse
        self.pre_tokens = pre_tokens
        self.next_tokens = next_tokens

    def forward(self, query, key, value, block_table, actual_seq_lengths_kv, query_rope=None, key_rope=None,
                actual_seq_lengths_query=None):
        return paged_attention(
            query, key, value, block_table, actual_seq_lengths_kv, scale_value=self.scale_value,
            query_rope=query_rope, key_rope=key_rope, actual_seq_lengths_query=actual_seq_lengths_query,
            sparse_mode=self.sparse_mode, pre_tokens=self.pre_tokens, next_tokens=self.next_tokens,
            return_softmax_lse=self.return_softmax_lse)

    construct = forward
