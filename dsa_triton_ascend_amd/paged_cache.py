"""Pages of a cache on MI355X: writing new tokens, forking, releasing and
extending sequences, and compaction.

The attention and indexer operators read caches in the PA_BSND layout,
``[pages, page_size, heads, columns]``, through a block table ``[B,
max_blocks]``; these functions fill and manage them.  Several caches (latent,
rope, indexer keys, of all layers) share one table: pass them as a list.

The state of a pool is three int32 tensors: the block table (-1: no page), the
lengths ``[B]`` and ``page_refs [pages]``, how often each page is referred to
(0: free).  A page that something outside the table holds too has that counted
in ``page_refs``.  Everything is decided on the device from these tensors,
without reading them on the host; the functions return new ones and leave the
given ones as they are, so a call can be captured and replayed.  The caches
are changed in place.

One decoding step:

    table, lens, refs = paged_cache_fork(caches, table, lens, refs, parents, new_tokens=1)   # once
    paged_cache_write([latent, k_rope, k_index], [...], table, lens)                         # per layer
    out, _, _ = paged_attention(q, latent_cache, None, table, lens + 1, ...)                 # per layer
    lens = lens + 1
"""
import ctypes

import torch

from . import _lib
from .sparse_flash_attention import _check_device

_INT = torch.int32


def _list(x, name):
    if isinstance(x, torch.Tensor):
        x = [x]
    x = list(x)
    for t in x:
        if not isinstance(t, torch.Tensor):
            raise ValueError(f"{name} must be tensors")
    return x


def _check_caches(caches, pages=None):
    """Number of pages and page size of caches that share a table."""
    size = None
    for t in caches:
        if t.dim() < 3:
            raise ValueError(f"a cache must be [pages, page_size, heads, columns], got {tuple(t.shape)}")
        if not t.is_contiguous():
            raise ValueError("caches must be contiguous (they are changed in place)")
        if size is None:
            size = (t.shape[0], t.shape[1])
        elif (t.shape[0], t.shape[1]) != size:
            raise ValueError(f"all caches must have the same pages and page size, got {size} and {tuple(t.shape[:2])}")
        if t.numel() == 0:
            raise ValueError(f"a cache must not be empty, got {tuple(t.shape)}")
    if pages is not None and size is not None and size[0] != pages:
        raise ValueError(f"page_refs must have one entry per page ({size[0]}), got {pages}")
    seen = {}
    for t in caches:
        if t.data_ptr() in seen:
            raise ValueError("the same cache is given twice")
        seen[t.data_ptr()] = True
    return size


def _ints(t, name, dim):
    if t.dtype != _INT:
        raise ValueError(f"{name} must be int32, got {t.dtype}")
    if t.dim() != dim or t.numel() == 0:
        raise ValueError(f"{name} must have {dim} dimension(s) and not be empty, got {tuple(t.shape)}")
    return t.contiguous()


def _pointers(tensors):
    return (ctypes.c_void_p * max(1, len(tensors)))(*[t.data_ptr() for t in tensors])


def _longs(values):
    return (ctypes.c_int64 * max(1, len(values)))(*values)


def _row_bytes(t):
    return t[0, 0].numel() * t.element_size()


def paged_cache_write(caches, rows, block_table, seq_lengths, row_lengths=None, layout="BSND"):
    """Write new tokens' rows into the pages of their sequences, in place.

    ``rows[i]`` [B, S, ...] (layout "BSND") or [T, ...] ("TND", packed) holds the new
    rows of ``caches[i]`` [pages, page_size, ...], of its dtype and trailing
    sizes; batch and token strides are free.  The first new token of sequence b
    goes to position ``seq_lengths[b]`` (tokens before the call).
    ``row_lengths``: new tokens of each sequence (BSND; all S by default), or
    cumulative (TND, required).  Tokens that have no page (past the table, a -1
    entry) and packed rows behind the last sequence are not written.  A page
    that several sequences share is not to be written: fork first.  Returns
    None.
    """
    caches, rows = _list(caches, "caches"), _list(rows, "rows")
    if len(caches) != len(rows) or not caches:
        raise ValueError(f"one tensor of rows per cache is needed, got {len(rows)} for {len(caches)}")
    if layout not in ("BSND", "TND"):
        raise ValueError(f"layout must be BSND or TND, got {layout}")
    pages, page = _check_caches(caches)
    table = _ints(block_table, "block_table", 2)
    batch = table.shape[0]
    lens = _ints(seq_lengths, "seq_lengths", 1)
    if lens.shape[0] != batch:
        raise ValueError(f"seq_lengths must have one entry per row of block_table ({batch}), got {lens.shape[0]}")
    if row_lengths is not None:
        row_lengths = _ints(row_lengths, "row_lengths", 1)
        if row_lengths.shape[0] != batch:
            raise ValueError(f"row_lengths must have one entry per sequence ({batch}), got {row_lengths.shape[0]}")
    elif layout == "TND":
        raise ValueError("TND layout requires row_lengths (cumulative)")
    lead = 1 if layout == "TND" else 2
    tokens = tuple(rows[0].shape[:lead])
    sizes, sb, st, kept = [], [], [], []
    for r, c in zip(rows, caches):
        if r.dim() != c.dim() - 2 + lead or tuple(r.shape[lead:]) != tuple(c.shape[2:]):
            raise ValueError(f"rows {tuple(r.shape)} do not fit a cache {tuple(c.shape)}")
        if tuple(r.shape[:lead]) != tokens or (lead == 2 and tokens[0] != batch):
            raise ValueError(f"rows must be [{'T' if lead == 1 else f'B={batch}, S'}, ...], alike for all caches, "
                             f"got {tuple(r.shape)}")
        if r.dtype != c.dtype:
            raise ValueError(f"rows dtype {r.dtype} differs from cache dtype {c.dtype}")
        if r.numel() and not r[(0,) * lead].is_contiguous():
            r = r.contiguous()
        kept.append(r)
        es = r.element_size()
        sizes.append(_row_bytes(c))
        sb.append(r.stride(0) * es if lead == 2 else 0)
        st.append(r.stride(lead - 1) * es)
    _check_device(*caches, *kept, table, lens, row_lengths)
    n_tok = tokens[0] if lead == 1 else tokens[0] * tokens[1]
    if n_tok == 0:
        return
    with _lib.on_device(table.device):
        status = _lib.load().dsa_paged_cache_write(
            len(caches), _pointers(kept), _pointers(caches), _longs(sizes), _longs(sb), _longs(st), table.data_ptr(),
            lens.data_ptr(), _lib.ptr(row_lengths), batch, 0 if lead == 1 else tokens[1], n_tok, table.shape[1], pages,
            page, _lib.LAYOUT[layout], _lib.stream_handle(table.device))
    _lib.check(status, "dsa_paged_cache_write")


def paged_cache_fork(caches, block_table, seq_lengths, page_refs, parents=None, new_tokens=0, page_size=None):
    """The block table of the next step: rows forked, reordered, released and
    given room.

    New row c continues row ``parents[c]`` (int32; negative: an empty row;
    None: every row continues itself) and has pages for ``new_tokens`` more
    tokens.  Rows that nobody continues are released.  Full pages are shared;
    a partly filled last page stays with the first row that continues it if
    nobody else refers to it, and is copied in all ``caches`` for every other.
    Pages come from those free before the call, lowest first, to rows in
    order.  A row for which they do not last, or that outgrows the table's
    width, gets no pages and the length -1; its sequence is released unless
    another row continues it, so keep the old state until lengths are checked.
    Pages of the old table past a sequence's last token are released.
    ``caches`` may be empty (tables only, with ``page_size``), which leaves the
    copies to the caller.

    Returns ``(block_table [C, max_blocks], seq_lengths [C], page_refs)``.
    """
    caches = _list(caches, "caches")
    refs = _ints(page_refs, "page_refs", 1)
    size = _check_caches(caches, refs.shape[0])
    if size is None:
        if page_size is None:
            raise ValueError("page_size is required without caches")
    elif page_size is not None and page_size != size[1]:
        raise ValueError(f"page_size ({page_size}) must equal the caches' ({size[1]})")
    page = size[1] if size is not None else int(page_size)
    table = _ints(block_table, "block_table", 2)
    rows, wide = table.shape
    lens = _ints(seq_lengths, "seq_lengths", 1)
    if lens.shape[0] != rows:
        raise ValueError(f"seq_lengths must have one entry per row of block_table ({rows}), got {lens.shape[0]}")
    if parents is not None:
        parents = _ints(parents, "parents", 1)
    if int(new_tokens) != new_tokens or not 0 <= new_tokens < 2 ** 31:
        raise ValueError(f"new_tokens must be an integer in [0, 2^31), got {new_tokens}")
    _check_device(table, *caches, lens, refs, parents)
    children = rows if parents is None else parents.shape[0]
    dev = table.device
    new_table = torch.empty(children, wide, dtype=_INT, device=dev)
    new_lens = torch.empty(children, dtype=_INT, device=dev)
    new_refs = torch.empty_like(refs)
    lib = _lib.load()
    nbytes = lib.dsa_paged_cache_fork_workspace_size(rows, children, refs.shape[0])
    ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=dev)
    with _lib.on_device(dev):
        status = lib.dsa_paged_cache_fork(
            len(caches), _pointers(caches), _longs([_row_bytes(c) for c in caches]), table.data_ptr(), lens.data_ptr(),
            refs.data_ptr(), _lib.ptr(parents), new_table.data_ptr(), new_lens.data_ptr(), new_refs.data_ptr(), rows,
            children, wide, wide, refs.shape[0], page, int(new_tokens), ws.data_ptr(), nbytes, _lib.stream_handle(dev))
    _lib.check(status, "dsa_paged_cache_fork")
    return new_table, new_lens, new_refs


def paged_cache_compact(caches, block_table, page_refs, page_size=None):
    """Move the pages in use to the lowest ids, in all ``caches``, in place.

    With n pages in use (``page_refs`` > 0), those at ids below n stay, and the
    k-th other one moves to the k-th free id below n.  Returns ``(block_table,
    page_refs, page_map)``: the table and the counts for the new ids, and each
    old page's new id (-1: it was free).
    """
    caches = _list(caches, "caches")
    refs = _ints(page_refs, "page_refs", 1)
    size = _check_caches(caches, refs.shape[0])
    if size is not None and page_size is not None and page_size != size[1]:
        raise ValueError(f"page_size ({page_size}) must equal the caches' ({size[1]})")
    table = _ints(block_table, "block_table", 2)
    rows, wide = table.shape
    _check_device(table, *caches, refs)
    dev = table.device
    new_table, new_refs, page_map = torch.empty_like(table), torch.empty_like(refs), torch.empty_like(refs)
    lib = _lib.load()
    nbytes = lib.dsa_paged_cache_compact_workspace_size(refs.shape[0])
    ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=dev)
    with _lib.on_device(dev):
        status = lib.dsa_paged_cache_compact(
            len(caches), _pointers(caches), _longs([_row_bytes(c) for c in caches]), table.data_ptr(), refs.data_ptr(),
            new_table.data_ptr(), new_refs.data_ptr(), page_map.data_ptr(), rows, wide, refs.shape[0],
            size[1] if size is not None else 1, ws.data_ptr(), nbytes, _lib.stream_handle(dev))
    _lib.check(status, "dsa_paged_cache_compact")
    return new_table, new_refs, page_map
