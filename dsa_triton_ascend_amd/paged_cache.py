"""Pages of a cache on MI355X: writing new tokens, forking, releasing and
extending sequences, planning a step of requests of many lengths, finding the
prefixes that sequences share, and compaction.

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
are changed in place.  None of the functions has derivatives: caches and rows
that require grad are refused outside ``torch.no_grad()``.

One decoding step:

    table, lens, refs = paged_cache_fork(caches, table, lens, refs, parents, new_tokens=1)   # once
    paged_cache_write([latent, k_rope, k_index], [...], table, lens)                         # per layer
    out, _, _ = paged_attention(q, latent_cache, None, table, lens + 1, ...)                 # per layer
    lens = lens + 1                                                                          # of rows in use

One step of requests with new tokens of their own number each: ``new[r]`` of
row r, S1 at most (a number known on the host), packed in ``tokens`` places for
rotation and writes.  Attention takes each row's own tokens, padded to S1:

    old = lens.clamp(min=0)
    table, lens, refs, slots, positions, ends = paged_cache_plan(table, lens, refs, new, page, tokens)   # once
    groups, shared = paged_cache_prefixes(table, lens, page)                                             # once
    counts = (lens - old).clamp(min=0)     # tokens taken, 0 for rows that were refused or have ended      once
    at = ((ends - new.clamp(min=0))[:, None] + torch.arange(S1, device=ends.device)).clamp(max=tokens - 1)  # once
    paged_cache_write_slots([latent, k_rope, k_index], [...], slots)                                     # per layer
    out, _, _ = paged_prefix_attention(q[at], latent_cache, None, table, lens, groups, shared,           # per layer
                                       query_rope=q_rope[at], key_rope=k_rope_cache, actual_seq_lengths_query=counts)

and token t of the packed ones has its output at ``out[r, t - (ends - new)[r]]``
with ``r = torch.searchsorted(ends, t, right=True)`` (tokens of refused rows: zeros).
"""
from array import array

import torch

from . import _lib

_INT = torch.int32


def _list(x, name):
    if isinstance(x, torch.Tensor):
        return [x]
    for t in x:
        if not isinstance(t, torch.Tensor):
            raise ValueError(f"{name} must be tensors")
    return x


def _check_caches(caches):
    """(pages, page size, addresses, bytes of a token's row) of caches that
    share a table; (None, None, [], []) without caches."""
    pages = page = None
    addresses, row_bytes = [], []
    for t in caches:
        shape = t.shape
        if len(shape) < 3:
            raise ValueError(f"a cache must be [pages, page_size, heads, columns], got {tuple(shape)}")
        if not t.is_contiguous():
            raise ValueError("caches must be contiguous (they are changed in place)")
        if pages is None:
            pages, page = shape[0], shape[1]
        elif shape[0] != pages or shape[1] != page:
            raise ValueError("all caches must have the same pages and page size, got "
                             f"{(pages, page)} and {tuple(shape[:2])}")
        n = t.numel()
        if n == 0:
            raise ValueError(f"a cache must not be empty, got {tuple(shape)}")
        addresses.append(t.data_ptr())
        row_bytes.append(n // (pages * page) * t.element_size())
    if len(addresses) > 1:
        spans = sorted(zip(addresses, row_bytes))
        end = 0
        for at, size in spans:
            if at < end:
                raise ValueError("the same cache is given twice, or two caches overlap")
            end = at + size * pages * page
    return pages, page, addresses, row_bytes


def _ints(t, name, dim):
    if t.dtype != _INT:
        raise ValueError(f"{name} must be int32, got {t.dtype}")
    if t.dim() != dim or t.numel() == 0:
        raise ValueError(f"{name} must have {dim} dimension(s) and not be empty, got {tuple(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _longs(*lists):
    """The lists as arrays of 64-bit integers in one allocation: the owner,
    which has to live until the call returns, and their addresses."""
    a = array("q", [x for values in lists for x in values])
    at, out = a.buffer_info()[0], []
    for values in lists:
        out.append(at)
        at += 8 * len(values)
    return a, out


def _sources(rows, caches, lead):
    """Addresses and byte strides (batch, token) of the new rows, whose first
    ``lead`` dimensions are tokens, and the tensors that hold them."""
    sources, sb, st, kept = [], [], [], []
    tokens = rows[0].shape[:lead]
    for r, c in zip(rows, caches):
        shape, inner = r.shape, c.shape[2:]
        if shape[lead:] != inner:
            raise ValueError(f"rows {tuple(shape)} do not fit a cache {tuple(c.shape)}")
        if shape[:lead] != tokens:
            raise ValueError(f"rows must have the same tokens for all caches, got {tuple(tokens)} and {tuple(shape)}")
        if r.dtype != c.dtype:
            raise ValueError(f"rows dtype {r.dtype} differs from cache dtype {c.dtype}")
        stride, step = r.stride(), 1
        for i in range(len(shape) - 1, lead - 1, -1):  # a token's row has to be in one piece
            if stride[i] != step and shape[i] != 1:
                r = r.contiguous()
                stride = r.stride()
                break
            step *= shape[i]
        es = r.element_size()
        kept.append(r)
        sources.append(r.data_ptr())
        sb.append(stride[0] * es if lead == 2 else 0)
        st.append(stride[lead - 1] * es)
    return sources, sb, st, kept


def paged_cache_write(caches, rows, block_table, seq_lengths, row_lengths=None, layout="BSND"):
    """Write new tokens' rows into the pages of their sequences, in place.

    ``rows[i]`` [B, S, ...] (layout "BSND") or [T, ...] ("TND", packed) holds the new
    rows of ``caches[i]`` [pages, page_size, ...], of its dtype and trailing
    sizes, outside the caches; batch and token strides are free.  The first new token of sequence b
    goes to position ``seq_lengths[b]`` (tokens before the call).
    ``row_lengths``: new tokens of each sequence (BSND; all S by default), or
    cumulative (TND, required).  Tokens that have no page (past the table, a -1
    entry) and packed rows behind the last sequence are not written.  A page
    that several sequences share is not to be written: fork first.  Returns
    None.
    """
    if _lib.calls().write(caches, rows, block_table, seq_lengths, row_lengths, layout):
        return
    caches, rows = _list(caches, "caches"), _list(rows, "rows")
    if len(caches) != len(rows) or not caches:
        raise ValueError(f"one tensor of rows per cache is needed, got {len(rows)} for {len(caches)}")
    if layout == "BSND":
        lead = 2
    elif layout == "TND":
        lead = 1
    else:
        raise ValueError(f"layout must be BSND or TND, got {layout}")
    pages, page, addresses, sizes = _check_caches(caches)
    table = _ints(block_table, "block_table", 2)
    batch, wide = table.shape
    lens = _ints(seq_lengths, "seq_lengths", 1)
    if lens.shape[0] != batch:
        raise ValueError(f"seq_lengths must have one entry per row of block_table ({batch}), got {lens.shape[0]}")
    if row_lengths is not None:
        row_lengths = _ints(row_lengths, "row_lengths", 1)
        if row_lengths.shape[0] != batch:
            raise ValueError(f"row_lengths must have one entry per sequence ({batch}), got {row_lengths.shape[0]}")
    elif lead == 1:
        raise ValueError("TND layout requires row_lengths (cumulative)")
    tokens = rows[0].shape[:lead]
    if lead == 2 and tokens and tokens[0] != batch:
        raise ValueError(f"rows must be [B={batch}, S, ...], got {tuple(rows[0].shape)}")
    sources, sb, st, kept = _sources(rows, caches, lead)
    _lib.no_derivatives("paged_cache_write", *caches, *rows)
    index = _lib.same_device(table, lens, row_lengths, *caches, *kept)
    n_tok = tokens[0] if lead == 1 else tokens[0] * tokens[1]
    if n_tok == 0:
        return
    owner, (a_src, a_dst, a_size, a_sb, a_st) = _longs(sources, addresses, sizes, sb, st)
    status = _lib.call_on(
        index, _lib.load().dsa_paged_cache_write, len(caches), a_src, a_dst, a_size, a_sb, a_st, table.data_ptr(),
        lens.data_ptr(), None if row_lengths is None else row_lengths.data_ptr(), batch,
        0 if lead == 1 else tokens[1], n_tok, wide, pages, page, 2 - lead, _lib.raw_stream(index))
    if status:
        _lib.check(status, "dsa_paged_cache_write")
    _lib.changed(*caches)


def paged_cache_fork(caches, block_table, seq_lengths, page_refs, parents=None, new_tokens=0, page_size=None):
    """The block table of the next step: rows forked, reordered, released and
    given room.

    New row c continues row ``parents[c]`` (int32; negative: an empty row,
    length 0 and no pages; None: every row continues itself) and has pages for
    ``new_tokens`` more tokens.  Rows that nobody continues are released.  Full pages are shared;
    a partly filled last page stays with the first row that continues it if
    nobody else refers to it, and is copied in all ``caches`` for every other.
    Pages come from those free before the call, lowest first, to rows in
    order.  A row for which they do not last, or that outgrows the table's
    width, gets no pages and the length -1; its sequence is released unless
    another row continues it, so keep the old state until lengths are checked.
    Pages of the old table past a sequence's last token are released, and what
    a row needs is taken from those free before the call: a page that it
    reserved and did not fill is exchanged for another one, so a pool needs one
    free page for every row in such a state.  Fork when the room is used up, or
    write into pages reserved earlier without a fork between.  A length below
    zero, as of a row that got no pages, counts as zero.
    ``caches`` may be empty (tables only, with ``page_size``), which leaves the
    copies to the caller.

    Returns ``(block_table [C, max_blocks], seq_lengths [C], page_refs)``.
    """
    state = _lib.calls().fork(caches, block_table, seq_lengths, page_refs, parents, new_tokens, page_size)
    if state is not None:
        return state
    caches = _list(caches, "caches")
    pages, page, addresses, sizes = _check_caches(caches)
    refs = _ints(page_refs, "page_refs", 1)
    n_pages = refs.shape[0]
    if pages is not None and pages != n_pages:
        raise ValueError(f"page_refs must have one entry per page ({pages}), got {n_pages}")
    if page is None:
        if page_size is None:
            raise ValueError("page_size is required without caches")
        page = int(page_size)
    elif page_size is not None and page_size != page:
        raise ValueError(f"page_size ({page_size}) must equal the caches' ({page})")
    table = _ints(block_table, "block_table", 2)
    rows, wide = table.shape
    lens = _ints(seq_lengths, "seq_lengths", 1)
    if lens.shape[0] != rows:
        raise ValueError(f"seq_lengths must have one entry per row of block_table ({rows}), got {lens.shape[0]}")
    children = rows
    if parents is not None:
        parents = _ints(parents, "parents", 1)
        children = parents.shape[0]
    if int(new_tokens) != new_tokens or not 0 <= new_tokens < 2 ** 31:
        raise ValueError(f"new_tokens must be an integer in [0, 2^31), got {new_tokens}")
    _lib.no_derivatives("paged_cache_fork", *caches)
    index = _lib.same_device(table, lens, refs, parents, *caches)
    new_table = table.new_empty((children, wide))
    new_lens = lens.new_empty(children)
    new_refs = torch.empty_like(refs)
    lib = _lib.load()
    nbytes = lib.dsa_paged_cache_fork_workspace_size(rows, children, n_pages)
    ws = refs.new_empty((nbytes + 3) // 4)
    owner, (a_caches, a_sizes) = _longs(addresses, sizes)
    status = _lib.call_on(
        index, lib.dsa_paged_cache_fork, len(caches), a_caches, a_sizes, table.data_ptr(), lens.data_ptr(),
        refs.data_ptr(), None if parents is None else parents.data_ptr(), new_table.data_ptr(), new_lens.data_ptr(),
        new_refs.data_ptr(), rows, children, wide, wide, n_pages, page, int(new_tokens), ws.data_ptr(), nbytes,
        _lib.raw_stream(index))
    if status:
        _lib.check(status, "dsa_paged_cache_fork")
    _lib.changed(*caches)
    return new_table, new_lens, new_refs


def paged_cache_plan(block_table, seq_lengths, page_refs, new_lengths, page_size, tokens):
    """Tables, slots and positions of a step that adds ``new_lengths[r]`` tokens
    to row r (int32 [R], a number of its own for each row; negative: the
    request has ended and its row is released).

    Row r gets pages for its new tokens, lowest free ones first, to rows in
    order.  A row for which they do not last, every later row that needs any,
    and a row that would outgrow the table are refused: they keep their pages
    and their length, and get no new tokens (the length shows it), so that they
    can wait in place.  Pages freed by the call are not handed out in it.
    Pages of the old table past a row's last token are released, as by
    ``paged_cache_fork``.  A partly filled last page that rows share is not to
    be written: fork first.  A length below zero counts as zero.

    The step's new tokens lie packed, row after row: ``tokens`` places (at least
    as many as there are new tokens; an integer, known without reading the
    device; more, as padding, are allowed).

    Returns ``(block_table, seq_lengths, page_refs, slots, positions,
    row_lengths)``, all int32: the state with the new tokens in it (an ended
    row: length 0, no pages); each token's place for ``paged_cache_write_slots``
    (-1: a refused row's, or padding) and its position for ``rotary_embedding``
    (0 for padding), [tokens]; and the cumulative numbers of new tokens [R], as
    the packed layouts ("TND") take them (those of refused rows are counted).
    """
    state = _lib.calls().plan(block_table, seq_lengths, page_refs, new_lengths, page_size, tokens)
    if state is not None:
        return state
    table = _ints(block_table, "block_table", 2)
    rows, wide = table.shape
    lens = _ints(seq_lengths, "seq_lengths", 1)
    more = _ints(new_lengths, "new_lengths", 1)
    refs = _ints(page_refs, "page_refs", 1)
    for name, t in (("seq_lengths", lens), ("new_lengths", more)):
        if t.shape[0] != rows:
            raise ValueError(f"{name} must have one entry per row of block_table ({rows}), got {t.shape[0]}")
    if int(page_size) != page_size or page_size < 1:
        raise ValueError(f"page_size must be a positive integer, got {page_size}")
    if int(tokens) != tokens or not 0 <= tokens <= 2 ** 30:
        raise ValueError(f"tokens must be an integer in [0, 2^30], got {tokens}")
    index = _lib.same_device(table, lens, more, refs)
    tokens, pages = int(tokens), refs.shape[0]
    new_table, new_lens, new_refs = torch.empty_like(table), torch.empty_like(lens), torch.empty_like(refs)
    slots, positions, ends = lens.new_empty(tokens), lens.new_empty(tokens), torch.empty_like(lens)
    lib = _lib.load()
    nbytes = lib.dsa_paged_cache_plan_workspace_size(rows, pages)
    ws = refs.new_empty((nbytes + 3) // 4)
    status = _lib.call_on(
        index, lib.dsa_paged_cache_plan, table.data_ptr(), lens.data_ptr(), refs.data_ptr(), more.data_ptr(),
        new_table.data_ptr(), new_lens.data_ptr(), new_refs.data_ptr(), slots.data_ptr(), positions.data_ptr(),
        ends.data_ptr(), rows, wide, pages, int(page_size), tokens, ws.data_ptr(), nbytes, _lib.raw_stream(index))
    if status:
        _lib.check(status, "dsa_paged_cache_plan")
    return new_table, new_lens, new_refs, slots, positions, ends


def paged_cache_write_slots(caches, rows, slots):
    """Write packed rows into the slots of a plan, in place.

    ``rows[i]`` [T, ...] or [B, S, ...] holds rows of ``caches[i]`` [pages,
    page_size, ...], of its dtype and trailing sizes, outside the caches; batch
    and token strides are free.  ``slots`` (int32 [T] or [B, S]) names each
    token's place, ``page * page_size + offset``; a token whose place lies
    outside the caches (-1) is not written.  No place may be given twice.
    Without a search of tables and lengths in it, this is the form for many
    layers that share one plan.  Returns None.
    """
    if _lib.calls().write_slots(caches, rows, slots):
        return
    caches, rows = _list(caches, "caches"), _list(rows, "rows")
    if len(caches) != len(rows) or not caches:
        raise ValueError(f"one tensor of rows per cache is needed, got {len(rows)} for {len(caches)}")
    pages, page, addresses, sizes = _check_caches(caches)
    if slots.dtype != _INT:
        raise ValueError(f"slots must be int32, got {slots.dtype}")
    lead = slots.dim()
    if lead not in (1, 2):
        raise ValueError(f"slots must be [T] or [B, S], got {tuple(slots.shape)}")
    slots = slots if slots.is_contiguous() else slots.contiguous()
    sources, sb, st, kept = _sources(rows, caches, lead)
    if rows[0].shape[:lead] != slots.shape:
        raise ValueError(f"rows must have the tokens of slots {tuple(slots.shape)}, got {tuple(rows[0].shape)}")
    _lib.no_derivatives("paged_cache_write_slots", *caches, *rows)
    index = _lib.same_device(slots, *caches, *kept)
    if slots.numel() == 0:
        return
    owner, (a_src, a_dst, a_size, a_sb, a_st) = _longs(sources, addresses, sizes, sb, st)
    status = _lib.call_on(
        index, _lib.load().dsa_paged_cache_write_slots, len(caches), a_src, a_dst, a_size, a_sb, a_st,
        slots.data_ptr(), 1 if lead == 1 else slots.shape[0], slots.shape[-1], pages, page, _lib.raw_stream(index))
    if status:
        _lib.check(status, "dsa_paged_cache_write_slots")
    _lib.changed(*caches)


def paged_cache_prefixes(block_table, seq_lengths, page_size, min_tokens=1):
    """Which neighbouring sequences begin with the same pages, for
    ``paged_prefix_attention``: of beams, after a fork, or of requests behind a
    common prompt.

    Row b is linked to the row before it if both sequences begin with the same
    full pages, one page and ``min_tokens`` tokens at least.  Returns
    ``(prefix_groups, prefix_lengths)``, int32 [R]: for each row the first row
    of its run of linked rows, and the tokens that all of the run share: the
    least that two neighbours in it do (whole pages; 0 for a row without links).
    Put rows that share much next to each other; where one neighbour shares
    little of a long common prefix, a ``min_tokens`` above that keeps it apart.
    """
    result = _lib.calls().prefixes(block_table, seq_lengths, page_size, min_tokens)
    if result is not None:
        return result
    table = _ints(block_table, "block_table", 2)
    rows, wide = table.shape
    lens = _ints(seq_lengths, "seq_lengths", 1)
    if lens.shape[0] != rows:
        raise ValueError(f"seq_lengths must have one entry per row of block_table ({rows}), got {lens.shape[0]}")
    if int(page_size) != page_size or page_size < 1:
        raise ValueError(f"page_size must be a positive integer, got {page_size}")
    if int(min_tokens) != min_tokens or not 0 <= min_tokens < 2 ** 31:
        raise ValueError(f"min_tokens must be an integer in [0, 2^31), got {min_tokens}")
    index = _lib.same_device(table, lens)
    groups, lengths = torch.empty_like(lens), torch.empty_like(lens)
    status = _lib.call_on(
        index, _lib.load().dsa_paged_cache_prefixes, table.data_ptr(), lens.data_ptr(), groups.data_ptr(),
        lengths.data_ptr(), rows, wide, int(page_size), int(min_tokens), _lib.raw_stream(index))
    if status:
        _lib.check(status, "dsa_paged_cache_prefixes")
    return groups, lengths


def paged_cache_compact(caches, block_table, page_refs, page_size=None):
    """Move the pages in use to the lowest ids, in all ``caches``, in place.

    With n pages in use (``page_refs`` > 0), those at ids below n stay, and the
    k-th other one moves to the k-th free id below n.  Returns ``(block_table,
    page_refs, page_map)``: the table and the counts for the new ids, and each
    old page's new id (-1: it was free).
    """
    state = _lib.calls().compact(caches, block_table, page_refs, page_size)
    if state is not None:
        return state
    caches = _list(caches, "caches")
    pages, page, addresses, sizes = _check_caches(caches)
    refs = _ints(page_refs, "page_refs", 1)
    n_pages = refs.shape[0]
    if pages is not None and pages != n_pages:
        raise ValueError(f"page_refs must have one entry per page ({pages}), got {n_pages}")
    if page is not None and page_size is not None and page_size != page:
        raise ValueError(f"page_size ({page_size}) must equal the caches' ({page})")
    table = _ints(block_table, "block_table", 2)
    rows, wide = table.shape
    _lib.no_derivatives("paged_cache_compact", *caches)
    index = _lib.same_device(table, refs, *caches)
    new_table, new_refs, page_map = torch.empty_like(table), torch.empty_like(refs), torch.empty_like(refs)
    lib = _lib.load()
    nbytes = lib.dsa_paged_cache_compact_workspace_size(n_pages)
    ws = refs.new_empty((nbytes + 3) // 4)
    owner, (a_caches, a_sizes) = _longs(addresses, sizes)
    status = _lib.call_on(
        index, lib.dsa_paged_cache_compact, len(caches), a_caches, a_sizes, table.data_ptr(), refs.data_ptr(),
        new_table.data_ptr(), new_refs.data_ptr(), page_map.data_ptr(), rows, wide, n_pages,
        1 if page is None else page, ws.data_ptr(), nbytes, _lib.raw_stream(index))
    if status:
        _lib.check(status, "dsa_paged_cache_compact")
    _lib.changed(*caches)
    return new_table, new_refs, page_map
