"""Refusals of the paged decoding operators (CPU only, no kernel launch): the
Python functions on CPU tensors, whose checks run before the device check, and
the C entry points with addresses that are never read."""
import ctypes
import os

import pytest
import torch

import dsa_triton_ascend_amd as dsa

BF = torch.bfloat16


def _i(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


# ---- rotary_embedding ----

def _rope(**kw):
    a = dict(query=torch.zeros(2, 3, 4, 64, dtype=BF), key=torch.zeros(2, 3, 1, 64, dtype=BF), positions=_i(2, 3),
             inv_freq=torch.ones(16, dtype=torch.float64))
    a.update(kw)
    return dsa.rotary_embedding(**a)


@pytest.mark.parametrize("kw,match", [
    (dict(layout="SBND"), "layout"),
    (dict(positions=None), "required"),
    (dict(inv_freq=None), "required"),
    (dict(query=torch.zeros(6, 4, 64, dtype=BF)), "query must be"),
    (dict(query=torch.zeros(2, 3, 4, 64, dtype=torch.float64)), "dtype"),
    (dict(key=torch.zeros(2, 3, 1, 64)), "key dtype"),
    (dict(key=torch.zeros(2, 4, 1, 64, dtype=BF)), "batch and tokens"),
    (dict(positions=_i(2, 4)), "positions"),
    (dict(positions=_i(4)), "positions"),
    (dict(positions=torch.zeros(2, 3)), "int32 or int64"),
    (dict(inv_freq=torch.ones(2, 8)), "vector"),
    (dict(inv_freq=torch.ones(0)), "vector"),
    (dict(inv_freq=torch.ones(33)), "do not lie inside"),
    (dict(rotary_offset=33), "do not lie inside"),
    (dict(rotary_offset=-1), "do not lie inside"),
    (dict(rotary_offset=0.5), "do not lie inside"),
    (dict(key_rotary_offset=40), "key"),
    (dict(query=torch.zeros(2, 3, 4, 64, requires_grad=True), key=None, inplace=True), "inference"),
    (dict(query=torch.zeros(2, 3, 1, 64, dtype=BF).expand(2, 3, 4, 64), inplace=True), "share memory"),
    (dict(query=torch.zeros(2, 3, 64, 4, dtype=BF).transpose(2, 3), inplace=True), "next to each other"),
    (dict(), "ROCm GPU device"),
])
def test_rotary_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        _rope(**kw)


def test_rotary_in_place_refuses_one_tensor_as_both():
    q = torch.zeros(2, 3, 4, 64, dtype=BF)
    with pytest.raises(ValueError, match="of their own"):
        _rope(query=q, key=q, inplace=True)


@pytest.mark.parametrize("kw,match", [
    (dict(dim=3), "even"), (dict(dim=0), "even"), (dict(dim=8, scaling="x"), "scaling"), (dict(dim=8, factor=0), "positive"),
    (dict(dim=8, base=-1), "positive"), (dict(dim=2, scaling="ntk", factor=2), "4 columns"),
    (dict(dim=8, scaling="yarn", beta_fast=1, beta_slow=2), "beta_fast"), (dict(dim=8, scaling="yarn", base=1.0), "base"),
])
def test_rotary_frequencies_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        dsa.rotary_frequencies(device="cpu", **kw)


# ---- pages ----

def _write(**kw):
    a = dict(caches=[torch.zeros(5, 4, 1, 8, dtype=BF)], rows=[torch.zeros(2, 3, 1, 8, dtype=BF)], block_table=_i(2, 3),
             seq_lengths=_i(2))
    a.update(kw)
    return dsa.paged_cache_write(**a)


@pytest.mark.parametrize("kw,match", [
    (dict(rows=[]), "one tensor of rows"),
    (dict(caches=[], rows=[]), "one tensor of rows"),
    (dict(layout="PA_BSND"), "layout"),
    (dict(layout="TND", rows=[torch.zeros(6, 1, 8, dtype=BF)]), "row_lengths"),
    (dict(caches=[torch.zeros(5, 4)]), "a cache must be"),
    (dict(caches=[torch.zeros(4, 5, 1, 8, dtype=BF).transpose(0, 1)]), "contiguous"),
    (dict(caches=[torch.zeros(5, 0, 1, 8, dtype=BF)]), "not be empty"),
    (dict(block_table=torch.zeros(2, 3)), "int32"),
    (dict(block_table=_i(2)), "block_table"),
    (dict(block_table=_i(2, 0)), "block_table"),
    (dict(seq_lengths=_i(3)), "seq_lengths"),
    (dict(seq_lengths=torch.zeros(2, dtype=torch.int64)), "int32"),
    (dict(row_lengths=_i(3)), "row_lengths"),
    (dict(rows=[torch.zeros(2, 3, 1, 9, dtype=BF)]), "do not fit"),
    (dict(rows=[torch.zeros(3, 3, 1, 8, dtype=BF)]), "B=2"),
    (dict(rows=[torch.zeros(2, 3, 1, 8)]), "dtype"),
    (dict(), "ROCm GPU device"),
])
def test_write_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        _write(**kw)


def test_write_refuses_caches_that_differ_or_repeat():
    c = torch.zeros(5, 4, 1, 8, dtype=BF)
    rows = [torch.zeros(2, 3, 1, 8, dtype=BF)] * 2
    with pytest.raises(ValueError, match="same pages"):
        _write(caches=[c, torch.zeros(6, 4, 1, 8, dtype=BF)], rows=rows)
    with pytest.raises(ValueError, match="given twice"):
        _write(caches=[c, c], rows=rows)
    with pytest.raises(ValueError, match="tensors"):
        _write(caches=[c, None], rows=rows)


@pytest.mark.parametrize("kw,match", [
    (dict(page_refs=_i(6)), "one entry per page"),
    (dict(page_refs=torch.zeros(5)), "int32"),
    (dict(block_table=_i(3, 2), seq_lengths=_i(2)), "seq_lengths"),
    (dict(parents=torch.zeros(4, dtype=torch.int64)), "int32"),
    (dict(parents=_i(0)), "parents"),
    (dict(new_tokens=-1), "new_tokens"),
    (dict(new_tokens=1.5), "new_tokens"),
    (dict(page_size=8), "page_size"),
    (dict(caches=[]), "page_size is required"),
    (dict(), "ROCm GPU device"),
])
def test_fork_refuses(kw, match):
    a = dict(caches=[torch.zeros(5, 4, 1, 8)], block_table=_i(2, 3), seq_lengths=_i(2), page_refs=_i(5))
    a.update(kw)
    with pytest.raises(ValueError, match=match):
        dsa.paged_cache_fork(**a)


@pytest.mark.parametrize("kw,match", [
    (dict(page_refs=_i(6)), "one entry per page"),
    (dict(block_table=_i(6)), "block_table"),
    (dict(page_size=8), "page_size"),
    (dict(), "ROCm GPU device"),
])
def test_compact_refuses(kw, match):
    a = dict(caches=[torch.zeros(5, 4, 1, 8)], block_table=_i(2, 3), page_refs=_i(5))
    a.update(kw)
    with pytest.raises(ValueError, match=match):
        dsa.paged_cache_compact(**a)


# ---- paged_attention ----

def _attn(latent=False, **kw):
    d, n2 = (512, 1) if latent else (128, 2)
    a = dict(query=torch.zeros(2, 1, 8, d, dtype=BF), key=torch.zeros(5, 4, n2, d, dtype=BF),
             value=None if latent else torch.zeros(5, 4, n2, d, dtype=BF), block_table=_i(2, 3),
             actual_seq_lengths_kv=[3, 4])
    if latent:
        a.update(query_rope=torch.zeros(2, 1, 8, 64, dtype=BF), key_rope=torch.zeros(5, 4, 1, 64, dtype=BF))
    a.update(kw)
    return dsa.paged_attention(**a)


@pytest.mark.parametrize("kw,match", [
    (dict(sparse_mode=1), "sparse_mode"),
    (dict(pre_tokens=0.5), "pre_tokens"),
    (dict(value=None), "latent form"),
    (dict(query_rope=torch.zeros(2, 1, 8, 64, dtype=BF)), "grouped form"),
    (dict(query=torch.zeros(2, 8, 128, dtype=BF)), "query must be"),
    (dict(key=torch.zeros(5, 4, 2, 64, dtype=BF)), "columns"),
    (dict(query=torch.zeros(2, 1, 8, 96, dtype=BF), key=torch.zeros(5, 4, 2, 96, dtype=BF)), "D must be"),
    (dict(query=torch.zeros(2, 1, 7, 128, dtype=BF)), "multiple"),
    (dict(query=torch.zeros(2, 1, 8, 128)), "bfloat16 or float16"),
    (dict(key=torch.zeros(5, 4, 2, 128)), "key dtype"),
    (dict(value=torch.zeros(5, 4, 2, 64, dtype=BF)), "value"),
    (dict(block_table=_i(1, 3)), "block_table"),
    (dict(block_table=None), "required"),
    (dict(actual_seq_lengths_kv=None), "required"),
    (dict(query=torch.zeros(2, 1, 8, 128, dtype=BF, requires_grad=True)), "no backward"),
    (dict(), "ROCm GPU device"),
])
def test_grouped_attention_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        _attn(**kw)


@pytest.mark.parametrize("kw,match", [
    (dict(key_rope=None), "latent form"),
    (dict(key=torch.zeros(5, 4, 2, 512, dtype=BF)), "one key head"),
    (dict(query=torch.zeros(2, 1, 8, 64, dtype=BF), key=torch.zeros(5, 4, 1, 64, dtype=BF)), "D must be"),
    (dict(query_rope=torch.zeros(2, 1, 8, 32, dtype=BF)), "query_rope"),
    (dict(key_rope=torch.zeros(4, 5, 1, 64, dtype=BF)), "key_rope"),
    (dict(key_rope=torch.zeros(5, 4, 1, 64)), "key_rope dtype"),
    (dict(), "ROCm GPU device"),
])
def test_latent_attention_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        _attn(latent=True, **kw)


# ---- C entry points ----

def _lib():
    from dsa_triton_ascend_amd import _lib as L
    if not os.path.exists(L.LIB_PATH):
        pytest.skip("libdsa_hip.so not built")
    return L.load()


A = 0x10000  # an address that is never read


def _c(defaults, kw):
    a = dict(defaults)
    a.update(kw)
    return list(a.values())


ROPE = dict(q=A, qo=A, s0=64, s1=64, s2=64, o0=64, o1=64, o2=64, qh=1, qd=64, qs=0, k=None, ko=None, k0=0, k1=0, k2=0,
            l0=0, l1=0, l2=0, kh=0, kd=0, ks=0, pos=A, p64=0, per=1, inv=A, b=1, s=1, rot=64, inter=0, inverse=0,
            dtype=0, scale=1.0, stream=None)


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), 1), (dict(qo=None), 1), (dict(pos=None), 1), (dict(inv=None), 1), (dict(k=A), 1), (dict(dtype=3), 2),
    (dict(rot=63), 2), (dict(rot=0), 2), (dict(rot=2048, qd=4096), 2), (dict(b=0), 1), (dict(s=0), 1), (dict(qh=0), 1),
    (dict(qs=1), 1), (dict(qs=-1), 1), (dict(s0=-1), 1), (dict(qd=1 << 21, qh=1), 1), (dict(k=A, ko=A, kh=1, kd=32), 1),
])
def test_c_rope_refuses(kw, code):
    lib = _lib()
    assert lib.dsa_rope(*_c(ROPE, kw)) == code and lib.dsa_last_error()


def _list(kind, *values):
    return (kind * max(1, len(values)))(*values)


def _wargs(**kw):
    p, n = ctypes.c_void_p, ctypes.c_int64
    return _c(dict(n=1, rows=_list(p, A), caches=_list(p, A), bytes=_list(n, 128), sb=_list(n, 128), st=_list(n, 128),
                   table=A, lens=A, new=None, b=2, s=3, tokens=6, blocks=4, pages=8, page=16, layout=0, stream=None), kw)


@pytest.mark.parametrize("kw,code", [
    (dict(n=0), 1), (dict(rows=None), 1), (dict(caches=None), 1), (dict(bytes=None), 1), (dict(table=None), 1),
    (dict(lens=None), 1), (dict(caches=_list(ctypes.c_void_p, None)), 1), (dict(rows=_list(ctypes.c_void_p, None)), 1),
    (dict(bytes=_list(ctypes.c_int64, 0)), 2), (dict(sb=_list(ctypes.c_int64, -1)), 1), (dict(page=0), 1),
    (dict(page=1 << 21), 1), (dict(pages=0), 1), (dict(blocks=0), 1), (dict(pages=1 << 30), 1), (dict(layout=2), 2),
    (dict(layout=1), 1), (dict(tokens=7), 1), (dict(tokens=0), 1), (dict(b=0), 1), (dict(n=1 << 20), 1),
])
def test_c_write_refuses(kw, code):
    lib = _lib()
    assert lib.dsa_paged_cache_write(*_wargs(**kw)) == code and lib.dsa_last_error()


def _fargs(**kw):
    p, n = ctypes.c_void_p, ctypes.c_int64
    return _c(dict(n=1, caches=_list(p, A), bytes=_list(n, 128), table=A, lens=A, refs=A, parents=A, nt=2 * A, nl=2 * A,
                   nr=2 * A, rows=2, kids=3, blocks=4, nblocks=4, pages=8, page=16, new=1, ws=A, bytes2=1 << 20,
                   stream=None), kw)


@pytest.mark.parametrize("kw,code", [
    (dict(table=None), 1), (dict(nr=None), 1), (dict(caches=None), 1), (dict(rows=0), 1), (dict(kids=0), 1),
    (dict(parents=None), 1), (dict(new=-1), 1), (dict(new=1 << 31), 1), (dict(nt=A), 1), (dict(nr=A), 1),
    (dict(nblocks=0), 1), (dict(nblocks=(1 << 20) + 1), 1), (dict(page=0), 1), (dict(ws=None), 4), (dict(bytes2=4), 4),
])
def test_c_fork_refuses(kw, code):
    lib = _lib()
    assert lib.dsa_paged_cache_fork(*_fargs(**kw)) == code and lib.dsa_last_error()


def _cargs(**kw):
    p, n = ctypes.c_void_p, ctypes.c_int64
    return _c(dict(n=1, caches=_list(p, A), bytes=_list(n, 128), table=A, refs=A, nt=A, nr=2 * A, map=3 * A, rows=2,
                   blocks=4, pages=8, page=16, ws=A, bytes2=1 << 20, stream=None), kw)


@pytest.mark.parametrize("kw,code", [
    (dict(table=None), 1), (dict(map=None), 1), (dict(nr=A), 1), (dict(map=2 * A), 1), (dict(rows=0), 1),
    (dict(pages=0), 1), (dict(ws=None), 4), (dict(bytes2=0), 4), (dict(n=-1), 1),
])
def test_c_compact_refuses(kw, code):
    lib = _lib()
    assert lib.dsa_paged_cache_compact(*_cargs(**kw)) == code and lib.dsa_last_error()


ATTN = dict(q=A, qr=None, k=A, kr=None, v=A, out=A, mx=A, sm=A, aq=None, ak=A, table=A, b=2, s1=1, n1=8, n2=2, d=128,
            dr=0, pages=8, page=16, blocks=4, mode=3, pre=1 << 62, nxt=1 << 62, dtype=0, scale=0.1, lse=1, ws=A,
            bytes=1 << 62, stream=None)


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), 1), (dict(k=None), 1), (dict(out=None), 1), (dict(ak=None), 1), (dict(table=None), 1),
    (dict(mx=None), 1), (dict(mx=None, sm=None), 1), (dict(dtype=2), 2), (dict(mode=1), 2), (dict(d=96), 2),
    (dict(d=512), 2), (dict(qr=A), 1), (dict(dr=64), 1), (dict(n1=7), 1), (dict(n2=0), 1), (dict(b=0), 1), (dict(s1=0), 1),
    (dict(v=None), 1), (dict(v=None, qr=A, kr=A, dr=64, n2=2), 2), (dict(v=None, qr=A, kr=A, dr=32, n2=1), 2),
    (dict(v=None, qr=A, kr=A, dr=64, n2=1, d=64), 2), (dict(page=0), 1), (dict(blocks=1 << 21), 1),
    (dict(pages=1 << 30), 1), (dict(k=A + 8), 1), (dict(ws=None), 4), (dict(bytes=16), 4), (dict(ws=A + 4), 1),
    (dict(b=1 << 20, s1=1 << 12, n1=8), 1),
])
def test_c_attention_refuses(kw, code):
    lib = _lib()
    assert lib.dsa_paged_attn(*_c(ATTN, kw)) == code and lib.dsa_last_error()


def test_workspace_sizes():
    lib = _lib()
    assert lib.dsa_paged_attn_workspace_size(2, 1, 8, 2, 128, 0, 4, 16) > 0
    assert lib.dsa_paged_attn_workspace_size(2, 1, 8, 2, 96, 0, 4, 16) == 0
    assert lib.dsa_paged_attn_workspace_size(1 << 24, 1 << 24, 8, 2, 128, 0, 4, 16) == 0
    assert lib.dsa_paged_cache_fork_workspace_size(0, 1, 1) == 0
    assert lib.dsa_paged_cache_fork_workspace_size(2, 3, 8) == 4 * (2 + 6 + 8)
    assert lib.dsa_paged_cache_compact_workspace_size(0) == 0
    assert lib.dsa_paged_cache_compact_workspace_size(1025) == 4 * (2 + 3 * 1025)


def test_tables_that_name_too_many_tokens_are_refused():
    lib = _lib()
    big = dict(b=1 << 11, blocks=1 << 20, page=32)  # 2^36
    assert lib.dsa_paged_attn(*_c(ATTN, big)) == 2 and b"2^35" in lib.dsa_last_error()
    assert lib.dsa_paged_attn_workspace_size(1 << 11, 1, 8, 2, 128, 0, 1 << 20, 32) == 0


def test_caches_that_overlap_are_refused():
    pool = torch.zeros(8, 4, 1, 8, dtype=BF)
    rows = [torch.zeros(2, 3, 1, 8, dtype=BF)] * 2
    with pytest.raises(ValueError, match="overlap"):
        _write(caches=[pool[3:8], pool[0:5]], rows=rows)


# ---- derivatives ----

@pytest.mark.parametrize("which", ["caches", "rows"])
def test_write_refuses_what_requires_grad(which):
    c, r = torch.zeros(5, 4, 1, 8), torch.zeros(2, 3, 1, 8)
    a = dict(caches=[c, c.clone()], rows=[r, r.clone()])
    a[which][1].requires_grad_()
    with pytest.raises(ValueError, match="paged_cache_write has no backward"):
        _write(**a)
    with torch.no_grad(), pytest.raises(ValueError, match="ROCm GPU device"):
        _write(**a)


def test_fork_and_compact_refuse_caches_that_require_grad():
    c = torch.zeros(5, 4, 1, 8, requires_grad=True)
    for f in (lambda: dsa.paged_cache_fork([c], _i(2, 3), _i(2), _i(5)),
              lambda: dsa.paged_cache_compact([c * 2], _i(2, 3), _i(5))):
        with pytest.raises(ValueError, match="has no backward"):
            f()
        with torch.no_grad(), pytest.raises(ValueError, match="ROCm GPU device"):
            f()


def test_operators_without_derivatives_refuse_tangents():
    import torch.autograd.forward_ad as fwad
    with fwad.dual_level(), torch.no_grad():
        def dual(*shape, dtype=torch.float32):
            return fwad.make_dual(torch.zeros(*shape, dtype=dtype), torch.ones(*shape, dtype=dtype))

        for f in (lambda: _write(caches=[torch.zeros(5, 4, 1, 8)], rows=[dual(2, 3, 1, 8)]),
                  lambda: _write(caches=[dual(5, 4, 1, 8)], rows=[torch.zeros(2, 3, 1, 8)]),
                  lambda: dsa.paged_cache_fork([dual(5, 4, 1, 8)], _i(2, 3), _i(2), _i(5)),
                  lambda: dsa.paged_cache_compact([dual(5, 4, 1, 8)], _i(2, 3), _i(5)),
                  lambda: _attn(query=dual(2, 1, 8, 128, dtype=BF)),
                  lambda: _attn(latent=True, key_rope=dual(5, 4, 1, 64, dtype=BF))):
            with pytest.raises(ValueError, match="tangents"):
                f()


# ---- in place: query and key in one piece of memory ----

def _views(rng, flat):
    """A query and a key as strided views of one buffer, often apart, often not:
    (query, its rotated columns' start, key, start, columns)."""
    B, S, cols = rng.randint(1, 3), rng.randint(1, 4), 2 * rng.randint(1, 3)
    heads = [rng.randint(1, 3), rng.randint(1, 3)]
    pitch = rng.choice([cols, cols + 1, 2 * cols, 3 * cols])
    row = rng.choice([sum(heads) * pitch, (sum(heads) + 2) * pitch, max(heads) * pitch])
    seq = rng.choice([S * row, S * row + 3, (S + 1) * row])
    out = []
    for h, at in zip(heads, (rng.randint(0, 5), rng.choice([heads[0] * pitch, rng.randint(0, 4 * row), B * seq]))):
        d = rng.randint(cols, pitch)
        step = (seq, row) if rng.random() < 0.7 else (row, B * row)
        t = torch.as_strided(flat, (B, S, h, d), (*step, pitch, 1), at)
        out += [t, rng.randint(0, d - cols)]
    return (*out, cols)


def _shared(q, qs, k, ks, cols):
    at = torch.arange(1 << 14)
    a, b = (torch.as_strided(at, (*t.shape[:-1], cols), t.stride(), t.storage_offset() + s) for t, s in ((q, qs), (k, ks)))
    return bool(set(a.flatten().tolist()) & set(b.flatten().tolist()))


def test_views_that_share_memory_are_told_from_those_that_do_not():
    import random

    from dsa_triton_ascend_amd.rotary_embedding import _overlaps_itself, _share_memory
    rng, flat, seen = random.Random(0), torch.zeros(1 << 14), [0, 0]
    for _ in range(3000):
        q, qs, k, ks, cols = _views(rng, flat)
        if not _overlaps_itself(q) and not _overlaps_itself(k):
            want = _shared(q, qs, k, ks, cols)
            assert _share_memory(q, qs, k, ks, cols) == want, (q.shape, q.stride(), qs, k.shape, k.stride(), ks, cols)
            seen[want] += 1
    assert min(seen) > 300, seen


def test_rotary_in_place_refuses_views_that_share_columns():
    proj = torch.zeros(2, 3, 6, 64, dtype=BF)
    with pytest.raises(ValueError, match="share memory"):
        _rope(query=proj[:, :, :4], key=proj[:, :, 3:], inplace=True)
    with pytest.raises(ValueError, match="share memory"):  # columns 32 .. 63 of one, 24 .. 55 of the other
        _rope(query=proj[:, :, :4], key=proj[..., 8:][:, :, :1], rotary_offset=32, key_rotary_offset=16, inplace=True)
    for q, k in ((proj[:, :, :4], proj[:, :, 4:]),          # heads of their own
                 (proj[..., :40], proj[:, :, :1, 32:])):    # columns 0 .. 31 and 32 .. 63
        with pytest.raises(ValueError, match="ROCm GPU device"):
            _rope(query=q, key=k, inplace=True)


# ---- launches: fewer than 2^32 threads, checked before the first kernel of a call ----

def test_launches_of_too_many_threads_are_refused():
    lib = _lib()
    p, n = ctypes.c_void_p, ctypes.c_int64
    many = dict(b=1, s=1 << 24, qh=64, per=0)                 # 2^24 tokens of 512 pieces of 16 bytes
    assert lib.dsa_rope(*_c(ROPE, many)) == 2 and b"launch" in lib.dsa_last_error()
    big = dict(bytes=_list(n, 4096), sb=_list(n, 4096), st=_list(n, 4096), b=1 << 24, s=1, tokens=1 << 24)
    assert lib.dsa_paged_cache_write(*_wargs(**big)) == 2 and b"too many rows" in lib.dsa_last_error()
    # the 33rd cache's launch is too large, that of the 32 before it is not
    wide = dict(n=33, rows=_list(p, *[A] * 33), caches=_list(p, *[A] * 33), sb=_list(n, *[4096] * 33),
                st=_list(n, *[4096] * 33), bytes=_list(n, *[1] * 32, 4096), b=1 << 24, s=1, tokens=1 << 24)
    assert lib.dsa_paged_cache_write(*_wargs(**wide)) == 2
    fork = dict(rows=1 << 24, kids=1 << 24, bytes2=1 << 40)
    assert lib.dsa_paged_cache_fork(*_fargs(**fork)) == 2 and b"too many rows" in lib.dsa_last_error()
    fork = dict(n=33, caches=_list(p, *[A] * 33), bytes=_list(n, *[128] * 32, 1 << 20), rows=1 << 18, kids=1 << 18,
                bytes2=1 << 40)
    assert lib.dsa_paged_cache_fork(*_fargs(**fork)) == 2
    for kw in (dict(b=1 << 16, n1=1024, n2=1), dict(b=1 << 16, s1=8, n1=128, n2=1, v=None, qr=A, kr=A, dr=64)):
        assert lib.dsa_paged_attn(*_c(ATTN, kw)) == 2 and b"launch" in lib.dsa_last_error()
    size = lib.dsa_paged_attn_workspace_size
    assert size(1 << 16, 1, 1024, 1, 128, 0, 4, 16) == 0 and size((1 << 16) - 1, 1, 1024, 1, 128, 0, 4, 16) > 0
    assert size(1 << 16, 8, 128, 1, 512, 1, 4, 16) == 0 and size((1 << 16) - 1, 8, 128, 1, 512, 1, 4, 16) > 0


# ---- the compiled calls ----

def test_compiled_calls_that_do_not_load_are_done_without(tmp_path):
    """In a process of its own, with the package beside a _torch_calls that the
    loader refuses, as it does one built for another torch."""
    import subprocess
    import sys
    _lib()
    pkg = os.path.dirname(os.path.abspath(dsa.__file__))
    (tmp_path / "dsa_triton_ascend_amd").mkdir()
    for name in os.listdir(pkg):
        if name not in ("_torch_calls.so", "__pycache__"):
            os.symlink(os.path.join(pkg, name), tmp_path / "dsa_triton_ascend_amd" / name)
    (tmp_path / "dsa_triton_ascend_amd" / "_torch_calls.so").write_bytes(b"not a library")
    code = ("import warnings, torch; warnings.simplefilter('always')\n"
            "import dsa_triton_ascend_amd as dsa\n"
            "from dsa_triton_ascend_amd import _lib\n"
            "print(_lib.calls() is _lib._NoCalls, _lib.calls() is _lib._NoCalls)\n"
            "try:\n    dsa.paged_cache_compact([], torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))\n"
            "except ValueError as e:\n    print(e)\n")
    env = dict(os.environ, PYTHONPATH=str(tmp_path), DSA_HIP_LIB=os.path.join(pkg, "libdsa_hip.so"))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, env=env, cwd=tmp_path, timeout=300)
    assert r.returncode == 0, r.stderr
    assert r.stdout.startswith("True True\n") and "ROCm GPU device" in r.stdout
    assert r.stderr.count("does not load") == 1


def test_compiled_calls_have_no_thread_local_data():
    """A module loaded after the library whose thread-local data nobody uses
    makes each such access of the process slow (with glibc before 2.39)."""
    import struct

    from dsa_triton_ascend_amd import _lib as L
    if not os.path.exists(L.CALLS_PATH):
        pytest.skip("_torch_calls.so not built")
    with open(L.CALLS_PATH, "rb") as f:
        elf = f.read()
    assert elf[:6] == b"\x7fELF\x02\x01"
    at, size, count = struct.unpack_from("<Q", elf, 32)[0], *struct.unpack_from("<HH", elf, 54)
    types = [struct.unpack_from("<I", elf, at + i * size)[0] for i in range(count)]
    assert 1 in types and 7 not in types  # PT_LOAD, PT_TLS
