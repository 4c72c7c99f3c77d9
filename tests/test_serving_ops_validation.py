"""Refusals of the operators that serve requests of many lengths (CPU only, no
kernel launch): the Python functions on CPU tensors, whose checks run before
the device check, and the C entry points with addresses that are never read."""
import ctypes
import os

import pytest
import torch

import dsa_triton_ascend_amd as dsa

BF = torch.bfloat16


def _i(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


# ---- rotary_embedding with sections ----

def _rope(**kw):
    a = dict(query=torch.zeros(2, 3, 4, 64, dtype=BF), key=torch.zeros(2, 3, 1, 64, dtype=BF), positions=_i(3, 2, 3),
             inv_freq=torch.ones(16, dtype=torch.float64), sections=(6, 5, 5))
    a.update(kw)
    return dsa.rotary_embedding(**a)


@pytest.mark.parametrize("kw,match", [
    (dict(sections=()), "one to four"),
    (dict(sections=(4, 4, 4, 2, 2)), "one to four"),
    (dict(sections=(18, -2)), "one to four"),
    (dict(sections=(8.5, 7.5)), "one to four"),
    (dict(sections=(6, 5, 6)), "add up"),
    (dict(sections=(5, 5, 6), sections_interleaved=True), "no room"),
    (dict(sections=(0, 16), positions=_i(2, 2, 3), sections_interleaved=True), "no room"),
    (dict(positions=_i(2, 3)), "positions"),
    (dict(positions=_i(2, 2, 3)), "positions"),
    (dict(positions=_i(3, 2)), "positions"),
    (dict(positions=_i(3, 2, 4)), "positions"),
    (dict(positions=_i(3, 2, 3), sections=None), "positions"),
    (dict(), "ROCm GPU device"),
    (dict(positions=_i(3, 3)), "ROCm GPU device"),
    (dict(sections=(6, 5, 5), sections_interleaved=True), "ROCm GPU device"),
])
def test_rotary_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        _rope(**kw)


# ---- plan, slots, prefixes ----

def _plan(**kw):
    a = dict(block_table=_i(2, 4), seq_lengths=_i(2), page_refs=_i(8), new_lengths=_i(2), page_size=16, tokens=5)
    a.update(kw)
    return dsa.paged_cache_plan(**a)


@pytest.mark.parametrize("kw,match", [
    (dict(block_table=_i(8)), "block_table"),
    (dict(block_table=torch.zeros(2, 4)), "block_table must be int32"),
    (dict(block_table=_i(2, 0)), "block_table"),
    (dict(seq_lengths=_i(3)), "seq_lengths must have one entry"),
    (dict(new_lengths=_i(1)), "new_lengths must have one entry"),
    (dict(new_lengths=torch.zeros(2, dtype=torch.int64)), "new_lengths must be int32"),
    (dict(page_refs=_i(0)), "page_refs"),
    (dict(page_size=0), "page_size"),
    (dict(page_size=1.5), "page_size"),
    (dict(tokens=-1), "tokens"),
    (dict(tokens=2 ** 30 + 1), "tokens"),
    (dict(tokens=0.5), "tokens"),
    (dict(), "ROCm GPU device"),
])
def test_plan_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        _plan(**kw)


def _slots(**kw):
    a = dict(caches=[torch.zeros(8, 16, 1, 64, dtype=BF), torch.zeros(8, 16, 1, 8)],
             rows=[torch.zeros(5, 1, 64, dtype=BF), torch.zeros(5, 1, 8)], slots=_i(5))
    a.update(kw)
    return dsa.paged_cache_write_slots(**a)


@pytest.mark.parametrize("kw,match", [
    (dict(caches=[], rows=[]), "one tensor of rows per cache"),
    (dict(rows=[torch.zeros(5, 1, 64, dtype=BF)]), "one tensor of rows per cache"),
    (dict(slots=torch.zeros(5, dtype=torch.int64)), "int32"),
    (dict(slots=_i(1, 5, 1)), r"\[T\] or \[B, S\]"),
    (dict(slots=_i(4)), "tokens of slots"),
    (dict(slots=_i(1, 5)), "do not fit"),
    (dict(rows=[torch.zeros(5, 1, 64, dtype=BF), torch.zeros(5, 1, 9)]), "do not fit"),
    (dict(rows=[torch.zeros(5, 1, 64, dtype=BF), torch.zeros(6, 1, 8)]), "same tokens"),
    (dict(rows=[torch.zeros(5, 1, 64), torch.zeros(5, 1, 8)]), "dtype"),
    (dict(rows=[torch.zeros(5, 1, 64, dtype=BF), torch.zeros(5, 1, 8, requires_grad=True)]), "no backward"),
    (dict(caches=[torch.zeros(8, 16, 2, 64, dtype=BF)[:, :, :1], torch.zeros(8, 16, 1, 8)]), "contiguous"),
    (dict(), "ROCm GPU device"),
])
def test_slots_refuse(kw, match):
    with pytest.raises(ValueError, match=match):
        _slots(**kw)


def test_slots_refuse_one_cache_twice():
    c = torch.zeros(8, 16, 1, 64)
    with pytest.raises(ValueError, match="overlap"):
        dsa.paged_cache_write_slots([c, c], [torch.zeros(5, 1, 64)] * 2, _i(5))


@pytest.mark.parametrize("kw,match", [
    (dict(block_table=_i(8)), "block_table"),
    (dict(seq_lengths=_i(3)), "one entry"),
    (dict(page_size=0), "page_size"),
    (dict(min_tokens=-1), "min_tokens"),
    (dict(min_tokens=2 ** 31), "min_tokens"),
    (dict(), "ROCm GPU device"),
])
def test_prefixes_refuse(kw, match):
    a = dict(block_table=_i(2, 4), seq_lengths=_i(2), page_size=16)
    a.update(kw)
    with pytest.raises(ValueError, match=match):
        dsa.paged_cache_prefixes(**a)


# ---- the C entry points ----

def _c(name, args, message):
    from dsa_triton_ascend_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    lib = _lib.load()
    status = getattr(lib, name)(*args)
    assert status in (1, 2, 4)
    assert message in lib.dsa_last_error().decode()


P = 0x1000  # an address that no check reads


@pytest.mark.parametrize("change,message", [
    ({0: None}, "null"), ({3: None}, "null"), ({7: None}, "null"), ({9: None}, "null"),
    ({4: P}, "must not be the old ones"), ({10: 0}, "rows"), ({10: 2 ** 24 + 1}, "rows"), ({11: 0}, "at least one"),
    ({11: 2 ** 20 + 1}, "max_blocks"), ({12: 0}, "at least one"), ({13: 0}, "page"), ({13: 2 ** 20 + 1}, "page"),
    ({12: 2 ** 31}, "2^31"), ({14: -1}, "tokens"), ({14: 2 ** 30 + 1}, "tokens"), ({16: 3}, "workspace"),
    ({15: None}, "workspace")])
def test_plan_entry_refuses(change, message):
    a = [P, P + 64, P + 128, P + 192, P + 256, P + 320, P + 384, P + 448, P + 512, P + 576, 4, 4, 16, 16, 8, P + 4096,
         1 << 20, None]
    for i, x in change.items():
        a[i] = x
    _c("dsa_paged_cache_plan", a, message)


@pytest.mark.parametrize("change,message", [
    ({0: None}, "null"), ({3: None}, "null"), ({2: P}, "arrays of their own"), ({4: 0}, "rows"), ({5: 0}, "at least one"),
    ({6: 0}, "page"), ({7: -1}, "min_tokens"), ({7: 2 ** 31}, "min_tokens")])
def test_prefixes_entry_refuses(change, message):
    a = [P + 128, P + 64, P + 192, P, 4, 4, 16, 1, None]
    for i, x in change.items():
        a[i] = x
    _c("dsa_paged_cache_prefixes", a, message)


def _longs(*x):
    return (ctypes.c_int64 * len(x))(*x)


@pytest.mark.parametrize("change,message", [
    ({0: 0}, "null row list"), ({1: None}, "null row list"), ({2: None}, "null cache list"), ({3: _longs(0)}, "cache row"),
    ({4: _longs(-1)}, "strides"), ({5: _longs(2 ** 48)}, "strides"), ({6: None}, "null"), ({7: 0}, "tokens"),
    ({8: 2 ** 31}, "tokens"), ({9: 0}, "at least one"), ({10: 0}, "page"), ({1: _longs(0)}, "null row")])
def test_slots_entry_refuses(change, message):
    a = [1, _longs(P), _longs(P), _longs(64), _longs(64), _longs(64), P, 1, 4, 8, 16, None]
    for i, x in change.items():
        a[i] = x
    _c("dsa_paged_cache_write_slots", a, message)


@pytest.mark.parametrize("change,message", [
    ({29: 0}, "axes"), ({29: 5}, "axes"), ({30: None}, "null sections"), ({30: _longs(6, 5, 6)}, "add up"),
    ({30: _longs(20, -2, -2)}, "sections"), ({30: _longs(5, 5, 6), 31: 1}, "no room"), ({28: 0}, "rotary dim"),
    ({28: 2 ** 40}, "rotary dim"), ({22: None}, "null"), ({26: 0}, "tokens")])
def test_rope_axes_entry_refuses(change, message):
    side = [P, P + 4096, 768, 256, 64, 768, 256, 64, 4, 64, 0]
    a = side + side + [P, 0, 1, P, 2, 3, 32]
    # indexes: 22 positions, 25 inv_freq, 26 batch, 27 s1, 28 rotary_dim
    a += [3, _longs(6, 5, 5), 0, 0, 0, 0, 1.0, None]
    for i, x in change.items():
        a[i] = x
    _c("dsa_rope_axes", a, message)


# ---- paged_prefix_attention ----

def _attn(latent=False, **kw):
    """Arguments of a call with three sequences, four pages of 16 tokens."""
    a = dict(query=torch.zeros(3, 1, 8, 512 if latent else 128, dtype=BF),
             key=torch.zeros(4, 16, 1, 512, dtype=BF) if latent else torch.zeros(4, 16, 2, 128, dtype=BF),
             value=None if latent else torch.zeros(4, 16, 2, 128, dtype=BF), block_table=_i(3, 2),
             actual_seq_lengths_kv=_i(3), prefix_groups=_i(3), prefix_lengths=_i(3))
    if latent:
        a.update(query_rope=torch.zeros(3, 1, 8, 64, dtype=BF), key_rope=torch.zeros(4, 16, 1, 64, dtype=BF))
    a.update(kw)
    return dsa.paged_prefix_attention(**a)


@pytest.mark.parametrize("latent", [False, True])
@pytest.mark.parametrize("kw,match", [
    (dict(prefix_groups=None), "prefix_groups and prefix_lengths are required"),
    (dict(prefix_lengths=None), "prefix_groups and prefix_lengths are required"),
    (dict(actual_seq_lengths_kv=None), "are required"),
    (dict(block_table=_i(2, 2)), "block_table"),
    (dict(sparse_mode=2), "sparse_mode"),
    (dict(query=torch.zeros(3, 1, 8, 96, dtype=BF)), "columns"),
    (dict(query=torch.zeros(3, 1, 8, 128)), "columns|dtype|must be"),
    (dict(query=torch.zeros(3, 8, 128, dtype=BF)), "query must be"),
    (dict(pre_tokens="x"), "pre_tokens|invalid literal"),
    (dict(min_tokens=-1), "min_tokens"),
    (dict(min_tokens=0.5), "min_tokens"),
    (dict(min_tokens=2 ** 63), "min_tokens"),
    (dict(), "ROCm GPU device"),
])
def test_prefix_attention_refuses(latent, kw, match):
    with pytest.raises(ValueError, match=match):
        _attn(latent, **kw)


@pytest.mark.parametrize("latent,kw,match", [
    (False, dict(value=None), "query_rope and key_rope"),
    (False, dict(query_rope=torch.zeros(3, 1, 8, 64, dtype=BF)), "no rope parts"),
    (False, dict(query=torch.zeros(3, 1, 7, 128, dtype=BF)), "multiple"),
    (False, dict(value=torch.zeros(4, 16, 2, 64, dtype=BF)), "value"),
    (False, dict(value=torch.zeros(4, 16, 2, 128)), "dtype"),
    (True, dict(query_rope=torch.zeros(3, 1, 8, 32, dtype=BF)), "query_rope"),
    (True, dict(key=torch.zeros(4, 16, 2, 512, dtype=BF), key_rope=torch.zeros(4, 16, 2, 64, dtype=BF)), "one key head"),
])
def test_prefix_attention_forms_refuse(latent, kw, match):
    with pytest.raises(ValueError, match=match):
        _attn(latent, **kw)


@pytest.mark.parametrize("name", ["query", "key", "value"])
def test_prefix_attention_has_no_backward(name):
    t = torch.zeros(3, 1, 8, 128, dtype=BF) if name == "query" else torch.zeros(4, 16, 2, 128, dtype=BF)
    with pytest.raises(ValueError, match="paged_prefix_attention has no backward"):
        _attn(**{name: t.requires_grad_()})


@pytest.mark.parametrize("change,message", [
    ({0: None}, "null"), ({2: None}, "null"), ({5: None}, "null"), ({9: None}, "null"), ({10: None}, "null"),
    ({11: None}, "null"), ({12: None}, "null"), ({1: P}, "no rope parts"), ({4: None}, "query_rope and key_rope"),
    ({7: None}, "softmax_max and softmax_sum"), ({13: 0}, "batch"), ({13: 2 ** 24 + 1}, "batch"), ({14: 0}, "S1"),
    ({15: 7}, "divisible"), ({17: 96}, "D must be"), ({19: 0}, "at least one"), ({20: 0}, "page"),
    ({21: 2 ** 20 + 1}, "max_blocks"), ({14: 2 ** 22}, "query rows"), ({22: 1}, "sparse_mode"), ({26: 2}, "dtype"),
    ({29: None}, "workspace"), ({30: 100}, "workspace"), ({29: P + 8}, "16-byte"), ({0: P + 2}, "16-byte")])
def test_prefix_attention_entry_refuses(change, message):
    a = [P, None, P, None, P, P, P, P, None, P, P, P, P, 3, 1, 8, 2, 128, 0, 8, 16, 4, 3, 2 ** 62, 2 ** 62, -1, 0, 0.1,
         1, P, 1 << 40, None]
    for i, x in change.items():
        a[i] = x
    _c("dsa_paged_prefix_attn", a, message)


@pytest.mark.parametrize("change", [
    {0: 0}, {0: 2 ** 24 + 1}, {1: 0}, {2: 7}, {3: 0}, {4: 96}, {4: 512}, {5: 1}, {6: 0}, {6: 2 ** 20 + 1}, {7: 0},
    {7: 2 ** 20 + 1}, {1: 2 ** 62}, {6: 2 ** 62}])
def test_prefix_attention_workspace_of_no_call_is_zero(change):
    from dsa_triton_ascend_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    a = [3, 1, 8, 2, 128, 0, 4, 16]
    size = _lib.load().dsa_paged_prefix_attn_workspace_size
    assert size(*a) > 0
    for i, x in change.items():
        a[i] = x
    assert size(*a) == 0
