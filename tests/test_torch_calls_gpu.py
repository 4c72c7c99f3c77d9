"""Ordinary calls of the paged decoding operators by way of _torch_calls and
by way of Python: the same results, bit for bit; what is not an ordinary call
is left to Python."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

I32 = torch.int32


def _state(dtype=torch.bfloat16, heads=1, cols=64):
    g = torch.Generator(device="cuda").manual_seed(3)
    caches = [torch.randn(9, 16, heads, c, generator=g, device="cuda").to(dtype) for c in (cols, 64)]
    table = torch.tensor([[3, 1, -1], [5, 8, 0]], dtype=I32, device="cuda")
    lens = torch.tensor([20, 40], dtype=I32, device="cuda")
    refs = torch.zeros(9, dtype=I32, device="cuda")
    refs[[3, 1, 5, 8, 0]] = 1
    return caches, table, lens, refs


def _both(monkeypatch, f):
    """f() with and without the module; whether the module took it is in _taken."""
    from dsa_triton_ascend_amd import _lib
    assert _lib.calls() is not _lib._NoCalls
    a = f()
    monkeypatch.setattr(_lib, "_calls", _lib._NoCalls)
    b = f()
    monkeypatch.undo()
    for x, y in zip(a, b):
        assert (x is None) == (y is None)
        if x is not None:
            assert x.shape == y.shape and x.dtype == y.dtype and x.stride() == y.stride() and torch.equal(x, y)


@pytest.mark.parametrize("layout,key,shared", [("BSND", True, False), ("BSND", False, True), ("TND", True, False)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rotary(monkeypatch, layout, key, shared, dtype):
    import dsa_triton_ascend_amd as dsa
    lead = (3, 5) if layout == "BSND" else (7,)
    q = torch.randn(*lead, 6, 96, device="cuda").to(dtype)[..., :5, 16:]  # strided
    k = torch.randn(*lead, 2, 64, device="cuda").to(dtype) if key else None
    pos = torch.arange(5, device="cuda") + 9 if shared else torch.randint(0, 9999, lead, device="cuda", dtype=I32)
    inv, _ = dsa.rotary_frequencies(32)
    _both(monkeypatch, lambda: dsa.rotary_embedding(q, k, pos, inv, interleaved=key, rotary_offset=32,
                                                    attention_scale=1.25, layout=layout, inverse=shared))

    def in_place():
        packed = torch.cat([q] * 2, -1)
        x, y = packed[..., :80], None if k is None else k.clone()
        return dsa.rotary_embedding(x, y, pos, inv, rotary_offset=32, layout=layout, inplace=True) + (packed,)

    _both(monkeypatch, in_place)


@pytest.mark.parametrize("sides", ["both", "query", "key", "query alone"])
@pytest.mark.parametrize("how", ["dense", "strided", "broadcast", "missing"])
def test_rotary_gradients(monkeypatch, sides, how):
    import dsa_triton_ascend_amd as dsa
    pos = torch.randint(0, 9999, (2, 5), device="cuda")
    inv, _ = dsa.rotary_frequencies(32)
    g = torch.Generator(device="cuda").manual_seed(5)
    base = [torch.randn(2, 5, n, 64, generator=g, device="cuda") for n in (4, 2)]
    up = [torch.randn(2, 5, n, 64, generator=g, device="cuda") for n in (4, 2)]
    if how == "strided":
        up = [x.transpose(2, 3).contiguous().transpose(2, 3) for x in up]  # columns apart
    elif how == "broadcast":
        up = [x[:, :1, :, :1].expand_as(x) for x in up]

    def run():
        q, k = (x.clone().requires_grad_(sides != other) for x, other in zip(base, ("key", "query")))
        out = dsa.rotary_embedding(q, None if sides == "query alone" else k, pos, inv, rotary_offset=16,
                                   key_rotary_offset=32, attention_scale=0.75)
        outs = [t for t in out if t is not None]
        assert all(t.requires_grad for t in outs)
        keep = slice(0, 1) if how == "missing" else slice(None)
        leaves = [t for t in (q, k) if t.requires_grad and not (t is k and sides == "query alone")]
        return torch.autograd.grad(outs[keep], leaves, up[:len(outs)][keep], allow_unused=how == "missing")

    _both(monkeypatch, run)


def test_rotary_gradients_in_a_graph_on_a_stream_and_after_a_change():
    import dsa_triton_ascend_amd as dsa
    q = torch.randn(2, 5, 4, 64, device="cuda", requires_grad=True)
    pos = torch.arange(5, device="cuda")
    inv, _ = dsa.rotary_frequencies(64)
    up = torch.randn_like(q)

    def step():
        out, _ = dsa.rotary_embedding(q, None, pos, inv)
        return out, torch.autograd.grad(out, q, up)[0]

    assert dsa.rotary_embedding(q, None, pos, inv)[0].grad_fn.name() == "RotaryEmbeddingBackward"
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        want = step()
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(step(), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for scale in (1.0, 2.0, 0.25):
        up.mul_(scale)
        with torch.no_grad():
            q.mul_(scale)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
    out, _ = dsa.rotary_embedding(q, None, pos, inv)
    pos.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    from torch.utils.checkpoint import checkpoint
    pos.sub_(1)
    checkpoint(lambda x: dsa.rotary_embedding(x, None, pos, inv)[0] * 2, q, use_reentrant=False).backward(up)
    assert torch.equal(q.grad, torch.autograd.grad(dsa.rotary_embedding(q, None, pos, inv)[0] * 2, q, up)[0])


@pytest.mark.parametrize("layout", ["BSND", "TND"])
def test_cache(monkeypatch, layout):
    import dsa_triton_ascend_amd as dsa
    caches, table, lens, refs = _state()
    keep = [c.clone() for c in caches]
    if layout == "BSND":
        rows = [torch.randn(2, 4, 1, 64, device="cuda").bfloat16(), torch.randn(2, 4, 3, 64, device="cuda").bfloat16()[:, :, 1:2]]
        counts = None
    else:
        rows = [torch.randn(9, 1, 64, device="cuda").bfloat16() for _ in range(2)]
        counts = torch.tensor([3, 8], dtype=I32, device="cuda")

    def write():
        for c, x in zip(caches, keep):
            c.copy_(x)
        dsa.paged_cache_write(caches, rows, table, lens, row_lengths=counts, layout=layout)
        return [c.clone() for c in caches]

    def fork():
        for c, x in zip(caches, keep):
            c.copy_(x)
        parents = torch.tensor([1, 0, 1], dtype=I32, device="cuda")
        return (*dsa.paged_cache_fork(caches, table, lens, refs, parents, new_tokens=2), *[c.clone() for c in caches])

    def compact():
        for c, x in zip(caches, keep):
            c.copy_(x)
        return (*dsa.paged_cache_compact(caches, table, refs), *[c.clone() for c in caches])

    for f in (write, fork, compact, lambda: dsa.paged_cache_fork(caches[0], table, lens, refs)):
        _both(monkeypatch, f)


@pytest.mark.parametrize("latent", [False, True])
def test_attention(monkeypatch, latent):
    import dsa_triton_ascend_amd as dsa
    caches, table, lens, _ = _state(heads=1, cols=128 if latent else 64)
    q = torch.randn(2, 2, 8, 128 if latent else 64, device="cuda").bfloat16()
    qr = torch.randn(2, 2, 8, 64, device="cuda").bfloat16() if latent else None
    new = torch.tensor([2, 1], dtype=I32, device="cuda")
    table = table.clamp(min=0)
    for lse in (True, False):
        _both(monkeypatch, lambda: dsa.paged_attention(
            q, caches[0], None if latent else caches[1], table, lens, scale_value=0.125, query_rope=qr,
            key_rope=caches[1] if latent else None, actual_seq_lengths_query=new if lse else None, sparse_mode=3,
            pre_tokens=30 if lse else 2 ** 63 - 1, return_softmax_lse=lse)[:3 if lse else 1])


def test_what_is_taken_and_what_is_left():
    from dsa_triton_ascend_amd import _lib, rotary_frequencies
    c = _lib.calls()
    caches, table, lens, refs = _state()
    inv, _ = rotary_frequencies(32)
    q = torch.randn(2, 3, 4, 64, device="cuda")
    pos = torch.arange(3, device="cuda")
    ok = (q, None, pos, inv, False, 0, None, 1.0, "BSND", False, False)
    assert c.rotate(*ok) is not None
    for i, x in ((0, q.double()), (0, q.cpu()), (0, q[:0]), (0, q.transpose(2, 3)),
                 (2, pos.float()), (2, pos[:2]), (2, None), (3, inv.float()), (5, 40), (5, -1), (5, 2 ** 70), (5, 0.0),
                 (7, "1"), (8, "SBND"), (9, 0), (1, q[:, :2]), (1, q.bfloat16())):
        assert c.rotate(*ok[:i], x, *ok[i + 1:]) is None, (i, x)
    with torch.no_grad():
        assert c.rotate(q.clone().requires_grad_(), *ok[1:]) is not None
    x = q.clone()
    out, _ = c.rotate(x, *ok[1:10], True)
    assert out is x and x._version == 1 and torch.equal(x, c.rotate(*ok)[0])
    for t in (q[:, :1].expand(2, 3, 4, 64), q[..., ::2], q.clone().requires_grad_()):
        assert c.rotate(t, None, pos, inv[:8].contiguous(), *ok[4:10], True) is None
    assert c.rotate(x, x, *ok[2:10], True) is None
    rows = [torch.randn(2, 4, 1, 64, device="cuda").bfloat16()] * 2
    ok = (caches, rows, table, lens, None, "BSND")
    assert c.write(*ok) is True
    for i, x in ((0, caches[:1]), (0, [caches[0], caches[0]]), (0, [caches[0], caches[0][1:]]), (0, []),
                 (0, [caches[0], caches[1].cpu()]), (1, rows[:1]), (1, [r.float() for r in rows]),
                 (1, [r[:, :, :, ::2] for r in rows]), (1, [r[:1] for r in rows]), (1, [rows[0], rows[0][:, :2]]),
                 (2, table.long()), (2, table[0]), (2, table.t()), (3, lens[:1]), (4, lens[:1]), (5, "TND"), (5, None),
                 (0, None), (1, None)):
        assert c.write(*ok[:i], x, *ok[i + 1:]) is None, (i, x)
    ok = (caches, table, lens, refs, None, 1, None)
    assert c.fork(*ok) is not None and c.fork(*ok[:6], 16) is not None
    for i, x in ((0, []), (1, table.long()), (2, lens[:1]), (3, refs[:5]), (4, lens.long()), (5, -1), (5, 2 ** 31),
                 (5, 1.0), (6, 8)):
        assert c.fork(*ok[:i], x, *ok[i + 1:]) is None, (i, x)
    ok = (caches, table, refs, None)
    assert c.compact(*ok) is not None
    for i, x in ((0, []), (1, table.long()), (2, refs[:5]), (3, 8)):
        assert c.compact(*ok[:i], x, *ok[i + 1:]) is None, (i, x)
    q = torch.randn(2, 1, 8, 64, device="cuda").bfloat16()
    ok = (q, caches[0], caches[1], table, lens, 0.1, None, None, None, 3, 2 ** 63 - 1, 2 ** 63 - 1, False)
    assert c.attention(*ok) is not None
    for i, x in ((0, q.float()), (0, q[:, :, :3, :48]), (0, q[:, :, ::2]), (1, caches[0].half()), (1, caches[0][:, ::2]),
                 (2, caches[1][:5]), (2, None), (3, table.long()), (3, table[:1]), (4, [20, 40]), (4, lens.long()),
                 (5, None), (6, q), (8, lens[:1]), (9, 1), (9, True), (9, 2 ** 32 + 3), (10, 2 ** 63), (11, None), (12, 1)):
        assert c.attention(*ok[:i], x, *ok[i + 1:]) is None, (i, x)
    assert c.attention(*ok[:12]) is None  # too few arguments
    torch.cuda.synchronize()


def test_two_threads_and_a_graph():
    import dsa_triton_ascend_amd as dsa
    caches, table, lens, _ = _state()
    q = torch.randn(2, 1, 8, 64, device="cuda").bfloat16()
    table = table.clamp(min=0)
    want = dsa.paged_attention(q, caches[0], caches[1], table, lens)[0]
    torch.cuda.synchronize()
    bad = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                out = dsa.paged_attention(q, caches[0], caches[1], table, lens)[0]
                if not torch.equal(out, want):
                    bad.append(1)

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = dsa.paged_attention(q, caches[0], caches[1], table, lens)[0]
    for scale in (1.0, 0.5, 2.0):
        q.mul_(scale)
        graph.replay()
        eager = dsa.paged_attention(q, caches[0], caches[1], table, lens)[0]
        assert torch.equal(out, eager)


@pytest.mark.parametrize("compiled", [True, False])
def test_an_error_left_behind_is_raised_and_no_rotation_made_twice(monkeypatch, compiled):
    """An error that an earlier HIP call left behind (here: no such device) is
    reported by the next launch, whose kernel has run by then."""
    import ctypes

    import dsa_triton_ascend_amd as dsa
    from dsa_triton_ascend_amd import _lib
    if not compiled:
        monkeypatch.setattr(_lib, "_calls", _lib._NoCalls)
    q = torch.randn(2, 3, 4, 64, device="cuda")
    pos = torch.arange(3, device="cuda")
    inv, _ = dsa.rotary_frequencies(64)
    once, _ = dsa.rotary_embedding(q, None, pos, inv)
    hip = ctypes.CDLL("libamdhip64.so")
    x = q.clone()
    torch.cuda.synchronize()
    hip.hipGetLastError()
    assert hip.hipSetDevice(10 ** 6) != 0
    try:
        with pytest.raises(RuntimeError, match="HIP error"):
            dsa.rotary_embedding(x, None, pos, inv, inplace=True)
    finally:
        hip.hipGetLastError()
    assert torch.equal(x, once)
    assert torch.equal(dsa.rotary_embedding(q, None, pos, inv)[0], once)  # and the next call is an ordinary one


def test_derivatives_are_left_to_python():
    """Where a derivative would be lost the module takes no call; under no_grad it does."""
    import torch.autograd.forward_ad as fwad

    from dsa_triton_ascend_amd import _lib
    c = _lib.calls()
    caches, table, lens, refs = _state()
    rows = [torch.randn(2, 4, 1, 64, device="cuda").bfloat16() for _ in range(2)]
    q = torch.randn(2, 1, 8, 64, device="cuda").bfloat16()
    inf = 2 ** 63 - 1

    def calls(caches, rows, q):
        return [c.write(caches, rows, table, lens, None, "BSND"), c.fork(caches, table, lens, refs, None, 1, None),
                c.compact(caches, table, refs, None),
                c.attention(q, caches[0], caches[1], table, lens, 0.1, None, None, None, 3, inf, inf, False)]

    assert all(x is not None for x in calls(caches, rows, q))
    leaf = [caches[0], caches[1].clone().requires_grad_()]
    assert all(x is None for x in calls(leaf, rows, q))
    assert calls(caches, [rows[0], rows[1].clone().requires_grad_()], q)[0] is None
    assert calls(caches, rows, q.clone().requires_grad_())[3] is None
    with torch.no_grad():
        assert all(x is not None for x in calls(leaf, [r.clone().requires_grad_() for r in rows], q.clone().requires_grad_()))
    with fwad.dual_level():
        assert all(x is None for x in calls([caches[0], fwad.make_dual(caches[1], caches[0])], rows, q))
        assert calls(caches, [fwad.make_dual(rows[0], rows[1]), rows[1]], q)[0] is None
        assert calls(caches, rows, fwad.make_dual(q, q.clone()))[3] is None


@pytest.mark.parametrize("compiled", [True, False])
def test_caches_are_marked_as_changed(monkeypatch, compiled):
    """A backward that saved a cache before a write, a fork or a compaction
    raises, as after torch's own operations in place."""
    import dsa_triton_ascend_amd as dsa
    from dsa_triton_ascend_amd import _lib
    if not compiled:
        monkeypatch.setattr(_lib, "_calls", _lib._NoCalls)
    caches, table, lens, refs = _state(dtype=torch.float32)
    rows = [torch.randn(2, 4, 1, 64, device="cuda") for _ in range(2)]
    w = torch.randn(64, device="cuda", requires_grad=True)
    for change in (lambda c: dsa.paged_cache_write(c, rows, table, lens),
                   lambda c: dsa.paged_cache_fork(c, table, lens, refs, new_tokens=1),
                   lambda c: dsa.paged_cache_compact(c, table, refs)):
        loss = (caches[1] * w).sum()
        before = [c._version for c in caches]
        change(caches)
        assert [c._version for c in caches] == [v + 1 for v in before]
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
        with torch.inference_mode():
            mine = [c.clone() for c in caches]
        change(mine)  # tensors without a version
    views = [caches[0][:9], caches[1][:9]]
    before = caches[0]._version
    dsa.paged_cache_write(views, rows, table, lens)
    assert caches[0]._version == before + 1


def test_in_place_views_of_one_buffer():
    """The module takes what shares no columns, and no other."""
    import random

    from test_decode_ops_validation import _shared, _views

    import dsa_triton_ascend_amd as dsa
    from dsa_triton_ascend_amd import _lib
    from dsa_triton_ascend_amd.rotary_embedding import _overlaps_itself
    rng, taken = random.Random(1), [0, 0]
    start = torch.randn(1 << 14, device="cuda")
    for _ in range(400):
        flat = start.clone()
        q, qs, k, ks, cols = _views(rng, flat)
        if _overlaps_itself(q) or _overlaps_itself(k):
            continue
        pos = torch.randint(0, 99, q.shape[:2], device="cuda")
        inv, _ = dsa.rotary_frequencies(cols)
        shared = _shared(q, qs, k, ks, cols) or q.data_ptr() == k.data_ptr()
        want = dsa.rotary_embedding(q, k, pos, inv, rotary_offset=qs, key_rotary_offset=ks)
        got = _lib.calls().rotate(q, k, pos, inv, False, qs, ks, 1.0, "BSND", False, True)
        assert (got is None) == shared
        if shared:
            with pytest.raises(ValueError, match="share memory"):
                dsa.rotary_embedding(q, k, pos, inv, rotary_offset=qs, key_rotary_offset=ks, inplace=True)
            assert torch.equal(flat, start)
        else:
            for a, b, s in zip((q, k), want, (qs, ks)):
                assert torch.equal(a[..., s:s + cols], b[..., s:s + cols])
        taken[shared] += 1
    assert min(taken) > 40, taken


def test_ordinary_calls_are_taken(monkeypatch):
    """The forms that are compared with Python above do go by the module: each
    call is recorded, and it returns something."""
    import dsa_triton_ascend_amd as dsa
    from dsa_triton_ascend_amd import _lib
    module, made = _lib.calls(), []

    class Recorder:
        def __getattr__(self, name):
            def call(*args):
                result = getattr(module, name)(*args)
                made.append((name, result is not None))
                return result
            return call

    monkeypatch.setattr(_lib, "_calls", Recorder())

    def taken(name, f):
        made.clear()
        f()
        assert made == [(name, True)], (name, made)

    caches, table, lens, refs = _state()
    latent, ltable, llens, _ = _state(cols=128)
    inv, _ = dsa.rotary_frequencies(32)
    for lead, layout in (((3, 5), "BSND"), ((7,), "TND")):
        pos = torch.randint(0, 9999, lead, device="cuda", dtype=I32)
        q = torch.randn(*lead, 6, 96, device="cuda").bfloat16()
        k = torch.randn(*lead, 2, 64, device="cuda").bfloat16()
        for kw in (dict(), dict(inplace=True), dict(inverse=True, interleaved=True)):
            taken("rotate", lambda: dsa.rotary_embedding(q[..., :5, 16:], k, pos, inv, rotary_offset=32, layout=layout, **kw))
        fused = torch.randn(*lead, 6, 64, device="cuda")
        taken("rotate", lambda: dsa.rotary_embedding(fused[..., :4, :], fused[..., 4:, :], pos, inv, layout=layout,
                                                     inplace=True))
        leaf = fused.clone().requires_grad_()
        taken("rotate", lambda: dsa.rotary_embedding(leaf, None, pos, inv, layout=layout)[0].sum().backward())
    rows = [torch.randn(2, 4, 1, 64, device="cuda").bfloat16(), torch.randn(2, 4, 3, 64, device="cuda").bfloat16()[:, :, 1:2]]
    packed = [torch.randn(9, 1, 64, device="cuda").bfloat16() for _ in range(2)]
    counts = torch.tensor([3, 8], dtype=I32, device="cuda")
    taken("write", lambda: dsa.paged_cache_write(caches, rows, table, lens))
    taken("write", lambda: dsa.paged_cache_write(tuple(caches), rows, table, lens, row_lengths=counts))
    taken("write", lambda: dsa.paged_cache_write(caches, packed, table, lens, row_lengths=counts, layout="TND"))
    taken("fork", lambda: dsa.paged_cache_fork(caches, table, lens, refs, torch.tensor([1, 0, 1], dtype=I32, device="cuda"),
                                               new_tokens=2))
    taken("fork", lambda: dsa.paged_cache_fork(caches[0], table, lens, refs))
    taken("compact", lambda: dsa.paged_cache_compact(caches, table, refs))
    for new in (None, torch.tensor([2, 1], dtype=I32, device="cuda")):
        q = torch.randn(2, 2, 8, 128, device="cuda").bfloat16()
        taken("attention", lambda: dsa.paged_attention(q[..., :64].contiguous(), caches[0], caches[1], table.clamp(min=0),
                                                       lens, actual_seq_lengths_query=new, pre_tokens=30))
        taken("attention", lambda: dsa.paged_attention(
            q, latent[0], None, ltable.clamp(min=0), llens, query_rope=q[..., :64].contiguous(), key_rope=latent[1],
            actual_seq_lengths_query=new, return_softmax_lse=True))
