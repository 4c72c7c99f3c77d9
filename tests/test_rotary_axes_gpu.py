"""rotary_embedding with positions on several axes, against the rotation in 64
bits.

Error bound: sine and cosine of an angle reduced in 64 bits are good to 2^-22,
each product and the sum of two to 2^-24 relative, so a rotated value is off by
at most 2^-20 (|a| + |b|) before it is rounded to its type (eps / 2 of it).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

I32 = torch.int32
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _axes(sections, mixed):
    if not mixed:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    n = len(sections)
    return [i % n if i < n * sections[i % n] else 0 for i in range(sum(sections))]


def _turn(x, pos, inv, sections, mixed, start, interleaved=False, scale=1.0, inverse=False):
    """The rotation of [..., heads, columns] in 64 bits, and the error bound of its columns."""
    rot = 2 * len(inv)
    angle = torch.stack([pos[a].double() * inv[i] for i, a in enumerate(_axes(sections, mixed))], -1)
    angle = angle.expand(*x.shape[:-2], rot // 2)[..., None, :] * (-1 if inverse else 1)
    c, s = torch.cos(angle) * scale, torch.sin(angle) * scale
    y = x.double().clone()
    part = y[..., start:start + rot]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :rot // 2], part[..., rot // 2:])
    out = [a * c - b * s, a * s + b * c]
    loose = (a.abs() + b.abs()) * scale * 2.0 ** -20
    bound = torch.zeros_like(y)
    join = (lambda u, v: torch.stack([u, v], -1).flatten(-2)) if interleaved else (lambda u, v: torch.cat([u, v], -1))
    y[..., start:start + rot] = join(*out)
    bound[..., start:start + rot] = join(loose, loose)
    bound += y.abs() * torch.finfo(x.dtype).eps / 2
    if start:
        bound[..., :start] = 0
    bound[..., start + rot:] = 0
    return y, bound


def _near(got, want_bound):
    want, bound = want_bound
    assert (got.double() - want).abs().le(bound).all()


def _inputs(lead, heads, kheads, d, kd, dtype, axes, seed=0, far=100000, pos_type=I32, shared=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randn(*lead, heads, d, generator=g, device="cuda").to(dtype)
    k = torch.randn(*lead, kheads, kd, generator=g, device="cuda").to(dtype)
    shape = (axes,) + (lead[-1:] if shared else lead)
    pos = torch.randint(-5, far, shape, generator=g, device="cuda").to(pos_type)
    return q, k, pos


@pytest.mark.parametrize("sections,mixed", [
    ((16, 24, 24), False), ((24, 20, 20), True), ((22, 42), False), ((32, 32), True), ((64,), False), ((64,), True),
    ((0, 30, 34), False), ((10, 20, 30, 4), False), ((31, 11, 11, 11), True), ((62, 1, 1), True), ((64, 0, 0), True)])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_axes(sections, mixed, dtype):
    import dsa_triton_ascend_amd as dsa
    q, k, pos = _inputs((2, 7), 3, 2, 160, 128, DTYPES[dtype], len(sections))
    inv, _ = dsa.rotary_frequencies(128)
    qo, ko = dsa.rotary_embedding(q, k, pos, inv, rotary_offset=16, key_rotary_offset=0, attention_scale=1.25,
                                  sections=sections, sections_interleaved=mixed)
    _near(qo, _turn(q, pos, inv, sections, mixed, 16, scale=1.25))
    _near(ko, _turn(k, pos, inv, sections, mixed, 0, scale=1.25))


@pytest.mark.parametrize("lead,heads,cols,rot,shared,pos_type", [
    ((1, 1), 1, 2, 2, False, I32), ((5,), 3, 33, 26, False, torch.int64), ((3, 1), 128, 64, 64, True, I32),
    ((2, 513), 5, 72, 64, True, torch.int64), ((1000,), 16, 80, 80, False, I32)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_sizes(lead, heads, cols, rot, shared, pos_type, interleaved):
    import dsa_triton_ascend_amd as dsa
    layout = "TND" if len(lead) == 1 else "BSND"
    q, k, pos = _inputs(lead, heads, 1, cols, cols, torch.float16, 2, far=2 ** 31 - 1, pos_type=pos_type, shared=shared)
    sections = (rot // 2 - rot // 6, rot // 6)
    inv, _ = dsa.rotary_frequencies(rot)
    qo, ko = dsa.rotary_embedding(q, k, pos, inv, interleaved=interleaved, layout=layout, inverse=True,
                                  rotary_offset=cols - rot, sections=list(sections), sections_interleaved=True)
    for x, y in ((q, qo), (k, ko)):
        _near(y, _turn(x, pos, inv, sections, True, cols - rot, interleaved, inverse=True))
    alone, none = dsa.rotary_embedding(q, None, pos, inv, interleaved=interleaved, layout=layout, inverse=True,
                                       rotary_offset=cols - rot, sections=sections, sections_interleaved=True)
    assert none is None and torch.equal(alone, qo)


def test_equal_positions_are_one_axis():
    import dsa_triton_ascend_amd as dsa
    q, k, pos = _inputs((2, 9), 4, 1, 128, 64, torch.bfloat16, 1)
    inv, _ = dsa.rotary_frequencies(64)
    one = dsa.rotary_embedding(q, k, pos[0], inv)
    for sections, mixed in (((32,), False), ((10, 10, 12), False), ((12, 10, 10), True)):
        many = dsa.rotary_embedding(q, k, pos.expand(len(sections), 2, 9), inv, sections=sections,
                                    sections_interleaved=mixed)
        assert torch.equal(one[0], many[0]) and torch.equal(one[1], many[1])


def test_in_place_and_strided():
    import dsa_triton_ascend_amd as dsa
    sections = (8, 12, 12)
    packed, _, pos = _inputs((2, 33), 5, 1, 256, 64, torch.bfloat16, 3)
    inv, _ = dsa.rotary_frequencies(64)
    q, k = packed[..., :4, 32:128], packed[..., 4:, 128:]
    want = [_turn(q, pos, inv, sections, False, 0), _turn(k, pos, inv, sections, False, 0)]
    before = packed.clone()
    out = dsa.rotary_embedding(q, k, pos, inv, sections=sections)
    for o, w in zip(out, want):
        _near(o, w)
    assert torch.equal(packed, before)
    same = dsa.rotary_embedding(q, k, pos, inv, sections=sections, inplace=True)
    assert same[0] is q and same[1] is k and torch.equal(q, out[0]) and torch.equal(k, out[1])
    assert torch.equal(packed[..., :32], before[..., :32])
    # positions that are a view
    wide = torch.stack([pos, pos + 1], -1)
    again = dsa.rotary_embedding(before[..., :4, 32:128], None, wide[..., 0], inv, sections=sections)[0]
    assert torch.equal(again, out[0])


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("layout", ["BSND", "TND"])
def test_gradients(dtype, layout):
    import dsa_triton_ascend_amd as dsa
    lead = (2, 37) if layout == "BSND" else (41,)
    sections = (24, 20, 20)
    q, k, pos = _inputs(lead, 6, 2, 160, 128, DTYPES[dtype], 3)
    inv, _ = dsa.rotary_frequencies(128)
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    kw = dict(rotary_offset=32, key_rotary_offset=0, attention_scale=0.75, layout=layout, sections=sections,
              sections_interleaved=True)
    q.requires_grad_(True), k.requires_grad_(True)
    qo, ko = dsa.rotary_embedding(q, k, pos, inv, **kw)
    gq, gk = torch.autograd.grad((qo, ko), (q, k), (dq, dk))
    _near(gq, _turn(dq, pos, inv, sections, True, 32, scale=0.75, inverse=True))
    _near(gk, _turn(dk, pos, inv, sections, True, 0, scale=0.75, inverse=True))
    # a key alone, and shapes of nodes of torch's own behind and before
    gk2, = torch.autograd.grad((dsa.rotary_embedding(q * 1, k * 1, pos, inv, **kw)[1].float() * dk.float()).sum(), k)
    assert torch.equal(gk2, gk)
    # the difference of two outputs along dq is the derivative (the rotation is linear), in the type's rounding
    with torch.no_grad():
        a = dsa.rotary_embedding((q + dq).detach(), None, pos, inv, **{**kw, "key_rotary_offset": None})[0].double()
        b = dsa.rotary_embedding(q.detach(), None, pos, inv, **{**kw, "key_rotary_offset": None})[0].double()
    turned, _ = _turn(dq, pos, inv, sections, True, 32, scale=0.75)
    eps = torch.finfo(q.dtype).eps
    size = (q.abs().amax() + dq.abs().amax()).double() * 2
    assert (a - b - turned).abs().max() <= size * (2 * eps + 2.0 ** -18)  # sum, both outputs and both turned inputs


def test_second_order_and_tangents():
    import dsa_triton_ascend_amd as dsa
    import torch.autograd.forward_ad as fwd
    sections = (6, 5, 5)
    q, k, pos = _inputs((1, 11), 2, 1, 32, 32, torch.float32, 3)
    inv, _ = dsa.rotary_frequencies(32)
    kw = dict(sections=sections, sections_interleaved=True)

    def f(x):
        return dsa.rotary_embedding(x, None, pos, inv, **kw)[0]

    x, w = q.clone().requires_grad_(True), torch.randn_like(q).requires_grad_(True)
    g, = torch.autograd.grad(f(x), x, w, create_graph=True)
    gg, = torch.autograd.grad(g, w, k.expand_as(g).contiguous())
    _near(gg, _turn(k.expand_as(g), pos, inv, sections, True, 0))
    t = torch.randn_like(q)
    with fwd.dual_level():
        out = fwd.unpack_dual(f(fwd.make_dual(q, t)))
    assert torch.equal(out.primal, f(q))
    assert torch.equal(out.tangent, f(t))


def test_compiled_and_python_calls_agree(monkeypatch):
    import dsa_triton_ascend_amd as dsa
    from dsa_triton_ascend_amd import _lib
    assert _lib.calls() is not _lib._NoCalls
    q, k, pos = _inputs((2, 7), 3, 2, 128, 128, torch.bfloat16, 3)
    inv, _ = dsa.rotary_frequencies(128)

    def f():
        x, y = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
        out = dsa.rotary_embedding(x, y, pos, inv, sections=(16, 24, 24))
        return out + torch.autograd.grad(out, (x, y), (q, k))

    args = (q, k, pos, inv, False, 0, None, 1.0, "BSND", False, False, (16, 24, 24), False)
    assert _lib.calls().rotate_axes(*args) is not None
    for i, bad in ((2, pos[:2].contiguous()), (2, pos[0]), (11, (16, 24, 23)), (11, (64.0,)), (11, None),
                   (11, (-1, 33, 32)), (12, 1)):
        assert _lib.calls().rotate_axes(*args[:i], bad, *args[i + 1:]) is None
    a = f()
    monkeypatch.setattr(_lib, "_calls", _lib._NoCalls)
    b = f()
    monkeypatch.undo()
    for u, v in zip(a, b):
        assert torch.equal(u, v)


def test_module_and_replay():
    import dsa_triton_ascend_amd as dsa
    q, k, pos = _inputs((4, 1), 8, 1, 64, 64, torch.bfloat16, 3)
    m = dsa.RotaryEmbedding(64, sections=(16, 8, 8), sections_interleaved=True)
    want = dsa.rotary_embedding(q, k, pos, m.inv_freq, sections=(16, 8, 8), sections_interleaved=True)
    assert torch.equal(m(q, k, pos)[0], want[0])
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        m(q, k, pos)
        with torch.cuda.graph(graph, stream=stream):
            out = m(q, k, pos)
    for step in range(3):
        pos.add_(step * 17)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = m(q, k, pos)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
