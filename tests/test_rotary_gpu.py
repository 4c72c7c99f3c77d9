"""rotary_embedding against the rotation in 64 bits.

Error bound of an element o = s (a cos -/+ b sin): the sine and cosine are
within 4 ulp of 32 bits (the angle itself is formed in 64 bits), the two
products and the sum round in 32 bits, so the value before the last rounding
is off by at most 2^-20 s (|a| + |b|); rounding to the type adds eps / 2 of
the value.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _turn(x, pos, inv, start, interleaved, scale, sign=1.0):
    """The rotation of x [B, S, N, D] in 64 bits; also sum of |pair| per column."""
    y, mag = x.double().cpu().clone(), x.double().cpu().abs() * 0
    half = inv.numel()
    ang = pos.double().cpu()[..., None] * inv.double().cpu()
    if ang.dim() == 2:
        ang = ang[None]
    c, s = (torch.cos(ang) * scale)[:, :, None], (torch.sin(ang) * scale * sign)[:, :, None]
    ia = start + (torch.arange(half) * 2 if interleaved else torch.arange(half))
    ib = ia + (1 if interleaved else half)
    a, b = y[..., ia].clone(), y[..., ib].clone()
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    mag[..., ia] = mag[..., ib] = (a.abs() + b.abs()) * abs(scale)
    return y, mag


def _check(got, want, mag, dtype, what):
    g = got.double().cpu()
    tol = mag * 2.0 ** -20 + (want.abs() + mag * 2.0 ** -20) * (torch.finfo(dtype).eps / 2) + 1e-30
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25  # half a step of its subnormal numbers
    tol = torch.where(mag == 0, torch.zeros_like(tol), tol)  # copied columns are equal
    bad = (g - want).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {((g - want).abs() - tol).max():.3g}"


CASES = [
    # B, S, N, D, KN, KD, R, q offset, k offset, interleaved, dtype
    (1, 1, 1, 2, 1, 2, 2, 0, 0, True, "fp32"),
    (1, 1, 1, 2, 1, 2, 2, 0, 0, False, "bf16"),
    (2, 3, 5, 64, 1, 64, 64, 0, 0, True, "bf16"),
    (3, 7, 16, 192, 1, 64, 64, 128, 0, False, "bf16"),
    (2, 5, 8, 128, 1, 128, 64, 0, 0, False, "fp16"),
    (1, 33, 3, 128, 2, 96, 32, 16, 64, True, "fp16"),
    (2, 9, 7, 70, 3, 33, 6, 5, 11, False, "fp32"),
    (2, 9, 7, 70, 3, 33, 6, 5, 11, True, "bf16"),
    (1, 4, 128, 576, 1, 576, 64, 512, 512, True, "bf16"),
    (4, 300, 2, 64, 1, 64, 64, 0, 0, False, "fp32"),
    (1, 2, 2, 1100, 1, 1024, 1024, 76, 0, False, "fp16"),
]


@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_forward_and_gradients(case):
    import dsa_triton_ascend_amd as dsa
    B, S, N, D, KN, KD, R, q0, k0, inter, dt = case
    dtype = DTYPES[dt]
    print(case, flush=True)
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn(B, S, N, D, generator=g, device="cuda", dtype=dtype, requires_grad=True)
    k = torch.randn(B, S, KN, KD, generator=g, device="cuda", dtype=dtype, requires_grad=True)
    pos = torch.randint(0, 131072, (B, S), generator=g, device="cuda", dtype=torch.int64)
    inv, scale = dsa.rotary_frequencies(R, scaling="yarn" if R >= 32 else "none", factor=8.0)
    qo, ko = dsa.rotary_embedding(q, k, pos, inv, interleaved=inter, rotary_offset=q0, key_rotary_offset=k0,
                                  attention_scale=scale)
    dq, dk = torch.randn_like(qo), torch.randn_like(ko)
    gq, gk = torch.autograd.grad((qo, ko), (q, k), (dq, dk))
    for name, got, x, start, sign in (("query", qo, q, q0, 1.0), ("key", ko, k, k0, 1.0), ("d query", gq, dq, q0, -1.0),
                                      ("d key", gk, dk, k0, -1.0)):
        want, mag = _turn(x.detach(), pos, inv, start, inter, scale, sign)
        _check(got.detach(), want, mag, dtype, name)


def test_gradient_against_differences():
    """The operator is linear, so a difference is exact: <d, f(x + h) - f(x)> = <grad, h>.
    fp32 values of size 1: every element is off by at most 2^-20 * 4, and 2 * 6 * 40 * 2
    of them enter either sum with weights of size up to 4."""
    import dsa_triton_ascend_amd as dsa
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(2, 6, 2, 40, generator=g, device="cuda", requires_grad=True)
    h, d = (torch.randn(2, 6, 2, 40, generator=g, device="cuda") for _ in range(2))
    pos = torch.arange(6, device="cuda", dtype=torch.int32) + 5000
    inv, _ = dsa.rotary_frequencies(16)
    for inter in (True, False):
        kw = dict(interleaved=inter, rotary_offset=7, attention_scale=1.5)
        y, none = dsa.rotary_embedding(x, None, pos, inv, **kw)
        assert none is None
        (grad,) = torch.autograd.grad(y, x, d)
        y2, _ = dsa.rotary_embedding((x + h).detach(), None, pos, inv, **kw)
        left = (d.double() * (y2.double() - y.detach().double())).sum()
        right = (grad.double() * h.double()).sum()
        assert abs(left - right) <= 2 * 6 * 40 * 2 * 2 * 16 * 2.0 ** -20


@pytest.mark.parametrize("sides", ["both", "query", "key"])
def test_second_gradient(sides):
    """<grad, h> as a function of the outputs' gradients d is <d, f(h)>: its gradient is f(h)."""
    import dsa_triton_ascend_amd as dsa
    g = torch.Generator(device="cuda").manual_seed(7)
    q = torch.randn(2, 5, 3, 48, generator=g, device="cuda", requires_grad=sides != "key")
    k = torch.randn(2, 5, 1, 32, generator=g, device="cuda", requires_grad=sides != "query")
    pos = torch.arange(5, device="cuda") + 77
    inv, _ = dsa.rotary_frequencies(16)
    outs = dsa.rotary_embedding(q, k, pos, inv, rotary_offset=8, key_rotary_offset=16, attention_scale=0.5)
    some = [i for i, t in enumerate((q, k)) if t.requires_grad]
    d = [torch.randn(outs[i].shape, generator=g, device="cuda", requires_grad=True) for i in some]
    h = [torch.randn(outs[i].shape, generator=g, device="cuda") for i in some]
    first = torch.autograd.grad([outs[i] for i in some], [(q, k)[i] for i in some], d, create_graph=True)
    second = torch.autograd.grad(first, d, h)
    for i, got, x in zip(some, second, h):
        want, mag = _turn(x, pos, inv, (8, 16)[i], False, 0.5)
        _check(got, want, mag, torch.float32, sides)


def test_only_one_side_differentiable():
    import dsa_triton_ascend_amd as dsa
    q = torch.randn(1, 3, 2, 32, device="cuda")
    k = torch.randn(1, 3, 1, 48, device="cuda", requires_grad=True)
    pos = torch.arange(3, device="cuda")
    inv, _ = dsa.rotary_frequencies(32)
    qo, ko = dsa.rotary_embedding(q, k, pos, inv, key_rotary_offset=16)
    assert not torch.equal(qo, q)
    d = torch.randn_like(ko)
    (gk,) = torch.autograd.grad(ko, k, d)
    want, mag = _turn(d, pos, inv, 16, False, 1.0, -1.0)
    _check(gk, want, mag, torch.float32, "d key")


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_strided_views_packed_and_in_place(dt):
    """The rope part of a projection [T, N, 128 + 64], read through its
    strides, out of place and in place; the rest of the projection stays."""
    import dsa_triton_ascend_amd as dsa
    dtype = DTYPES[dt]
    proj = torch.randn(37, 5, 192, device="cuda").to(dtype)
    kproj = torch.randn(37, 576, device="cuda").to(dtype)
    pos = torch.randint(0, 10 ** 6, (37,), device="cuda", dtype=torch.int32)
    inv, scale = dsa.rotary_frequencies(64)
    q, k = proj[..., 128:], kproj[:, None, 512:]
    qo, ko = dsa.rotary_embedding(q, k, pos, inv, interleaved=True, layout="TND")
    wq, mq = _turn(q[None], pos[None], inv, 0, True, scale)
    wk, mk = _turn(k[None], pos[None], inv, 0, True, scale)
    _check(qo[None], wq, mq, dtype, "query")
    _check(ko[None], wk, mk, dtype, "key")
    kept, kkept = proj[..., :128].clone(), kproj[:, :512].clone()
    qi, ki = dsa.rotary_embedding(q, k, pos, inv, interleaved=True, layout="TND", inplace=True)
    assert qi is q and ki is k
    assert torch.equal(q, qo) and torch.equal(k, ko)
    assert torch.equal(proj[..., :128], kept) and torch.equal(kproj[:, :512], kkept)
    # transposed heads and tokens, and columns apart (copied)
    t = torch.randn(2, 4, 9, 64, device="cuda").to(dtype).transpose(1, 2)
    a, _ = dsa.rotary_embedding(t, None, pos[:9], inv)
    b, _ = dsa.rotary_embedding(t.contiguous(), None, pos[:9], inv)
    assert torch.equal(a, b) and a.is_contiguous()
    c, _ = dsa.rotary_embedding(t.transpose(-1, -2).contiguous().transpose(-1, -2), None, pos[:9], inv)
    assert torch.equal(c, b)
    # unaligned addresses
    flat = torch.randn(1 + 2 * 3 * 64, device="cuda").to(dtype)[1:].view(1, 2, 3, 64)
    d, _ = dsa.rotary_embedding(flat, None, pos[:2], inv)
    e, _ = dsa.rotary_embedding(flat.clone(), None, pos[:2], inv)
    assert torch.equal(d, e)


def test_inverse_and_broadcast_input():
    import dsa_triton_ascend_amd as dsa
    x = torch.randn(1, 1, 1, 64, device="cuda").expand(2, 3, 4, 64)
    pos = torch.tensor([[0, 1, 77], [131071, 3, -5]], device="cuda")
    inv, _ = dsa.rotary_frequencies(64)
    y, _ = dsa.rotary_embedding(x, None, pos, inv)
    want, mag = _turn(x, pos, inv, 0, False, 1.0)
    _check(y, want, mag, torch.float32, "broadcast")
    z, _ = dsa.rotary_embedding(y, None, pos, inv, inverse=True)
    # two rotations: each off by 2^-20 (|a| + |b|) + eps / 2 |value|, |a| + |b| <= 1.5 * the pair's norm
    pair = (x[..., :32] ** 2 + x[..., 32:] ** 2).sqrt()
    tol = torch.cat([pair, pair], -1) * (2 * 1.5 * 2.0 ** -20 + 2 * 2.0 ** -24 * 1.5)
    assert ((z - x).abs() <= tol).all()
    # a leaf that is broadcast gets the sum of its copies' gradients
    w = torch.randn(1, 1, 1, 64, device="cuda", requires_grad=True)
    out, _ = dsa.rotary_embedding(w.expand(2, 3, 4, 64), None, pos, inv)
    d = torch.randn_like(out)
    out.backward(d)
    ref, mg = _turn(d, pos, inv, 0, False, 1.0, -1.0)
    # 24 gradients, each off by 2^-20 mag + 2^-24 |value|, and 23 roundings of partial sums
    total = ref.sum((0, 1, 2))
    tol = (mg * 2.0 ** -20 + ref.abs() * 2.0 ** -24 * 24).sum((0, 1, 2))
    assert ((w.grad.double().cpu()[0, 0, 0] - total).abs() <= tol + 1e-12).all()


def test_far_positions():
    """Position 2^30 at frequency 1: the angle in 64 bits."""
    import dsa_triton_ascend_amd as dsa
    x = torch.randn(1, 4, 1, 8, device="cuda")
    pos = torch.tensor([2 ** 30, 2 ** 30 + 1, 2 ** 31 - 1, 2 ** 40], device="cuda", dtype=torch.int64)
    inv, _ = dsa.rotary_frequencies(8)
    y, _ = dsa.rotary_embedding(x, None, pos, inv)
    # angle * 2^-53 of relative error in turns on either side: 2^40 / 6.3 * 2^-52 turns = 2^-14.6,
    # times 2 pi; the first three are 2^9 times nearer
    want, mag = _turn(x, pos, inv, 0, False, 1.0)
    err = (y.double().cpu() - want).abs()
    assert (err[:, :3] <= mag[:, :3] * 2.0 ** -19 + want[:, :3].abs() * 2.0 ** -24).all()
    assert (err[:, 3] <= mag[:, 3] * 2.0 ** -11).all()


def test_empty_and_module():
    import dsa_triton_ascend_amd as dsa
    inv, _ = dsa.rotary_frequencies(16)
    q = torch.empty(0, 3, 2, 16, device="cuda")
    qo, ko = dsa.rotary_embedding(q, q, torch.empty(0, 3, device="cuda", dtype=torch.int32), inv)
    assert qo.shape == q.shape and ko.shape == q.shape
    mod = dsa.RotaryEmbedding(16, scaling="linear", factor=4.0, interleaved=True, device="cuda").to(torch.bfloat16)
    assert mod.inv_freq.dtype == torch.float64
    x = torch.randn(1, 5, 2, 16, device="cuda")
    pos = torch.arange(5, device="cuda")
    y, _ = mod(x, None, pos)
    want, mag = _turn(x, pos.double() / 4, inv, 0, True, 1.0)
    _check(y, want, mag, torch.float32, "module")


def test_graph_replays():
    """Captured forward, and a captured forward and backward of leaves of its own."""
    import dsa_triton_ascend_amd as dsa
    q = torch.randn(2, 5, 4, 64, device="cuda").bfloat16()
    k = torch.randn(2, 5, 1, 64, device="cuda").bfloat16()
    pos = torch.randint(0, 9999, (2, 5), device="cuda", dtype=torch.int32)
    inv, _ = dsa.rotary_frequencies(64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        dsa.rotary_embedding(q, k, pos, inv)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qo, ko = dsa.rotary_embedding(q, k, pos, inv)
    for i in range(3):
        q.copy_(torch.randn_like(q))
        pos.add_(17 + i)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eq, ek = dsa.rotary_embedding(q, k, pos, inv)
        assert torch.equal(qo, eq) and torch.equal(ko, ek)


def test_frequencies():
    import dsa_triton_ascend_amd as dsa
    plain, one = dsa.rotary_frequencies(64)
    assert one == 1.0 and plain.dtype == torch.float64 and plain[0] == 1.0
    lin, _ = dsa.rotary_frequencies(64, scaling="linear", factor=4.0)
    assert np.allclose(lin.cpu() * 4, plain.cpu(), rtol=1e-15)
    ntk, _ = dsa.rotary_frequencies(64, scaling="ntk", factor=4.0)
    assert ntk[0] == 1.0 and math.isclose(float(ntk[-1] * 4), float(plain[-1]), rel_tol=1e-12)
    yarn, scale = dsa.rotary_frequencies(64, scaling="yarn", factor=40.0, mscale_all_dim=0.0)
    assert math.isclose(scale, 0.1 * math.log(40.0) + 1.0)
    assert yarn[0] == plain[0] and math.isclose(float(yarn[-1] * 40), float(plain[-1]), rel_tol=1e-12)
    assert (yarn <= plain).all() and (yarn * 40 >= plain * (1 - 1e-12)).all()
    assert dsa.rotary_frequencies(64, scaling="yarn", factor=40.0, mscale=0.7, mscale_all_dim=0.7)[1] == 1.0


@pytest.mark.parametrize("sides", ["both", "query", "key", "query alone"])
@pytest.mark.parametrize("compiled", [True, False])
@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode(monkeypatch, sides, compiled, requires_grad):
    """The rotation is linear: a tangent turns as its input does, whether or not
    a gradient is asked for too, and a gradient's tangent as the gradient."""
    import torch.autograd.forward_ad as fwad

    import dsa_triton_ascend_amd as dsa
    from dsa_triton_ascend_amd import _lib
    if not compiled:
        monkeypatch.setattr(_lib, "_calls", _lib._NoCalls)
    pos = torch.randint(0, 9999, (2, 5), device="cuda")
    inv, _ = dsa.rotary_frequencies(32)
    args = dict(positions=pos, inv_freq=inv, rotary_offset=16, key_rotary_offset=32, attention_scale=0.75)
    x, t, up, up_t = ([torch.randn(2, 5, n, 64, device="cuda") for n in (4, 2)] for _ in range(4))
    with_key = sides != "query alone"
    has = (sides != "key", sides in ("both", "key"))

    def turn(q, k, **kw):
        return [o for o in dsa.rotary_embedding(q, k if with_key else None, **args, **kw) if o is not None]

    plain, turned, back, back_t = turn(*x), turn(*t), turn(*up, inverse=True), turn(*up_t, inverse=True)
    with fwad.dual_level():
        leaves = [a.clone().requires_grad_(requires_grad) for a in x]
        ins = [fwad.make_dual(a, b) if h else a for a, b, h in zip(leaves, t, has)]
        outs = turn(*ins)
        for i, o in enumerate(outs):
            got = fwad.unpack_dual(o)
            assert torch.equal(got.primal, plain[i])
            if has[i]:
                assert torch.equal(got.tangent, turned[i])
            else:
                assert got.tangent is None or not got.tangent.any()
        if requires_grad:
            grads = torch.autograd.grad(outs, ins[:len(outs)], [fwad.make_dual(a, b) for a, b in zip(up, up_t)][:len(outs)])
            for g, a, b in zip(grads, back, back_t):
                g = fwad.unpack_dual(g)
                assert torch.equal(g.primal, a) and torch.equal(g.tangent, b)
        with torch.no_grad(), pytest.raises(ValueError, match="tangents"):
            dsa.rotary_embedding(fwad.make_dual(x[0].clone(), t[0]), None, **args, inplace=True)


@pytest.mark.parametrize("compiled", [True, False])
def test_a_gradient_s_tangent_where_the_input_has_none(monkeypatch, compiled):
    import torch.autograd.forward_ad as fwad

    import dsa_triton_ascend_amd as dsa
    from dsa_triton_ascend_amd import _lib
    if not compiled:
        monkeypatch.setattr(_lib, "_calls", _lib._NoCalls)
    pos = torch.arange(5, device="cuda")
    inv, _ = dsa.rotary_frequencies(64)
    q = torch.randn(1, 5, 2, 64, device="cuda", requires_grad=True)
    k = torch.randn(1, 5, 1, 64, device="cuda", requires_grad=True)
    w, t = torch.randn(1, 5, 2, 64, device="cuda"), torch.randn(1, 5, 2, 64, device="cuda")
    with fwad.dual_level():
        qo, ko = dsa.rotary_embedding(q, k, pos, inv)
        g = fwad.unpack_dual(torch.autograd.grad((qo * fwad.make_dual(w, t)).sum(), q)[0])
    assert torch.equal(g.primal, dsa.rotary_embedding(w, None, pos, inv, inverse=True)[0])
    assert torch.equal(g.tangent, dsa.rotary_embedding(t, None, pos, inv, inverse=True)[0])


@pytest.mark.parametrize("compiled", [True, False])
def test_gradients_and_tangents_without_memory(monkeypatch, compiled):
    """torch's zero tensors, which stand for zeros that nobody has written."""
    import torch.autograd.forward_ad as fwad

    import dsa_triton_ascend_amd as dsa
    from dsa_triton_ascend_amd import _lib
    if not compiled:
        monkeypatch.setattr(_lib, "_calls", _lib._NoCalls)
    pos = torch.arange(5, device="cuda")
    inv, _ = dsa.rotary_frequencies(64)
    q = torch.randn(1, 5, 2, 64, device="cuda", requires_grad=True)
    zero = torch._efficientzerotensor(1, 5, 2, 64, device="cuda")
    out, _ = dsa.rotary_embedding(q, None, pos, inv)
    (g,) = torch.autograd.grad(out, q, zero)
    assert g.shape == q.shape and not g.any()
    t = torch.randn(1, 5, 2, 64, device="cuda")
    with fwad.dual_level():
        out, _ = dsa.rotary_embedding(q, None, pos, inv)
        g = fwad.unpack_dual(torch.autograd.grad(out, q, fwad.make_dual(torch.zeros_like(t), t))[0])
        assert not g.primal.any() and torch.equal(g.tangent, dsa.rotary_embedding(t, None, pos, inv, inverse=True)[0])
        y, _ = dsa.rotary_embedding(fwad.make_dual(t, zero), None, pos, inv)
        y = fwad.unpack_dual(y)
        assert torch.equal(y.primal, dsa.rotary_embedding(t, None, pos, inv)[0])
        assert y.tangent is None or not y.tangent.any()
    torch.cuda.synchronize()
