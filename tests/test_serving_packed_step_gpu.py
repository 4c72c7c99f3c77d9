"""The packed step of requests of many lengths as the module's documentation of paged_cache shows it: plan, prefixes,
writes, and attention over each row's tokens taken from the packed ones, without a host loop; captured too."""
import pytest
import torch

from tests.test_prefix_attention_gpu import _compare
from tests.test_serving_step_gpu import PAGE, _ints, _Model

pytestmark = pytest.mark.gpu


def _step(dsa, m, state, new, tokens, S1, q, qr, kv):
    table, lens, refs = state
    old = lens.clamp(min=0)
    table, lens, refs, slots, positions, ends = dsa.paged_cache_plan(table, lens, refs, new, PAGE, tokens)
    groups, shared = dsa.paged_cache_prefixes(table, lens, PAGE)
    counts = (lens - old).clamp(min=0)
    at = ((ends - new.clamp(min=0))[:, None] + torch.arange(S1, device=ends.device)).clamp(max=tokens - 1)
    dsa.paged_cache_write_slots(m.caches, kv, slots)
    args = m.attend(q[at], None if qr is None else qr[at], table, lens, groups, shared, counts)
    out, mx, sm = dsa.paged_prefix_attention(**args)
    t = torch.arange(tokens, device=ends.device)
    r = torch.searchsorted(ends, t, right=True).clamp(max=ends.numel() - 1)
    packed = out[r, (t - (ends - new.clamp(min=0))[r]).clamp(0, S1 - 1)]
    return (table, lens, refs), counts, args, (out, mx, sm), packed


@pytest.mark.parametrize("latent,dtype,heads", [(False, torch.float16, 8), (True, torch.bfloat16, 16)])
def test_documented_packed_step(latent, dtype, heads):
    import dsa_triton_ascend_amd as dsa
    pages, wide, rows = 30, 9, 6
    m = _Model(latent, dtype, pages, heads)
    state = (_ints([[-1] * wide] * rows), _ints([-1] * rows), _ints([0] * pages))
    history = [[torch.empty(0, m.kv_heads, c, device="cuda", dtype=dtype) for c in m.cols] for _ in range(rows)]
    refused = 0
    for new in ([70, 5, 0, 33, 1, 0], [1, 1, 40, 1, -1, 9], [1, 30, 1, 120, 20, 1], [2, 1, 1, 1, 3, 1]):
        total = sum(max(n, 0) for n in new)
        q, qr, kv = m.tokens(total + 2)
        before = [max(n, 0) for n in state[1].tolist()]  # (a length below zero counts as zero)
        state, counts, args, got, packed = _step(dsa, m, state, _ints(new), total + 2, max(new), q, qr, kv)
        at = 0
        after = state[1].tolist()
        for r, n in enumerate(new):
            took = max(after[r] - before[r], 0)
            assert took in (0, max(n, 0)) and counts.tolist()[r] == took
            refused += n > 0 and not took
            if n < 0:
                history[r] = [x[:0] for x in history[r]]
            elif took:
                history[r] = [torch.cat([h, x[at:at + n]]) for h, x in zip(history[r], kv)]
                assert torch.equal(packed[at:at + n], got[0][r, :n])
            else:
                assert not packed[at:at + n].any()
            at += max(n, 0)
        _compare(args, history, after, act_q=counts.tolist(), got=got)
    assert refused


@pytest.mark.parametrize("latent,dtype,heads", [(False, torch.bfloat16, 8), (True, torch.float16, 16)])
def test_documented_packed_step_captured(latent, dtype, heads):
    """Other lengths and other tokens at each replay, against the same step made eagerly."""
    import dsa_triton_ascend_amd as dsa
    pages, wide, rows, tokens, S1 = 30, 9, 6, 40, 12
    m = _Model(latent, dtype, pages, heads)
    for c in m.caches:
        c.copy_(m.normal(*c.shape))
    state = (_ints([[-1] * wide] * rows), _ints([-1] * rows), _ints([0] * pages))
    state = dsa.paged_cache_plan(*state, _ints([70, 30, 0, 0, 17, 0]), PAGE, 117)[:3]
    state = dsa.paged_cache_fork(m.caches, *state, _ints([0, 0, 0, 1, 1, 4]))
    new = _ints([1] * rows)
    q, qr, kv = m.tokens(tokens)
    contents = [c.clone() for c in m.caches]
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        _step(dsa, m, state, new, tokens, S1, q, qr, kv)
        with torch.cuda.graph(graph, stream=stream):
            kept = _step(dsa, m, state, new, tokens, S1, q, qr, kv)
    torch.cuda.synchronize()
    for lengths in ([1] * 6, [12, 1, 1, -1, 2, 0], [3, 3, 3, 3, 3, 3], [0, 12, 0, 12, 1, 1]):
        new.copy_(_ints(lengths))
        for x in (q, *kv) + (() if qr is None else (qr,)):
            x.copy_(m.normal(*x.shape))
        for x, y in zip(m.caches, contents):
            x.copy_(y)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (*kept[0], *kept[3], kept[4], *m.caches)]
        for x, y in zip(m.caches, contents):
            x.copy_(y)
        want = _step(dsa, m, state, new, tokens, S1, q, qr, kv)
        for x, y in zip(got, (*want[0], *want[3], want[4], *m.caches)):
            assert torch.equal(x, y)
