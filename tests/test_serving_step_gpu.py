"""Serving requests of many lengths with the operators together: plan, rotate
(positions on three axes), write to slots, find the prefixes, attend; beams
fork behind a common prompt with an image in it, requests come, wait for pages
and end, pages are compacted on the way.  Against histories per request: the
tables exactly, the rotation and the attention in 64 bits (bounds of their own
tests)."""
import math
import random

import pytest
import torch

from tests.test_prefix_attention_gpu import INT64_MAX, _compare
from tests.test_rotary_axes_gpu import _near, _turn

pytestmark = pytest.mark.gpu

PAGE, SECTIONS = 16, (12, 10, 10)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class _Model:
    """Random projections of a step's tokens; caches of one layer."""

    def __init__(self, latent, dtype, pages, heads):
        import dsa_triton_ascend_amd as dsa
        self.latent, self.dtype, self.heads = latent, dtype, heads
        self.g = torch.Generator(device="cuda").manual_seed(5)
        self.cols = [512, 64] if latent else [128, 128]
        self.kv_heads = 1 if latent else 2
        self.caches = [torch.full((pages, PAGE, self.kv_heads, c), float("nan"), device="cuda", dtype=dtype)
                       for c in self.cols]
        self.inv, _ = dsa.rotary_frequencies(64)

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.g, device="cuda").to(self.dtype)

    def tokens(self, n):
        q = self.normal(n, self.heads, self.cols[0])
        qr = self.normal(n, self.heads, 64) if self.latent else None
        return q, qr, [self.normal(n, self.kv_heads, c) for c in self.cols]

    def rotate(self, dsa, q, qr, rows, axes, check=True):
        """(query, its rope part, the caches' rows), rotated."""
        x, y = (qr, rows[1]) if self.latent else (q, rows[0])
        xo, yo = dsa.rotary_embedding(x, y, axes, self.inv, layout="TND", sections=SECTIONS, sections_interleaved=True)
        if check:
            _near(xo, _turn(x, axes, self.inv, SECTIONS, True, 0))
            _near(yo, _turn(y, axes, self.inv, SECTIONS, True, 0))
        return (q, xo, [rows[0], yo]) if self.latent else (xo, None, [yo, rows[1]])

    def attend(self, q, qr, table, lens, groups, shared, counts=None):
        scale = 1.0 / math.sqrt(self.cols[0] + (64 if self.latent else 0))
        return dict(query=q, key=self.caches[0], value=None if self.latent else self.caches[1], block_table=table,
                    actual_seq_lengths_kv=lens, prefix_groups=groups, prefix_lengths=shared, scale_value=scale,
                    query_rope=qr, key_rope=self.caches[1] if self.latent else None,
                    actual_seq_lengths_query=counts, sparse_mode=3, pre_tokens=INT64_MAX, next_tokens=INT64_MAX,
                    return_softmax_lse=True)


def _axes(positions):
    """Positions in time, height and width: an image at tokens 8 to 43 of each request."""
    image = (positions >= 8) & (positions < 44)
    at = positions - 8
    return torch.stack([torch.where(image, 8 + 0 * at, positions), torch.where(image, 8 + at // 6, positions),
                        torch.where(image, 8 + at % 6, positions)]).int()


@pytest.mark.parametrize("latent,dtype,heads", [(False, torch.float16, 8), (True, torch.bfloat16, 16)])
@pytest.mark.parametrize("side", [False, True])
def test_serving_loop(latent, dtype, heads, side):
    import dsa_triton_ascend_amd as dsa
    stream = torch.cuda.Stream() if side else torch.cuda.current_stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        _loop(dsa, latent, dtype, heads)
    torch.cuda.synchronize()


def _loop(dsa, latent, dtype, heads):
    rng = random.Random(7)
    pages, wide, rows = 40, 12, 7
    m = _Model(latent, dtype, pages, heads)
    table = _ints([[-1] * wide] * rows)
    lens, refs = _ints([0] * rows), _ints([0] * pages)
    history = [[torch.empty(0, m.kv_heads, c, device="cuda", dtype=dtype) for c in m.cols] for _ in range(rows)]
    steps = [[75, 0, 0, 0, 0, 0, 0],      # the common prompt
             "fork",                      # three beams behind it
             [1, 1, 1, 0, 33, 0, 0],      # a prompt begins while they decode
             [3, 1, 2, 0, 1, 70, 0],      # speculated tokens, another prompt
             [1, 1, 1, 0, 1, 1, 30],
             [1, -1, 1, 5, 1, 1, 1],      # a beam ends, its row takes none; row 3 begins
             "compact",
             [30, 1, 1, 1, 20, 40, 9],
             [70, 60, 1, 50, 20, 30, 40],  # the pages do not last
             [1, 1, 1, 1, -1, 1, 1],
             [1, 40, 1, 1, 16, 1, 1]]
    waited, beams = 0, True
    for step in steps:
        if step == "fork":
            table, lens, refs = dsa.paged_cache_fork(m.caches, table, lens, refs, _ints([0, 0, 0, -1, -1, -1, -1]))
            history = [[x.clone() for x in history[0]] for _ in range(3)] + history[3:]
            continue
        if step == "compact":
            table, refs, _ = dsa.paged_cache_compact(m.caches, table, refs)
            used = int((refs > 0).sum())
            assert (refs[:used] > 0).all() and not refs[used:].any()
            continue
        new = list(step)
        total = sum(max(n, 0) for n in new)
        padded = total + rng.randint(0, 3)
        before = lens.tolist()
        table, lens, refs, slots, positions, ends = dsa.paged_cache_plan(table, lens, refs, _ints(new), PAGE, padded)
        # the table's pages are counted, no page belongs to two rows but for the full ones that a fork shared
        listed = [e for row in table.tolist() for e in row if e >= 0]
        assert refs.tolist() == [listed.count(i) for i in range(pages)]
        after = lens.tolist()
        served = [n >= 0 and a == b + n for n, a, b in zip(new, after, before)]
        for r, n in enumerate(new):
            assert after[r] == (0 if n < 0 else before[r] + (n if served[r] else 0))
        waited += sum(n > 0 and not s for n, s in zip(new, served))
        ends = [0] + ends.tolist()
        assert ends[-1] == total
        axes = _axes(positions)
        raw = m.tokens(padded)
        q, qr, kv = m.rotate(dsa, *raw, axes)
        dsa.paged_cache_write_slots(m.caches, kv, slots)
        for r, n in enumerate(new):
            assert positions[ends[r]:ends[r + 1]].tolist() == list(range(before[r], before[r] + max(n, 0)))
            if n < 0:
                history[r] = [x[:0] for x in history[r]]
            elif served[r]:
                history[r] = [torch.cat([h, x[ends[r]:ends[r + 1]]]) for h, x in zip(history[r], kv)]
        groups, shared = dsa.paged_cache_prefixes(table, lens, PAGE)
        hosted, kept = table.tolist(), lens.tolist()
        for r in range(1, rows):
            same = 0
            while (same < min(kept[r], kept[r - 1]) // PAGE and hosted[r][same] == hosted[r - 1][same] >= 0):
                same += 1
            assert (groups[r] == groups[r - 1]) == (same > 0) and (not same or shared[r] <= same * PAGE)
        beams = beams and step[1] >= 0  # until the second one ends
        if beams and after[1]:
            assert groups[:3].tolist() == [0, 0, 0] and shared[:3].tolist() == [64, 64, 64]
        # a request's tokens, padded to the longest of the step
        counts = [max(n, 0) if s else 0 for n, s in zip(new, served)]
        S1 = max(counts)
        if not S1:
            continue
        pad = [torch.zeros(rows, S1, *x.shape[1:], device="cuda", dtype=dtype) if x is not None else None for x in (q, qr)]
        for r, n in enumerate(counts):
            for x, y in zip(pad, (q, qr)):
                if y is not None:
                    x[r, :n] = y[ends[r]:ends[r] + n]
        args = m.attend(pad[0], pad[1], table, lens, groups, shared, _ints(counts))
        _compare(args, history, after, act_q=counts)
        _compare(dict(args, min_tokens=1), history, after, act_q=counts)
    assert waited  # some request was refused and waited in place


@pytest.mark.parametrize("latent,dtype,heads", [(False, torch.bfloat16, 8), (True, torch.float16, 16)])
@pytest.mark.parametrize("least", [None, 1])
def test_captured_decoding_step(latent, dtype, heads, least):
    """A decoding step whose state stays on the device, replayed beside the same steps made eagerly."""
    import dsa_triton_ascend_amd as dsa
    pages, wide, rows = 40, 8, 4
    m = _Model(latent, dtype, pages, heads)
    state = [_ints([[-1] * wide] * rows), _ints([0] * rows), _ints([0] * pages)]
    state = list(dsa.paged_cache_plan(*state, _ints([70, 0, 0, 0]), PAGE, 70)[:3])
    for c in m.caches:
        c.copy_(m.normal(*c.shape))
    state = list(dsa.paged_cache_fork(m.caches, *state, _ints([0] * rows)))
    start, contents = [x.clone() for x in state], [c.clone() for c in m.caches]
    q, qr, kv = m.tokens(rows)
    one = _ints([1] * rows)

    def step():
        *after, slots, positions, _ = dsa.paged_cache_plan(*state, one, PAGE, rows)
        for x, y in zip(state, after):
            x.copy_(y)
        a, b, rows_ = m.rotate(dsa, q, qr, kv, _axes(positions), check=False)
        dsa.paged_cache_write_slots(m.caches, rows_, slots)
        groups, shared = dsa.paged_cache_prefixes(state[0], state[1], PAGE)
        return dsa.paged_prefix_attention(**m.attend(a[:, None], None if b is None else b[:, None], state[0], state[1],
                                                     groups, shared), min_tokens=least)

    inputs = [[torch.randn_like(x.float()).to(dtype) for x in (q, qr, *kv) if x is not None] for _ in range(12)]

    def put(i):
        for x, y in zip([x for x in (q, qr, *kv) if x is not None], inputs[i]):
            x.copy_(y)

    def reset():
        for x, y in zip(state + m.caches, start + contents):
            x.copy_(y)

    want = []
    for i in range(12):
        put(i)
        want.append([x.clone() for x in step()])
    held = [x.clone() for x in state]
    reset()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        step()
        with torch.cuda.graph(graph, stream=stream):
            out = step()
    torch.cuda.synchronize()
    reset()
    for i in range(12):
        put(i)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(out, want[i]):
            assert torch.equal(x, y), f"replay {i}"
    for x, y in zip(state, held):
        assert torch.equal(x, y)
    assert state[1].tolist() == [82] * rows
