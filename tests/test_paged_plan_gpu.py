"""paged_cache_plan, paged_cache_write_slots and paged_cache_prefixes against
loops over the requests; everything is exact."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

I32 = torch.int32


def _i(x):
    return torch.tensor(x, dtype=I32, device="cuda")


def _plan(table, lens, refs, new, page, tokens):
    """The step, request by request."""
    wide, pages = len(table[0]), len(refs)
    free = [i for i, r in enumerate(refs) if r == 0]
    refs = list(refs)
    at, total = 0, 0
    out, out_lens, ends = [], [], []
    slots, positions = [-1] * tokens, [0] * tokens

    def known(e):
        return e if 0 <= e < pages else -1

    for row, n, m in zip(table, lens, new):
        n = min(max(n, 0), wide * page)
        held = -(-n // page)
        if m < 0:
            held, kept, served = 0, [], False
        else:
            kept = [known(e) for e in row[:held]]
            fits = n + m <= wide * page
            need = -(-(n + m) // page) - held if fits else 0
            served = fits and (need == 0 or at + need <= len(free))
            if served:
                kept = kept + free[at:at + need]
                for e in free[at:at + need]:
                    refs[e] += 1
            at += need
        for e in row[held:]:
            if known(e) >= 0:
                refs[e] -= 1
        for i in range(max(m, 0)):
            if total + i >= tokens:
                break
            p = n + i
            positions[total + i] = p
            if served and kept[p // page] >= 0:
                slots[total + i] = kept[p // page] * page + p % page
        total += max(m, 0)
        ends.append(min(total, 2 ** 31 - 1))
        out.append(kept + [-1] * (wide - len(kept)))
        out_lens.append(0 if m < 0 else n + m if served else n)
    return out, out_lens, refs, slots, positions, ends


def _state(rng, rows, page, wide, pages, spare=0.0):
    """Rows of random lengths over scattered pages, some with a page reserved behind their tokens."""
    ids = list(range(pages))
    rng.shuffle(ids)
    table, lens = [], []
    for _ in range(rows):
        n = rng.choice([0, 1, page - 1, page, page + 1, rng.randint(0, max(1, wide * page // 2))])
        held = min(-(-n // page) + (rng.random() < spare), wide)
        if held > len(ids):
            n, held = 0, 0
        n = min(n, held * page)
        table.append([ids.pop() for _ in range(held)] + [-1] * (wide - held))
        lens.append(n)
    refs = [0] * pages
    for r in table:
        for e in r:
            if e >= 0:
                refs[e] += 1
    return table, lens, refs


def _check(table, lens, refs, new, page, tokens):
    import dsa_triton_ascend_amd as dsa
    given = [_i(table), _i(lens), _i(refs), _i(new)]
    kept = [t.clone() for t in given]
    got = dsa.paged_cache_plan(*given, page, tokens)
    want = _plan(table, lens, refs, new, page, tokens)
    for name, g, w in zip(("table", "lens", "refs", "slots", "positions", "ends"), got, want):
        assert g.dtype == I32 and g.tolist() == w, name
    for a, b in zip(given, kept):
        assert torch.equal(a, b)
    return got


@pytest.mark.parametrize("rows,page,wide,pages", [
    (1, 1, 1, 1), (1, 16, 4, 9), (7, 16, 9, 40), (64, 64, 33, 900), (65, 1, 70, 3000), (300, 48, 11, 1500),
    (1100, 16, 6, 4200), (2049, 7, 3, 9000), (4200, 16, 3, 6000)])
def test_plans(rows, page, wide, pages):
    rng = random.Random(rows * 31 + page)
    for kind in range(4):
        table, lens, refs = _state(rng, rows, page, wide, pages, 0.2 if kind else 0.0)
        new = [rng.choice([1, 1, 1, 0, -1, rng.randint(1, 2 * page)]) if kind else 1 for _ in range(rows)]
        tokens = sum(max(m, 0) for m in new)
        _check(table, lens, refs, new, page, max(0, tokens + rng.choice([0, 5, -3])))


def test_long_rows():
    rng = random.Random(5)
    page, wide = 16, 700
    for pages in (2000, 3999, 9001):
        table, lens, refs = _state(rng, 5, page, wide, pages)
        _check(table, lens, refs, [3517, 0, 1, -1, 2999], page, 3517 + 1 + 2999 + 37)


def test_pages_that_do_not_last():
    # two free pages: the first row gets one, the second needs two, the third none
    table = [[0, -1, -1], [1, -1, -1], [2, -1, -1], [3, -1, -1]]
    got = _check(table, [4, 4, 2, 4], [1, 1, 1, 1, 0, 0], [1, 5, 2, 1], 4, 9)
    assert got[1].tolist() == [5, 4, 4, 4]
    # a row that outgrows the table takes nothing from those after it
    got = _check(table, [4, 4, 2, 4], [1, 1, 1, 1, 0, 0], [9, 1, 1, 1], 4, 12)
    assert got[1].tolist() == [4, 5, 3, 5]
    # pages of an ended row are not handed out by the same call
    got = _check(table, [4, 4, 2, 4], [1, 1, 1, 1, 0, 0], [-1, 1, 1, 5], 4, 7)
    assert got[1].tolist() == [0, 5, 3, 4] and got[2].tolist() == [0, 1, 1, 1, 1, 0]


def test_odd_states():
    # negative and overlong lengths, entries outside the pool, holes, counts that others hold
    table = [[0, 7, -1], [-5, 2, -1], [3, 99, 1], [4, -1, -1]]
    _check(table, [-3, 6, 50, 3], [2, 1, 3, 1, 1, 0, 0, 1], [2, 4, 0, 1], 4, 7)
    _check(table, [-3, 6, 50, 3], [2, 1, 3, 1, 1, 0, 0, 1], [2, 4, 1, -7], 4, 3)
    big = 2 ** 31 - 1
    got = _check(table, [1, 5, 12, 3], [1, 1, 1, 1, 1, 0, 0, 1], [1, big, big, big], 4, 100)
    assert got[5].tolist() == [1, big, big, big]


def test_no_tokens_and_padding_only():
    table, refs = [[0, 1], [2, -1]], [1, 1, 1, 0]
    _check(table, [8, 3], refs, [0, 0], 4, 0)
    _check(table, [8, 3], refs, [0, -1], 4, 5)


def test_plan_replays():
    import dsa_triton_ascend_amd as dsa
    rng = random.Random(2)
    page, wide = 16, 20
    table, lens, refs = _state(rng, 9, page, wide, 200)
    t, l, r = _i(table), _i(lens), _i(refs)
    new = _i([1] * 9)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        dsa.paged_cache_plan(t, l, r, new, page, 64)
        dsa.paged_cache_prefixes(t, l, page)
        with torch.cuda.graph(graph, stream=stream):
            out = dsa.paged_cache_plan(t, l, r, new, page, 64)
            pre = dsa.paged_cache_prefixes(out[0], out[1], page)
    for step in range(4):
        m = [rng.choice([1, 1, 7, 0, -1]) for _ in range(9)]
        new.copy_(_i(m))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = _plan(t.tolist(), l.tolist(), r.tolist(), m, page, 64)
        for g, w in zip(out, want):
            assert g.tolist() == w
        assert [x.tolist() for x in pre] == list(_prefixes(want[0], want[1], page))
        t.copy_(out[0]), l.copy_(out[1]), r.copy_(out[2])


# ---- slots ----

@pytest.mark.parametrize("cols,dtype", [((512, 64, 128), torch.bfloat16), ((3,), torch.uint8), ((1, 7), torch.float16),
                                        ((33, 2, 4), torch.float32), ((16,) * 40, torch.float16)])
@pytest.mark.parametrize("lead", [(1,), (137,), (3, 5), (4, 1)])
def test_slots(cols, dtype, lead):
    import dsa_triton_ascend_amd as dsa
    g = torch.Generator().manual_seed(len(cols) + lead[0])
    pages, page, heads = 21, 9, 2
    n = 1
    for x in lead:
        n *= x

    def values(*shape):
        return torch.randint(0, 200, shape, generator=g).to(dtype).cuda()

    caches = [values(pages, page, heads, c) for c in cols]
    # rows with gaps between tokens and between sequences
    wide = [values(*(x + 1 for x in lead), heads, c) for c in cols]
    rows = [w[1:] if len(lead) == 1 else w[:lead[0], 1:] for w in wide]
    slots = torch.randperm(pages * page, generator=g)[:n].int().view(lead).clone()
    flat = slots.view(-1)
    for i, bad in ((2, -1), (7, pages * page), (9, -2 ** 31), (11, 2 ** 31 - 1)):
        if i < n:
            flat[i] = bad
    want = [c.clone() for c in caches]
    for w, r in zip(want, rows):
        for i, s in enumerate(flat.tolist()):
            if 0 <= s < pages * page:
                w.view(pages * page, -1)[s] = r.reshape(n, -1)[i]
    versions = [c._version for c in caches]
    dsa.paged_cache_write_slots(caches, rows, slots.cuda())
    for c, w, v in zip(caches, want, versions):
        assert torch.equal(c, w) and c._version > v


def test_slots_of_a_plan_are_where_write_puts_the_rows():
    import dsa_triton_ascend_amd as dsa
    rng = random.Random(11)
    page = 16
    table, lens, refs = _state(rng, 6, page, 12, 60)
    new = [1, 30, 0, 17, 1, 5]
    out, out_lens, _, slots, positions, ends = dsa.paged_cache_plan(_i(table), _i(lens), _i(refs), _i(new), page, 60)
    assert out_lens.tolist() == [a + b for a, b in zip(lens, new)]
    rows = torch.randn(60, 1, 64, device="cuda")
    a, b = torch.zeros(60, page, 1, 64, device="cuda"), torch.zeros(60, page, 1, 64, device="cuda")
    dsa.paged_cache_write_slots(a, rows, slots)
    dsa.paged_cache_write(b, rows, out, _i(lens), row_lengths=ends, layout="TND")
    assert torch.equal(a, b) and a.any()


def test_slots_in_a_large_cache():
    """Offsets past 2^32 bytes."""
    import dsa_triton_ascend_amd as dsa
    cache = torch.zeros(2 ** 17 + 3, 64, 1, 512, dtype=torch.float16, device="cuda")  # 8.6 GB
    flat = cache.view(-1, 512)
    slots = _i([flat.shape[0] - 1, 0, 2 ** 22 + 5, flat.shape[0]])
    rows = torch.randn(4, 1, 512, device="cuda", dtype=torch.float16)
    dsa.paged_cache_write_slots(cache, rows, slots)
    assert torch.equal(flat[slots[:3].long()], rows[:3, 0])
    assert int((flat[:, 0] != 0).sum()) <= 3


# ---- prefixes ----

def _prefixes(table, lens, page, least=1):
    groups, shared, links = [], [], []

    def close():
        shared.extend([min(links) * page if links else 0] * (len(groups) - len(shared)))
        links.clear()

    for b, row in enumerate(table):
        n = 0
        if b:
            whole = min(max(0, min(lens[b], lens[b - 1])) // page, len(row))
            while n < whole and row[n] == table[b - 1][n] and row[n] >= 0:
                n += 1
        if n and n * page >= least:
            links.append(n)
            groups.append(groups[-1])
        else:
            close()
            groups.append(b)
    close()
    return groups, shared


@pytest.mark.parametrize("rows,page,wide", [(1, 16, 3), (2, 1, 1), (5, 16, 9), (16, 8, 512),
                                            (17, 8, 512), (16, 8, 513), (3, 1, 1200), (64, 4, 70), (70, 16, 600),
                                            (1030, 8, 5), (3000, 16, 3)])
@pytest.mark.parametrize("least", [0, 1, 40])
def test_prefixes(rows, page, wide, least):
    import dsa_triton_ascend_amd as dsa
    rng = random.Random(rows + least)
    table, lens, at = [], [], 0
    while len(table) < rows:
        trunk = rng.randint(0, wide)
        family = [rng.randint(0, 10 ** 6) for _ in range(trunk)]
        for _ in range(rng.choice([1, 2, 3, 17, 200])):
            share = trunk if rng.random() < 0.8 else rng.randint(0, trunk)
            row = family[:share]
            row += [rng.randint(0, 10 ** 6) for _ in range(rng.randint(0, wide - len(row)))]
            if row and rng.random() < 0.05:
                row[rng.randrange(len(row))] = -1
            n = rng.choice([len(row) * page, max(0, len(row) * page - rng.randint(0, page)), rng.randint(-3, wide * page)])
            table.append(row + [-1] * (wide - len(row)))
            lens.append(n)
    table, lens = table[:rows], lens[:rows]
    groups, shared = dsa.paged_cache_prefixes(_i(table), _i(lens), page, min_tokens=least)
    want = _prefixes(table, lens, page, least)
    assert groups.tolist() == want[0] and shared.tolist() == want[1]


def test_prefixes_of_beams():
    """After a fork the beams of a prompt share what they had before they parted."""
    import dsa_triton_ascend_amd as dsa
    page = 4
    table = _i([[0, 1, 2, 3], [4, 5, -1, -1]])
    lens, refs = _i([14, 7]), _i([1] * 6 + [0] * 10)
    t, l, r = dsa.paged_cache_fork([], table, lens, refs, parents=_i([0, 0, 0, 1, 1]), new_tokens=1, page_size=page)
    groups, shared = dsa.paged_cache_prefixes(t, l, page)
    assert groups.tolist() == [0, 0, 0, 3, 3] and shared.tolist() == [12, 12, 12, 4, 4]


def test_compiled_and_python_calls_agree(monkeypatch):
    import dsa_triton_ascend_amd as dsa
    from dsa_triton_ascend_amd import _lib
    assert _lib.calls() is not _lib._NoCalls
    table, lens, refs = _i([[3, 1, -1], [3, 8, 0]]), _i([20, 40]), _i([1, 1, 0, 2, 0, 0, 0, 0, 1])
    new = _i([3, 8])
    rows = torch.randn(12, 1, 64, device="cuda")

    def f():
        out = dsa.paged_cache_plan(table, lens, refs, new, 16, 12)
        cache = torch.zeros(9, 16, 1, 64, device="cuda")
        dsa.paged_cache_write_slots([cache], [rows], out[3])
        return out + dsa.paged_cache_prefixes(table, lens, 16) + (cache,)

    c = _lib.calls()
    assert c.plan(table, lens, refs, new, 16, 12) is not None and c.prefixes(table, lens, 16, 1) is not None
    for bad in ((table.long(), lens, refs, new, 16, 12), (table, lens[:1], refs, new, 16, 12),
                (table, lens, refs, new, 0, 12), (table, lens, refs, new, 16, -1), (table, lens, refs, new.cpu(), 16, 12)):
        assert c.plan(*bad) is None
    a = f()
    monkeypatch.setattr(_lib, "_calls", _lib._NoCalls)
    b = f()
    monkeypatch.undo()
    for u, v in zip(a, b):
        assert torch.equal(u, v)
