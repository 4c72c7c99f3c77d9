"""Writing, forking and compacting the pages of a cache against plain Python.
Everything is copies and whole numbers: results are equal."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _caches(pages, page, rows, dtypes):
    return [(torch.randn(pages, page, *r, device="cuda") * 100).to(d) for r, d in zip(rows, dtypes)]


ROWS = [((1, 512), (1, 64), (1, 128)), ((3, 5),), ((2, 8), (1, 1), (1, 12))]
TYPES = [(torch.bfloat16,) * 3, (torch.float16,), (torch.float32, torch.uint8, torch.bfloat16)]


@pytest.mark.parametrize("page", [1, 3, 16, 64])
@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("layout", ["BSND", "TND"])
def test_write(page, kind, layout):
    import dsa_triton_ascend_amd as dsa
    rng = random.Random(page * 10 + kind)
    B, S = 5, 7
    old = [0, 1, page - 1, 3 * page, 50]
    new = [S, 0, 3, 1, 5]
    wide = (max(o + n for o, n in zip(old, new)) + page - 1) // page
    pages = B * wide + 3
    ids = rng.sample(range(pages), B * wide)
    table = [ids[b * wide:(b + 1) * wide] for b in range(B)]
    table[4][(50 // page)] = -1            # tokens without a page are dropped
    caches = _caches(pages, page, ROWS[kind], TYPES[kind])
    want = [c.clone() for c in caches]
    if layout == "BSND":
        rows = [(torch.randn(B, S, *r, device="cuda") * 100).to(d) for r, d in zip(ROWS[kind], TYPES[kind])]
        lengths = _ints(new)
        take = [[r[b, s] for r in rows] for b in range(B) for s in range(new[b])]
    else:
        total = sum(new) + 4               # four rows behind the last sequence
        rows = [(torch.randn(total, *r, device="cuda") * 100).to(d) for r, d in zip(ROWS[kind], TYPES[kind])]
        lengths = _ints([sum(new[:b + 1]) for b in range(B)])
        take = [[r[t] for r in rows] for t in range(sum(new))]
    i = 0
    for b in range(B):
        for s in range(new[b]):
            p = old[b] + s
            blk = table[b][p // page]
            if blk >= 0:
                for w, r in zip(want, take[i]):
                    w[blk, p % page] = r
            i += 1
    dsa.paged_cache_write(caches, rows, _ints(table), _ints(old), row_lengths=lengths, layout=layout)
    for c, w in zip(caches, want):
        assert torch.equal(c, w)


def test_write_strided_rows_past_the_table_and_many_caches():
    import dsa_triton_ascend_amd as dsa
    page, pages = 4, 9
    proj = torch.randn(2, 3, 576, device="cuda").bfloat16()
    rows = [proj[..., None, :512], proj[..., None, 512:]]
    caches = _caches(pages, page, [(1, 512), (1, 64)], [torch.bfloat16] * 2)
    want = [c.clone() for c in caches]
    table = _ints([[3, 5], [7, 0]])
    dsa.paged_cache_write(caches, rows, table, _ints([2, 6]))   # sequence 1 runs past its two pages
    for w, r in zip(want, rows):
        w[3, 2], w[3, 3], w[5, 0] = r[0, 0], r[0, 1], r[0, 2]
        w[0, 2], w[0, 3] = r[1, 0], r[1, 1]
    assert all(torch.equal(c, w) for c, w in zip(caches, want))
    # negative lengths count as none; more caches than one launch takes
    many = _caches(pages, page, [(1, 8 + i) for i in range(70)], [torch.float16] * 70)
    rows = [torch.randn(2, 1, *c.shape[2:], device="cuda").half() for c in many]
    want = [c.clone() for c in many]
    for w, r in zip(want, rows):
        w[3, 0], w[7, 1] = r[0, 0], r[1, 0]
    dsa.paged_cache_write(many, rows, table, _ints([-3, 1]))
    assert all(torch.equal(c, w) for c, w in zip(many, want))
    # no tokens
    dsa.paged_cache_write(many[:1], [rows[0][:, :0]], table, _ints([0, 0]))


def _fork(table, lens, refs, parents, new, page):
    """(new table, new lengths, new counts, moves) from the definition."""
    wide = len(table[0])
    free = [i for i, r in enumerate(refs) if r == 0]
    out, out_lens, moves, taken, seen = [], [], [], 0, set()
    for c, p in enumerate(parents):
        empty = [-1] * wide
        if not 0 <= p < len(table):
            out.append(empty)
            out_lens.append(0)
            continue
        n = min(max(lens[p], 0), wide * page)
        held, want = -(-n // page), -(-(n + new) // page)
        first = p not in seen
        seen.add(p)
        row = list(table[p][:held])
        copy = bool(n % page) and row[-1] >= 0 and not (first and refs[row[-1]] == 1)
        if want > wide:
            out.append(empty)
            out_lens.append(-1)
            continue
        need = copy + want - held
        start = taken
        taken += need
        if need and start + need > len(free):
            out.append(empty)
            out_lens.append(-1)
            continue
        mine = free[start:start + need]
        if copy:
            moves.append((row[-1], mine[0], n % page))
            row[-1] = mine[0]
            mine = mine[1:]
        row += mine
        out.append(row + [-1] * (wide - len(row)))
        out_lens.append(n)
    counts = list(refs)
    for rows, sign in ((out, 1), (table, -1)):
        for r in rows:
            for e in r:
                if e >= 0:
                    counts[e] += sign
    return out, out_lens, counts, moves


def _pool(rng, rows, page, hi, spare, extra=0):
    """Sequences in groups that share their first pages."""
    table, lens, trunks = [], [], []
    wide = -(-hi // page) + 2
    pages = rows * wide + spare
    ids = rng.sample(range(pages), pages)
    for b in range(rows):
        n = rng.randint(0, hi)
        if b and rng.random() < 0.5:
            n, trunk = lens[b - 1], trunks[b - 1]
        else:
            trunk = [ids.pop() for _ in range(rng.randint(0, n // page))]
        row = trunk + [ids.pop() for _ in range(-(-n // page) - len(trunk))]
        row += [ids.pop() for _ in range(rng.randint(0, extra))]  # reserved pages past the tokens
        table.append((row + [-1] * wide)[:wide])
        lens.append(n)
        trunks.append(trunk)
    refs = [0] * pages
    for r in table:
        for e in r:
            if e >= 0:
                refs[e] += 1
    return table, lens, refs


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("page", [1, 5, 16])
def test_fork(seed, page):
    import dsa_triton_ascend_amd as dsa
    rng = random.Random(seed * 100 + page)
    rows = rng.choice([1, 4, 40])
    table, lens, refs = _pool(rng, rows, page, rng.choice([3, 60]), 10, extra=seed % 3)
    if seed % 2:
        for e in rng.sample([i for i, r in enumerate(refs) if r], min(3, sum(r > 0 for r in refs))):
            refs[e] += 1                    # held by something outside the table
    kids = rng.choice([1, rows, 3 * rows, 1100])
    parents = [rng.randint(-1, rows) for _ in range(kids)]  # -1 and rows: empty rows
    new = rng.choice([0, 1, page, 2 * page + 1])
    caches = _caches(len(refs), page, ROWS[seed % 3], TYPES[seed % 3])
    w_table, w_lens, w_refs, moves = _fork(table, lens, refs, parents, new, page)
    want = [c.clone() for c in caches]
    for w in want:
        for src, dst, n in moves:
            w[dst, :n] = w[src, :n]
    old = [_ints(table), _ints(lens), _ints(refs)]
    t, l, r = dsa.paged_cache_fork(caches, *old, parents=_ints(parents), new_tokens=new)
    assert t.tolist() == w_table and l.tolist() == w_lens and r.tolist() == w_refs
    assert all(torch.equal(c, w) for c, w in zip(caches, want))
    assert [x.tolist() for x in old] == [table, lens, refs]
    # tables only
    t2, l2, r2 = dsa.paged_cache_fork([], *old, parents=_ints(parents), new_tokens=new, page_size=page)
    assert torch.equal(t2, t) and torch.equal(l2, l) and torch.equal(r2, r)


def test_fork_without_parents_extends_and_releases():
    import dsa_triton_ascend_amd as dsa
    page = 4
    table = [[0, 1, -1], [2, 5, 6], [-1, -1, -1], [3, -1, -1]]
    lens = [6, 4, 0, 4]
    refs = [1, 1, 1, 1, 0, 1, 1, 0, 0]     # row 1 holds two pages past its tokens
    cache = torch.randn(9, page, 1, 8, device="cuda")
    kept = cache.clone()
    t, l, r = dsa.paged_cache_fork(cache, _ints(table), _ints(lens), _ints(refs), new_tokens=3)
    assert t.tolist() == [[0, 1, 4], [2, 7, -1], [8, -1, -1], [-1, -1, -1]]
    assert l.tolist() == [6, 4, 0, -1]      # three free pages: the last row gets none
    assert r.tolist() == [1, 1, 1, 0, 1, 0, 0, 1, 1]
    assert torch.equal(cache, kept)


@pytest.mark.parametrize("pages,live", [(1, 1.0), (1, 0.0), (7, 0.5), (1024, 0.3), (1025, 0.9), (5000, 0.02),
                                        (5000, 0.5), (3000, 0.0), (2048, 1.0)])
def test_compact(pages, live):
    import dsa_triton_ascend_amd as dsa
    rng = random.Random(pages)
    page, kind = rng.choice([1, 3, 8]), pages % 3
    used = sorted(rng.sample(range(pages), int(pages * live)))
    refs = [0] * pages
    for i in used:
        refs[i] = rng.randint(1, 4)
    table = [[rng.choice(used) if used and rng.random() < 0.8 else rng.choice([-1, -7, pages, pages + 5])
              for _ in range(9)] for _ in range(6)]
    caches = _caches(pages, page, ROWS[kind], TYPES[kind])
    n = len(used)
    holes = [i for i in range(n) if refs[i] == 0]
    high = [i for i in used if i >= n]
    page_map = [(i if i < n else holes[high.index(i)]) if refs[i] else -1 for i in range(pages)]
    want = [c.clone() for c in caches]
    for w in want:
        for src, dst in zip(high, holes):
            w[dst] = w[src]
    w_refs = [0] * pages
    for i, to in enumerate(page_map):
        if to >= 0:
            w_refs[to] = refs[i]
    w_table = [[page_map[e] if 0 <= e < pages else -1 for e in r] for r in table]
    t, r, m = dsa.paged_cache_compact(caches, _ints(table), _ints(refs))
    assert t.tolist() == w_table and r.tolist() == w_refs and m.tolist() == page_map
    assert all(torch.equal(c, w) for c, w in zip(caches, want))


def test_many_caches_fork_and_compact():
    import dsa_triton_ascend_amd as dsa
    page = 4
    caches = _caches(12, page, [(1, 3 + i % 7) for i in range(67)], [torch.float16] * 67)
    want = [c.clone() for c in caches]
    t, l, r = dsa.paged_cache_fork(caches, _ints([[9, 10, -1]]), _ints([6]), _ints([0] * 9 + [1, 1, 0]),
                                   parents=_ints([0, 0]))
    for w in want:
        w[0, :2] = w[10, :2]
    assert t.tolist() == [[9, 10, -1], [9, 0, -1]]
    assert all(torch.equal(c, w) for c, w in zip(caches, want))
    t, r, m = dsa.paged_cache_compact(caches, t, r)
    for w in want:
        w[1], w[2] = w[9], w[10]
    assert t.tolist() == [[1, 2, -1], [1, 0, -1]]
    assert all(torch.equal(c, w) for c, w in zip(caches, want))


def test_graph_replays():
    """One captured step (fork, write, compact) replayed against the eager one."""
    import dsa_triton_ascend_amd as dsa
    rng = random.Random(4)
    page = 8
    table, lens, refs = _pool(rng, 6, page, 40, 20)
    state = [_ints(table), _ints(lens), _ints(refs)]
    parents = _ints([1, 1, 0, 4, 4, -1])
    start = _caches(len(refs), page, ROWS[0], TYPES[0])
    caches = [c.clone() for c in start]
    rows = [torch.randn(6, 1, *c.shape[2:], device="cuda").bfloat16() for c in caches]

    def step(cs):
        t, l, r = dsa.paged_cache_fork(cs, *state, parents=parents, new_tokens=1)
        dsa.paged_cache_write(cs, rows, t, l)
        return [l, *dsa.paged_cache_compact(cs, t, r)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step([c.clone() for c in start])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(caches)
    for i in range(3):
        for c, s in zip(caches, start):
            c.copy_(s)
        parents.copy_(_ints([i, 1, i, 4 - i, 4, -1]))
        for r in rows:
            r.copy_(torch.randn_like(r))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        mine = [s.clone() for s in start]
        eager = step(mine)
        assert all(torch.equal(a, b) for a, b in zip(got, eager))
        assert all(torch.equal(a, b) for a, b in zip(caches, mine))


def test_write_counts_that_do_not_rise():
    """Whatever the cumulative counts are, what lies around the pages keeps its values."""
    import dsa_triton_ascend_amd as dsa
    pool = torch.full((6, 4, 1, 8), 7.0, device="cuda")
    cache = pool[2:4]  # two pages, with two before and two behind them
    table = torch.tensor([[0], [1], [1]], dtype=torch.int32, device="cuda")
    lens = torch.zeros(3, dtype=torch.int32, device="cuda")
    rows = torch.arange(6 * 8, device="cuda", dtype=torch.float32).view(6, 1, 8)
    counts = torch.tensor([2, 30, 4], dtype=torch.int32, device="cuda")
    dsa.paged_cache_write(cache, rows, table, lens, row_lengths=counts, layout="TND")
    assert (pool[:2] == 7).all() and (pool[4:] == 7).all()
    assert torch.equal(pool[2, :2], rows[:2]) and (pool[2, 2:] == 7).all()
    assert torch.equal(pool[3], rows[2:6])
    for counts in ([5, 1, 6], [-2 ** 31, 4, 6], [-1, -2 ** 31, 6]):
        pool.fill_(7.0)
        dsa.paged_cache_write(cache, rows, table, lens, layout="TND",
                              row_lengths=torch.tensor(counts, dtype=torch.int32, device="cuda"))
        assert (pool[:2] == 7).all() and (pool[4:] == 7).all()


@pytest.mark.parametrize("page", [1, 16])
def test_fork_for_more_tokens_than_any_table_holds(page):
    import dsa_triton_ascend_amd as dsa
    cache = torch.zeros(8, page, 1, 8, device="cuda")
    table = torch.tensor([[2, 5], [-1, -1]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([2, 0], dtype=torch.int32, device="cuda")
    refs = torch.zeros(8, dtype=torch.int32, device="cuda")
    refs[2] = refs[5] = 1
    new_table, new_lens, new_refs = dsa.paged_cache_fork(cache, table, lens, refs, new_tokens=2 ** 31 - 1)
    assert (new_table == -1).all() and (new_lens == -1).all() and (new_refs == 0).all()


@pytest.mark.parametrize("rows,kids", [(4096, 5000), (4097, 4500), (9000, 3)])
def test_fork_of_many_rows(rows, kids):
    import dsa_triton_ascend_amd as dsa
    rng = random.Random(rows)
    page = 8
    table, lens, refs = _pool(rng, rows, page, 20, 1500)
    parents = [rng.randint(-1, rows) for _ in range(kids)]
    caches = _caches(len(refs), page, ROWS[0], TYPES[0])
    w_table, w_lens, w_refs, moves = _fork(table, lens, refs, parents, 1, page)
    want = [c.clone() for c in caches]
    moved = torch.tensor(moves, device="cuda").view(-1, 3)
    for w in want:
        for k in moved[:, 2].unique().tolist():
            m = moved[moved[:, 2] == k]
            w[m[:, 1], :k] = w[m[:, 0], :k]
    t, l, r = dsa.paged_cache_fork(caches, _ints(table), _ints(lens), _ints(refs), parents=_ints(parents), new_tokens=1)
    assert t.tolist() == w_table and l.tolist() == w_lens and r.tolist() == w_refs
    assert all(torch.equal(c, w) for c, w in zip(caches, want))


@pytest.mark.parametrize("pages", [16384, 16385, 20480, 40001])
@pytest.mark.parametrize("live", ["none", "one", "some", "a chunk's end", "half", "most", "all but one", "all"])
def test_compact_of_many_pages(pages, live):
    """Around and above the number of pages up to which one launch counts and
    ranks; the number in use falls on and off the ends of chunks of 1024."""
    import dsa_triton_ascend_amd as dsa
    rng = random.Random(pages)
    n = {"none": 0, "one": 1, "some": 777, "a chunk's end": 5 * 1024, "half": pages // 2, "most": pages - 1500,
         "all but one": pages - 1, "all": pages}[live]
    used = sorted(rng.sample(range(pages), n))
    refs = torch.zeros(pages, dtype=torch.int32)
    refs[used] = torch.randint(1, 5, (n,), dtype=torch.int32, generator=torch.Generator().manual_seed(n))
    holes = (refs[:n] == 0).nonzero().flatten()
    high = torch.tensor([i for i in used if i >= n], dtype=torch.int64)
    page_map = torch.where(refs > 0, torch.arange(pages, dtype=torch.int32), -1)
    page_map[high] = holes.int()
    table = torch.tensor([[rng.choice([rng.randrange(pages), rng.choice(used) if used else 0, -1, pages]) for _ in range(33)]
                          for _ in range(7)], dtype=torch.int32)
    inside = (table >= 0) & (table < pages)
    w_table = torch.where(inside, page_map[table.clamp(0, pages - 1).long()], -1)
    w_refs = torch.zeros_like(refs)
    w_refs[page_map[refs > 0].long()] = refs[refs > 0]
    caches = [torch.arange(pages * 2 * k, device="cuda", dtype=torch.int32).view(pages, 2, 1, k) for k in (1, 4)]
    want = [c.clone() for c in caches]
    for w in want:
        w[holes.cuda()] = w[high.cuda()]
    t, r, m = dsa.paged_cache_compact(caches, table.cuda(), refs.cuda())
    assert torch.equal(t.cpu(), w_table) and torch.equal(r.cpu(), w_refs) and torch.equal(m.cpu(), page_map)
    assert all(torch.equal(c, w) for c, w in zip(caches, want))
