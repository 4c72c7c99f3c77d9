"""paged_prefix_attention against the softmax in 64 bits.

Caches are NaN wherever no row of a family (for its own tokens: of a sequence)
sees a token, and the table names no page for what a sequence has from its
family, so that a read of one shows.

Error bound of an output as in test_paged_attention_gpu.py, with u = eps / 2: the
numerators of a prefix are rounded to the input type once.
"""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
INT64_MAX = 9223372036854775807


def _bounds(mode, act_q, act_k, s, pre, nxt):
    diag = s if mode == 0 else act_k - act_q + s
    hi = min(act_k, diag + nxt + 1, act_k if mode == 0 else diag + 1)
    return max(diag - pre, 0), max(hi, 0)


def _make(families, S1, N1, N2, D, page, dtype, latent, seed=0, act_q=None, mode=3, pre=INT64_MAX, nxt=INT64_MAX,
          spread=2.0, missing=(), wide=0):
    """``families``: (id, shared tokens, lengths of the members).  ``missing``: (sequence, column, entry) of the table."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    cols = [D, 64] if latent else [D, D]
    lens, ids, shared, leader = [], [], [], []
    for fid, P, members in families:
        first = len(lens)
        alone = fid < 0 or P <= 0 or len(members) < 2
        for n in members:
            leader.append(len(lens) if alone else first)
            lens.append(n), ids.append(fid), shared.append(P)
    B = len(lens)
    own = [0 if leader[b] == b and (b + 1 == B or leader[b + 1] != b) else shared[b] for b in range(B)]  # shared in fact
    held = [max(n, p) if leader[b] == b else n for b, (n, p) in enumerate(zip(lens, own))]
    wide = max([wide, 1] + [-(-n // page) for n in held])
    need = sum(-(-n // page) for n in held)
    pool = need + 3
    free = rng.sample(range(pool), need)
    table = [[-1] * wide for _ in range(B)]
    for b in range(B):
        for c in range(0 if leader[b] == b else own[b] // page, -(-held[b] // page)):
            table[b][c] = free.pop()
    for b, c, e in missing:
        table[b][c] = e
    caches = [torch.full((pool, page, N2, c), float("nan"), device="cuda", dtype=dtype) for c in cols]

    def span(bs):
        lo, hi = 2 ** 40, 0
        for b in bs:
            q_b = S1 if act_q is None else act_q[b]
            for s in range(q_b):
                x, y = _bounds(mode, q_b, lens[b], s, pre, nxt)
                if y > x:
                    lo, hi = min(lo, x), max(hi, y)
        return lo, hi

    def put(b, t0, t1, rows):
        t = t0
        while t < t1:
            z = min(t1, (t // page + 1) * page)
            blk = table[b][t // page]
            if 0 <= blk < pool:
                for c, r in zip(caches, rows):
                    c[blk, t % page:t % page + z - t] = r[t:z]
            else:
                for r in rows:
                    r[t:z] = 0
            t = z

    data = [None] * B
    for b in range(B):
        n = max(held[b], lens[b])
        rows = [torch.randn(n, N2, c, generator=g, device="cuda").to(dtype) for c in cols]
        a = leader[b]
        if a == b:
            members = [i for i in range(B) if leader[i] == b]
            lo, hi = span(members)
            put(b, max(0, lo), min(own[b], hi), rows)
        else:
            for r, x in zip(rows, data[a]):
                r[:min(own[b], n)] = x[:min(own[b], n)]
        lo, hi = span([b])
        put(b, max(own[b], lo), min(lens[b], hi), rows)
        data[b] = rows
    q = (torch.randn(B, S1, N1, D, generator=g, device="cuda") * spread).to(dtype)
    qr = (torch.randn(B, S1, N1, 64, generator=g, device="cuda") * spread).to(dtype) if latent else None

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    args = dict(query=q, key=caches[0], value=None if latent else caches[1], block_table=ints(table),
                actual_seq_lengths_kv=ints(lens), prefix_groups=ints(ids), prefix_lengths=ints(shared),
                scale_value=1.0 / math.sqrt(D + 64 if latent else D), query_rope=qr, key_rope=caches[1] if latent else None,
                actual_seq_lengths_query=None if act_q is None else ints(act_q), sparse_mode=mode, pre_tokens=pre,
                next_tokens=nxt, return_softmax_lse=True, min_tokens=1)
    return args, data, lens


def _compare(args, data, lens, act_q=None, got=None):
    import dsa_triton_ascend_amd as dsa
    if got is None:
        got = dsa.paged_prefix_attention(**args)
        torch.cuda.synchronize()
    q, latent = args["query"], args["value"] is None
    B, S1, N1, D = q.shape
    N2 = args["key"].shape[2]
    G = N1 // N2
    dtype = q.dtype
    half = torch.finfo(dtype).eps / 2
    cols = D + 64 if latent else D
    for b, n in enumerate(lens):
        q_b = S1 if act_q is None else act_q[b]
        k0, k1 = (x.double() for x in data[b])
        for s in range(S1):
            lo, hi = _bounds(args["sparse_mode"], q_b, n, s, args["pre_tokens"], args["next_tokens"])
            o, mx, sm = got[0][b, s].double(), got[1][b, :, s].double().flatten(), got[2][b, :, s].double().flatten()
            if s >= q_b or hi <= lo:
                assert (o == 0).all() and (mx == 0).all() and (sm == 0).all(), f"row {b}, {s} sees nothing"
                continue
            qs = q[b, s].double().view(N2, G, D)
            kk = k0[lo:hi].transpose(0, 1)                       # [N2, n, D]
            vv = kk if latent else k1[lo:hi].transpose(0, 1)
            if latent:
                qs = torch.cat([qs, args["query_rope"][b, s].double().view(1, N1, 64)], -1)
                kk = torch.cat([kk, k1[lo:hi].transpose(0, 1)], -1)
            score = torch.matmul(qs, kk.transpose(1, 2).contiguous()) * args["scale_value"]
            size = torch.matmul(qs.abs(), kk.abs().transpose(1, 2).contiguous()) * abs(args["scale_value"])
            ds = size.amax(-1) * (cols + 4) * 2.0 ** -24          # [N2, G]
            top = score.amax(-1)
            p = torch.exp(score - top[..., None])
            total = p.sum(-1)
            w = p / total[..., None]
            want = torch.matmul(w, vv.contiguous()).reshape(N1, D)
            mag = torch.matmul(w, vv.abs().contiguous()).reshape(N1, D)
            rel = (2 * ds.flatten() + 2 * half + 2.0 ** -20)[:, None]
            tol = mag * rel + (want.abs() + mag * rel) * half + (2.0 ** -24 if dtype == torch.float16 else 0) + 1e-30
            err = (o - want).abs()
            assert (err <= tol).all(), (f"sequence {b} ({n}), token {s}: {int((~(err <= tol)).sum())} of {err.numel()} "
                                        f"off, worst ratio {(err / tol).max():.3g}")
            e1 = (mx - top.flatten()).abs()
            assert (e1 <= ds.flatten() + top.flatten().abs() * 2.0 ** -22).all(), f"max of {b}, {s}: {e1.max():.3g}"
            e2 = (sm / total.flatten() - 1).abs()
            assert (e2 <= 2 * ds.flatten() + 2.0 ** -20).all(), f"sum of {b}, {s}: {e2.max():.3g}"
    return got


GROUPED = [
    # N1, N2, D, S1, page, dtype, families
    (1, 1, 64, 1, 16, "bf16", [(0, 16, [17, 18])]),
    (8, 2, 128, 1, 16, "fp16", [(0, 640, [663, 697, 681, 673])]),
    (8, 8, 64, 1, 1, "bf16", [(0, 33, [34, 40, 33, 60]), (1, 1, [2, 5]), (2, 100, [130, 101, 200])]),
    (20, 4, 128, 1, 3, "bf16", [(0, 31, [40, 33]), (-1, 50, [60, 70]), (1, 64, [65, 64, 90])]),
    (16, 1, 256, 1, 64, "fp16", [(0, 500, [999, 501, 640, 700]), (0, 128, [200, 300])]),
    (34, 2, 128, 1, 64, "bf16", [(0, 192, [193] * 9 + [400])]),        # 170 rows a key head
    (64, 1, 64, 1, 48, "fp16", [(0, 96, [97] * 9), (1, 960, [1000] * 3)]),   # more than a block of 256 rows
    (80, 1, 128, 1, 128, "bf16", [(5, 1280, [1500, 1281, 1400, 1300]), (6, 0, [10, 20])]),
    (40, 1, 256, 1, 16, "bf16", [(0, 320, [333, 390, 321, 400, 350])]),  # more than a block of 128 rows
    (10, 2, 128, 4, 16, "bf16", [(0, 64, [68, 100, 70, 66]), (1, 32, [36, 40])]),
    (12, 3, 64, 3, 7, "fp16", [(0, 98, [101, 140, 110]), (1, 15, [20, 18])]),
    (4, 2, 128, 1, 16, "bf16", [(f, 32 * (f % 5), [32 * (f % 5) + 1 + i % 7 for i in range(1 + (f * 7) % 40)])
                                for f in range(12)]),                  # more sequences than lanes
    (2, 1, 64, 1, 16, "bf16", [(0, 48, [49 + i % 5 for i in range(100)]), (1, 16, [17 + i % 3 for i in range(200)])]),
    (5, 5, 128, 2, 16, "fp16", [(0, 400, [402, 450, 403])]),           # workers that do not divide
]


@pytest.mark.parametrize("i", range(len(GROUPED)))
@pytest.mark.parametrize("mode", [3, 0])
def test_grouped(i, mode):
    N1, N2, D, S1, page, dt, families = GROUPED[i]
    print("grouped", GROUPED[i][:6], mode, flush=True)
    args, data, lens = _make(families, S1, N1, N2, D, page, DTYPES[dt], False, seed=i, mode=mode)
    _compare(args, data, lens)


LATENT = [
    (1, 128, 1, 16, "bf16", [(0, 16, [17, 18])]),
    (16, 512, 1, 64, "bf16", [(0, 640, [663, 697, 681, 673])]),
    (16, 512, 2, 64, "fp16", [(0, 128, [130, 200, 131]), (1, 0, [50]), (2, 320, [330] * 9)]),
    (128, 512, 1, 64, "bf16", [(0, 1000, [1001, 1300, 1100]), (1, 77, [78, 200])]),
    (64, 256, 1, 3, "fp16", [(0, 31, [40, 33]), (-1, 50, [60, 70]), (1, 64, [65, 64, 90])]),
    (128, 128, 3, 16, "bf16", [(0, 96, [99, 120, 100])]),
    (9, 256, 1, 1, "bf16", [(0, 300, [301, 330])]),
    (3, 128, 1, 16, "fp16", [(f, 32 * (f % 5), [32 * (f % 5) + 1 + i % 7 for i in range(1 + (f * 7) % 40)])
                             for f in range(12)]),
    (100, 512, 1, 48, "bf16", [(0, 480, [481, 500, 600, 490, 485, 700])]),
]


@pytest.mark.parametrize("i", range(len(LATENT)))
@pytest.mark.parametrize("mode", [3, 0])
def test_latent(i, mode):
    N1, D, S1, page, dt, families = LATENT[i]
    print("latent", LATENT[i][:5], mode, flush=True)
    args, data, lens = _make(families, S1, N1, 1, D, page, DTYPES[dt], True, seed=i, mode=mode)
    _compare(args, data, lens)


def _form(latent, D=None):
    return dict(latent=latent, D=D or (512 if latent else 128), N1=16, N2=1 if latent else 2)


@pytest.mark.parametrize("latent", [False, True])
def test_prefixes_longer_than_sequences(latent):
    families = [(0, 200, [150, 230, 1, 0, 199, 201]), (3, 70, [5, 60]), (4, 64, [0, 0])]
    args, data, lens = _make(families, 1, page=16, dtype=torch.bfloat16, **_form(latent))
    _compare(args, data, lens)


@pytest.mark.parametrize("latent", [False, True])
@pytest.mark.parametrize("mode,pre,nxt", [(3, 40, INT64_MAX), (3, 0, 0), (0, 3, 50), (3, INT64_MAX, -5), (3, 2, -1000)])
def test_band(latent, mode, pre, nxt):
    families = [(0, 200, [203, 230, 260]), (1, 96, [97, 99, 500]), (2, 64, [66, 67])]
    args, data, lens = _make(families, 2, page=16, dtype=torch.float16, mode=mode, pre=pre, nxt=nxt, **_form(latent))
    _compare(args, data, lens)


@pytest.mark.parametrize("latent", [False, True])
@pytest.mark.parametrize("entry", [-1, 10 ** 6, -2 ** 31])
def test_missing_pages_are_zero_rows_and_new_tokens_vary(latent, entry):
    families = [(0, 128, [130, 150, 140]), (1, 300, [320, 310])]
    act_q = [2, 0, 3, 1, 3]
    args, data, lens = _make(families, 3, page=16, dtype=torch.bfloat16, act_q=act_q, seed=3,
                             missing=[(0, 2, entry), (3, 0, entry), (3, 18, entry), (2, 8, entry)], **_form(latent))
    _compare(args, data, lens, act_q)


@pytest.mark.parametrize("latent,N1,D", [(False, 16, 128), (False, 16, 256), (True, 32, 512)])
@pytest.mark.parametrize("rising", [True, False])
def test_scores_that_move_the_reference(latent, N1, D, rising):
    families = [(0, 1024, [1100, 1050, 1030, 1025])]
    args, data, lens = _make(families, 1, N1, 1 if latent else 2, D, 16, torch.bfloat16, latent, seed=9, spread=1.0)
    # the first column carries a ramp of a few hundred units of the exponent
    ramp = torch.linspace(0, 60, 1100, device="cuda")
    ramp = ramp if rising else ramp.flip(0)
    args["query"][..., 0] = 8.0
    for b, n in enumerate(lens):
        data[b][0][:, :, 0] = ramp[:data[b][0].shape[0], None].to(torch.bfloat16)
        for t in range(0, n):
            row = b if t >= 1024 else 0
            blk = int(args["block_table"][row, t // 16])
            args["key"][blk, t % 16] = data[b][0][t]
    _compare(args, data, lens)


@pytest.mark.parametrize("latent", [False, True])
def test_one_family_of_many_rows_and_a_long_table(latent):
    """More pages than the kernels hold at a time, and more jobs than workgroups."""
    families = [(0, 1500, [1501 + i % 4 for i in range(70)])]
    f = _form(latent, 128)
    f["N1"] = 64
    args, data, lens = _make(families, 1, page=1, dtype=torch.bfloat16, seed=5, wide=1600, **f)
    _compare(args, data, lens)


@pytest.mark.parametrize("latent", [False, True])
def test_more_blocks_of_rows_than_workgroups(latent):
    """600 sequences of four new tokens: the workgroups take several jobs each."""
    families = [(0, 64, [70 + i % 3 for i in range(300)]), (1, 160, [165 + i % 9 for i in range(300)])]
    N1, N2 = (128, 1) if latent else (64, 2)
    args, data, lens = _make(families, 4, N1, N2, 128, 16, torch.bfloat16, latent, seed=6)
    got = _compare_some(args, data, lens, [0, 1, 150, 299, 300, 301, 450, 599])
    assert torch.isfinite(got[0].float()).all()


def _compare_some(args, data, lens, which):
    import dsa_triton_ascend_amd as dsa
    got = dsa.paged_prefix_attention(**args)
    torch.cuda.synchronize()
    some = dict(args)
    for name in ("query", "query_rope"):
        some[name] = None if args[name] is None else args[name][which]
    _compare(some, [data[b] for b in which], [lens[b] for b in which], got=[x[which] for x in got])
    return got


@pytest.mark.parametrize("latent", [False, True])
def test_offsets_past_32_bits(latent):
    """Pages at the far end of a cache of more than 2^32 bytes."""
    import dsa_triton_ascend_amd as dsa
    dtype, page = torch.float16, 64
    N1, N2, D = (16, 1, 512) if latent else (16, 8, 128)
    pages = 2 ** 32 // (page * N2 * D * 2) + 40
    key = torch.empty(pages, page, N2, D, dtype=dtype, device="cuda")
    other = torch.empty(pages, page, N2, 64 if latent else D, dtype=dtype, device="cuda")
    families = [(0, 256, [300, 260, 290])]
    args, data, lens = _make(families, 1, N1, N2, D, page, dtype, latent, seed=4)
    small = [args["key"], args["key_rope"] if latent else args["value"]]
    n = small[0].shape[0]
    for big, s in zip((key, other), small):
        big[-n:] = s
    args["key"], args["key_rope" if latent else "value"] = key, other
    args["block_table"] = torch.where(args["block_table"] >= 0, args["block_table"] + (pages - n), -1).int()
    _compare(args, data, lens)


@pytest.mark.parametrize("latent", [False, True])
def test_equals_paged_attention_of_the_same_pages(latent):
    """Sequences whose tables name the prefix's pages themselves; sequences alone take the same way bit for bit."""
    import dsa_triton_ascend_amd as dsa
    families = [(0, 320, [330, 400, 350]), (1, 0, [500]), (-1, 100, [77, 300])]
    args, data, lens = _make(families, 1, page=16, dtype=torch.bfloat16, seed=8, **_form(latent))
    a = dsa.paged_prefix_attention(**args)
    table = args["block_table"].clone()
    table[1:3, :20] = table[0, :20]
    plain = {k: v for k, v in args.items() if not k.startswith("prefix") and k != "min_tokens"}
    plain["block_table"] = table
    b = dsa.paged_attention(**plain)
    for x, y in zip(a, b):
        assert torch.allclose(x.float(), y.float(), rtol=2.0 ** -6, atol=2.0 ** -6)
    alone = dict(args, prefix_groups=torch.arange(6, dtype=torch.int32, device="cuda"), block_table=table)
    for x, y in zip(dsa.paged_prefix_attention(**alone), b):
        assert torch.equal(x, y)
    # with the prefixes that the table itself shows, in families of their own
    groups, shared = dsa.paged_cache_prefixes(table, args["actual_seq_lengths_kv"], 16)
    assert groups.tolist() == [0, 0, 0, 3, 4, 5] and shared.tolist() == [320, 320, 320, 0, 0, 0]
    c = dsa.paged_prefix_attention(**dict(alone, prefix_groups=groups, prefix_lengths=shared))
    for x, y in zip(a, c):
        assert torch.equal(x, y)


@pytest.mark.parametrize("latent", [False, True])
def test_graph_replays_lengths_and_streams(latent):
    import dsa_triton_ascend_amd as dsa
    families = [(0, 96, [100, 150, 130]), (1, 64, [65, 200])]
    args, data, lens = _make(families, 1, page=16, dtype=torch.bfloat16, seed=2, **_form(latent))
    args["key"].nan_to_num_(0.5)
    (args["key_rope"] if latent else args["value"]).nan_to_num_(0.5)
    table = args["block_table"]
    table[1:3, :6], table[4, :4] = table[0, :6], table[3, :4]
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        dsa.paged_prefix_attention(**args)
        with torch.cuda.graph(graph, stream=stream):
            out = dsa.paged_prefix_attention(**args)
            again = dsa.paged_prefix_attention(**args)
    rng = random.Random(1)
    for step in range(4):
        args["actual_seq_lengths_kv"].copy_(torch.tensor([rng.randint(1, n) for n in lens], dtype=torch.int32))
        args["prefix_lengths"].copy_(torch.tensor([16 * (step + 1)] * 3 + [17] * 2, dtype=torch.int32))
        args["query"].normal_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = dsa.paged_prefix_attention(**args)
        for x, y, z in zip(out, want, again):
            assert torch.equal(x, y) and torch.equal(x, z)


def test_negative_and_zero_scale_and_no_statistics():
    import dsa_triton_ascend_amd as dsa
    for latent in (False, True):
        for scale in (-0.05, 0.0):
            families = [(0, 96, [100, 150, 130])]
            args, data, lens = _make(families, 1, page=16, dtype=torch.bfloat16, seed=2, **_form(latent))
            args["scale_value"] = scale
            got = _compare(args, data, lens)
        args["return_softmax_lse"] = False
        other = dsa.paged_prefix_attention(**args)
        assert torch.equal(other[0], got[0]) and not other[1].any() and not other[2].any()


def test_rows_that_see_nothing_beside_values_that_are_not_finite():
    """A prefix that holds infinities and that some of the sequences do not see at all: those are zero."""
    import dsa_triton_ascend_amd as dsa
    for latent in (False, True):
        families = [(0, 64, [0, 100, 0, 80])]
        args, data, lens = _make(families, 1, page=16, dtype=torch.bfloat16, seed=2, **_form(latent))
        (args["key"] if latent else args["value"])[int(args["block_table"][0, 1]), 3] = float("inf")
        out, mx, sm = dsa.paged_prefix_attention(**args)
        assert not out[[0, 2]].any() and not mx[[0, 2]].any() and not sm[[0, 2]].any()


def test_compiled_and_python_calls_agree(monkeypatch):
    import dsa_triton_ascend_amd as dsa
    from dsa_triton_ascend_amd import _lib
    assert _lib.calls() is not _lib._NoCalls
    for latent in (False, True):
        families = [(0, 96, [100, 150, 130])]
        args, data, lens = _make(families, 1, page=16, dtype=torch.float16, seed=2, **_form(latent))
        a = dsa.paged_prefix_attention(**args)
        monkeypatch.setattr(_lib, "_calls", _lib._NoCalls)
        b = dsa.paged_prefix_attention(**args)
        lists = dict(args, prefix_groups=[0, 0, 0], prefix_lengths=[96, 96, 96], actual_seq_lengths_kv=lens,
                     block_table=args["block_table"].long())
        c = dsa.paged_prefix_attention(**lists)
        m = dsa.PagedPrefixAttention(scale_value=args["scale_value"], return_softmax_lse=True, min_tokens=1)
        d = m(args["query"], args["key"], args["value"], args["block_table"], args["actual_seq_lengths_kv"],
              args["prefix_groups"], args["prefix_lengths"], args["query_rope"], args["key_rope"])
        monkeypatch.undo()
        for x, y, z, w in zip(a, b, c, d):
            assert torch.equal(x, y) and torch.equal(x, z) and torch.equal(x, w)


def test_empty_caches_and_batches():
    import dsa_triton_ascend_amd as dsa
    q = torch.randn(2, 1, 8, 128, device="cuda").half()
    none = torch.empty(0, 16, 2, 128, device="cuda").half()
    i = torch.zeros(2, dtype=torch.int32, device="cuda")
    out, mx, sm = dsa.paged_prefix_attention(q, none, none, torch.zeros(2, 1, dtype=torch.int32, device="cuda"), i, i, i)
    assert not out.any() and not mx.any() and not sm.any()


@pytest.mark.parametrize("change,match", [
    (dict(prefix_groups=2), "one entry per sequence"), (dict(prefix_lengths=4), "one entry per sequence"),
    (dict(actual_seq_lengths_kv=2), "one entry per batch"), (dict(actual_seq_lengths_query=5), "one entry per batch")])
def test_refuses_lengths_of_other_batches(change, match):
    import dsa_triton_ascend_amd as dsa
    args, _, _ = _make([(0, 96, [100, 150, 130])], 1, page=16, dtype=torch.float16, latent=False, N1=8, N2=2, D=128)
    for name, n in change.items():
        with pytest.raises(ValueError, match=match):
            dsa.paged_prefix_attention(**dict(args, **{name: torch.zeros(n, dtype=torch.int32, device="cuda")}))
        with pytest.raises(ValueError, match=match):
            dsa.paged_prefix_attention(**dict(args, **{name: [0] * n}))


def test_refuses_strided_caches():
    import dsa_triton_ascend_amd as dsa
    args, _, _ = _make([(0, 96, [100, 150, 130])], 1, page=16, dtype=torch.float16, latent=False, N1=8, N2=2, D=128)
    for name in ("key", "value"):
        wide = torch.zeros(*args[name].shape[:2], 4, 128, dtype=torch.float16, device="cuda")
        with pytest.raises(ValueError, match="contiguous"):
            dsa.paged_prefix_attention(**dict(args, **{name: wide[:, :, ::2]}))


@pytest.mark.parametrize("latent", [False, True])
def test_strided_queries_and_other_tables(latent):
    """Heads of a wider projection, tables of more rows and of 64 bits, a batch of one."""
    import dsa_triton_ascend_amd as dsa
    for families in ([(0, 96, [100, 150, 130])], [(0, 50, [75])]):
        args, data, lens = _make(families, 1, page=16, dtype=torch.bfloat16, seed=2, **_form(latent))
        want = _compare(args, data, lens)
        q = args["query"]
        wide = torch.randn(*q.shape[:2], q.shape[2] + 3, q.shape[3], device="cuda").to(q.dtype)
        wide[:, :, 2:-1] = q
        table = torch.cat([args["block_table"], args["block_table"][:1] * 0 - 7])
        got = dsa.paged_prefix_attention(**dict(args, query=wide[:, :, 2:-1], block_table=table.long()))
        for x, y in zip(got, want):
            assert torch.equal(x, y)


@pytest.mark.parametrize("i", range(len(GROUPED) + len(LATENT)))
def test_short_prefixes_sequence_by_sequence(i):
    """Families below min_tokens: each sequence for itself, the prefix from the pages of the family's first."""
    latent = i >= len(GROUPED)
    if latent:
        N1, D, S1, page, dtype, families = LATENT[i - len(GROUPED)]
        N2 = 1
    else:
        N1, N2, D, S1, page, dtype, families = GROUPED[i]
    args, data, lens = _make(families, S1, N1, N2, D, page, DTYPES[dtype], latent, seed=i)
    for least in (2 ** 40, 50):  # none together; some
        _compare(dict(args, min_tokens=least), data, lens)


@pytest.mark.parametrize("latent", [False, True])
@pytest.mark.parametrize("shared", [64, 75])
def test_sequence_by_sequence_is_paged_attention(latent, shared):
    """Bit for bit where the tables name the same pages, and whatever the tables of the others name there."""
    import dsa_triton_ascend_amd as dsa
    families = [(0, shared, [330, 400, 20]), (1, 0, [500]), (2, shared, [77, 300])]
    args, data, lens = _make(families, 1, page=16, dtype=torch.bfloat16, seed=8, **_form(latent))
    a = dsa.paged_prefix_attention(**dict(args, min_tokens=1000))
    if shared % 16:
        _compare(args, data, lens, got=a)
        return
    table = args["block_table"].clone()
    table[1:3, :shared // 16], table[5, :shared // 16] = table[0, :shared // 16], table[4, :shared // 16]
    plain = {k: v for k, v in args.items() if not k.startswith("prefix") and k != "min_tokens"}
    b = dsa.paged_attention(**dict(plain, block_table=table))
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_prefixes_longer_than_the_table_and_min_tokens():
    """A shared length past the table's room counts as the room, also against min_tokens."""
    for latent in (False, True):
        args, data, lens = _make([(0, 96, [96, 80, 50])], 1, page=16, dtype=torch.float16, seed=3, **_form(latent))
        assert args["block_table"].shape[1] == 6
        args["prefix_lengths"].fill_(2 ** 31 - 1)
        for least in (1, 96, 97, 10 ** 6, None):
            _compare(dict(args, min_tokens=least), data, lens)


@pytest.mark.parametrize("latent,N1,N2,D", [(False, 32, 8, 128), (True, 16, 1, 512), (True, 64, 1, 512)])
def test_families_chosen_by_size(latent, N1, N2, D):
    """Without min_tokens: long prefixes of many, of few and of two, short ones, and sequences alone, in one batch."""
    P = 4800 if latent else 2400
    families = [(0, P, [P + 17 * i for i in range(33)]), (1, P + 16, [P + 20, P + 90]), (2, 160, [170 + i for i in range(20)]),
                (-1, 50, [300]), (3, P - 16, [P, P + 3, P + 100, P - 500, P + 40])]
    args, data, lens = _make(families, 1, N1, N2, D, 16, torch.bfloat16, latent, seed=4)
    _compare(dict(args, min_tokens=None), data, lens)


@pytest.mark.parametrize("latent", [False, True])
@pytest.mark.parametrize("before", [0, 1, 40, 62, 63, 64])
@pytest.mark.parametrize("least", [1, 1000])
def test_families_across_64s(latent, before, least):
    """Together in parts of 64 sequences, and for each, the prefix in the pages of the first of all."""
    families = [(-1, 0, [10 + i % 3 for i in range(before)]), (0, 48, [50 + i % 40 for i in range(90)]),
                (1, 32, [33, 40])]
    form = dict(latent=latent, D=128, N1=2, N2=1)
    args, data, lens = _make([f for f in families if f[2]], 1, page=16, dtype=torch.bfloat16, seed=6, **form)
    _compare(dict(args, min_tokens=least), data, lens)


def test_families_chosen_by_size_of_large_batches():
    """More sequences than a wave has lanes, families that go on behind the 64th, prefixes just long enough and not."""
    B, token_bytes = 130, 4096
    least = (256 << 20) // (B * token_bytes)
    families = [(0, least + 8, [least + 10 + i for i in range(70)]), (1, least - 8, [least + i for i in range(20)]),
                (2, least + 1, [least + 40 - 3 * i for i in range(38)]), (3, 2 * least, [2 * least + 5] * 2)]
    assert sum(len(m) for _, _, m in families) == B
    args, data, lens = _make(families, 1, 16, 8, 128, 16, torch.bfloat16, False, seed=9)
    _compare(dict(args, min_tokens=None), data, lens)
