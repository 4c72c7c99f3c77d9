"""paged_attention against the softmax in 64 bits.

Caches are NaN wherever no visible token lies, so that a read of one shows.

Error bound of an output o = sum w v, with A = sum w |v|: a score is off by at
most ds = (columns + 4) 2^-24 sum |q k| scale (products and sums of 32 bits,
scale, exponent), a weight by 2 ds (its own and the sum's), by the rounding u
of the numerator to the type (twice: its own and the divisor's), and by 2^-20
for exponential, sums and joins; the output rounds by eps / 2.  u is eps / 2
where the numerators are rounded once (latent form, more than 32 rows) and
(eps / 2)^2 where they are kept as two values.  Largest score: off by ds and
2^-22 of itself; sum: 2 ds + 2^-20 relative.
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


def _make(B, S1, N1, N2, D, page, lens, dtype, latent, seed=0, hole=None, act_q=None, mode=3, pre=INT64_MAX,
          nxt=INT64_MAX, spread=2.0, wide=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    wide = wide or max(1, max(-(-n // page) for n in lens))
    need = sum(-(-n // page) for n in lens)
    pool = need + 3
    ids = rng.sample(range(pool), need)
    table = torch.full((B, wide), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(lens):
        m = -(-n // page)
        table[b, :m] = torch.tensor(ids[at:at + m], dtype=torch.int32)
        at += m
    cols = [D, 64] if latent else [D, D]
    caches = [torch.full((pool, page, N2, c), float("nan"), device="cuda", dtype=dtype) for c in cols]
    data = []  # per sequence: the two caches' rows in 64 bits, zero where there is no page
    for b, n in enumerate(lens):
        rows = [torch.randn(n, N2, c, generator=g, device="cuda").to(dtype) for c in cols]
        lo, hi = n, 0
        q_b = S1 if act_q is None else act_q[b]
        for s in range(q_b):
            x, y = _bounds(mode, q_b, n, s, pre, nxt)
            lo, hi = min(lo, x), max(hi, y)
        if hole is not None and b == hole[0] and hole[1] < -(-n // page):
            table[b, hole[1]] = hole[2]
            for r in rows:
                r[hole[1] * page:(hole[1] + 1) * page] = 0
        for t0 in range(0, n, page):
            blk = int(table[b, t0 // page])
            a, z = max(t0, lo), min(t0 + page, hi, n)
            if 0 <= blk < pool and a < z:
                for c, r in zip(caches, rows):
                    c[blk, a - t0:z - t0] = r[a:z]
        data.append(rows)
    q = (torch.randn(B, S1, N1, D, generator=g, device="cuda") * spread).to(dtype)
    qr = (torch.randn(B, S1, N1, 64, generator=g, device="cuda") * spread).to(dtype) if latent else None
    scale = 1.0 / math.sqrt(D + 64 if latent else D)
    args = dict(query=q, key=caches[0], value=None if latent else caches[1], block_table=table.cuda(),
                actual_seq_lengths_kv=torch.tensor(lens, dtype=torch.int32, device="cuda"), scale_value=scale,
                query_rope=qr, key_rope=caches[1] if latent else None,
                actual_seq_lengths_query=None if act_q is None else torch.tensor(act_q, dtype=torch.int32,
                                                                                 device="cuda"),
                sparse_mode=mode, pre_tokens=pre, next_tokens=nxt, return_softmax_lse=True)
    return args, data


def _compare(args, data, lens, act_q=None):
    import dsa_triton_ascend_amd as dsa
    got = dsa.paged_attention(**args)
    torch.cuda.synchronize()
    q, latent = args["query"], args["value"] is None
    B, S1, N1, D = q.shape
    N2 = args["key"].shape[2]
    G = N1 // N2
    dtype = q.dtype
    half = torch.finfo(dtype).eps / 2
    u = half if latent and S1 * N1 > 32 else half * half
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
            rel = (2 * ds.flatten() + 2 * u + 2.0 ** -20)[:, None]
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
    # N1, N2, D, S1, page, dtype, lengths
    (1, 1, 64, 1, 16, "bf16", [1]),
    (8, 2, 128, 1, 16, "fp16", [777]),
    (8, 8, 64, 1, 1, "bf16", [0, 1, 31, 32, 33, 64, 65, 130]),
    (20, 4, 128, 1, 3, "bf16", [5, 0, 300, 129, 128]),
    (16, 1, 256, 1, 64, "fp16", [999, 63, 64, 65, 1]),
    (34, 2, 128, 1, 64, "bf16", [700, 3]),              # 17 heads: two row tiles
    (33, 1, 64, 1, 48, "fp16", [257, 2000]),            # three row tiles in four
    (80, 1, 128, 1, 128, "bf16", [1500, 0, 40]),        # two row groups
    (40, 1, 256, 1, 16, "bf16", [333, 90]),             # two row groups of 32
    (10, 2, 128, 4, 16, "bf16", [3, 500, 4, 1, 77]),    # four new tokens, one length below that
    (12, 3, 64, 3, 7, "fp16", [100, 2, 1000, 33]),
    (4, 2, 128, 1, 16, "bf16", [(37 * i) % 211 for i in range(150)]),  # more sequences than lanes
]


@pytest.mark.parametrize("i", range(len(GROUPED)))
@pytest.mark.parametrize("mode", [3, 0])
def test_grouped(i, mode):
    N1, N2, D, S1, page, dt, lens = GROUPED[i]
    print("grouped", GROUPED[i][:6], mode, flush=True)
    args, data = _make(len(lens), S1, N1, N2, D, page, lens, DTYPES[dt], False, seed=i, mode=mode)
    _compare(args, data, lens)


LATENT = [
    # N1, D, S1, page, dtype, lengths
    (1, 512, 1, 64, "bf16", [1]),
    (16, 512, 1, 64, "bf16", [0, 1, 31, 32, 33, 64, 65, 700]),
    (16, 512, 2, 64, "fp16", [901, 2, 1, 300]),
    (32, 512, 1, 16, "bf16", [513, 3, 0, 129]),
    (64, 512, 1, 1, "fp16", [400, 77]),
    (17, 512, 3, 48, "bf16", [600, 2, 97]),              # 51 rows
    (128, 512, 1, 64, "bf16", [1000, 1, 0, 33, 255]),
    (128, 512, 1, 64, "fp16", [1, 2, 3, 4, 5, 6, 1030]),
    (100, 512, 1, 3, "bf16", [300, 31]),                 # idle rows
    (128, 512, 3, 64, "bf16", [500, 2]),                 # three row groups
    (16, 128, 1, 16, "bf16", [300, 64, 5]),
    (32, 128, 1, 16, "fp16", [300, 64, 5]),
    (64, 128, 1, 16, "bf16", [300, 64, 5]),
    (128, 128, 2, 16, "bf16", [300, 64, 1]),
    (8, 256, 1, 64, "fp16", [290, 1]),
    (30, 256, 1, 64, "bf16", [290, 1]),
    (64, 256, 1, 64, "bf16", [290, 1]),
    (128, 256, 1, 64, "fp16", [290, 1, 600]),
]


@pytest.mark.parametrize("i", range(len(LATENT)))
def test_latent(i):
    N1, D, S1, page, dt, lens = LATENT[i]
    print("latent", LATENT[i][:5], flush=True)
    args, data = _make(len(lens), S1, N1, 1, D, page, lens, DTYPES[dt], True, seed=i)
    _compare(args, data, lens)


@pytest.mark.parametrize("latent", [False, True])
@pytest.mark.parametrize("mode,pre,nxt", [(3, 99, INT64_MAX), (3, 0, INT64_MAX), (0, 300, 40), (0, INT64_MAX, -3),
                                          (3, -1, INT64_MAX), (3, 40, -7), (3, 2 ** 62, 2 ** 62)])
def test_band(latent, mode, pre, nxt):
    """Sliding windows and bands; tokens outside are NaN, and some rows' bands are empty."""
    lens = [700, 5, 1, 0, 64, 333]
    args, data = _make(6, 3, 8, 1 if latent else 2, 512 if latent else 128, 16, lens, torch.bfloat16, latent, seed=9,
                       mode=mode, pre=pre, nxt=nxt)
    _compare(args, data, lens)


@pytest.mark.parametrize("latent", [False, True])
@pytest.mark.parametrize("entry", [-1, 10 ** 6])
def test_missing_pages_are_zero_rows_and_new_tokens_vary(latent, entry):
    lens, act_q = [100, 300, 40, 7], [1, 3, 0, 2]
    args, data = _make(4, 3, 16, 1 if latent else 4, 512 if latent else 128, 16, lens, torch.bfloat16, latent, seed=11,
                       hole=(1, 4, entry), act_q=act_q)
    _compare(args, data, lens, act_q)


@pytest.mark.parametrize("latent,N1,dt", [(False, 8, "bf16"), (False, 8, "fp16"), (True, 16, "fp16"), (True, 64, "bf16"),
                                          (True, 128, "bf16"), (True, 128, "fp16")])
@pytest.mark.parametrize("rising", [True, False])
def test_scores_that_move_the_reference(latent, N1, dt, rising):
    """Scores that grow (or fall) by 60 binades over the tokens."""
    lens = [500, 900]
    args, data = _make(2, 1, N1, 1, 512 if latent else 128, 64, lens, DTYPES[dt], latent, seed=13, spread=0.5)
    q = args["query"]
    q[..., 0] = 4.0
    page = 64
    for b, n in enumerate(lens):
        ramp = torch.linspace(-1, 1, n, device="cuda") * (1 if rising else -1)
        col = (ramp * 10.0 / 4.0 / args["scale_value"]).to(q.dtype)  # +- 10 in natural units at scale 1
        data[b][0][:, :, 0] = col[:, None]
        for t0 in range(0, n, page):
            args["key"][int(args["block_table"][b, t0 // page]), :min(page, n - t0), :, 0] = col[t0:t0 + page, None]
    args["scale_value"] *= 2.0
    _compare(args, data, lens)


@pytest.mark.parametrize("latent", [False, True])
def test_long_table_of_repeated_pages(latent):
    """300001 tokens over a table that names a few pages again and again: long
    runs, and more table entries than a run holds at a time."""
    g = torch.Generator(device="cuda").manual_seed(1)
    n, pool, page = 300001, 11, 1
    D, N1, N2 = (512, 16, 1) if latent else (128, 8, 2)
    k0 = torch.randn(pool, page, N2, D, generator=g, device="cuda").bfloat16()
    k1 = torch.randn(pool, page, N2, 64 if latent else D, generator=g, device="cuda").bfloat16()
    table = torch.randint(0, pool, (1, n + 5), generator=g, device="cuda", dtype=torch.int32)
    q = torch.randn(1, 1, N1, D, generator=g, device="cuda").bfloat16()
    qr = torch.randn(1, 1, N1, 64, generator=g, device="cuda").bfloat16() if latent else None
    rows = [x[table[0, :n].long(), 0] for x in (k0, k1)]
    args = dict(query=q, key=k0, value=None if latent else k1, block_table=table, actual_seq_lengths_kv=[n],
                scale_value=0.05, query_rope=qr, key_rope=k1 if latent else None, sparse_mode=3, pre_tokens=INT64_MAX,
                next_tokens=INT64_MAX, return_softmax_lse=True)
    _compare(args, [rows], [n])


@pytest.mark.parametrize("latent", [False, True])
def test_offsets_past_32_bits(latent):
    """Pages behind 4 GiB of their cache."""
    D, N1, N2, page = (512, 16, 1, 64) if latent else (128, 16, 8, 64)
    pool = (9 << 29) // (page * N2 * D * 2)  # 4.5 GiB
    lens = [400, 131]
    args, data = _make(2, 1, N1, N2, D, page, lens, torch.bfloat16, latent, seed=21)
    far = torch.arange(pool - 10, pool, dtype=torch.int32, device="cuda")
    table = args["block_table"]
    for name in ("key", "key_rope" if latent else "value"):
        small = args[name]
        big = torch.empty(pool, *small.shape[1:], dtype=small.dtype, device="cuda")
        for b, n in enumerate(lens):
            for i in range(-(-n // page)):
                big[pool - 10 + b * 7 + i] = small[int(table[b, i])]
        args[name] = big
    new = torch.full_like(table, -1)
    new[0, :7], new[1, :3] = far[:7], far[7:]
    args["block_table"] = new
    _compare(args, data, lens)


@pytest.mark.parametrize("latent", [False, True])
def test_graph_replays_lengths_and_streams(latent):
    """A captured call replayed while lengths, table and queries change, two
    graphs in turn, and a call on another stream; all bit-identical to eager."""
    import dsa_triton_ascend_amd as dsa
    lens = [300, 64, 900, 5]
    args, _ = _make(4, 2, 16, 1 if latent else 4, 512 if latent else 128, 16, lens, torch.bfloat16, latent, seed=31)
    for name in ("key", "value", "key_rope"):
        if args[name] is not None:
            args[name].nan_to_num_(0.5)
    lengths = args["actual_seq_lengths_kv"]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        aside = dsa.paged_attention(**args)
    torch.cuda.current_stream().wait_stream(side)
    eager = dsa.paged_attention(**args)
    assert all(torch.equal(a, b) for a, b in zip(aside, eager))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = dsa.paged_attention(**args)
        graphs.append((g, out))
    for i, now in enumerate(([300, 64, 900, 5], [1, 0, 17, 64], [299, 40, 512, 2], [0, 0, 0, 0])):
        lengths.copy_(torch.tensor(now, dtype=torch.int32))
        args["query"].copy_(torch.randn_like(args["query"]))
        junk = torch.randn(1 << 20, device="cuda").sum()
        torch.cuda.synchronize()
        for g, out in graphs:
            for o in out:
                o.fill_(float("nan"))
            g.replay()
        torch.cuda.synchronize()
        assert torch.isfinite(junk)
        eager = dsa.paged_attention(**args)
        for g, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, eager)), i


def test_statistics_off_lists_and_strides():
    import dsa_triton_ascend_amd as dsa
    lens = [300, 64]
    args, data = _make(2, 1, 16, 4, 128, 16, lens, torch.bfloat16, False, seed=41)
    out, mx, sm = dsa.paged_attention(**args)
    args["return_softmax_lse"] = False
    args["actual_seq_lengths_kv"] = lens                      # a list
    wide = torch.zeros(2, 1, 16, 192, device="cuda", dtype=torch.bfloat16)
    wide[..., 64:] = args["query"]
    args["query"] = wide[..., 64:]                            # a view
    args["block_table"] = args["block_table"].long()
    o2, m2, s2 = dsa.paged_attention(**args)
    assert torch.equal(out, o2) and (m2 == 0).all() and (s2 == 0).all()
    assert (mx != 0).any() and (sm != 0).any()
    mod = dsa.PagedAttention(scale_value=args["scale_value"])
    o3, _, _ = mod(args["query"], args["key"], args["value"], args["block_table"], args["actual_seq_lengths_kv"])
    assert torch.equal(out, o3)


def test_matches_sparse_flash_attention_where_all_tokens_are_selected():
    """The sparse operator with every token selected is this one: both round
    the same sums differently, so outputs agree to two roundings."""
    import dsa_triton_ascend_amd as dsa
    lens, page = [512, 300], 64
    args, data = _make(2, 1, 128, 1, 512, page, lens, torch.bfloat16, True, seed=51)
    for name in ("key", "key_rope"):
        args[name].nan_to_num_(0.0)
    si = torch.full((2, 1, 1, 512), -1, dtype=torch.int32, device="cuda")
    for b, n in enumerate(lens):
        si[b, 0, 0, :n] = torch.arange(n, device="cuda")
    ref, rmax, rsum = dsa.sparse_flash_attention_triton(
        args["query"], args["key"], None, si, scale_value=args["scale_value"], block_table=args["block_table"],
        actual_seq_lengths_kv=args["actual_seq_lengths_kv"], query_rope=args["query_rope"],
        key_rope=args["key_rope"], layout_kv="PA_BSND", return_softmax_lse=True)
    out, mx, sm = _compare(args, data, lens)
    assert mx.shape == rmax.shape
    for b in range(2):
        v = data[b][0].double().abs().max()
        # each off by at most 2^-8 of the value and twice 2^-8 of the mean |v|
        assert (out[b].double() - ref[b].double()).abs().max() <= 2 * 3 * 2.0 ** -8 * v
    assert torch.allclose(mx, rmax, rtol=2.0 ** -20, atol=1e-4) and torch.allclose(sm, rsum, rtol=1e-3)


@pytest.mark.parametrize("latent,N1,N2,D", [(False, 16, 8, 128), (False, 40, 2, 64), (False, 6, 3, 256), (True, 16, 1, 512),
                                            (True, 32, 1, 512), (True, 64, 1, 512), (True, 128, 1, 512)])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_streaming_loads(latent, N1, N2, D, dt):
    """A pool and a table for more tokens than the caches hold, whose loads
    stream, with short sequences in it (one of them without a page in the
    middle)."""
    page, lens = 64, [400, 131, 0, 64]
    args, data = _make(4, 1, N1, N2, D, page, lens, DTYPES[dt], latent, seed=23, hole=(0, 2, -1))
    cols = N2 * (D + 64 if latent else 2 * D)
    pool = (300 << 20) // (page * cols * 2) + 1
    table = torch.full((4, pool), -1, dtype=torch.int32, device="cuda")
    ids = torch.randperm(pool, device="cuda")[:16].int()
    for name in ("key", "key_rope" if latent else "value"):
        small = args[name]
        big = torch.full((pool, *small.shape[1:]), float("nan"), dtype=small.dtype, device="cuda")
        at = 0
        for b, n in enumerate(lens):
            for i in range(-(-n // page)):
                old = int(args["block_table"][b, i])
                if old >= 0:
                    table[b, i] = ids[at]
                    big[int(ids[at])] = small[old]
                at += 1
        args[name] = big
    args["block_table"] = table
    _compare(args, data, lens)


def test_negative_and_zero_scale():
    lens = [100, 333]
    for latent in (False, True):
        for scale in (-0.07, 0.0):
            args, data = _make(2, 2, 16, 1 if latent else 4, 512 if latent else 128, 16, lens, torch.bfloat16, latent,
                               seed=61)
            args["scale_value"] = scale
            _compare(args, data, lens)


def test_lengths_past_the_table_and_negative():
    """More tokens than the table holds count as those it holds, fewer than none as none."""
    import dsa_triton_ascend_amd as dsa
    lens = [128, 64, 0]
    for latent in (False, True):
        args, data = _make(3, 1, 8, 1 if latent else 2, 512 if latent else 128, 64, lens, torch.bfloat16, latent,
                           seed=71)
        for name in ("key", "value", "key_rope"):
            if args[name] is not None:
                args[name].nan_to_num_(0.25)
        args["actual_seq_lengths_kv"] = torch.tensor([128, 64, 0], dtype=torch.int32, device="cuda")
        want = dsa.paged_attention(**args)
        args["actual_seq_lengths_kv"] = torch.tensor([2 ** 31 - 1, 64, -7], dtype=torch.int32, device="cuda")
        got = dsa.paged_attention(**args)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("N1,D,latent", [(16, 128, True), (64, 128, True), (8, 64, False)])
@pytest.mark.parametrize("lens", [
    [96] * 3,                                             # every sequence three tiles, runs of two
    [1 + 37 * i % 211 for i in range(300)],               # more sequences than workgroups
    [40] * 520,                                           # two of them in a run
    [0] * 70 + [33] + [0] * 70 + [4000, 0, 1],            # long empty stretches
    [2500] * 9,                                           # runs a little longer than an equal share
])
def test_runs_over_many_shapes_of_batches(N1, D, latent, lens):
    args, data = _make(len(lens), 1, N1, 1 if latent else 2, D, 16, lens, torch.bfloat16, latent, seed=81)
    _compare(args, data, lens)


@pytest.mark.parametrize("latent,N1,D", [(False, 8, 64), (False, 4, 256), (True, 8, 512), (True, 16, 512),
                                         (True, 128, 512), (True, 64, 128)])
@pytest.mark.parametrize("n", [70, 3000])
def test_rows_that_see_nothing_beside_values_that_are_not_finite(latent, N1, D, n):
    """Padding rows are zero next to a token of infinities; a row that sees a NaN says so."""
    import dsa_triton_ascend_amd as dsa
    args, _ = _make(2, 3, N1, 1 if latent else 2, D, 64, [n, n], torch.bfloat16, latent, seed=83, act_q=[1, 2])
    last = int(args["block_table"][0, (n - 1) // 64]), (n - 1) % 64
    want = dsa.paged_attention(**args)
    for value in (float("inf"), float("nan")):
        args["key" if latent else "value"][last] = value
        out, mx, sm = dsa.paged_attention(**args)
        assert not torch.isfinite(out[0, 0]).any()
        assert (out[0, 1:] == 0).all() and (mx[0, :, 1:] == 0).all() and (sm[0, :, 1:] == 0).all()
        assert all(torch.equal(a[1], b[1]) for a, b in zip((out, mx, sm), want))  # the other sequence
    args["key"][last] = float("nan")
    out, mx, sm = dsa.paged_attention(**args)
    assert torch.isnan(out[0, 0]).all() and torch.isnan(sm[0, :, 0]).all() and (out[0, 1:] == 0).all()


@pytest.mark.parametrize("latent,N1,N2,D,S1,page,lens,act_q", [
    (False, 4, 2, 64, 100, 1000, [100, 1500, 70], [100, 100, 70]),
    (False, 6, 1, 256, 33, 24, [33, 400, 0], None),
    (True, 4, 1, 128, 100, 24, [100, 130, 900], [100, 1, 64]),
    (True, 40, 1, 512, 17, 64, [17, 333, 5], [17, 17, 5]),
])
@pytest.mark.parametrize("mode,pre", [(3, INT64_MAX), (3, 40), (0, INT64_MAX)])
def test_many_new_tokens(latent, N1, N2, D, S1, page, lens, act_q, mode, pre):
    args, data = _make(len(lens), S1, N1, N2, D, page, lens, torch.bfloat16, latent, seed=91, act_q=act_q, mode=mode,
                       pre=pre)
    _compare(args, data, lens, act_q=act_q)


@pytest.mark.parametrize("latent,N1,D", [(False, 8, 128), (True, 16, 512), (True, 64, 512), (True, 128, 512),
                                         (True, 128, 128), (True, 40, 256)])
@pytest.mark.parametrize("dt,large,small", [("bf16", 2.0 ** 12, 2.0 ** -12), ("fp16", 2.0 ** 14, 2.0 ** -8)])
def test_small_columns_beside_a_large_one(latent, N1, D, dt, large, small):
    """A column of values 2^22 or 2^24 times the others': the others keep their
    own precision, also where a sequence is joined from many runs."""
    lens = [4000, 130, 3]
    args, data = _make(3, 1, N1, 1, D, 64, lens, DTYPES[dt], latent, seed=95)
    args["query"][..., 0] = 0
    i = 0 if latent else 1
    for x in [args["key" if latent else "value"]] + [d[i] for d in data]:
        x *= small
        x[..., 0] = large
    _compare(args, data, lens)


@pytest.mark.parametrize("latent", [False, True])
def test_64_bit_tables_and_lengths(latent):
    """Entries and lengths that 32 bits do not hold are outside the cache, past the table or below zero."""
    import dsa_triton_ascend_amd as dsa
    lens = [128, 100, 64]
    args, _ = _make(3, 1, 8, 1 if latent else 2, 512 if latent else 128, 64, lens, torch.bfloat16, latent, seed=97)
    for name in ("key", "value", "key_rope"):
        if args[name] is not None:
            args[name].nan_to_num_(0.25)
    args["block_table"][0, 1] = -1
    args["actual_seq_lengths_kv"] = torch.tensor([128, 128, 0], dtype=torch.int32, device="cuda")
    want = dsa.paged_attention(**args)
    args["actual_seq_lengths_kv"] = torch.tensor([128, 2 ** 32 + 3, -2 ** 32 + 9], device="cuda")
    page = int(args["block_table"][1, 0])
    args["block_table"] = args["block_table"].long()
    for entry in (2 ** 32 + page, -2 ** 32 + page, 2 ** 31, 2 ** 63 - 1, -2 ** 63):
        args["block_table"][0, 1] = entry
        assert all(torch.equal(a, b) for a, b in zip(dsa.paged_attention(**args), want)), entry


@pytest.mark.parametrize("latent", [False, True])
def test_queries_at_any_address(latent):
    import dsa_triton_ascend_amd as dsa
    args, _ = _make(2, 1, 8, 1 if latent else 2, 512 if latent else 128, 64, [128, 100], torch.bfloat16, latent, seed=99)
    want = dsa.paged_attention(**args)
    for name in ("query", "query_rope") if latent else ("query",):
        t = args[name]
        args[name] = torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)
        assert args[name].data_ptr() % 16 and args[name].is_contiguous()
    assert all(torch.equal(a, b) for a, b in zip(dsa.paged_attention(**args), want))
    cache = args["key"]
    args["key"] = torch.cat([cache.new_zeros(1), cache.flatten()])[1:].view(cache.shape)
    with pytest.raises(ValueError, match="aligned"):
        dsa.paged_attention(**args)
