"""Measured workloads of the paged decoding operators.

``listed()`` names twelve, ``draw(rng)`` gives more of the same ranges.  Each is
one call of an operator (for training one forward and backward):

* rope     rotary positions of a query and a key
* write    new tokens' rows into the pages of a cache
* fork     next step's block table: rows forked, released, given room; partial pages copied
* compact  live pages moved to the lowest ids
* attn     attention of the newest tokens over the pages, grouped heads or shared latent

Sizes are those of the repository's benchmark and tests (128 heads of 512 + 64
columns, indexer keys of 128, pages of 64, 32K context) and of tensor-parallel
shards of them; the grouped heads are generic.  Sequence lengths are text:
"a,b,c" gives one per sequence.

``own`` selects the framework's operators; else ``run`` computes them from
elementary torch operations.  ``exact`` restates them in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LATENT = (512, 64, 128)  # columns per token of a layer's caches: latent, rope, indexer key


def listed():
    return [
        # one decoding step at full width: rope parts of 32 sequences' queries and latent keys
        dict(name="rope_decode", op="rope", b=32, s=1, heads=128, d=64, kd=64, rot=64, interleaved=True, factor=8.0,
             grad=False, far=32768, dtype="bf16"),
        # one layer of a training step: queries of 128 + 64 columns, the last 64 rotated, forward and backward
        dict(name="rope_train", op="rope", b=1, s=4096, heads=128, d=192, kd=64, rot=64, interleaved=False, factor=1.0,
             grad=True, far=4096, dtype="bf16"),
        # one decoding step: a token of 32 sequences into a layer's three caches
        dict(name="write_decode", op="write", q=_rep(1, 32), k=_spread(801, 32767, 32), page=64, packed=False,
             dtype="bf16"),
        # packed prompts of odd lengths into a layer's three caches
        dict(name="write_prefill", op="write", q="3517,77,2999,1599", k="0,0,129,1", page=64, packed=True,
             dtype="bf16"),
        # four beams of four prompts, one layer: the smallest fork
        dict(name="fork_small", op="fork", groups=4, beams=4, hi=1203, page=16, layers=1, new=1, dtype="bf16"),
        # four beams of 64 prompts reordered, two layers
        dict(name="fork_beams", op="fork", groups=64, beams=4, hi=4001, page=64, layers=2, new=1, dtype="bf16"),
        # a small pool after a few sequences ended
        dict(name="compact_small", op="compact", pages=300, live=0.6, page=16, layers=1, dtype="fp16"),
        # a pool half empty, two thirds of a gigabyte
        dict(name="compact_half", op="compact", pages=8192, live=0.5, page=64, layers=1, dtype="bf16"),
        # one short sequence, two key heads: launch and host latency
        dict(name="attn_small", op="attn", q=1, k="777", heads=8, kvheads=2, d=128, page=16, latent=False,
             dtype="fp16"),
        # 32 sequences of 32K context, eight key heads shared by eight query heads each
        dict(name="attn_grouped", op="attn", q=1, k=_rep(32768, 32), heads=64, kvheads=8, d=128, page=64,
             latent=False, dtype="bf16"),
        # 32 sequences of 32K context over the latent cache, all 128 heads
        dict(name="attn_latent", op="attn", q=1, k=_rep(32768, 32), heads=128, kvheads=1, d=512, page=64, latent=True,
             dtype="bf16"),
        # a 16-head shard, two tokens per sequence (speculative decoding), contexts of many lengths
        dict(name="attn_latent_shard", op="attn", q=2, k=_spread(901, 24013, 24), heads=16, kvheads=1, d=512, page=64,
             latent=True, dtype="fp16"),
    ]


def draw(rng):
    """One more case of the listed ranges."""
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    dtype = rng.choice(["bf16", "bf16", "fp16"])
    kind = rng.choice(["rope", "rope", "write", "fork", "compact", "attn", "attn", "attn", "attn"])
    if kind == "rope":
        grad = rng.random() < 0.5
        b, s = (rng.randint(1, 4), log(30, 1000)) if grad else (log(1, 64), log(1, 60))
        d = rng.choice([64, 128, 192, 128])
        return dict(op="rope", b=b, s=s, heads=rng.choice([8, 16, 32, 64, 128]), d=d, kd=rng.choice([64, d]),
                    rot=rng.choice([32, 64, 64]), interleaved=rng.random() < 0.5, factor=rng.choice([1.0, 4.0, 8.0, 40.0]),
                    grad=grad, far=log(2000, 131072), dtype=rng.choice([dtype, dtype, "fp32"]))
    if kind == "write":
        packed = rng.random() < 0.5
        b = rng.randint(1, 6) if packed else log(1, 64)
        step = rng.randint(1, 4)
        q = [log(1, 2000) if packed else step for _ in range(b)]
        k = [0 if rng.random() < 0.3 else log(1, 8000) for _ in range(b)]
        return dict(op="write", q=_text(q), k=_text(k), page=rng.choice([16, 48, 64, 128]), packed=packed, dtype=dtype)
    if kind == "fork":
        return dict(op="fork", groups=log(1, 48), beams=rng.randint(1, 5), hi=log(20, 3500),
                    page=rng.choice([16, 48, 64]), layers=rng.randint(1, 2), new=rng.randint(0, 5), dtype=dtype)
    if kind == "compact":
        return dict(op="compact", pages=log(20, 6000), live=round(rng.uniform(0.05, 0.95), 3),
                    page=rng.choice([16, 48, 64]), layers=1, dtype=dtype)
    hi, latent = log(30, 32768), rng.random() < 0.5
    b = min(log(1, 48), max(1, (250000 if latent else 500000) // hi))
    k = _rep(hi, b) if rng.random() < 0.4 else _spread(max(1, hi // rng.randint(2, 20)), hi, b)
    q, page = rng.choice([1, 1, 1, 2, 3, 4]), rng.choice([16, 48, 64, 64, 128])
    if latent:
        return dict(op="attn", q=q, k=k, heads=rng.choice([16, 32, 64, 128]), kvheads=1, d=512, page=page, latent=True,
                    dtype=dtype)
    kv = rng.choice([1, 2, 4, 8])
    return dict(op="attn", q=q, k=k, heads=kv * rng.choice([1, 4, 5, 8]), kvheads=kv, d=rng.choice([64, 128, 128, 256]),
                page=page, latent=False, dtype=dtype)


def _text(lens):
    return ",".join(str(x) for x in lens)


def _rep(n, times):
    return _text([n] * times)


def _spread(lo, hi, n):
    """``n`` lengths from ``lo`` to ``hi``, evenly spread in a scattered order."""
    return _text([lo + (hi - lo) * ((i * 7) % n) // max(1, n - 1) for i in range(n)])


def _lens(text):
    return [int(x) for x in text.split(",")]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed), torch.Generator().manual_seed(seed)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _table(lens, page, pool, host):
    """A block table over scattered pages for sequences of these lengths, -1 past their ends."""
    need = [-(-n // page) for n in lens]
    ids = torch.randperm(pool, generator=host)[:sum(need)].tolist()
    wide, rows, at = max(max(need), 1), [], 0
    for n in need:
        rows.append(ids[at:at + n] + [-1] * (wide - n))
        at += n
    return rows


def _frequencies(case):
    """Inverse frequencies and output scale of a case: positions stretched by ``factor`` with YaRN's blend."""
    rot, factor, base, orig = case["rot"], case["factor"], 10000.0, 4096
    half = rot // 2
    inv = [base ** (-2.0 * i / rot) for i in range(half)]
    if factor == 1.0:
        return inv, 1.0

    def at(turns):
        return rot * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(base))

    lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
    out = []
    for i, f in enumerate(inv):
        ramp = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
        out.append(f / factor * ramp + f * (1.0 - ramp))
    return out, 0.1 * math.log(factor) + 1.0


def prepare(case, seed):
    gen, host = _gen(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)

    st = dict(case=case)
    op = case["op"]
    if op == "rope":
        b, s = case["b"], case["s"]
        q, k = normal(b, s, case["heads"], case["d"]), normal(b, s, 1, case["kd"])
        first = torch.randint(0, max(1, case["far"] - s + 1), (b, 1), generator=host)
        st["positions"] = (first + torch.arange(s)).to(device="cuda", dtype=torch.int32)
        st["dq"], st["dk"] = (normal(*q.shape), normal(*k.shape)) if case["grad"] else (None, None)
        if case["grad"]:
            q.requires_grad_(True)
            k.requires_grad_(True)
        st["q"], st["k"] = q, k
        if own:
            import dsa_triton_ascend_amd as dsa
            st["inv_freq"], st["scale"] = dsa.rotary_frequencies(
                case["rot"], scaling="none" if case["factor"] == 1.0 else "yarn", factor=case["factor"], device="cuda")
        else:
            inv, st["scale"] = _frequencies(case)
            st["inv_freq"] = torch.tensor(inv, dtype=torch.float64, device="cuda")
    elif op == "write":
        new, old, page = _lens(case["q"]), _lens(case["k"]), case["page"]
        need = sum(-(-(a + b) // page) for a, b in zip(new, old))
        pool = need + 5
        st["table"] = _ints(_table([a + b for a, b in zip(new, old)], page, pool, host))
        st["lens"] = _ints(old)
        st["caches"] = [normal(pool, page, 1, c) for c in LATENT]
        if case["packed"]:
            st["rows"] = [normal(sum(new), 1, c) for c in LATENT]
            st["new"] = torch.cumsum(torch.tensor(new), 0).to(device="cuda", dtype=torch.int32)
        else:
            st["rows"] = [normal(len(new), new[0], 1, c) for c in LATENT]
            st["new"] = None
        st["new_host"] = new
    elif op == "fork":
        # beams of a prompt share its pages up to where they parted, then have their own
        page, beams = case["page"], case["beams"]
        pool = case["groups"] * ((-(-case["hi"] // page)) + beams * 5) + case["groups"] * beams * 3 + 8
        ids = torch.randperm(pool, generator=host).tolist()
        rows, lens, parents = [], [], []
        for g in range(case["groups"]):
            n = int(torch.randint(max(1, case["hi"] // 4), case["hi"] + 1, (1,), generator=host))
            total = -(-n // page)
            shared = max(0, min(n // page, total - 1 - int(torch.randint(0, 4, (1,), generator=host))))
            trunk = [ids.pop() for _ in range(shared)]
            for _ in range(beams):
                rows.append(trunk + [ids.pop() for _ in range(total - shared)])
                lens.append(n)
            pick = torch.randint(0, beams, (beams,), generator=host).tolist()
            ended = int(torch.randint(0, 8, (1,), generator=host)) == 0  # one group in eight is done
            parents += [-1 if ended else g * beams + p for p in pick]
        wide = -(-(case["hi"] + case["new"]) // page) + 1
        st["table"] = _ints([r + [-1] * (wide - len(r)) for r in rows])
        st["lens"], st["parents"] = _ints(lens), _ints(parents)
        refs = torch.zeros(pool, dtype=torch.int32)
        for r in rows:
            refs[torch.tensor(r, dtype=torch.long)] += 1
        st["refs"] = refs.cuda()
        st["caches"] = [normal(pool, page, 1, c) for _ in range(case["layers"]) for c in LATENT]
    elif op == "compact":
        pool, page = case["pages"], case["page"]
        live = torch.randperm(pool, generator=host)[:max(1, int(pool * case["live"]))].tolist()
        wide = max(1, min(128, len(live) // 4))
        rows, at = [], 0
        while at < len(live):
            rows.append(live[at:at + wide])
            at += wide
        rows.append(rows[0][:len(rows[0]) // 2] + rows[-1][-1:])  # a row that shares others' pages
        st["table"] = _ints([r + [-1] * (wide + 1 - len(r)) for r in rows])
        refs = torch.zeros(pool, dtype=torch.int32)
        for r in rows:
            refs[torch.tensor(r, dtype=torch.long)] += 1
        st["refs"] = refs.cuda()
        st["caches"] = [normal(pool, page, 1, c) for _ in range(case["layers"]) for c in LATENT]
    else:
        lens, page, n2, d = _lens(case["k"]), case["page"], case["kvheads"], case["d"]
        pool = sum(-(-n // page) for n in lens) + 3
        st["table"] = _ints(_table(lens, page, pool, host))
        st["lens"], st["lens_host"] = _ints(lens), lens
        # queries of twice the keys' spread: the softmax settles on a few hundred of 32K tokens
        st["q"] = normal(len(lens), case["q"], case["heads"], d) * 2
        st["k"] = normal(pool, page, n2, d)
        st["v"] = None if case["latent"] else normal(pool, page, n2, d)
        st["qr"] = normal(len(lens), case["q"], case["heads"], 64) * 2 if case["latent"] else None
        st["kr"] = normal(pool, page, n2, 64) if case["latent"] else None
        st["scale"] = 1.0 / math.sqrt(d + 64 if case["latent"] else d)
    return st


def run(st):
    if own:
        return _run_own(st)
    case = st["case"]
    op = case["op"]
    if op == "rope":
        return _rope_plain(st)
    if op == "write":
        _write(st["caches"], st["rows"], st["table"], st["lens"], st["new_host"], case["packed"])
        return list(st["caches"])
    if op == "fork":
        return _fork_plain(st)
    if op == "compact":
        return _compact_plain(st)
    return _attention(st, torch.float32)


def _run_own(st):
    import dsa_triton_ascend_amd as dsa
    case = st["case"]
    op = case["op"]
    if op == "rope":
        q, k = dsa.rotary_embedding(
            st["q"], st["k"], st["positions"], st["inv_freq"], interleaved=case["interleaved"],
            rotary_offset=case["d"] - case["rot"], key_rotary_offset=case["kd"] - case["rot"],
            attention_scale=st["scale"])
        if not case["grad"]:
            return q, k
        dq, dk = torch.autograd.grad((q, k), (st["q"], st["k"]), (st["dq"], st["dk"]))
        return q.detach(), k.detach(), dq, dk
    if op == "write":
        dsa.paged_cache_write(st["caches"], st["rows"], st["table"], st["lens"], row_lengths=st["new"],
                              layout="TND" if case["packed"] else "BSND")
        return list(st["caches"])
    if op == "fork":
        table, lens, refs = dsa.paged_cache_fork(st["caches"], st["table"], st["lens"], st["refs"],
                                                 parents=st["parents"], new_tokens=case["new"])
        return [table, lens, refs] + list(st["caches"])
    if op == "compact":
        table, refs, page_map = dsa.paged_cache_compact(st["caches"], st["table"], st["refs"])
        return [table, refs, page_map] + list(st["caches"])
    return dsa.paged_attention(st["q"], st["k"], st["v"], st["table"], st["lens"], scale_value=st["scale"],
                               query_rope=st["qr"], key_rope=st["kr"], return_softmax_lse=True)


# ---- the operators from elementary torch operations, sums in 32 bits ----

def _turn(x, cos, sin, start, rot, interleaved):
    """``x`` with the columns start .. start + rot of every head rotated."""
    part = x[..., start:start + rot].float()
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
    else:
        a, b = part[..., :rot // 2], part[..., rot // 2:]
    a2, b2 = a * cos - b * sin, a * sin + b * cos
    part = torch.stack([a2, b2], -1).flatten(-2) if interleaved else torch.cat([a2, b2], -1)
    return torch.cat([x[..., :start], part.to(x.dtype), x[..., start + rot:]], -1)


def _rope_plain(st):
    case = st["case"]
    # angles of far positions need 64 bits
    angle = st["positions"].double()[..., None] * st["inv_freq"]
    cos = (torch.cos(angle) * st["scale"]).float()[:, :, None, :]
    sin = (torch.sin(angle) * st["scale"]).float()[:, :, None, :]
    rot, inter = case["rot"], case["interleaved"]
    q0, k0 = case["d"] - rot, case["kd"] - rot
    with torch.no_grad():
        out = [_turn(st["q"], cos, sin, q0, rot, inter), _turn(st["k"], cos, sin, k0, rot, inter)]
        if case["grad"]:
            out += [_turn(st["dq"], cos, -sin, q0, rot, inter), _turn(st["dk"], cos, -sin, k0, rot, inter)]
    return tuple(out)


def _write(caches, rows, table, lens, new, packed):
    page = caches[0].shape[1]
    device = table.device
    counts = torch.tensor(new, device=device)
    seq = torch.repeat_interleave(torch.arange(len(new), device=device), counts)
    first = torch.cumsum(counts, 0) - counts
    pos = lens.long()[seq] + torch.arange(seq.numel(), device=device) - first[seq]
    slot = table.long()[seq, pos // page] * page + pos % page
    for cache, row in zip(caches, rows):
        cache.view(-1, cache.shape[-1])[slot] = row.reshape(-1, cache.shape[-1])


def _fork_plain(st):
    case, table, lens, refs, parents = st["case"], st["table"], st["lens"], st["refs"], st["parents"]
    page, new = case["page"], case["new"]
    rows, wide = table.shape
    pool = refs.numel()
    device = table.device
    live = parents >= 0
    par = parents.clamp(min=0).long()
    n = torch.where(live, lens[par], 0).long()
    full, held, want = n // page, -(-n // page), torch.where(live, -(-(n + new) // page), 0)
    c = torch.arange(parents.numel(), device=device)
    first = torch.full((rows,), parents.numel(), dtype=torch.long, device=device)
    first.scatter_reduce_(0, par, torch.where(live, c, parents.numel()), "amin")
    last = table[par, full.clamp(max=wide - 1)].long()
    partial = live & (full < held)
    copy = partial & ~((first[par] == c) & (refs[last.clamp(min=0)] == 1))
    need = copy.long() + want - held
    start = torch.cumsum(need, 0) - need
    free = torch.nonzero(refs == 0).flatten()
    col = torch.arange(wide, device=device)[None]
    out = torch.where(col < held[:, None], table[par].long(), -1)
    out = torch.where(live[:, None], out, -1)
    fresh = (start + copy.long())[:, None] + col - held[:, None]
    out = torch.where((col >= held[:, None]) & (col < want[:, None]), free[fresh.clamp(0, free.numel() - 1)], out)
    dst = free[start.clamp(max=free.numel() - 1)]
    out = torch.where(copy[:, None] & (col == full[:, None]), dst[:, None], out)
    counted = refs.long()
    counted = counted + torch.bincount(out[out >= 0], minlength=pool) - torch.bincount(table[table >= 0].long(),
                                                                                       minlength=pool)
    tok = torch.arange(page, device=device)[None]
    which = (copy[:, None] & (tok < (n % page)[:, None])).nonzero()
    src_slot = last[which[:, 0]] * page + which[:, 1]
    dst_slot = dst[which[:, 0]] * page + which[:, 1]
    for cache in st["caches"]:
        flat = cache.view(-1, cache.shape[-1])
        flat[dst_slot] = flat[src_slot]
    return [out.int(), n.int(), counted.int()] + list(st["caches"])


def _compact_plain(st):
    table, refs = st["table"], st["refs"]
    live = refs > 0
    n = int(live.sum())
    ids = torch.arange(refs.numel(), device=refs.device)
    high, hole = ids[live & (ids >= n)], ids[~live & (ids < n)]
    page_map = torch.where(live, ids, -1)
    page_map[high] = hole
    for cache in st["caches"]:
        cache[hole] = cache[high]
    out_refs = torch.zeros_like(refs)
    out_refs[page_map[live]] = refs[live]
    out = torch.where(table >= 0, page_map[table.clamp(min=0).long()], -1)
    return [out.int(), out_refs, page_map.int()] + list(st["caches"])


def _attention(st, real):
    """The attention in the floating type ``real``; outputs in the query's type when that is 32 bits."""
    case, q = st["case"], st["q"]
    b, s1, heads, d = q.shape
    n2 = case["kvheads"]
    group = heads // n2
    page = case["page"]
    out = torch.zeros(q.shape, dtype=q.dtype if real == torch.float32 else real, device=q.device)
    smax = torch.zeros(b, n2, s1, group, dtype=real, device=q.device)
    ssum = torch.zeros_like(smax)
    for i, n in enumerate(st["lens_host"]):
        pages = st["table"][i, :-(-n // page)].long()

        def gather(cache):  # [n2, n, columns]
            return cache[pages].reshape(-1, n2, cache.shape[-1])[:n].to(real).transpose(0, 1).contiguous()

        key = gather(st["k"])
        query = q[i].to(real)
        if case["latent"]:
            value = key
            key = torch.cat([key, gather(st["kr"])], -1)
            query = torch.cat([query, st["qr"][i].to(real)], -1)
        else:
            value = gather(st["v"])
        # [n2, s1 * group, columns]
        query = query.view(s1, n2, group, -1).transpose(0, 1).reshape(n2, s1 * group, -1)
        score = torch.matmul(query, key.transpose(1, 2).contiguous()) * st["scale"]
        limit = n - s1 + 1 + torch.arange(s1, device=q.device).repeat_interleave(group)  # tokens that a row sees
        hidden = torch.arange(n, device=q.device)[None] >= limit[:, None]
        score = score.masked_fill(hidden, float("-inf"))
        top = score.amax(-1, keepdim=True)
        seen = torch.isfinite(top)
        p = torch.where(seen, torch.exp(score - torch.where(seen, top, 0)), 0)
        total = p.sum(-1, keepdim=True)
        o = torch.matmul(p, value) / torch.where(total > 0, total, 1)
        out[i] = o.view(n2, s1, group, d).transpose(0, 1).reshape(s1, heads, d).to(out.dtype)
        smax[i] = torch.where(seen, top, 0).view(n2, s1, group)
        ssum[i] = total.view(n2, s1, group)
    return out, smax, ssum


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    op = case["op"]
    if op == "rope":
        rows = case["b"] * case["s"]
        elements = rows * (case["heads"] * case["d"] + case["kd"])
        passes = 2 if case["grad"] else 1
        return {"bytes": passes * (2 * elements * size + rows * 4),
                "flops": passes * 3 * rows * (case["heads"] + 1) * case["rot"]}
    columns = sum(LATENT)
    if op == "write":
        return {"bytes": sum(_lens(case["q"])) * columns * 2 * size, "flops": 0}
    if op == "fork":
        # of a prompt's beams about a third continue a parent that another one keeps; half a page each
        rows = case["groups"] * case["beams"]
        tokens = rows * (1 - 1 / case["beams"]) * 0.6 * (case["page"] / 2)
        tables = rows * (-(-case["hi"] // case["page"])) * 8
        return {"bytes": int(tokens * columns * case["layers"] * 2 * size + tables) + 64, "flops": 0}
    if op == "compact":
        moved = case["pages"] * case["live"] * (1 - case["live"])
        return {"bytes": int(moved * case["page"] * columns * case["layers"] * 2 * size) + case["pages"] * 12, "flops": 0}
    tokens, d = sum(_lens(case["k"])), case["d"]
    rows = len(_lens(case["k"])) * case["q"] * case["heads"]
    dk, per = (d + 64, d + 64) if case["latent"] else (d, 2 * d)
    return {"bytes": tokens * case["kvheads"] * per * size + rows * ((dk + d) * size + 8),
            "flops": 2 * tokens * case["q"] * case["heads"] * (dk + d)}


# ---- definitions in 64 bits ----

def exact(case, seed):
    # the same inputs, made without the framework
    global own
    kept, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = kept
    op = case["op"]
    with torch.no_grad():
        if op == "rope":
            return _rope_exact(st)
        if op == "write":
            return _write_exact(st)
        if op == "fork":
            return _fork_exact(st)
        if op == "compact":
            return _compact_exact(st)
        return _attention_exact(st)


def _rope_exact(st):
    case = st["case"]
    rot = case["rot"]
    theta = st["positions"].double()[:, :, None, None] * st["inv_freq"]
    turn = torch.polar(torch.full_like(theta, st["scale"]), theta)

    def apply(x, start, factor):
        y = x.double().clone()
        part = y[..., start:start + rot]
        if case["interleaved"]:
            z = torch.view_as_complex(part.reshape(*part.shape[:-1], rot // 2, 2).contiguous()) * factor
            y[..., start:start + rot] = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(part[..., :rot // 2].contiguous(), part[..., rot // 2:].contiguous()) * factor
            y[..., start:start + rot] = torch.cat([z.real, z.imag], -1)
        return y

    out = [apply(st["q"], case["d"] - rot, turn), apply(st["k"], case["kd"] - rot, turn)]
    if case["grad"]:
        out += [apply(st["dq"], case["d"] - rot, turn.conj()), apply(st["dk"], case["kd"] - rot, turn.conj())]
    return tuple(out)


def _write_exact(st):
    table, page, at = st["table"].tolist(), st["case"]["page"], 0
    out = [c.double() for c in st["caches"]]
    rows = [r.double().reshape(-1, r.shape[-1]) for r in st["rows"]]
    for b, (n, old) in enumerate(zip(st["new_host"], st["lens"].tolist())):
        done = 0
        while done < n:
            slot, begin = divmod(old + done, page)
            take = min(page - begin, n - done)
            for o, r in zip(out, rows):
                o[table[b][slot], begin:begin + take, 0] = r[at + done:at + done + take]
            done += take
        at += n
    return out


def _fork_exact(st):
    case = st["case"]
    page, new = case["page"], case["new"]
    table, lens, refs = st["table"].tolist(), st["lens"].tolist(), st["refs"].tolist()
    free = iter([i for i, r in enumerate(refs) if r == 0])
    before, used, moves = list(refs), set(), []
    out, out_lens = [], []
    for p in st["parents"].tolist():
        if p < 0:
            out.append([-1] * len(table[0]))
            out_lens.append(0)
            continue
        n = lens[p]
        held = -(-n // page)
        row = table[p][:held]
        if n % page and (p in used or before[row[-1]] != 1):
            to = next(free)
            moves.append((row[-1], to, n % page))
            row = row[:-1] + [to]
        used.add(p)
        while len(row) < -(-(n + new) // page):
            row.append(next(free))
        out.append(row + [-1] * (len(table[0]) - len(row)))
        out_lens.append(n)
    for row in out:
        for e in row:
            if e >= 0:
                refs[e] += 1
    for row in table:
        for e in row:
            if e >= 0:
                refs[e] -= 1
    caches = [c.double() for c in st["caches"]]
    for c in caches:
        for src, dst, count in moves:
            c[dst, :count] = c[src, :count]
    return [_ints(out), _ints(out_lens), _ints(refs)] + caches


def _compact_exact(st):
    table, refs = st["table"].tolist(), st["refs"].tolist()
    n = sum(r > 0 for r in refs)
    holes = iter([i for i in range(n) if refs[i] == 0])
    page_map = [-1 if r == 0 else (i if i < n else next(holes)) for i, r in enumerate(refs)]
    out_refs = [0] * len(refs)
    for i, to in enumerate(page_map):
        if to >= 0:
            out_refs[to] = refs[i]
    src = [i for i, to in enumerate(page_map) if to >= 0 and to != i]
    dst = [page_map[i] for i in src]
    caches = [c.double() for c in st["caches"]]
    for c in caches:
        c[dst] = c[src]
    out = [[page_map[e] if e >= 0 else -1 for e in row] for row in table]
    return [_ints(out), _ints(out_refs), _ints(page_map)] + caches


def _attention_exact(st):
    """Head by head, the log of the softmax's sum taken by logsumexp."""
    case, q = st["case"], st["q"].double()
    b, s1, heads, d = q.shape
    n2, page = case["kvheads"], case["page"]
    group = heads // n2
    out = torch.zeros_like(q)
    smax = torch.zeros(b, n2, s1, group, dtype=torch.float64, device=q.device)
    ssum = torch.zeros_like(smax)
    for i, n in enumerate(st["lens_host"]):
        slots = torch.arange(n, device=q.device)
        slots = st["table"][i].long()[slots // page] * page + slots % page
        for h in range(n2):
            key = st["k"].view(-1, n2, d)[slots, h].double()
            value = key if case["latent"] else st["v"].view(-1, n2, d)[slots, h].double()
            for s in range(s1):
                m = n - s1 + 1 + s
                if m <= 0:
                    continue
                mine = slice(h * group, (h + 1) * group)
                score = key[:m] @ q[i, s, mine].T
                if case["latent"]:
                    score += st["kr"].view(-1, 64)[slots[:m]].double() @ st["qr"][i, s, mine].double().T
                score *= st["scale"]
                norm = torch.logsumexp(score, 0)
                out[i, s, mine] = torch.exp(score - norm).T @ value[:m]
                smax[i, h, s] = score.max(0).values
                ssum[i, h, s] = torch.exp(norm - smax[i, h, s])
    return out, smax, ssum
