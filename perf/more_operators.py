"""Measured workloads of the operators that serve requests of many lengths
with shared prompts.

``listed()`` names twelve, ``draw(rng)`` gives more of the same ranges.  Each is
one call of an operator (for training one forward and backward):

* axes      rotary positions with several axes (time, height, width)
* plan      next step's block table, slots and positions from the requests' lengths
* slots     packed rows into the slots of a plan
* prefixes  which neighbouring sequences share their first pages
* attn      attention of the newest tokens, a shared prefix read once for its sequences

Sizes are those of the repository's benchmark and tests (128 heads of 512 + 64
columns, indexer keys of 128, pages of 64, 32K context) and of tensor-parallel
shards of them; the grouped heads are generic.  Lengths are text: "a,b,c".

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
        # one decoding step at full width: rope parts of 32 sequences behind images, queries and latent keys
        dict(name="axes_decode", op="axes", b=32, s=1, heads=128, d=64, kd=64, kheads=1, sections="16,8,8", mixed=True,
             grad=False, packed=False, dtype="bf16"),
        # a layer of a training step on text and an image grid: queries and eight key heads, forward and backward
        dict(name="axes_train", op="axes", b=1, s=4096, heads=64, d=128, kd=128, kheads=8, sections="16,24,24",
             mixed=False, grad=True, packed=False, dtype="bf16"),
        # one decoding step of 32 requests: the smallest plan
        dict(name="plan_decode", op="plan", rows=32, prompts=0, ended=0, hi=32768, new=1, page=64, pad=0),
        # a mixed step: 192 requests decode, 32 prompts begin, some have ended; a pool of small pages
        dict(name="plan_mixed", op="plan", rows=256, prompts=32, ended=16, hi=8000, new=1500, page=16, pad=37),
        # one decoding step: a token of 32 sequences into a layer's three caches
        dict(name="slots_decode", op="slots", tokens=32, pool=2048, page=64, dtype="bf16"),
        # a packed step of 8192 tokens, some of them padding, into a layer's three caches
        dict(name="slots_prefill", op="slots", tokens=8192, pool=160, page=64, dtype="bf16"),
        # four beams of four prompts
        dict(name="prefixes_small", op="prefixes", members="4,4,4,4", hi=1203, page=16),
        # 256 requests in families of many sizes over prompts of up to 32K tokens
        dict(name="prefixes_many", op="prefixes", members="64,1,31,8,2,50,1,1,98", hi=32768, page=16),
        # four beams of one prompt, two key heads: launch and host latency
        dict(name="attn_small", op="attn", q=1, members="4", prefix="640", suffix="23,57,41,33", heads=8, kvheads=2,
             d=128, page=16, latent=False, dtype="fp16"),
        # 32 requests behind a 32K prompt, eight key heads shared by eight query heads each
        dict(name="attn_grouped", op="attn", q=1, members="32", prefix="32768", suffix=_spread(33, 2011, 32), heads=64,
             kvheads=8, d=128, page=64, latent=False, dtype="bf16"),
        # 32 requests behind a 32K prompt over the latent cache, all 128 heads
        dict(name="attn_latent", op="attn", q=1, members="32", prefix="32768", suffix=_spread(33, 2011, 32), heads=128,
             kvheads=1, d=512, page=64, latent=True, dtype="bf16"),
        # a 16-head shard, two tokens per sequence (speculative decoding), families of many sizes
        dict(name="attn_latent_shard", op="attn", q=2, members="12,1,7,3,9", prefix="16000,0,24016,4992,9600",
             suffix=_spread(41, 3001, 32), heads=16, kvheads=1, d=512, page=64, latent=True, dtype="fp16"),
    ]


def draw(rng):
    """One more case of the listed ranges."""
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    dtype = rng.choice(["bf16", "bf16", "fp16"])
    kind = rng.choice(["axes", "axes", "plan", "plan", "slots", "prefixes", "attn", "attn", "attn", "attn"])
    if kind == "axes":
        grad, packed = rng.random() < 0.5, rng.random() < 0.3
        b, s = (rng.randint(1, 3), log(30, 1300)) if grad else (log(1, 64), log(1, 60))
        d = rng.choice([64, 128, 192])
        rot = rng.choice([32, 64, 64, d])
        if rng.random() < 0.3:  # height and width of an image encoder
            h = rng.randint(1, rot // 2 - 1)
            sections, mixed = [rot // 2 - h, h], False
        else:
            w = rng.randint(1, rot // 6)
            sections, mixed = [rot // 2 - 2 * w, w, w], rng.random() < 0.5
        return dict(op="axes", b=b, s=s, heads=rng.choice([8, 16, 32, 64]), d=d, kd=max(rot, rng.choice([64, d])),
                    kheads=rng.choice([1, 1, 4, 8]), sections=_text(sections), mixed=mixed, grad=grad, packed=packed,
                    dtype=rng.choice([dtype, dtype, "fp32"]))
    if kind == "plan":
        rows = log(4, 400)
        return dict(op="plan", rows=rows, prompts=rng.randint(0, rows // 2), ended=rng.randint(0, rows // 4),
                    hi=log(200, 9000), new=log(2, 2000) if rows < 100 else log(2, 400), page=rng.choice([16, 48, 64, 128]),
                    pad=rng.choice([0, 0, 1, 77]))
    if kind == "slots":
        tokens, page = log(1, 8192), rng.choice([16, 48, 64, 128])
        return dict(op="slots", tokens=tokens, pool=-(-tokens // page) + rng.randint(1, 100), page=page, dtype=dtype)
    if kind == "prefixes":
        members = [log(2, 64) for _ in range(rng.randint(2, 7))]
        return dict(op="prefixes", members=_text(members), hi=log(2000, 30000), page=rng.choice([16, 48, 64]))
    latent = rng.random() < 0.5
    families, q, page = rng.randint(1, 4), rng.choice([1, 1, 1, 2, 3]), rng.choice([16, 48, 64, 64, 128])
    members = [log(1, 12) for _ in range(families)]
    longest = log(50, 24000)
    prefix = [max(page, rng.randint(longest // 3, longest)) // page * page for _ in members]
    if rng.random() < 0.3:
        prefix[rng.randrange(families)] = 0
    b = sum(members)
    suffix = [q + log(1, 2000) - 1 for _ in range(b)]
    shape = dict(heads=rng.choice([16, 32, 64, 128]), kvheads=1, d=512)
    if not latent:
        kv = rng.choice([1, 2, 4, 8])
        shape = dict(heads=kv * rng.choice([1, 4, 5, 8]), kvheads=kv, d=rng.choice([64, 128, 128, 256]))
    return dict(op="attn", q=q, members=_text(members), prefix=_text(prefix), suffix=_text(suffix), page=page,
                latent=latent, dtype=dtype, **shape)


def _text(values):
    return ",".join(str(x) for x in values)


def _spread(lo, hi, n):
    """``n`` lengths from ``lo`` to ``hi``, evenly spread in a scattered order."""
    return _text([lo + (hi - lo) * ((i * 7) % n) // max(1, n - 1) for i in range(n)])


def _ints_of(text):
    return [int(x) for x in text.split(",")]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed), torch.Generator().manual_seed(seed)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _sizes(case):
    """A generator for lengths that belong to the case: other seeds give other contents of the same sizes."""
    return torch.Generator().manual_seed(sum((i + 1) * ord(c) for i, c in enumerate(repr(sorted(case.items())))))


def _between(host, lo, hi):
    return int(torch.randint(lo, hi + 1, (1,), generator=host))


def _axis_positions(n, axes, host):
    """Positions [axes, n] of text with images in it: text counts on all axes, a
    grid stays on the first and runs over the others, as video frames would."""
    out, at = [], _between(host, 0, 2000)
    while len(out) < n:
        run = _between(host, 1, 300)
        out += [[at + i] * axes for i in range(run)]
        at += run
        h, w = _between(host, 1, 40), _between(host, 1, 40)
        out += [[at, at + y, at + x] if axes == 3 else [at + y, at + x] for y in range(h) for x in range(w)]
        at += max(h, w)
    return torch.tensor(out[:n], dtype=torch.int32).T.contiguous()


def _pair_axes(case):
    """Axis of each pair of columns."""
    sections = _ints_of(case["sections"])
    if not case["mixed"]:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    a = len(sections)
    return [i % a if i < a * sections[i % a] else 0 for i in range(sum(sections))]


def prepare(case, seed):
    gen, host = _gen(seed)
    dtype = DTYPES[case.get("dtype", "bf16")]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)

    st = dict(case=case)
    op = case["op"]
    if op == "axes":
        b, s = case["b"], case["s"]
        lead = (b * s,) if case["packed"] else (b, s)
        q, k = normal(*lead, case["heads"], case["d"]), normal(*lead, case["kheads"], case["kd"])
        sections = _ints_of(case["sections"])
        pos = torch.cat([_axis_positions(s, len(sections), host) for _ in range(b)], 1)
        st["positions"] = pos.view(len(sections), *lead).cuda()
        st["dq"], st["dk"] = (normal(*q.shape), normal(*k.shape)) if case["grad"] else (None, None)
        if case["grad"]:
            q.requires_grad_(True)
            k.requires_grad_(True)
        st["q"], st["k"] = q, k
        rot = 2 * sum(sections)
        st["rot"], st["sections"] = rot, tuple(sections)
        st["inv_freq"] = torch.tensor([10000.0 ** (-2.0 * i / rot) for i in range(rot // 2)], dtype=torch.float64,
                                      device="cuda")
        st["pair_axes"] = torch.tensor(_pair_axes(case), device="cuda")
    elif op == "plan":
        rows, page, sizes = case["rows"], case["page"], _sizes(case)
        kinds = ["prompt"] * case["prompts"] + ["ended"] * case["ended"]
        kinds += ["decode"] * (rows - len(kinds))
        order = torch.randperm(rows, generator=sizes).tolist()
        old, new = [], []
        for i in order:
            prompt = kinds[i] == "prompt"
            # some prompts arrive in chunks, behind tokens of their own
            old.append(_between(sizes, 0, 300) if prompt and _between(sizes, 0, 2) == 0 else
                       0 if prompt else _between(sizes, 1, case["hi"]))
            new.append(-1 if kinds[i] == "ended" else _between(sizes, 1, case["new"]) if prompt else 1)
        held = [-(-n // page) for n in old]
        want = sum(-(-(n + max(m, 0)) // page) for n, m in zip(old, new))
        pool = sum(held) + want // 8 + sum(-(-max(m, 0) // page) for m in new) + 4
        ids = torch.randperm(pool, generator=host)[:sum(held)].tolist()
        wide = max(-(-(n + max(m, 0)) // page) for n, m in zip(old, new)) + 1
        table, refs, at = [], torch.zeros(pool, dtype=torch.int32), 0
        for n in held:
            table.append(ids[at:at + n] + [-1] * (wide - n))
            at += n
        refs[torch.tensor(ids, dtype=torch.long)] = 1
        st["table"], st["lens"], st["refs"], st["new"] = _ints(table), _ints(old), refs.cuda(), _ints(new)
        st["tokens"] = sum(max(m, 0) for m in new) + case["pad"]
    elif op == "slots":
        n, page, pool = case["tokens"], case["page"], case["pool"]
        slots = torch.randperm(pool * page, generator=host)[:n].to(torch.int32)
        # whole pages in order, as a prompt takes them, and one row in 50 is padding
        if n > page:
            full = (n // page) * page
            slots[:full] = (torch.randperm(pool, generator=host)[:n // page, None] * page
                            + torch.arange(page)[None]).flatten().int()
            used = torch.zeros(pool * page, dtype=torch.bool)
            used[slots[:full].long()] = True
            slots[full:] = (~used).nonzero().flatten()[:n - full].int()
            slots[torch.randperm(n, generator=host)[:n // 50]] = -1
        st["slots"] = slots.cuda()
        st["caches"] = [normal(pool, page, 1, c) for c in LATENT]
        st["rows"] = [normal(n, 1, c) for c in LATENT]
    elif op == "prefixes":
        page = case["page"]
        members = _ints_of(case["members"])
        rows, lens, used = [], [], 0
        for m in members:
            full = _between(host, max(1, case["hi"] // 4), case["hi"]) // page
            trunk, used = list(range(used, used + full)), used + full
            for _ in range(m):
                n = full * page + _between(host, 1, 5 * page)
                mine = -(-n // page) - full
                rows.append(trunk + list(range(used, used + mine)))
                used += mine
                lens.append(n)
        scattered = torch.randperm(used, generator=host)
        wide = case["hi"] // page + 7
        table = torch.full((len(rows), wide), -1, dtype=torch.int32)
        for i, r in enumerate(rows):
            table[i, :len(r)] = scattered[torch.tensor(r, dtype=torch.long)].int()
        st["table"], st["lens"] = table.cuda(), _ints(lens)
    else:
        page, n2, d = case["page"], case["kvheads"], case["d"]
        members, prefix, suffix = (_ints_of(case[x]) for x in ("members", "prefix", "suffix"))
        shared = [p for p, m in zip(prefix, members) for _ in range(m)]
        lens = [p + x for p, x in zip(shared, suffix)]
        total = [-(-n // page) for n in lens]
        pool = sum(p // page for p in prefix) + sum(t - p // page for t, p in zip(total, shared)) + 3
        ids = torch.randperm(pool, generator=host).tolist()
        table, leader, b = [], [], 0
        for p, m in zip(prefix, members):
            trunk = [ids.pop() for _ in range(p // page)]
            first = b
            for _ in range(m):
                table.append(trunk + [ids.pop() for _ in range(total[b] - p // page)])
                leader.append(first)
                b += 1
        wide = max(total)
        st["table"] = _ints([r + [-1] * (wide - len(r)) for r in table])
        st["lens"], st["lens_host"] = _ints(lens), lens
        # what the plan of a step gives: each sequence's family and the tokens it shares
        st["groups"], st["shared"] = _ints(leader), _ints(shared)
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
    if op == "axes":
        return _axes_plain(st)
    if op == "plan":
        return _plan_plain(st)
    if op == "slots":
        keep = (st["slots"] >= 0).nonzero().flatten()
        at = st["slots"][keep].long()
        for cache, row in zip(st["caches"], st["rows"]):
            cache.view(-1, cache.shape[-1])[at] = row.view(-1, row.shape[-1])[keep]
        return list(st["caches"])
    if op == "prefixes":
        return _prefixes_plain(st)
    return _attention(st)


def _run_own(st):
    import dsa_triton_ascend_amd as dsa
    case = st["case"]
    op = case["op"]
    if op == "axes":
        q, k = dsa.rotary_embedding(
            st["q"], st["k"], st["positions"], st["inv_freq"], rotary_offset=case["d"] - st["rot"],
            key_rotary_offset=case["kd"] - st["rot"], layout="TND" if case["packed"] else "BSND",
            sections=st["sections"], sections_interleaved=case["mixed"])
        if not case["grad"]:
            return q, k
        dq, dk = torch.autograd.grad((q, k), (st["q"], st["k"]), (st["dq"], st["dk"]))
        return q.detach(), k.detach(), dq, dk
    if op == "plan":
        return dsa.paged_cache_plan(st["table"], st["lens"], st["refs"], st["new"], case["page"], st["tokens"])
    if op == "slots":
        dsa.paged_cache_write_slots(st["caches"], st["rows"], st["slots"])
        return list(st["caches"])
    if op == "prefixes":
        return dsa.paged_cache_prefixes(st["table"], st["lens"], case["page"])
    return dsa.paged_prefix_attention(st["q"], st["k"], st["v"], st["table"], st["lens"], st["groups"], st["shared"],
                                      scale_value=st["scale"], query_rope=st["qr"], key_rope=st["kr"],
                                      return_softmax_lse=True)


# ---- the operators from elementary torch operations, sums in 32 bits ----

def _turn(x, cos, sin, start, rot):
    """``x`` with the columns start .. start + rot of every head rotated, pairs (i, i + rot / 2)."""
    part = x[..., start:start + rot].float()
    a, b = part[..., :rot // 2], part[..., rot // 2:]
    part = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([x[..., :start], part.to(x.dtype), x[..., start + rot:]], -1)


def _axes_plain(st):
    case, rot = st["case"], st["rot"]
    # angles of far positions need 64 bits
    angle = st["positions"][st["pair_axes"]].double().movedim(0, -1) * st["inv_freq"]
    cos, sin = torch.cos(angle).float()[..., None, :], torch.sin(angle).float()[..., None, :]
    q0, k0 = case["d"] - rot, case["kd"] - rot
    with torch.no_grad():
        out = [_turn(st["q"], cos, sin, q0, rot), _turn(st["k"], cos, sin, k0, rot)]
        if case["grad"]:
            out += [_turn(st["dq"], cos, -sin, q0, rot), _turn(st["dk"], cos, -sin, k0, rot)]
    return tuple(out)


def _plan_plain(st):
    table, lens, refs, new = st["table"], st["lens"].long(), st["refs"], st["new"].long()
    page, tokens = st["case"]["page"], st["tokens"]
    rows, wide = table.shape
    device = table.device
    more = new.clamp(min=0)
    held, want = -(-lens // page), -(-(lens + more) // page)
    live = new >= 0
    free = torch.nonzero(refs == 0).flatten()
    need = torch.where(live & (want <= wide), want - held, 0)
    start = torch.cumsum(need, 0) - need
    ok = live & (want <= wide) & (start + need <= free.numel())
    col = torch.arange(wide, device=device)[None]
    out = torch.where(live[:, None] & (col < held[:, None]), table.long(), -1)
    taken = ok[:, None] & (col >= held[:, None]) & (col < want[:, None])
    fresh = (start[:, None] + col - held[:, None]).clamp(0, max(free.numel() - 1, 0))
    if free.numel():
        out = torch.where(taken, free[fresh], out)
    pool = refs.numel()
    counted = refs.long() + torch.bincount(out[out >= 0], minlength=pool)
    counted = counted - torch.bincount(table[table >= 0].long(), minlength=pool)
    ends = torch.cumsum(more, 0)
    t = torch.arange(tokens, device=device)
    seq = torch.searchsorted(ends, t, right=True)
    inside = seq < rows
    seq = seq.clamp(max=rows - 1)
    pos = lens[seq] + t - (ends - more)[seq]
    blk = out[seq, (pos // page).clamp(max=wide - 1)]
    slot = torch.where(inside & ok[seq], blk * page + pos % page, -1)
    new_lens = torch.where(ok, lens + more, torch.where(live, lens, 0))
    return (out.int(), new_lens.int(), counted.int(), slot.int(), torch.where(inside, pos, 0).int(), ends.int())


def _prefixes_plain(st):
    table, lens, page = st["table"], st["lens"].long(), st["case"]["page"]
    b, wide = table.shape
    device = table.device
    whole = (torch.minimum(lens[1:], lens[:-1]) // page)[:, None]
    same = (table[1:] == table[:-1]) & (table[1:] >= 0) & (torch.arange(wide, device=device)[None] < whole)
    common = torch.cumprod(same.int(), 1).sum(1)
    linked = torch.cat([torch.zeros(1, dtype=torch.bool, device=device), common > 0])
    row = torch.arange(b, device=device)
    first = torch.cummax(torch.where(linked, 0, row), 0).values
    least = torch.full((b,), wide + 1, dtype=torch.long, device=device)
    if b > 1:
        least.scatter_reduce_(0, first[1:], torch.where(linked[1:], common, wide + 1), "amin")
    pages = least[first]
    return first.int(), torch.where(pages <= wide, pages * page, 0).int()


def _attention(st):
    case, q = st["case"], st["q"]
    b, s1, heads, d = q.shape
    n2, page = case["kvheads"], case["page"]
    group = heads // n2
    out = torch.empty_like(q)
    smax = torch.zeros(b, n2, s1, group, dtype=torch.float32, device=q.device)
    ssum = torch.zeros_like(smax)
    for i, n in enumerate(st["lens_host"]):
        pages = st["table"][i, :-(-n // page)].long()

        def gather(cache):  # [n2, n, columns]
            return cache[pages].reshape(-1, n2, cache.shape[-1])[:n].float().transpose(0, 1).contiguous()

        key, query = gather(st["k"]), q[i].float()
        if case["latent"]:
            value = key
            key = torch.cat([key, gather(st["kr"])], -1)
            query = torch.cat([query, st["qr"][i].float()], -1)
        else:
            value = gather(st["v"])
        # [n2, s1 * group, columns]
        query = query.view(s1, n2, group, -1).transpose(0, 1).reshape(n2, s1 * group, -1)
        score = torch.matmul(query, key.transpose(1, 2).contiguous()) * st["scale"]
        limit = n - s1 + 1 + torch.arange(s1, device=q.device).repeat_interleave(group)  # tokens that a row sees
        hidden = torch.arange(n, device=q.device)[None] >= limit[:, None]
        score = score.masked_fill(hidden, float("-inf"))
        top = score.amax(-1, keepdim=True)
        p = torch.exp(score - top)
        total = p.sum(-1, keepdim=True)
        o = torch.matmul(p, value) / total
        out[i] = o.view(n2, s1, group, d).transpose(0, 1).reshape(s1, heads, d).to(out.dtype)
        smax[i] = top.view(n2, s1, group)
        ssum[i] = total.view(n2, s1, group)
    return out, smax, ssum


def work(case):
    size = 4 if case.get("dtype") == "fp32" else 2
    op = case["op"]
    columns = sum(LATENT)
    if op == "axes":
        rows = case["b"] * case["s"]
        sections = _ints_of(case["sections"])
        elements = rows * (case["heads"] * case["d"] + case["kheads"] * case["kd"])
        passes = 2 if case["grad"] else 1
        return {"bytes": passes * (2 * elements * size + rows * 4 * len(sections)),
                "flops": passes * 3 * rows * (case["heads"] + case["kheads"]) * 2 * sum(sections)}
    if op == "plan":
        rows, page = case["rows"], case["page"]
        pages = (rows - case["prompts"]) * case["hi"] / 2 / page + case["prompts"] * case["new"] / 2 / page
        tokens = rows + case["prompts"] * case["new"] / 2
        return {"bytes": int(pages * 16 + tokens * 8 + rows * 20), "flops": 0}
    if op == "slots":
        return {"bytes": case["tokens"] * (columns * 2 * size + 4), "flops": 0}
    if op == "prefixes":
        rows = sum(_ints_of(case["members"]))
        return {"bytes": int(rows * (case["hi"] * 0.6 / case["page"] * 4 + 12)), "flops": 0}
    members, prefix, suffix = (_ints_of(case[x]) for x in ("members", "prefix", "suffix"))
    read = sum(prefix) + sum(suffix)
    seen = sum(p * m for p, m in zip(prefix, members)) + sum(suffix)
    d = case["d"]
    rows = sum(members) * case["q"] * case["heads"]
    dk, per = (d + 64, d + 64) if case["latent"] else (d, 2 * d)
    return {"bytes": read * case["kvheads"] * per * size + rows * ((dk + d) * size + 8),
            "flops": 2 * seen * case["q"] * case["heads"] * (dk + d)}


# ---- definitions in 64 bits ----

def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        if op == "axes":
            return _axes_exact(st)
        if op == "plan":
            return _plan_exact(st)
        if op == "slots":
            out = [c.double() for c in st["caches"]]
            where = st["slots"].tolist()
            source = [t for t, x in enumerate(where) if x >= 0]
            target = [where[t] for t in source]
            for o, r in zip(out, st["rows"]):
                o.view(-1, o.shape[-1]).index_copy_(0, torch.tensor(target, device="cuda"),
                                                    r.double()[torch.tensor(source, device="cuda"), 0])
            return out
        if op == "prefixes":
            return _prefixes_exact(st)
        return _attention_exact(st)


def _axes_exact(st):
    case, rot = st["case"], st["rot"]
    axes = _pair_axes(case)
    theta = torch.stack([st["positions"][a].double() * st["inv_freq"][i] for i, a in enumerate(axes)], -1)[..., None, :]
    turn = torch.polar(torch.ones_like(theta), theta)

    def apply(x, start, factor):
        y = x.double().clone()
        part = y[..., start:start + rot]
        z = torch.complex(part[..., :rot // 2].contiguous(), part[..., rot // 2:].contiguous()) * factor
        y[..., start:start + rot] = torch.cat([z.real, z.imag], -1)
        return y

    q0, k0 = case["d"] - rot, case["kd"] - rot
    out = [apply(st["q"], q0, turn), apply(st["k"], k0, turn)]
    if case["grad"]:
        out += [apply(st["dq"], q0, turn.conj()), apply(st["dk"], k0, turn.conj())]
    return tuple(out)


def _plan_exact(st):
    """Request by request, as a host would do it."""
    page, tokens = st["case"]["page"], st["tokens"]
    table, lens, refs, new = (st[x].tolist() for x in ("table", "lens", "refs", "new"))
    wide = len(table[0])
    free = [i for i, r in enumerate(refs) if r == 0]
    at = 0
    out, out_lens, slots, positions, ends = [], [], [], [], []
    for row, n, m in zip(table, lens, new):
        held = -(-n // page)
        for e in row[held if m >= 0 else 0:]:
            if e >= 0:
                refs[e] -= 1
        if m < 0:
            out.append([-1] * wide)
            out_lens.append(0)
            ends.append(len(positions))
            continue
        want = -(-(n + m) // page)
        row = row[:held]
        served = want <= wide and at + want - held <= len(free)
        if want <= wide:
            if served:
                row = row + free[at:at + want - held]
                for e in row[held:]:
                    refs[e] += 1
            at += want - held
        positions += range(n, n + m)
        slots += [row[p // page] * page + p % page if served else -1 for p in range(n, n + m)]
        out_lens.append(n + m if served else n)
        out.append(row + [-1] * (wide - len(row)))
        ends.append(len(positions))
    pad = tokens - len(positions)
    return (_ints(out), _ints(out_lens), _ints(refs), _ints(slots + [-1] * pad), _ints(positions + [0] * pad),
            _ints(ends))


def _prefixes_exact(st):
    page = st["case"]["page"]
    table, lens = st["table"].tolist(), st["lens"].tolist()
    groups, shared, members = [], [], []

    def close():
        pages = min(members) if members else 0
        shared.extend([pages * page] * (len(groups) - len(shared)))
        members.clear()

    for b, row in enumerate(table):
        common = 0
        if b:
            whole = min(lens[b], lens[b - 1]) // page
            while common < whole and row[common] == table[b - 1][common] and row[common] >= 0:
                common += 1
        if common:
            members.append(common)
            groups.append(groups[-1])
        else:
            close()
            groups.append(b)
    close()
    return _ints(groups), _ints(shared)


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
