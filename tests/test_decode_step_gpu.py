"""Decoding with the paged operators together, as a serving loop uses them:
packed prompts rotated and written into pages, then steps of fork (beams of a
prompt part, end and go on), rotate, write, attend, with a compaction on the
way, against plain histories per sequence in 64 bits.  The sparse operators
read the same caches."""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
N1, D, DR, PAGE = 16, 512, 64, 16


def _turn(x, pos, inv, scale):
    """Interleaved rotation of [tokens, heads, 64] in 64 bits, rounded to bf16."""
    ang = pos.double()[:, None] * inv.double()
    c, s = (torch.cos(ang) * scale)[:, None], (torch.sin(ang) * scale)[:, None]
    a, b = x.double()[..., 0::2], x.double()[..., 1::2]
    return torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2).to(BF)


def _near(x, want):
    """Equal, or neighbours where 32 and 64 bits round apart (one step: 2^-7 of the value at most)."""
    err = (x.double() - want.double()).abs()
    assert (err <= want.double().abs() * 2.0 ** -7 + 2.0 ** -20).all()


def test_serving_loop():
    import dsa_triton_ascend_amd as dsa
    rng = random.Random(3)
    g = torch.Generator(device="cuda").manual_seed(3)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(BF)

    pages, wide = 120, 12
    latent = torch.full((pages, PAGE, 1, D), float("nan"), device="cuda", dtype=BF)
    rope = torch.full((pages, PAGE, 1, DR), float("nan"), device="cuda", dtype=BF)
    caches = [latent, rope]
    inv, scale = dsa.rotary_frequencies(DR, scaling="yarn", factor=4.0)
    lens_h = [37, 1, 80, 16]
    table = torch.full((4, wide), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(4, dtype=torch.int32, device="cuda")
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    # room for the longest prompt in every row, then the prompts, packed, with two rows behind the last
    table, lens, refs = dsa.paged_cache_fork(caches, table, lens, refs, new_tokens=max(lens_h))
    total = sum(lens_h)
    kv = normal(total + 2, D + DR)
    pos = torch.cat([torch.arange(n) for n in lens_h] + [torch.zeros(2)]).to("cuda", torch.int32)
    _, kr = dsa.rotary_embedding(kv[:, None, D:], kv[:, None, D:], pos, inv, interleaved=True, attention_scale=scale,
                                 layout="TND")
    cu = torch.tensor([sum(lens_h[:i + 1]) for i in range(4)], dtype=torch.int32, device="cuda")
    dsa.paged_cache_write(caches, [kv[:, None, :D], kr], table, lens, row_lengths=cu, layout="TND")
    lens = lens + torch.tensor(lens_h, dtype=torch.int32, device="cuda")
    _near(kr, _turn(kv[:, None, D:], pos, inv, scale))
    history, at = [], 0
    for n in lens_h:
        history.append((kv[at:at + n, :D], kr[at:at + n, 0]))
        at += n
    soft = 1.0 / math.sqrt(D + DR)
    for step in range(7):
        rows = len(history)
        parents = [rng.randrange(rows) for _ in range(rng.choice([4, 6]))]
        if step == 3:
            parents[1] = -1
        table, lens, refs = dsa.paged_cache_fork(caches, table, lens, refs, new_tokens=2,
                                                 parents=torch.tensor(parents, dtype=torch.int32, device="cuda"))
        history = [history[p] if p >= 0 else (kv[:0, :D], kr[:0, 0]) for p in parents]
        assert lens.tolist() == [h[0].shape[0] for h in history]
        # every page is referred to as often as the table names it
        named = torch.bincount(table[table >= 0].long(), minlength=pages)
        assert torch.equal(named.int(), refs)
        if step == 4:
            table, refs, _ = dsa.paged_cache_compact(caches, table, refs)
            used = int((refs > 0).sum())
            assert (refs[:used] > 0).all() and int(table.max()) < used
        B = len(parents)
        new = normal(B, 2, D + DR)
        q, qr = normal(B, 2, N1, D), normal(B, 2, N1, DR)
        pos = lens[:, None] + torch.arange(2, device="cuda", dtype=torch.int32)
        qr2, kr2 = dsa.rotary_embedding(qr, new[:, :, None, D:], pos, inv, interleaved=True, attention_scale=scale)
        dsa.paged_cache_write(caches, [new[:, :, None, :D], kr2], table, lens)
        # (an empty row has no pages: its tokens are dropped, and its length stays 0)
        lens = lens + torch.tensor([2 * (p >= 0) for p in parents], dtype=torch.int32, device="cuda")
        out, _, _ = dsa.paged_attention(q, latent, None, table, lens, scale_value=soft, query_rope=qr2, key_rope=rope)
        idx = torch.full((B, 2, 1, 160), -1, dtype=torch.int32, device="cuda")
        for b in range(B):
            if parents[b] < 0:
                assert (out[b] == 0).all()
                continue
            _near(kr2[b], _turn(new[b, :, None, D:], pos[b], inv, scale))
            _near(qr2[b], _turn(qr[b], pos[b], inv, scale))
            history[b] = (torch.cat([history[b][0], new[b, :, :D]]), torch.cat([history[b][1], kr2[b, :, 0]]))
            k = torch.cat([history[b][0], history[b][1]], -1).double()
            n = k.shape[0]
            for s in range(2):
                m = n - 1 + s
                idx[b, s, 0, :m] = torch.arange(m, device="cuda")
                qs = torch.cat([q[b, s], qr2[b, s]], -1).double()
                score = qs @ k[:m].T * soft
                w = torch.softmax(score, -1)
                want, mag = w @ k[:m, :D], w @ k[:m, :D].abs()
                # a score is off by at most ds, a weight by 2 ds and 2^-15 (two values per numerator, sums),
                # the output by the rounding of its type
                ds = ((qs.abs() @ k[:m].abs().T) * soft * (D + DR + 4) * 2.0 ** -24).amax(-1, keepdim=True)
                rel = 2 * ds + 2.0 ** -15
                err = (out[b, s].double() - want).abs()
                assert (err <= mag * rel + (want.abs() + mag * rel) * 2.0 ** -8).all(), (step, b, s, float(err.max()))
        sparse, _, _ = dsa.sparse_flash_attention_triton(
            q, latent.nan_to_num(0.0), None, idx, scale_value=soft, block_table=table, actual_seq_lengths_kv=lens,
            query_rope=qr2, key_rope=rope.nan_to_num(0.0), layout_kv="PA_BSND", sparse_mode=3)
        # the sparse operator over all tokens: each rounds the output once and weights at most once
        v = latent[table[table >= 0].long()].nan_to_num(0.0).abs().max()
        assert (sparse.double() - out.double()).abs().max() <= 4 * 2.0 ** -8 * v
