"""Workspace of paged_prefix_attention: that of paged_attention where nothing is worked on together, bounded where
prompts are, with sequences worked on so many at a time."""
import os

import pytest
import torch

from tests.test_prefix_attention_gpu import DTYPES, _compare_some, _make

MOST = 2 ** 29


def _sizes(batch, s1, n1, n2, d, latent, blocks, page, least):
    from dsa_triton_ascend_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    lib = _lib.load()
    args = (batch, s1, n1, n2, d, latent, blocks, page)
    return (lib.dsa_paged_attn_workspace_size(*args), lib.dsa_paged_prefix_attn_workspace_bytes(*args, least),
            lib.dsa_paged_prefix_attn_workspace_size(*args))


@pytest.mark.parametrize("args,least", [
    ((256, 1, 128, 1, 512, 1, 512, 64), -1), ((8, 1024, 128, 1, 512, 1, 512, 64), -1),   # from 64 latent rows on: never
    ((8, 1024, 16, 1, 512, 1, 512, 64), -1), ((32, 1, 64, 8, 128, 0, 512, 64), 512 * 64 + 1),
    ((32, 1, 16, 1, 512, 1, 512, 64), 2 ** 62), ((4, 1, 8, 2, 128, 0, 4, 16), -1),        # no room for so long a prefix
    ((2, 10 ** 6, 16, 4, 256, 0, 8, 64), 0), ((3, 65536, 128, 1, 512, 1, 512, 64), 1)])   # two sequences take too much
def test_nothing_together_takes_what_paged_attention_takes(args, least):
    plain, own, _ = _sizes(*args, least)
    assert plain < own <= plain + 64 * args[0] + 64


@pytest.mark.parametrize("args", [
    (32, 1, 64, 8, 128, 0, 512, 64), (256, 1, 128, 1, 512, 1, 512, 64), (8, 1024, 64, 8, 128, 0, 512, 64),
    (8, 1024, 128, 1, 512, 1, 512, 64), (256, 1500, 64, 8, 128, 0, 512, 64), (200, 64, 64, 2, 128, 0, 8, 16),
    (1 << 20, 1, 2, 1, 64, 0, 32, 1), (1, 1, 1, 1, 64, 0, 1, 1), (5, 7, 36, 12, 256, 0, 100, 48)])
def test_bounded(args):
    top = 0
    for least in (-1, 0, 1, 64, 10 ** 5, 2 ** 62):
        plain, own, any_ = _sizes(*args, least)
        assert 0 < own <= plain + MOST + MOST // 8  # (an eighth: the lists of jobs and sequences)
        top = max(top, own)
    assert top <= any_ <= plain + MOST + MOST // 8
    # (the last min_tokens leaves nothing to work on together; of 8 x 1024 tokens of 128 latent heads the outputs of two
    # sequences alone, 2 * 131072 * 2064 bytes, pass the bound)
    assert own < any_ or args[0] == 1 or args[:3] == (8, 1024, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("latent,N1,N2,dtype", [(False, 64, 2, "bf16"), (True, 96, 1, "fp16")])
def test_sequences_worked_on_so_many_at_a_time(latent, N1, N2, dtype):
    """Families that begin in one launch and go on in the next ones, some whole, some alone in a launch's part."""
    P = [96, 40, 256, 0]
    families = [(0, P[0], [P[0] + 64 + i % 7 for i in range(130)]), (1, P[1], [P[1] + 70] * 2),
                (2, P[2], [P[2] + 64 + i % 40 for i in range(60)]), (-1, 0, [64]), (3, 16, [90] * 9)]
    args, data, lens = _make(families, 64, N1, N2, 128, 16, DTYPES[dtype], latent, seed=3)
    B, S1 = args["query"].shape[:2]
    wide = args["block_table"].shape[1]
    plain, own, _ = _sizes(B, S1, N1, N2, 128, latent, wide, 16, 1)
    rows = B * S1 * N1 * (128 + 4) * 4
    assert 3 * rows > MOST and own <= plain + MOST + MOST // 8
    got = _compare_some(args, data, lens, [0, 1, 63, 64, 65, 66, 67, 68, 69, 77, 78, 79, 100, 129, 130, 131, 132, 160, 191,
                                           192, 193, 194, 201])
    assert torch.isfinite(got[0].float()).all()
    # the parts end elsewhere: the same results to the bit where nothing is worked on together
    import dsa_triton_ascend_amd as dsa
    whole = dsa.paged_prefix_attention(**dict(args, min_tokens=2 ** 40))
    for x, y in zip(whole, got):
        assert torch.allclose(x.float(), y.float(), rtol=2.0 ** -6, atol=2.0 ** -6)


@pytest.mark.gpu
@pytest.mark.parametrize("latent", [False, True])
def test_prompts_that_would_take_too_much_together(latent):
    """Two sequences whose outputs in 32 bits alone pass the bound."""
    import dsa_triton_ascend_amd as dsa
    N1, N2, S1 = (128, 1, 4096) if latent else (128, 2, 4096)
    D = 128
    args, data, lens = _make([(0, 64, [64 + S1, S1])], S1, N1, N2, D, 64, torch.float16, latent, seed=1)
    args["query"].normal_()
    plain, own, _ = _sizes(2, S1, N1, N2, D, latent, args["block_table"].shape[1], 64, 1)
    assert own <= plain + 256
    got = dsa.paged_prefix_attention(**args)
    table = args["block_table"].clone()
    table[1, 0] = table[0, 0]
    same = {k: v for k, v in args.items() if not k.startswith("prefix") and k != "min_tokens"}
    for x, y in zip(got, dsa.paged_attention(**dict(same, block_table=table))):
        assert torch.equal(x, y)


def test_any_min_tokens_and_sizes_of_no_call():
    from dsa_triton_ascend_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    size = _lib.load().dsa_paged_prefix_attn_workspace_bytes
    a = (32, 64, 64, 8, 128, 0, 512, 64)
    assert size(*a, -2 ** 63) == size(*a, -1) > size(*a, 2 ** 63 - 1) > 0
    assert size(*a, 0) == size(*a, 1) == size(*a, 512 * 64) > size(*a, 512 * 64 + 1) == size(*a, 2 ** 31)
    for i, x in ((0, 0), (0, -1), (1, 2 ** 62), (3, 7), (4, 96), (6, 0), (7, 2 ** 20 + 1)):
        assert size(*a[:i], x, *a[i + 1:], 1) == 0
