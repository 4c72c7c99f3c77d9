"""paged_prefix_attention over caches and tables of more than 256 MB, from which the kernels of what is behind the
prefixes (and of prefixes read by each sequence for itself) load without keeping anything in the caches."""
import pytest
import torch

from tests.test_prefix_attention_gpu import DTYPES, _compare, _make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N1,N2,D,S1,page,dtype,latent", [
    (8, 8, 128, 1, 64, "bf16", False), (64, 8, 128, 3, 16, "fp16", False), (72, 8, 128, 4, 64, "bf16", False),
    (16, 16, 64, 1, 48, "fp16", False), (40, 8, 64, 4, 16, "bf16", False), (16, 4, 256, 1, 64, "bf16", False),
    (32, 4, 256, 4, 16, "fp16", False),
    (16, 1, 512, 1, 64, "bf16", True), (9, 1, 512, 3, 16, "fp16", True), (64, 1, 512, 1, 48, "bf16", True),
    (40, 1, 512, 3, 64, "fp16", True)])
@pytest.mark.parametrize("least", [1, None, 2 ** 40])
def test_large_pools_and_tables(N1, N2, D, S1, page, dtype, latent, least):
    families = [(0, 310, [330, 400, 350, 314]), (-1, 0, [500]), (1, 96, [100, 230]), (1, 64, [70, 900])]
    dtype = DTYPES[dtype]
    tokens = (260 << 20) // ((D + 64) * 2 if latent else N2 * D * 4)
    B = sum(len(m) for _, _, m in families)
    wide = tokens // (B * page) + 1
    args, data, lens = _make(families, S1, N1, N2, D, page, dtype, latent, seed=6, wide=wide)
    pages = tokens // page + 1
    other = "key_rope" if latent else "value"
    for name in ("key", other):
        small = args[name]
        big = torch.full((pages, *small.shape[1:]), float("nan"), dtype=dtype, device="cuda")
        big[-small.shape[0]:] = small
        args[name] = big
    args["block_table"] = torch.where(args["block_table"] >= 0, args["block_table"] + (pages - small.shape[0]), -1).int()
    # (the sizes by which the kernels are chosen)
    assert min(pages, B * args["block_table"].shape[1]) * page * (D + 64 if latent else 2 * N2 * D) * 2 > 256 << 20
    _compare(dict(args, min_tokens=least), data, lens)
