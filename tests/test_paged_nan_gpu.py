"""Queries that are not numbers: their rows come out as NaN however a sequence's tokens are split, the others as without."""
import pytest
import torch

from tests.test_prefix_attention_gpu import _make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("latent,N1,D", [(False, 16, 128), (False, 8, 64), (True, 16, 512), (True, 128, 512), (True, 3, 128)])
@pytest.mark.parametrize("families", [[(0, 640, [700, 641, 960])], [(-1, 0, [20000])], [(-1, 0, [70])],
                                      [(0, 4000, [4001 + i for i in range(9)])]])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_rows_of_queries_that_are_not_numbers(latent, N1, D, families, value):
    import dsa_triton_ascend_amd as dsa
    args, _, lens = _make(families, 2, N1, 1 if latent else 2, D, 16, torch.bfloat16, latent, seed=4)
    b, s, h = len(lens) - 1, 1, N1 // 2
    bad = dict(args, query=args["query"].clone())
    bad["query"][b, s, h, 3] = value
    table = args["block_table"].clone()
    if len(lens) > 1:
        p = families[0][1] // 16
        table[1:, :p] = table[0, :p]
    plain = ("prefix_groups", "prefix_lengths", "min_tokens")
    for call in (lambda a: dsa.paged_prefix_attention(**a), lambda a: dsa.paged_prefix_attention(**dict(a, min_tokens=2 ** 40)),
                 lambda a: dsa.paged_attention(**{k: v for k, v in dict(a, block_table=table).items() if k not in plain})):
        want, got = call(args), call(bad)
        assert torch.isnan(got[0][b, s, h]).all()
        assert torch.isnan(got[2][b].view(-1)[_stat(args, s, h)])
        keep = torch.ones_like(want[0], dtype=torch.bool)
        keep[b, s, h] = False
        assert torch.equal(want[0][keep], got[0][keep])
        keep = torch.ones(want[1].shape, dtype=torch.bool, device="cuda")
        keep[b].view(-1)[_stat(args, s, h)] = False
        assert torch.equal(want[1][keep], got[1][keep]) and torch.equal(want[2][keep], got[2][keep])


def _stat(args, s, h):
    """Place of a row in a sequence's statistics [N2, S1, N1 / N2]."""
    S1, N1, N2 = args["query"].shape[1], args["query"].shape[2], args["key"].shape[2]
    g = N1 // N2
    return (h // g * S1 + s) * g + h % g
